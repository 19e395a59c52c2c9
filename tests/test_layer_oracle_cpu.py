"""The attention oracle itself: its two ways to find visible keys agree, and fp32 checks by the norm would notice a lost part of the operands."""
import pytest
import torch

from oracle import layer_oracle as O

_t = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
MASKS = [{}, dict(causal=True), dict(window=0), dict(window=4), dict(causal=True, window=3), dict(causal=True, offset=2), dict(lengths=_t([20, 0])),
         dict(lengths=_t([30, 7]), offset=_t([-3, 15]), causal=True), dict(docs=_t([[0, 5, 5, 18], [2, 9, 12, 20]])), dict(prefix=_t([9, 0]), causal=True),
         dict(docs=_t([[0, 5, 5, 18], [-4, 9, 12, 40]]), causal=True, prefix=_t([[2, 1, 30], [0, 1, -5]])), dict(docs=_t([[3, 9], [0, 20]]), window=2),
         dict(offset=_t([2 ** 31 - 1, -2 ** 31]))]


@pytest.mark.parametrize("kw", MASKS, ids=lambda d: "-".join(sorted(d)) or "all")
@pytest.mark.parametrize("Tq", [20, 6, 1])
def test_visible_keys_two_ways(kw, Tq):
    if isinstance(kw.get("offset"), int) and kw["offset"] > 20 - Tq:
        pytest.skip("an offset beyond the key axis")
    a, b = O.visible(2, Tq, 20, **kw), O.visible_matrix(2, Tq, 20, **kw)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("H,G,dk,Tq,Tk,kw", [(2, 1, 96, 200, 200, {}), (2, 2, 64, 257, 257, dict(causal=True)), (2, 2, 32, 200, 200, dict(window=50))])
def test_operands_of_two_parts_would_fail_the_norm(H, G, dk, Tq, Tk, kw):
    """Inputs cut to the sum of two bf16 numbers (16 bits): every result is further from the exact one than 32 x 2^-24 of the norm."""
    g = torch.Generator().manual_seed(dk)
    q, k, v, do = (x * torch.randn(1, n * dk, T, generator=g) for x, n, T in ((1.5, H, Tq), (1, G, Tk), (1, G, Tk), (1, H, Tq)))

    def cut(x):
        a = x.bfloat16().float()
        return a + (x - a).bfloat16().float()

    a = O.attention(q, k, v, H, dout=do, **kw)
    b = O.attention(cut(q), cut(k), cut(v), H, dout=cut(do), **kw)
    for n in ("out", "dq", "dk", "dv"):
        err = ((a[n] - b[n]).norm() / a[n].norm()).item()
        assert err > 32 * 2.0 ** -24, (n, err)


def test_p_in_one_bf16_operand_would_fail_the_table_gradients_norm(monkeypatch):
    """The table's gradient holds D = sum dO out: with P in one bf16 operand it is 1.4e-3 of its norm off, far above 32 x 2^-24; two leave about that bound (1.5e-6),
    three 2e-9."""
    g = torch.Generator().manual_seed(11)
    q, k, v, do = (x * torch.randn(2, n * 96, 200, generator=g).bfloat16().float() for x, n in ((1.5, 2), (1, 1), (1, 1), (1, 2)))
    bias = 0.7 * torch.randn(2, 81, generator=g)
    want = O.attention(q, k, v, 2, dout=do, bias=bias)["dbias"]
    plain, err = torch.einsum, {}
    for n in (1, 3):
        def einsum(eq, a, b):
            if eq == "bhts,bhds->bhdt":                     # out = P v
                whole, rest = torch.zeros_like(a), a
                for _ in range(n):
                    part = rest.float().bfloat16().double()
                    whole, rest = whole + part, rest - part
                a = whole
            return plain(eq, a, b)
        monkeypatch.setattr(torch, "einsum", einsum)
        err[n] = ((O.attention(q, k, v, 2, dout=do, bias=bias)["dbias"] - want).norm() / want.norm()).item()
        monkeypatch.setattr(torch, "einsum", plain)
    assert err[1] > 100 * 32 * 2.0 ** -24 and err[3] < 2.0 ** -24, err
