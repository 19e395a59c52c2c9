"""attention_scored at the sizes whose launches differ from small ones: key heads placed by XCD (items * key heads divisible by 8, or 64 and more, with
query heads that share them), walks of many tiles, keys in many parts — against the float64 definition with the bounds of
tests/test_attention_scored_gpu.py.  And fp32 results by their norm, which bounds of worst cases leave loose."""
import pytest
import torch

from oracle import layer_oracle as O
from test_attention_scored_gpu import TYPES, _both, _i32, _inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _vector_mask(monkeypatch):
    """The oracle's visible keys by comparisons of whole matrices instead of entry by entry (tests/test_layer_ops_cpu.py's sizes are small; the same
    keys, tests/test_layer_oracle_cpu.py)."""
    monkeypatch.setattr(O, "visible", O.visible_matrix)


# (B, H, G, dk, Tq, Tk, W, p, options)
PLACED = [
    (4, 4, 2, 32, 150, 150, 20, 0.1, dict(causal=True, softcap=4.0)),                # 8 groups, 2 query heads each
    (8, 2, 1, 96, 130, 131, None, 0.0, dict(window=40)),
    (2, 12, 4, 64, 300, 300, 30, 0.0, dict(docs=_i32([[0, 70, 200, 290], [0, 128, 129, 300]]))),
    (1, 8, 8, 128, 257, 257, None, 0.0, dict(causal=True)),
    (65, 1, 1, 32, 140, 140, None, 0.0, dict(causal=True)),                         # 64 and more, not a multiple of 8: workgroups without work
    (67, 2, 1, 32, 133, 133, 5, 0.2, dict(lengths=_i32([133 - b for b in range(67)]))),
    (71, 3, 1, 17, 129, 129, None, 0.0, dict(causal=True)),
    (36, 4, 2, 64, 129, 129, None, 0.0, dict(window=3)),                            # 72
    (3, 6, 2, 64, 260, 260, 9, 0.0, dict(causal=True)),                             # 6: not placed by XCD
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", PLACED, ids=lambda c: f"{c[:7]}")
def test_every_placement(dev, case, dt):
    _both(dev, TYPES[dt], *case[:6], W=case[6], p=case[7], seed=2, **case[8])


@pytest.mark.parametrize("dt,T", [("fp32", 2100), ("fp32", 4200), ("bf16", 4200), ("fp16", 4200)])
@pytest.mark.parametrize("kw", [dict(causal=True), dict(window=70), dict(docs=_i32([[0, 100, 1900, 1901, 2090]]))], ids=["causal", "window", "docs"])
def test_deep_walks(dev, dt, T, kw):
    """More than 64 query tiles (64 rows of a 16-bit type, 32 of fp32) in dk's and dv's walk, two query heads one after the other."""
    _both(dev, TYPES[dt], 1, 2, 1, 32, T, T, W=64, seed=1, gain=1.0, **kw)


@pytest.mark.parametrize("p", [0.0, 0.1])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", [(1, 2, 1, 96, 1, 5001, 30, dict(causal=True)), (2, 4, 1, 64, 3, 3000, None, dict(window=1700, softcap=6.0)),
                                  (3, 2, 2, 32, 64, 2100, 9, dict(causal=True, lengths=_i32([2100, 1500, 700]), offset=_i32([2036, 1436, 636]))),
                                  (2, 8, 2, 128, 9, 4097, None, dict(offset=300, causal=True)), (1, 2, 1, 96, 65, 2500, 30, dict(causal=True))],
                         ids=lambda c: f"{c[:7]}")
def test_few_queries_in_many_parts(dev, case, dt, p):
    """Up to twenty parts of the keys and their joining; 65 queries are the first that are not cut."""
    _both(dev, TYPES[dt], *case[:6], W=case[6], p=p, seed=4, **case[7])


# 2^-24 is half a step of fp32.  A score's dk products are added in dk / 2 (or dk / 16 x 6) steps, each off by at most half a step of the partial sum,
# evenly spread and independent: about 2^-24 sqrt(dk / 2) / sqrt(3) |score|, some 4 half steps at 96 channels and |score| of 1.5; exp2, the sums of P and
# the second product add as much again, and dS = P (dP - D) has two such factors and a difference: 16 half steps in all, doubled for what is not
# independent: 32 x 2^-24 = 1.9e-6 of the norm.  Inputs cut to two bf16 parts (2^-17 each) are off by 4e-6 and more (test_layer_oracle_cpu.py).
NORM = 32 * 2.0 ** -24


@pytest.mark.parametrize("case", [(2, 2, 1, 96, 200, 200, None, {}), (1, 2, 2, 64, 257, 257, 40, dict(causal=True)), (2, 2, 2, 128, 150, 150, None, dict(softcap=8.0)),
                                  (2, 2, 2, 32, 200, 200, 20, dict(window=50)), (2, 2, 1, 96, 40, 200, None, dict(causal=True))], ids=lambda c: f"{c[:7]}")
def test_fp32_by_its_norm(dev, case):
    import svc_autograd as A
    B, H, G, dk, Tq, Tk, W, kw = case
    q, k, v, do, bias = _inputs(dev, torch.float32, B, H, G, dk, Tq, Tk, W, seed=5)
    ref = O.attention(q, k, v, H, dout=do, bias=bias, **kw)
    leaves = [t.requires_grad_() for t in (q, k, v)] + ([bias.requires_grad_()] if W else [])
    out = A.attention_scored(q, k, v, H, bias=bias, **kw)
    for n, x in zip(("out", "dq", "dk", "dv", "dbias"), (out, *torch.autograd.grad(out, leaves, do))):
        err = ((x.detach().double().cpu() - ref[n]).norm() / ref[n].norm()).item()
        print(f"{n} {err:.2e}", flush=True)
        assert err <= NORM, (n, err)


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("case", [(2, 2, 1, 96, 200, 200, 40, {}), (1, 2, 2, 64, 257, 257, 40, dict(causal=True, softcap=5.0))], ids=lambda c: f"{c[:7]}")
def test_table_gradients_of_16_bit_calls_by_their_norm(dev, case, dt):
    """An fp32 result: P in two operands (fp16: 11 + 11 bits and 2^8) or three (bf16), the library's tanh, dO.v from exact products.  Entries of the table sum dS of
    either sign; the norm of the absolute sums stands for the result's."""
    import svc_autograd as A
    B, H, G, dk, Tq, Tk, W, kw = case
    q, k, v, do, bias = _inputs(dev, TYPES[dt], B, H, G, dk, Tq, Tk, W, seed=5)
    ref = O.attention(q, k, v, H, dout=do, bias=bias, **kw)
    out = A.attention_scored(q, k, v, H, bias=bias.requires_grad_(), **kw)
    g, = torch.autograd.grad(out, bias, do)
    err = ((g.double().cpu() - ref["dbias"]).norm() / ref["dbias"].norm()).item()
    print(f"dbias {err:.2e}", flush=True)
    assert err <= NORM
