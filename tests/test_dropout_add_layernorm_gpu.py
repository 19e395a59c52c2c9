"""dropout_add_layernorm on the GPU against the float64 definition (oracle/layer_oracle.py).

Bounds (u = torch.finfo(t).eps / 2, e = 2^-24, C channels): h carries two roundings, mean and variance sums over C in fp32 at most (C + 8) half steps
of their magnitudes, so x^ is off by at most a = e ((C + 16)(1 + |x^|) + 4 max |h| rs) — the last for the cancellation in h - mean.
  y: u |y| + a |gamma| + 4 e (|x^ gamma| + |beta|);   dr, dx: u |d| + rs (K e) (|g| + max |g| (1 + |x^|) + ...) with K = 4 (C + 16) (1 + max |h| rs)
  dgamma, dbeta: fp32 sums of at most 64 terms in order, then float64: (a_max + 80 e) sum |.|."""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
E = 2.0 ** -24


def _data(dev, dt, B, C, T, seed=0):
    g = torch.Generator().manual_seed(seed + C + T)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, rr, dy = r(B, C, T).to(dt), (r(B, C, T) + 0.5 * r(1, C, 1)).to(dt), r(B, C, T).to(dt)
    return [t.to(dev) for t in (x, rr, 1 + 0.2 * r(C), 0.3 * r(C), dy)]


def _near(x, ref, bound, name):
    x = x.detach().double().cpu()
    assert x.shape == ref.shape and torch.isfinite(x).all(), name
    worst = ((x - ref).abs() / (bound + 1e-30)).max().item() if x.numel() else 0.0
    assert worst <= 1.0, (name, worst)


def _compare(ref, got, dt, gamma, beta, C):
    u = torch.finfo(dt).eps / 2 if dt != torch.float32 else E
    tiny = 2.0 ** -25 if dt == torch.float16 else 0.0
    gm, bt = gamma.double().cpu().abs()[:, None], beta.double().cpu().abs()[:, None]
    xh, big = ref["xh"].abs(), (ref["h"].abs().amax(1, keepdim=True) * ref["rs"])
    a = E * ((C + 16) * (1 + xh) + 4 * big)
    _near(got["y"], ref["y"], u * ref["y"].abs() + a * gm + 4 * E * (xh * gm + bt) + tiny, "y")
    if "dr" not in got:
        return
    g = ref["g"].abs()
    top = g.amax(1, keepdim=True)
    err = ref["rs"] * 4 * (C + 16) * E * (1 + big) * (g + top * (1 + xh) ** 2)
    for n in ("dr", "dx"):
        if got[n] is not None:
            _near(got[n], ref[n], u * ref[n].abs() + err * 4 + tiny, n)
    _near(got["dgamma"], ref["dgamma"], (a.max() * 2 + 80 * E) * (ref["mag_dgamma"] + ref["mag_dbeta"]) + E * ref["dgamma"].abs(), "dgamma")
    _near(got["dbeta"], ref["dbeta"], 80 * E * ref["mag_dbeta"] + E * ref["dbeta"].abs(), "dbeta")


def _run(dev, dt, B, C, T, p=0.0, mask=None, with_r=True, seed=0):
    import svc_autograd as A
    import svc_hip as S
    print(f"case {dt} B{B} C{C} T{T} p{p} mask{mask is not None} r{with_r}", flush=True)
    x, r, gamma, beta, dy = _data(dev, dt, B, C, T, seed)
    r = r if with_r else None
    draw = S.HashDraw(torch.tensor([77 + seed], dtype=torch.int64, device=dev), 2) if p else None
    ref = O.junction(x, r, gamma, beta, dy, draw=draw, p=p, mask=mask)
    m = None if mask is None else mask.to(dev)
    if not p:
        _compare(ref, {"y": S.dropout_add_layernorm(x, r, gamma, beta, mask=m)}, dt, gamma, beta, C)
    leaves = [t.requires_grad_() for t in (x, gamma, beta)] + ([r.requires_grad_()] if with_r else [])
    y = A.dropout_add_layernorm(x, r, gamma, beta, draw=draw, p=p, mask=m)
    g = torch.autograd.grad(y, leaves, dy)
    _compare(ref, {"y": y, "dx": g[0], "dgamma": g[1], "dbeta": g[2], "dr": g[3] if with_r else None}, dt, gamma, beta, C)


def _mask(B, T, seed=1):
    g = torch.Generator().manual_seed(seed)
    m = (torch.rand(B, T, generator=g) < 0.7).float()
    m[0, T // 2:] = 0
    return m


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,C,T", [(1, 1, 1), (1, 192, 1), (2, 7, 5), (1, 64, 64), (2, 192, 65), (1, 193, 131), (3, 33, 257), (1, 512, 100), (2, 768, 63), (1, 1025, 70),
                                   (1, 2500, 40), (4, 48, 500)])
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_against_float64(dev, dt, B, C, T, p):
    _run(dev, TYPES[dt], B, C, T, p=p, mask=_mask(B, T) if (C + T) % 2 else None)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_without_residual(dev, dt, p):
    _run(dev, TYPES[dt], 2, 96, 70, p=p, with_r=False)


def test_draws_are_those_of_the_dropout_launch(dev):
    import svc_hip as S
    x, r, gamma, beta, _ = _data(dev, torch.float32, 2, 192, 333)
    draw = S.HashDraw(torch.tensor([9], device=dev), 4)
    a = S.dropout_add_layernorm(x, r, gamma, beta, draw=draw, p=0.4)
    b = S.dropout_add_layernorm(S.dropout_rng(x, draw, 0.4), r, gamma, beta)
    assert (a - b).abs().max() <= 16 * E * 8         # the same numbers added; x * 1/(1-p) may round once more, |y| < 8


def test_masked_places_are_not_used(dev):
    """NaN and infinities where the mask is 0: zero outputs and gradients there, everything else as without them."""
    import svc_hip as S
    x, r, gamma, beta, dy = _data(dev, torch.bfloat16, 2, 96, 150)
    m = _mask(2, 150).to(dev)
    draw = S.HashDraw(torch.tensor([3], device=dev), 0)

    def go(x, r, dy):
        y, (mu, rs) = S.dropout_add_layernorm(x, r, gamma, beta, mask=m, draw=draw, p=0.2, stats=True)
        return (y, *S.dropout_add_layernorm_bwd(dy, x, r, gamma, beta, mu, rs, mask=m, draw=draw, p=0.2))

    want = go(x, r, dy)
    hole = (m == 0)[:, None]
    got = go(x.masked_fill(hole, float("nan")), r.masked_fill(hole, float("inf")), dy.masked_fill(hole, float("-inf")))
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    for t in got[:3]:
        assert not t.masked_select(hole).any()


def test_constant_columns_and_large_means(dev):
    """A column of equal values has variance 0; a mean of 1000 leaves h - mean 10 bits fewer (the bound's max |h| rs term)."""
    import svc_hip as S
    gamma, beta = torch.ones(64, device=dev), torch.zeros(64, device=dev)
    y = S.dropout_add_layernorm(torch.full((1, 64, 5), 3.0, device=dev), None, gamma, beta)
    assert y.abs().max() <= 1e-2                     # x^ = rounding of the mean (<= 2^-22) over sqrt(eps)
    x, r, gamma, beta, _ = _data(dev, torch.float32, 1, 192, 50)
    ref = O.junction(x + 1000, r, gamma, beta)
    _compare(ref, {"y": S.dropout_add_layernorm(x + 1000, r, gamma, beta)}, torch.float32, gamma, beta, 192)


def test_strided_inputs_and_mask_forms(dev):
    import svc_hip as S
    x, r, gamma, beta, dy = _data(dev, torch.float16, 2, 40, 66)
    m = _mask(2, 66).to(dev)
    want = S.dropout_add_layernorm(x, r, gamma, beta, mask=m)
    big = torch.cat([x, r], 1)
    assert torch.equal(S.dropout_add_layernorm(big[:, :40], big[:, 40:], gamma, beta, mask=m[:, None]), want)
    assert torch.equal(S.dropout_add_layernorm(x.transpose(1, 2).contiguous().transpose(1, 2), r, gamma, beta, mask=m), want)


def test_two_runs_are_bit_equal_and_replays_too(dev):
    import svc_hip as S
    x, r, gamma, beta, dy = _data(dev, torch.float32, 4, 192, 333)
    seed = torch.tensor([9], device=dev)
    draw = S.HashDraw(seed, 4)

    def step():
        y, (mu, rs) = S.dropout_add_layernorm(x, r, gamma, beta, draw=draw, p=0.1, stats=True)
        return (y, *S.dropout_add_layernorm_bwd(dy, x, r, gamma, beta, mu, rs, draw=draw, p=0.1))

    want = {s: None for s in (9, 10, 11)}
    for s in want:
        seed.fill_(s)
        want[s] = [t.clone() for t in step()]
        assert all(torch.equal(a, b) for a, b in zip(step(), want[s]))
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        out = step()
    for s in (10, 9, 11, 10):
        seed.fill_(s)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[s]))
        torch.randn(500, 500, device=dev).sum()


def test_refusals_and_empty(dev):
    import svc_autograd as A
    import svc_hip as S
    x, r, gamma, beta, dy = _data(dev, torch.float32, 2, 8, 6)
    for bad in ((x, r[:, :, :5], gamma, beta), (x, r.half(), gamma, beta), (x, r, gamma[:7], beta), (x, r, gamma.half(), beta), (x[0], r[0], gamma, beta),
                (x, r, gamma, beta.cpu())):
        with pytest.raises(S.SvcError):
            S.dropout_add_layernorm(*bad)
    for kw in (dict(mask=torch.ones(2, 5, device=dev)), dict(mask=torch.ones(2, 6, device=dev, dtype=torch.bool)), dict(p=0.1), dict(eps=0.0),
               dict(p=1.0, draw=S.HashDraw(torch.zeros(1, dtype=torch.int64, device=dev), 0)), dict(p=0.1, draw=torch.rand_like(x))):
        with pytest.raises(S.SvcError):
            S.dropout_add_layernorm(x, r, gamma, beta, **kw)
    e = torch.zeros(2, 8, 0, device=dev, requires_grad=True)
    y = A.dropout_add_layernorm(e, e, gamma.requires_grad_(), beta.requires_grad_())
    assert y.shape == e.shape
    g = torch.autograd.grad(y.sum(), (e, gamma, beta))
    assert not g[1].any() and not g[2].any()
