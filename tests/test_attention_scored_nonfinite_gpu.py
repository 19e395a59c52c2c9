"""attention_scored where values are not finite or very large: what a query sees decides what it answers, in every kernel alike."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
NAN, INF = float("nan"), float("inf")


def _inputs(dev, dt, B, H, G, dk, Tq, Tk, seed=0):
    g = torch.Generator().manual_seed(seed + Tq + 7 * Tk + dk)
    return [torch.randn(B, n * dk, T, generator=g).to(dt).to(dev) for n, T in ((H, Tq), (G, Tk), (G, Tk), (H, Tq))]


def _pass(q, k, v, do, H, **kw):
    """(out, lse, dq, dk, dv, dbias or None) of a training pass."""
    import svc_hip as S
    out, lse, o32 = S.attention_scored_fwd(q, k, v, H, want_dbias="bias" in kw, **kw)
    return (out, lse, *S.attention_scored_bwd(do, q, k, v, out if o32 is None else o32, lse, H, want_dbias="bias" in kw, **kw))


@pytest.mark.parametrize("p", [0.0, 0.2])
@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("dk", [64, 96, 128])
@pytest.mark.parametrize("dt", TYPES)
def test_capped_scores_at_keys_that_no_query_sees(dev, dt, dk, table, p):
    """Keys behind the last query's position, and before the first one's window, inside the key blocks of keys that are seen: with a cap the factor
    1 - tanh^2 of a NaN score is NaN, whatever its P."""
    import svc_hip as S
    q, k, v, do = _inputs(dev, TYPES[dt], 2, 2, 1, dk, 75, 150)
    kw = dict(softcap=4.0, offset=41)
    if table:
        kw["bias"] = torch.linspace(-1, 1, 2 * 11, device=dev).view(2, 11)
    if p:
        kw.update(draw=S.HashDraw(torch.tensor([3], device=dev), 1), p_drop=p)
    for seen, more in ((slice(0, 116), dict(causal=True)), (slice(36, 121), dict(window=5))):
        want = _pass(q, k, v, do, 2, **kw, **more)
        for bad in (NAN, INF):
            k2, v2 = torch.full_like(k, bad), torch.full_like(v, bad)
            k2[:, :, seen], v2[:, :, seen] = k[:, :, seen], v[:, :, seen]
            for a, b in zip(want, _pass(q, k2, v2, do, 2, **kw, **more)):
                assert a is None or torch.equal(a, b)
        for g in want[3:5]:
            g = g.clone()
            g[:, :, seen] = 0
            assert not g.any()


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("T", [40, 64, 65, 150])
@pytest.mark.parametrize("dk", [32, 96, 128])
@pytest.mark.parametrize("dt", TYPES)
def test_a_nan_query_spoils_its_row_alone(dev, dt, dk, T, cap):
    """Up to 64 queries and beyond (two forward kernels): out, lse and dq are NaN at the query, dv at the keys that it sees, nothing else is."""
    q, k, v, do = _inputs(dev, TYPES[dt], 1, 2, 1, dk, T, T)
    t0, w = 21, 5
    q[0, 3, t0] = NAN                                                  # head 0
    out, lse, dq, _, dv, _ = _pass(q, k, v, do, 2, window=w, softcap=cap)
    rows = torch.zeros(1, 2, T, dtype=torch.bool, device=dev)
    rows[0, 0, t0] = True
    wide = rows[:, :, None].expand(1, 2, dk, T).reshape(1, 2 * dk, T)
    keys = ((torch.arange(T, device=dev) - t0).abs() <= w).expand(1, dk, T)
    assert torch.equal(torch.isnan(lse), rows)
    for x, where in ((out, wide), (dq, wide), (dv, keys)):
        assert torch.equal(torch.isnan(x), where) and not torch.isinf(x).any()


@pytest.mark.parametrize("cap", [0.0, 5.0])
@pytest.mark.parametrize("T", [60, 150])
@pytest.mark.parametrize("dk", [32, 96, 128])
@pytest.mark.parametrize("dt", TYPES)
def test_a_nan_key_spoils_the_rows_that_see_it(dev, dt, dk, T, cap):
    """Rows that see it are NaN, and so are dk and dv of every key that one of these rows sees: P of such a row is NaN at all of them."""
    q, k, v, do = _inputs(dev, TYPES[dt], 1, 2, 1, dk, T, T)
    s0, w = 30, 4
    k[0, 1, s0] = NAN
    out, lse, _, dk_, dv, _ = _pass(q, k, v, do, 2, window=w, softcap=cap)
    at = (torch.arange(T, device=dev) - s0).abs()
    assert torch.equal(torch.isnan(lse), (at <= w).expand(1, 2, T))
    assert torch.equal(torch.isnan(out), (at <= w).expand(1, 2 * dk, T))
    for x in (dk_, dv):
        assert torch.equal(torch.isnan(x), (at <= 2 * w).expand(1, dk, T))


@pytest.mark.parametrize("T", [1, 40, 150])
@pytest.mark.parametrize("dt", TYPES)
def test_a_row_whose_every_score_is_nan_has_a_nan_lse(dev, dt, T):
    q, k, v, do = _inputs(dev, TYPES[dt], 1, 1, 1, 64, T, 700)
    q[0, 0] = NAN
    for x in _pass(q, k, v, do, 1)[:3]:
        assert torch.isnan(x).all()


def _exact(q, k, v, H, see):
    """float64, over the seen keys alone: a masked key takes no part, whatever it holds."""
    B, C, Tq = q.shape
    dk = C // H
    G = k.shape[1] // dk
    q, k, v = (x.double().cpu() for x in (q, k, v))
    out = torch.zeros_like(q)
    for b in range(B):
        for h in range(H):
            Q, K, V = q[b, h * dk:(h + 1) * dk], k[b, h // (H // G) * dk:][:dk], v[b, h // (H // G) * dk:][:dk]
            for t in range(Tq):
                s = torch.nonzero(see[t])[:, 0]
                a = (Q[:, t, None] * K[:, s]).sum(0) * dk ** -0.5
                P = torch.exp(a - a.max())
                live = P > 0
                out[b, h * dk:(h + 1) * dk, t] = (V[:, s[live]] * P[live]).sum(1) / P.sum()
    return out


@pytest.mark.parametrize("dk", [20, 64, 96, 128])
@pytest.mark.parametrize("T", [30, 150])
@pytest.mark.parametrize("dt", TYPES)
def test_infinite_values(dev, dt, T, dk):
    """An infinity that is seen gives infinities of its sign, not NaN: fp32's products of three parts as well."""
    import svc_hip as S
    q, k, v, _ = _inputs(dev, TYPES[dt], 1, 2, 1, dk, T, T)
    v[0, 0, 17], v[0, 5, 3], v[0, 6, T - 1] = INF, -INF, INF
    v[0, 7] = 1.0                                                      # a part of 1.0 behind the first is 0
    v[0, 7, 4] = -INF
    want = _exact(q, k, v, 2, torch.ones(T, T, dtype=torch.bool))
    got = S.attention_scored(q, k, v, 2).double().cpu()
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not torch.isnan(got).any()
    hot = torch.isinf(want)
    assert torch.equal(got[hot], want[hot])
    u = max(torch.finfo(TYPES[dt]).eps / 2, 2.0 ** -24 * 8 * dk)
    # u for the result, u for P as an operand, of sums of |v| P with |v| < 6
    assert (got - want)[~hot].abs().max() <= 2 * u * 6
    # a training pass of a 16-bit type has P in several operands, whose rests are of either sign or 0: not finite at the same places, and the same elsewhere
    train = S.attention_scored_fwd(q, k, v, 2)[0].double().cpu()
    assert torch.equal(~torch.isfinite(train), hot) and (train - want)[~hot].abs().max() <= 2 * u * 6
    assert dt != "fp32" or torch.equal(train, got)


@pytest.mark.parametrize("T", [30, 150])
@pytest.mark.parametrize("dt", TYPES)
def test_infinite_keys(dev, dt, T):
    """A score of minus infinity is a key without weight: the other keys' rows, and dk and dv, are as if it were not there."""
    import svc_hip as S
    dt = TYPES[dt]
    q, k, v, do = _inputs(dev, dt, 1, 2, 1, 64, T, T)
    q[0, 2], q[0, 64 + 2] = q[0, 2].abs() + 0.5, q[0, 64 + 2].abs() + 0.5
    k[0, 2, 11] = -INF
    see = torch.ones(T, T, dtype=torch.bool)
    see[:, 11] = False
    want = _exact(q, k, v, 2, see)
    out, lse, dq, dk_, dv, _ = _pass(q, k, v, do, 2)
    u = max(torch.finfo(dt).eps / 2, 2.0 ** -24 * 8 * 64)
    for got in (out, S.attention_scored(q, k, v, 2)):
        assert (got.double().cpu() - want).abs().max() <= 2 * u * 6
    assert torch.isfinite(lse).all() and torch.isfinite(dk_).all() and torch.isfinite(dv).all()
    assert not dk_[0, :, 11].any() and not dv[0, :, 11].any()
    dq = dq.view(1, 2, 64, T)
    assert torch.isfinite(dq[:, :, :2]).all() and torch.isfinite(dq[:, :, 3:]).all()      # (channel 2: 0 * infinity)


def test_the_largest_fp32_values(dev):
    """A row of one key answers with its v, up to where the type ends: 3.399e38 rounds to infinity in bf16.  (P is 2 to the rounding of the maximum, some half
    steps from 1, and divided by itself; at the type's very last number a P of 1 + 2^-23 would overflow.)"""
    import svc_hip as S
    top = 3.399e38
    q, k, v, _ = _inputs(dev, torch.float32, 2, 2, 1, 48, 100, 100)
    v[0, :, 0], v[1, :, 0] = top, -top
    v[0, 3, 0], v[1, 4, 0] = 3.3e38, 2.0 ** 127
    n = torch.tensor([1, 1], dtype=torch.int32, device=dev)
    out = S.attention_scored(q, k, v, 2, lengths=n)
    for h in (out[:, :48, 0], out[:, 48:, 0]):
        assert ((h.double() - v[:, :, 0].double()).abs() <= 8 * 2.0 ** -24 * v[:, :, 0].double().abs()).all()
    assert not out[:, :, 1:].any()


@pytest.mark.parametrize("T", [50, 150])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("dt", TYPES)
def test_caps_far_above_the_scores_change_nothing(dev, dt, dk, T):
    """cap tanh(a / cap) = a - a^3 / 3 cap^2: at a cap of 2^20 and |a| < 8 that is 1e-10, so capped and uncapped calls agree to their roundings: twice u for
    the result, and twice u for P (for out) or for dS and D (for gradients), of the sums of absolute values."""
    from oracle import layer_oracle as O
    dt = TYPES[dt]
    q, k, v, do = _inputs(dev, dt, 1, 2, 1, dk, T, T)
    ref = O.attention(q, k, v, 2, dout=do)
    a, b = _pass(q, k, v, do, 2), _pass(q, k, v, do, 2, softcap=2.0 ** 20)
    u = max(torch.finfo(dt).eps / 2, 2.0 ** -24 * 8 * dk)
    for x, y, n, f in zip((a[0], *a[2:5]), (b[0], *b[2:5]), ("out", "dq", "dk", "dv"), (2, 4, 4, 2)):
        bound = 2 * u * ref[n].abs() + f * u * ref["mag_" + n] + 2.0 ** -24
        assert ((x.double() - y.double()).abs().cpu() <= bound).all(), n
        assert ((y.double().cpu() - ref[n]).abs() <= bound).all(), n


@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("size", [100.0, 12000.0])
def test_large_fp16_values_keep_the_gradients(dev, size, dk, p):
    """fp16 v of thousands: dS is far inside fp32, and its fp16 operand has to stay inside fp16.  Bounds as in tests/test_attention_scored_gpu.py, with the
    operand's steps among fp16's subnormals: it is scaled so that the largest |dO| lies in [1, 2), or, where that is less, so that 2 keep dk max |dO| max |v|
    lies between 32752 and 65504."""
    import svc_hip as S
    from oracle import layer_oracle as O
    q, k, v, do = _inputs(dev, torch.float16, 2, 4, 2, dk, 150, 150)
    v, do = (v.float() * size).clamp(-60000, 60000).half(), (do.sign() * 1.9 * 2.0 ** -10).half()
    kw = dict(draw=S.HashDraw(torch.tensor([3], device=dev), 1), p_drop=p) if p else {}
    ref = O.attention(q, k, v, 4, dout=do, **kw)
    got = _pass(q, k, v, do, 4, **kw)
    u = 2.0 ** -11
    f = 2.0 ** -24 * (4 * (dk + 8) * (1 + ref["score"]) + 150 + 64)
    top = lambda x: x.double().abs().max().item()  # noqa: E731
    allowed = 2 / (1 - p) * dk * top(do) * top(v)
    step = max(top(do), allowed / 32752) * 2.0 ** -25
    floor = {"out": 300 * 2.0 ** -33 * top(v), "dv": 300 * 2.0 ** -33 * top(do), "dq": 150 * step * top(k) * dk ** -0.5, "dk": 300 * step * top(q) * dk ** -0.5}
    for x, n, m in zip((got[0], *got[2:5]), ("out", "dq", "dk", "dv"), (1.0, 2.0, 2.0, 1.0)):
        assert torch.isfinite(x).all(), n
        bound = u * ref[n].abs() + m * (u + f) * ref["mag_" + n] + floor[n] + 2.0 ** -25
        worst = ((x.double().cpu() - ref[n]).abs() / bound).max().item()
        assert worst <= 1, (n, worst)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_saved_tensors_that_come_back_at_the_same_address_with_other_strides(dev, dt):
    """Hooks that move saved tensors away and back may be given the old memory again: the backward has to look at the strides, not at the address alone."""
    import svc_autograd as A
    B, C, T = 2, 64, 40
    dt = TYPES[dt]
    g = torch.Generator().manual_seed(1)
    hold = torch.randn(B, 2 * C, T, generator=g).to(dt).to(dev)              # q: the first half of the channels
    k, v, do = (torch.randn(B, C, T, generator=g).to(dt).to(dev) for _ in range(3))
    go = lambda q: (A.attention_scored(q, k, v, 2, causal=True), q)  # noqa: E731
    k.requires_grad_(), v.requires_grad_()
    y, q = go(hold[:, :C].clone().requires_grad_())
    want = torch.autograd.grad(y, (q, k, v), do)
    q = hold[:, :C].detach().requires_grad_()

    def pack(t):
        return (t.detach().clone(), True) if t.data_ptr() == q.data_ptr() else (t, False)

    def unpack(pair):
        t, moved = pair
        if not moved:
            return t
        back = hold.view(-1)[:B * C * T].view(B, C, T)                       # at its old address, contiguous
        back.copy_(t)
        hold[1] = 7.0                                                        # (the rest of the old memory is someone else's by now)
        return back

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        y, _ = go(q)
    got = torch.autograd.grad(y, (q, k, v), do)
    for a, b in zip(want, got):
        assert torch.equal(a, b)
