"""attention_scored on the GPU against the float64 definition (oracle/layer_oracle.py).

Bounds, element by element.  u = half a step of the type (2^-24, 2^-8, 2^-11: torch.finfo(t).eps / 2).  The score's relative error in P is at most
twice its absolute error: accumulating dk products in fp32 leaves dk + 8 half steps of sum |q||k| scale (`score`), the cap's tanh some half steps
of the cap, exponentials, sums over Tk keys and the final division one each: f = 2^-24 (4 (dk + 8)(1 + score) + 16 cap + Tk + 64).  With mag_x the
oracle's sum of absolute values behind x:
  out, dv: u |ref| (the result's rounding) + (u + f) mag (P's rounding as an operand).
  dq, dk: u |ref| + (2 u + 2 f) mag: dS is rounded once as an operand (u |dS| <= u mag), and it contains D = sum dO out, whose out is off by
    u mag_out from P's rounding: u sum |dO| mag_out, and mag holds P sum |dO| mag_out.
  dbias, an fp32 result: P goes into the out that D is made of in two operands at least (u^2 mag_out, and u^2 / 2 for the second operand's own
    rounding): (2 f + 2 u^2) mag.
  fp16 numbers below 2^-14 have steps of 2^-24.  P goes in multiplied by 2^8 (relative to the row's largest in the forward, as it is in the
    backward): at most 2^-33 of each entry more, so n 2^-33 max |v| (or |dO|) over n = max(Tq, Tk) entries, times the heads that share a key; the
    second operand of out32 the same, once more through D: Tk 2^-33 sum |dO||v| <= 2^-33 Tk mag / P, bounded by 2^-33 Tk n dk max |dO| max |v|.  dS
    goes in multiplied by 2^e with 2^e max |dO| in [1, 2) : at most 2^-25 max |dO| of each entry, n 2^-25 max |dO| max |k or q| scale.
(fp32: nothing is rounded to the type, and u counts as one more of f's half steps.)"""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def _i32(v, dev="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _inputs(dev, dt, B, H, G, dk, Tq, Tk, W=None, bias_heads=None, seed=0, gain=1.5):
    g = torch.Generator().manual_seed(seed + 31 * Tq + Tk + dk)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v, do = (gain * r(B, H * dk, Tq)).to(dt), r(B, G * dk, Tk).to(dt), r(B, G * dk, Tk).to(dt), r(B, H * dk, Tq).to(dt)
    bias = None if W is None else 0.7 * r(bias_heads or H, 2 * W + 1)
    return [None if t is None else t.to(dev) for t in (q, k, v, do, bias)]


def _check(got, ref, name, f, dt, factor=1.0, operands=1.0, rounded=True):
    u = torch.finfo(dt).eps / 2
    u = u if rounded else 2 * u * u
    r, mag = ref[name], ref["mag_" + name]
    x = got.detach().double().cpu()
    assert x.shape == r.shape, (name, x.shape, r.shape)
    assert torch.isfinite(x).all(), name
    bound = u * r.abs() + (operands * u + factor * f) * mag + 1e-30
    if dt == torch.float16:
        bound = bound + ref["floor"][name] + (2.0 ** -25 * 1.001 if rounded else 0.0)              # half a step among fp16's subnormals
    off = (x - r).abs()
    worst = (off / bound).max().item() if x.numel() else 0.0
    assert worst <= 1.0, (name, worst, off.max().item())
    return worst


def _f(ref, dk, Tk, cap):
    return 2.0 ** -24 * (4 * (dk + 8) * (1 + ref["score"]) + 16 * cap + Tk + 64)


def _both(dev, dt, B, H, G, dk, Tq, Tk, W=None, bias_heads=None, p=0.0, seed=0, train=True, gain=1.5, **kw):
    import svc_autograd as A
    import svc_hip as S
    q, k, v, do, bias = _inputs(dev, dt, B, H, G, dk, Tq, Tk, W, bias_heads, seed, gain)
    draw = S.HashDraw(torch.tensor([1234 + seed], dtype=torch.int64, device=dev), 5) if p else None
    on = {n: x.to(dev) if isinstance(x, torch.Tensor) else x for n, x in kw.items()}
    print(f"case {dt} B{B} H{H} G{G} dk{dk} Tq{Tq} Tk{Tk} W{W} p{p} {sorted(kw)}", flush=True)
    ref = O.attention(q, k, v, H, dout=do if train else None, bias=bias, draw=draw, p_drop=p, **kw)
    f = _f(ref, dk, Tk, kw.get("softcap", 0.0))
    if p == 0:
        _check(S.attention_scored(q, k, v, H, bias=bias, **on), ref, "out", f, dt)
    if not train:
        return
    leaves = [t.requires_grad_() for t in (q, k, v)] + ([bias.requires_grad_()] if bias is not None else [])
    out = A.attention_scored(q, k, v, H, bias=bias, draw=draw, p_drop=p, **on)
    grads = torch.autograd.grad(out, leaves, do)
    _check(out, ref, "out", f, dt)
    _check(grads[2], ref, "dv", f, dt)
    _check(grads[0], ref, "dq", f, dt, 2.0, 2.0)
    _check(grads[1], ref, "dk", f, dt, 2.0, 2.0)
    if bias is not None:
        _check(grads[3], ref, "dbias", f, dt, 2.0, rounded=False)


# (B, H, G, dk, Tq, Tk, W, options)
CASES = [
    (1, 1, 1, 32, 1, 1, None, {}),
    (1, 2, 2, 96, 1, 33, None, dict(causal=True)),
    (2, 4, 1, 64, 1, 200, 5, dict(causal=True, softcap=5.0)),
    (2, 2, 1, 17, 5, 70, 2, dict(causal=True, window=9)),
    (1, 1, 1, 128, 32, 32, None, {}),
    (1, 2, 2, 96, 64, 64, 0, dict(causal=True)),
    (2, 2, 2, 96, 129, 129, 40, {}),
    (1, 4, 2, 64, 257, 257, 300, dict(causal=True, softcap=3.0)),
    (1, 3, 1, 40, 190, 190, 7, dict(window=20)),
    (2, 2, 1, 33, 131, 131, None, dict(window=0)),
    (2, 2, 2, 128, 150, 150, 16, dict(causal=True, prefix=_i32([40, 0]))),
    (2, 2, 2, 80, 161, 161, 9, dict(causal=True, docs=_i32([[0, 30, 30, 140], [10, 64, 128, 150]]))),
    (2, 2, 1, 64, 161, 161, 33, dict(docs=_i32([[0, 100, 161], [0, 1, 2]]))),
    (2, 2, 1, 64, 161, 161, 33, dict(causal=True, docs=_i32([[0, 90, 161], [3, 70, 130]]), prefix=_i32([[20, 0], [500, 11]]))),
    (3, 2, 2, 96, 140, 140, 25, dict(lengths=_i32([140, 67, 0]))),
    (3, 2, 1, 48, 20, 300, 12, dict(causal=True, lengths=_i32([300, 100, 64]), offset=_i32([280, 80, 44]))),
    (2, 2, 2, 32, 40, 170, None, dict(causal=True, offset=3, scale=0.3)),
    (2, 2, 2, 64, 70, 90, 4, dict(lengths=_i32([80, 15]), window=30)),
]
IDS = [f"{c[:7]}-{'-'.join(sorted(c[7]))}" for c in CASES]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_against_float64(dev, case, dt):
    _both(dev, TYPES[dt], *case[:6], W=case[6], **case[7])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("p", [0.1, 0.5])
@pytest.mark.parametrize("case", [CASES[i] for i in (1, 3, 6, 7, 11, 14)], ids=[IDS[i] for i in (1, 3, 6, 7, 11, 14)])
def test_dropout_against_float64(dev, case, dt, p):
    _both(dev, TYPES[dt], *case[:6], W=case[6], p=p, seed=3, **case[7])


@pytest.mark.parametrize("dt", TYPES)
def test_table_shared_by_all_heads(dev, dt):
    _both(dev, TYPES[dt], 2, 4, 2, 64, 100, 100, W=30, bias_heads=1, causal=True)


@pytest.mark.parametrize("dt", TYPES)
def test_large_scores(dev, dt):
    """Scores of some +-100: rows with one key that matters, exponentials that underflow."""
    _both(dev, TYPES[dt], 1, 2, 2, 64, 200, 200, gain=30.0, causal=True)


def test_small_fp16_gradients_keep_their_precision(dev):
    """dO of 1e-3: dS is far among fp16's subnormals unless the kernel scales it."""
    import svc_hip as S
    q, k, v, do, _ = _inputs(dev, torch.float16, 1, 2, 2, 64, 300, 300)
    do = (do.float() * 1e-3).half()
    out, lse, o32 = S.attention_scored_fwd(q, k, v, 2)
    got = S.attention_scored_bwd(do, q, k, v, o32, lse, 2)
    ref = O.attention(q, k, v, 2, dout=do)
    f = _f(ref, 64, 300, 0.0)
    for x, n, m in zip(got, ("dq", "dk", "dv"), (2.0, 2.0, 1.0)):
        _check(x, ref, n, f, torch.float16, m, m)


@pytest.mark.parametrize("dt", TYPES)
def test_what_lies_at_unseen_keys_is_not_used(dev, dt):
    """NaN and infinities in unwritten cache, behind the last document, and in the queries there."""
    import svc_hip as S
    dt = TYPES[dt]
    q, k, v, do, bias = _inputs(dev, dt, 2, 2, 2, 64, 150, 150, 20)
    docs = _i32([[5, 60, 120], [0, 40, 90]], dev)
    clean = S.attention_scored_fwd(q, k, v, 2, bias=bias, docs=docs, want_dbias=True)
    cg = S.attention_scored_bwd(do, q, k, v, clean[0] if dt == torch.float32 else clean[2], clean[1], 2, bias=bias, docs=docs, want_dbias=True)
    bad = [t.clone() for t in (q, k, v, do)]
    for t, x in zip(bad, (float("nan"), float("inf"), float("nan"), float("-inf"))):
        t[0, :, :5], t[0, :, 120:], t[1, :, 90:] = x, x, x
    out = S.attention_scored_fwd(*bad[:3], 2, bias=bias, docs=docs, want_dbias=True)
    gr = S.attention_scored_bwd(bad[3], *bad[:3], out[0] if dt == torch.float32 else out[2], out[1], 2, bias=bias, docs=docs, want_dbias=True)
    for a, b in zip((clean[0], *cg), (out[0], *gr)):
        assert torch.equal(a, b)
    cache_k, cache_v = k.clone(), v.clone()
    cache_k[0, :, 70:], cache_v[0, :, 70:], cache_k[1, :, 33:], cache_v[1, :, 33:] = (float("nan"),) * 4
    n = _i32([70, 33], dev)
    one = S.attention_scored(q[:, :, :1], k, v, 2, causal=True, lengths=n, offset=n - 1)
    assert torch.equal(one, S.attention_scored(q[:, :, :1], cache_k, cache_v, 2, causal=True, lengths=n, offset=n - 1))


def test_rows_without_keys_are_zero_and_pass_nothing(dev):
    import svc_hip as S
    q, k, v, do, bias = _inputs(dev, torch.float32, 2, 2, 1, 32, 40, 40, 3)
    for kw in (dict(lengths=_i32([0, 0], dev)), dict(docs=_i32([[40, 40], [-5, 0]], dev)), dict(offset=_i32([40, -40], dev))):
        out, lse, _ = S.attention_scored_fwd(q, k, v, 2, bias=bias, **kw)
        grads = S.attention_scored_bwd(do, q, k, v, out, lse, 2, bias=bias, want_dbias=True, **kw)
        assert not out.any() and not any(g.any() for g in grads), kw


def test_offsets_out_of_every_range(dev):
    import svc_hip as S
    q, k, v, _, _ = _inputs(dev, torch.bfloat16, 4, 2, 1, 32, 4, 40)
    off = _i32([2 ** 31 - 1, -2 ** 31, 36, 10], dev)
    out = S.attention_scored(q, k, v, 2, causal=True, offset=off)
    assert not out[:2].any()
    assert torch.equal(out[2:], torch.cat([S.attention_scored(q[i:i + 1], k[i:i + 1], v[i:i + 1], 2, causal=True, offset=o) for i, o in ((2, 36), (3, 10))]))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("Tq", [1, 5, 70])
@pytest.mark.parametrize("dk", [1, 7, 9, 20, 33, 47, 65, 81, 97, 113])
def test_a_head_reads_its_own_channels_only(dev, dt, Tq, dk):
    """Head sizes between the built ones: the next head's channels (nan here) stand where a tile's rows behind dk would be."""
    import svc_hip as S
    g = torch.Generator().manual_seed(dk + Tq)
    q, k, v = (torch.randn(1, 2 * dk, T, generator=g).to(TYPES[dt]).to(dev) for T in (Tq, 90, 90))
    want = S.attention_scored(*(x[:, :dk].contiguous() for x in (q, k, v)), 1, causal=True)
    for x in (q, k, v):
        x[:, dk:] = float("nan")
    got = S.attention_scored(q, k, v, 2, causal=True)
    assert torch.equal(got[:, :dk], want)
    assert torch.isnan(got[:, dk:]).all()


@pytest.mark.parametrize("dt", TYPES)
def test_views_and_alignment(dev, dt):
    """q, k, v as channel slices of one projection and as time slices at odd starts, channels in reverse order of a larger tensor; out as a view whose
    surroundings stay as they were."""
    import svc_hip as S
    dt = TYPES[dt]
    T, dk = 77, 48
    q, k, v, _, _ = _inputs(dev, dt, 2, 2, 2, dk, T, T)
    want = S.attention_scored(q, k, v, 2, causal=True)
    qkv = torch.cat([q, k, v], 1)
    C = 2 * dk
    assert torch.equal(S.attention_scored(qkv[:, :C], qkv[:, C:2 * C], qkv[:, 2 * C:], 2, causal=True), want)
    for at in (1, 3, 8):
        big = torch.full((2, 3 * C, T + 11), float("nan"), device=dev, dtype=dt)
        big[:, :, at:at + T] = qkv
        w = big[:, :, at:at + T]
        hold = torch.full((2, C + 2, T + 9), 7.0, device=dev, dtype=dt)
        S.attention_scored(w[:, :C], w[:, C:2 * C], w[:, 2 * C:], 2, causal=True, out=hold[:, 1:C + 1, at:at + T])
        assert torch.equal(hold[:, 1:C + 1, at:at + T], want)
        hold[:, 1:C + 1, at:at + T] = 7.0
        assert (hold == 7.0).all()
    swapped = torch.stack([q[:, :dk], q[:, dk:]], 0)          # heads apart: batch and channel strides of another order
    assert torch.equal(S.attention_scored(q.transpose(0, 1).contiguous().transpose(0, 1), k, v, 2, causal=True), want) and swapped.numel()


def test_offsets_beyond_32_bits(dev):
    """A cache whose channels lie 2^26 elements apart: 64 channels reach past 2^32."""
    import svc_hip as S
    cs, T, dk = 1 << 26, 50, 64
    k0 = torch.empty((dk + 1) * cs, device=dev, dtype=torch.bfloat16)
    k = torch.as_strided(k0, (1, dk, T), (0, cs, 1), 11)
    q, kk, v, _, _ = _inputs(dev, torch.bfloat16, 1, 2, 1, dk, T, T)
    k.copy_(kk)
    assert torch.equal(S.attention_scored(q, k, v, 2, causal=True), S.attention_scored(q, kk, v, 2, causal=True))


def test_empty_calls(dev):
    import svc_hip as S
    z = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
    assert S.attention_scored(z(0, 8, 3), z(0, 8, 3), z(0, 8, 3), 2).shape == (0, 8, 3)
    assert S.attention_scored(z(2, 8, 0), z(2, 8, 5), z(2, 8, 5), 2).shape == (2, 8, 0)
    out, lse, _ = S.attention_scored_fwd(z(2, 8, 0), z(2, 8, 5), z(2, 8, 5), 2)
    g = S.attention_scored_bwd(z(2, 8, 0), z(2, 8, 0), z(2, 8, 5), z(2, 8, 5), out, lse, 2)
    assert g[1].shape == (2, 8, 5) and not g[1].any() and g[3] is None


@pytest.mark.parametrize("kw,what", [
    (dict(window=-1), "window"), (dict(prefix="b"), "prefix"), (dict(offset=3), "offset"), (dict(offset=-1), "offset"), (dict(bias="even"), "bias"),
    (dict(bias="heads"), "bias"), (dict(bias="half"), "bias"), (dict(lengths="long"), "lengths"), (dict(lengths="cpu"), "lengths"),
    (dict(docs="flat"), "docs"), (dict(docs="one"), "docs"), (dict(prefix="b", causal=True, window=3), "prefix"), (dict(prefix="n", causal=True), "prefix")])
def test_binding_refuses(dev, kw, what):
    import svc_hip as S
    q, k, v, _, _ = _inputs(dev, torch.float32, 2, 4, 2, 16, 8, 10)
    made = {"even": torch.zeros(4, 6, device=dev), "heads": torch.zeros(3, 5, device=dev), "half": torch.zeros(4, 5, device=dev).half(),
            "long": torch.zeros(2, device=dev, dtype=torch.long), "cpu": _i32([1, 1]), "flat": _i32([0, 5], dev), "one": _i32([[0], [0]], dev),
            "b": _i32([1, 1], dev), "n": _i32([[1, 1], [1, 1]], dev)}
    with pytest.raises(S.SvcError, match=what):
        S.attention_scored(q, k, v, 4, **{n: made[x] if isinstance(x, str) else x for n, x in kw.items()})


def test_binding_refuses_shapes_and_types(dev):
    import svc_autograd as A
    import svc_hip as S
    q, k, v, _, _ = _inputs(dev, torch.float32, 2, 4, 2, 16, 8, 10)
    for bad in ((q, k, v, 5), (q, k, v, 0), (q, k[:, :24], v[:, :24], 4), (q, k, v[:, :, :9], 4), (k.repeat(1, 2, 1), q[:, :32], q[:, :32], 4), (q[:1], k, v, 4),
                (q, k.half(), v, 4), (q.transpose(1, 2), k, v, 4), (q.repeat(1, 5, 1)[:, :258], k, v, 2)):
        with pytest.raises(S.SvcError):
            S.attention_scored(*bad)
    with pytest.raises(S.SvcError, match="HashDraw"):
        A.attention_scored(q, k, v, 4, p_drop=0.1)
    with pytest.raises(S.SvcError, match="rate"):
        A.attention_scored(q, k, v, 4, p_drop=1.0, draw=S.HashDraw(torch.zeros(1, dtype=torch.int64, device=dev), 0))


def test_two_runs_are_bit_equal(dev):
    import svc_hip as S
    q, k, v, do, bias = _inputs(dev, torch.bfloat16, 2, 4, 2, 64, 300, 300, 50)
    draw = S.HashDraw(torch.tensor([5], device=dev), 1)
    kw = dict(bias=bias, causal=True, draw=draw, p_drop=0.2, want_dbias=True)
    runs = []
    for _ in range(2):
        out, lse, o32 = S.attention_scored_fwd(q, k, v, 4, **kw)
        runs.append((out, lse, *S.attention_scored_bwd(do, q, k, v, o32, lse, 4, **kw)))
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", ["fp32", "bf16"])
def test_captured_and_replayed(dev, dt):
    """Forward and backward in one graph, replayed on new data between eager work; two graphs at once."""
    import svc_hip as S
    dt = TYPES[dt]
    data = [_inputs(dev, dt, 2, 4, 2, 64, 130, 130, 9, seed=s) for s in range(3)]
    n = _i32([130, 90], dev)

    def step(q, k, v, do, bias):
        out, lse, o32 = S.attention_scored_fwd(q, k, v, 4, bias=bias, causal=True, lengths=n, want_dbias=True)
        return (out, *S.attention_scored_bwd(do, q, k, v, out if o32 is None else o32, lse, 4, bias=bias, causal=True, lengths=n, want_dbias=True))

    want = [step(*d) for d in data]
    held = [[t.clone() for t in data[0]] for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for h in held:
            step(*h)
    torch.cuda.synchronize()
    for h in held:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(step(*h))
        graphs.append(gr)
    for i in (1, 2, 0, 1):
        for h, j in zip(held, (i, (i + 1) % 3)):
            for t, s in zip(h, data[j]):
                t.copy_(s)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        junk = torch.randn(1000, 1000, device=dev) @ torch.randn(1000, 1000, device=dev)  # noqa: F841
        for o, j in zip(outs, (i, (i + 1) % 3)):
            for a, b in zip(o, want[j]):
                assert torch.equal(a, b)


def test_other_streams(dev):
    import svc_hip as S
    q, k, v, _, _ = _inputs(dev, torch.float16, 2, 4, 4, 64, 200, 200)
    want = S.attention_scored(q, k, v, 4, causal=True)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append(S.attention_scored(q, k, v, 4, causal=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_chunks_and_single_steps_equal_the_whole(dev):
    """A causal sequence written into a cache in chunks, then position by position: each call's rows are the whole call's."""
    import svc_hip as S
    B, H, G, dk, T = 2, 4, 2, 64, 90
    q, k, v, _, bias = _inputs(dev, torch.float32, B, H, G, dk, T, T, 20)
    whole = S.attention_scored(q, k, v, H, causal=True, bias=bias)
    ck, cv = (torch.full((B, G * dk, 128), float("nan"), device=dev) for _ in range(2))
    at = 0
    for n in (40, 33, 1, 1, 1, 14):
        ck[:, :, at:at + n], cv[:, :, at:at + n] = k[:, :, at:at + n], v[:, :, at:at + n]
        got = S.attention_scored(q[:, :, at:at + n], ck, cv, H, causal=True, bias=bias, lengths=_i32([at + n] * B, dev), offset=_i32([at] * B, dev))
        # both are within f of the definition (module docstring); |v| < 6 here
        assert (got - whole[:, :, at:at + n]).abs().max() < 2 * 2.0 ** -24 * (4 * 72 * 40 + 90 + 64) * 6
        at += n


def test_gradient_against_differences(dev):
    """Directional differences of the fp32 forward itself: step 2^-6 along a random direction, truncation error measured by halving the step."""
    import svc_hip as S
    B, H, G, dk, T = 1, 2, 1, 32, 48
    q, k, v, do, bias = _inputs(dev, torch.float32, B, H, G, dk, T, T, 6)
    kw = dict(softcap=4.0, causal=True)
    out, lse, _ = S.attention_scored_fwd(q, k, v, H, bias=bias, **kw)
    grads = S.attention_scored_bwd(do, q, k, v, out, lse, H, bias=bias, want_dbias=True, **kw)
    g = torch.Generator().manual_seed(8)
    way = [torch.randn(t.shape, generator=g).to(dev) for t in (q, k, v, bias)]
    f = lambda e: (S.attention_scored(*[t + e * w for t, w in zip((q, k, v), way)], H, bias=bias + e * way[3], **kw).double() * do.double()).sum().item()  # noqa: E731
    d1, d2 = ((f(e) - f(-e)) / (2 * e) for e in (2.0 ** -6, 2.0 ** -7))
    want = sum((x.double() * w.double()).sum().item() for x, w in zip(grads, way))
    # d2 is off by about (d1 - d2) / 3 (third-order term), plus rounding: some 1e-6 of sum |out||do| over 2 e
    assert abs(d2 - want) < abs(d1 - d2) + 1e-6 * (out.abs() * do.abs()).sum().item() * 64


def test_zero_dim_gradients_of_expanded_output(dev):
    """out.sum(): the incoming gradient is an expanded scalar."""
    import svc_autograd as A
    q, k, v, _, _ = _inputs(dev, torch.float32, 1, 2, 2, 32, 20, 20)
    q, k, v = (t.requires_grad_() for t in (q, k, v))
    a = torch.autograd.grad(A.attention_scored(q, k, v, 2).sum(), (q, k, v))
    b = torch.autograd.grad(A.attention_scored(q, k, v, 2), (q, k, v), torch.ones_like(q))
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("low", [-65504.0, -1e9, float(torch.finfo(torch.float32).min), float("-inf")])
@pytest.mark.parametrize("dt", TYPES)
def test_lowest_values_in_the_table_mask_their_distance(dev, dt, low):
    """A table that masks distances beyond 3, some of its heads' every distance: rows with nothing left are 0 and pass nothing, as single steps too."""
    import svc_hip as S
    dt = TYPES[dt]
    q, k, v, do, bias = _inputs(dev, dt, 2, 2, 1, 64, 100, 100, 8)
    bias[:, :5], bias[:, 12:] = low, low
    bias[1] = low
    out, lse, o32 = S.attention_scored_fwd(q, k, v, 2, bias=bias, want_dbias=True)
    grads = S.attention_scored_bwd(do, q, k, v, out if o32 is None else o32, lse, 2, bias=bias, want_dbias=True)
    ref = O.attention(q, k, v, 2, dout=do, bias=bias)
    f = _f(ref, 64, 100, 0.0)
    for x, n, m in zip((out, *grads), ("out", "dq", "dk", "dv", "dbias"), (1.0, 2.0, 2.0, 1.0, 2.0)):
        _check(x, ref, n, f, dt, m, m, rounded=n != "dbias")
    assert not out[:, 64:].any() and not grads[3][1].any()
    one = S.attention_scored(q[:, :, 99:], k, v, 2, bias=bias)
    _check(one, {n: x[:, :, 99:] if isinstance(x, torch.Tensor) and n.endswith("out") else x for n, x in ref.items()}, "out", f, dt)


@pytest.mark.parametrize("dt", ["fp32", "fp16"])
def test_autograd_captured_and_replayed(dev, dt):
    """A training pass through autograd in a graph (leaves made for it alone), replayed on new data."""
    import svc_autograd as A
    import svc_hip as S
    dt = TYPES[dt]
    seed = torch.tensor([1], dtype=torch.int64, device=dev)
    draw = S.HashDraw(seed, 2)

    def step(t):
        return torch.autograd.grad(A.attention_scored(*t[:3], 4, bias=t[4], causal=True, draw=draw, p_drop=0.1), (*t[:3], t[4]), t[3])

    def leaves(s):
        return [x.requires_grad_(i != 3) for i, x in enumerate(_inputs(dev, dt, 2, 4, 2, 64, 90, 90, 7, seed=s))]

    want = {}
    for s in (0, 1):
        seed.fill_(s)
        want[s] = [x.clone() for x in step(leaves(s))]
    held = leaves(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        got = step(held)
    for s in (1, 0, 1):
        seed.fill_(s)
        with torch.no_grad():
            for h, x in zip(held, leaves(s)):
                h.copy_(x)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[s]))


def test_second_derivatives_are_refused_and_gradients_are_per_input(dev):
    import svc_autograd as A
    q, k, v, _, bias = _inputs(dev, torch.float32, 1, 2, 2, 32, 20, 20, 3)
    q.requires_grad_()
    g, = torch.autograd.grad(A.attention_scored(q, k, v, 2, bias=bias).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
    bias.requires_grad_()
    only, = torch.autograd.grad(A.attention_scored(q.detach(), k, v, 2, bias=bias).sum(), bias)
    assert only.shape == bias.shape
