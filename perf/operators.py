"""Measured cases of the transformer-layer operators on [B, C, T] tensors:

  attention   svc_autograd.attention_scored / svc_hip.attention_scored: attention with a tanh cap, a distance bias, causal / prefix /
              document / window masks, ragged lengths and counter-based dropout; training pass, forward pass, chunk and single
              token over a cache
  norm        svc_autograd.dropout_add_layernorm / svc_hip.dropout_add_layernorm: y = LN_C(r + dropout(x)) * gamma + beta, masked;
              training pass and forward pass

`own` chooses between the elementary torch form (False) and the framework's kernels (True); both take the same state."""
import math
import os
import sys

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SITE = 3      # the dropout site's number
# the generator's constants as signed 64-bit numbers: the site's start, the counter's step, two mixing factors
START, STEP, MIX1, MIX2 = (v - (1 << 64) if v >> 63 else v for v in
                           ((SITE + 1) * 0x9E3779B97F4A7C15 % (1 << 64), 0xD1B54A32D192ED03, 0xBF58476D1CE4E5B9, 0x94D049BB133111EB))


def _att(name, dtype, B, H, G, dk, Tq, Tk, train=False, causal=True, prefix=0, docs=0, window=0, cap=0.0, bias=0, ragged=False, p=0.0):
    return {"name": name, "op": "attention", "dtype": dtype, "B": B, "H": H, "G": G, "dk": dk, "Tq": Tq, "Tk": Tk, "train": train,
            "causal": causal, "prefix": prefix, "docs": docs, "window": window, "cap": cap, "bias": bias, "ragged": ragged, "p": p}


def _norm(name, dtype, B, C, T, train=False, p=0.0, mask=True):
    return {"name": name, "op": "norm", "dtype": dtype, "B": B, "C": C, "T": T, "train": train, "p": p, "mask": mask}


def listed():
    return [
        # one frame of a streaming causal stack (2 heads x 96, the F0 decoder's shape) over a 10 s cache: a latency
        _att("step_fp32", "fp32", 1, 2, 2, 96, 1, 862),
        # one token for each of 16 streams over long caches of different fill, four query heads to a key head, capped scores: bandwidth
        _att("step_long_bf16", "bf16", 16, 16, 4, 128, 1, 8191, cap=30.0, ragged=True),
        # a chunk of frames appended to a cache, look-back limited, learned distance bias
        _att("chunk_fp16", "fp16", 4, 12, 12, 64, 37, 1500, window=200, bias=64),
        # prompt with a bidirectional prefix, capped scores, shared key heads
        _att("prompt_prefix_bf16", "bf16", 4, 16, 4, 128, 2049, 2049, prefix=500, cap=50.0),
        # training step of the 2 x 96 encoder on a ragged batch: bidirectional, distance bias with its gradient, attention dropout
        _att("train_ragged_fp32", "fp32", 16, 2, 2, 96, 790, 790, train=True, causal=False, bias=100, ragged=True, p=0.1),
        # packed rows of several utterances (12 x 64 unit-encoder heads), causal inside each document, bias and dropout
        _att("train_docs_bf16", "bf16", 2, 12, 12, 64, 4099, 4099, train=True, docs=9, bias=128, p=0.1),
        # local attention of a 30 s clip, shared key heads, bias
        _att("train_window_fp16", "fp16", 8, 12, 4, 64, 1501, 1501, train=True, causal=False, window=128, bias=128),
        # the largest: long causal rows with capped scores
        _att("train_long_bf16", "bf16", 4, 16, 4, 128, 4096, 4096, train=True, cap=30.0),
        # the residual junction of one clip at inference (192 channels, 862 frames): a latency
        _norm("junction_fp32", "fp32", 1, 192, 862),
        # the junction of a training batch of the 192-channel encoder
        _norm("train_junction_fp32", "fp32", 16, 192, 790, train=True, p=0.1),
        # 768 channels, 32 clips of 30 s
        _norm("train_junction_bf16", "bf16", 32, 768, 1499, train=True, p=0.1),
        # an odd width without dropout
        _norm("train_junction_odd_fp16", "fp16", 8, 1001, 2047, train=True, mask=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    kind = rng.choice(["step", "chunk", "prompt", "train", "train", "norm", "norm"])
    if kind == "norm":
        B, C = _log_int(rng, 1, 32), _log_int(rng, 33, 1025)
        T = min(_log_int(rng, 5, 4000), 36000000 // (B * C))
        train = rng.random() < 0.7
        c = _norm("", dtype, B, C, T, train, rng.choice([0.0, 0.1, 0.25]) if train else 0.0, rng.random() < 0.5)
    else:
        G = rng.choice([1, 2, 4, 6])
        H = G * rng.choice([1, 1, 2, 4])
        dk = rng.choice([32, 40, 64, 80, 96, 128, rng.randint(17, 128)])
        more = dict(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.choice([0, 0, 16, 100, 300]), ragged=rng.random() < 0.4)
        if kind == "step":
            c = _att("", dtype, _log_int(rng, 1, 16), H, G, dk, rng.choice([1, 1, 1, 4]), _log_int(rng, 60, 8000), window=rng.choice([0, 0, 300]), **more)
        elif kind == "chunk":
            c = _att("", dtype, _log_int(rng, 1, 8), H, G, dk, rng.randint(9, 100), _log_int(rng, 110, 4000), window=rng.choice([0, 0, 300]), **more)
        else:
            train = kind == "train"
            causal = rng.random() < 0.6
            form = rng.choice(["plain", "docs", "window", "prefix" if causal else "plain"])
            T = _log_int(rng, 40, 2400)
            B = max(1, min(_log_int(rng, 1, 16), int(4e7 / (H * T * T))))
            c = _att("", dtype, B, H, G, dk, T, T, train=train, causal=causal, docs=rng.randint(2, 9) if form == "docs" else 0,
                     window=rng.randint(4, 200) if form == "window" else 0, prefix=rng.randint(1, T) if form == "prefix" else 0,
                     p=rng.choice([0.0, 0.0, 0.1, 0.2]) if train else 0.0, **more)
            if c["docs"]:
                c["ragged"] = False
    del c["name"]
    return c


def _lengths(c, roll=0):
    """Valid keys of each item: all, or from the whole cache down to about half of it; at least the queries of a call."""
    if not c["ragged"]:
        return None
    n = [max(c["Tk"] - (b * c["Tk"]) // (2 * c["B"]), c["Tq"] if c["Tq"] < c["Tk"] else 1) for b in range(c["B"])]
    return n[roll % len(n):] + n[:roll % len(n)]


def _bounds(c, roll=0):
    """Document boundaries of a packed row: documents of different lengths, the last 1/64 of the row behind the last of them."""
    if not c["docs"]:
        return None
    N, end = c["docs"], c["Tk"] - c["Tk"] // 64
    cut = [0] + [end * (i + 1) * (i + 3) // (N * (N + 2)) for i in range(N)]
    size = [b - a for a, b in zip(cut, cut[1:])]
    rows = []
    for b in range(c["B"]):
        r = (roll + b) % N
        at = [0]
        for n in size[r:] + size[:r]:
            at.append(at[-1] + n)
        rows.append(at)
    return rows


def prepare(case, seed):
    c = dict(case)
    dev, dt = torch.device("cuda"), DTYPES[c["dtype"]]
    g = torch.Generator(device=dev)
    g.manual_seed(1000003 * seed + 17)
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev)  # noqa: E731
    s = {"case": c, "seed": torch.tensor([seed * 7919 + 12345], dtype=torch.int64, device=dev)}
    if c["op"] == "norm":
        s["x"] = (0.7 * normal(c["B"], c["C"], c["T"])).to(dt)
        s["r"] = (normal(c["B"], c["C"], c["T"]) + 0.3 * normal(1, c["C"], 1)).to(dt)
        s["gamma"], s["beta"] = 1 + 0.1 * normal(c["C"]), 0.1 * normal(c["C"])
        s["mask"] = None
        if c["mask"]:       # frames behind the end of each clip
            n = torch.tensor([max(1, c["T"] - b * c["T"] // (2 * c["B"])) for b in range(c["B"])], device=dev)
            s["mask"] = (torch.arange(c["T"], device=dev) < n[:, None]).float()
        s["dy"] = normal(c["B"], c["C"], c["T"]).to(dt) if c["train"] else None
        return s
    s["q"] = (2.5 * normal(c["B"], c["H"] * c["dk"], c["Tq"])).to(dt)
    s["k"] = normal(c["B"], c["G"] * c["dk"], c["Tk"]).to(dt)
    s["v"] = normal(c["B"], c["G"] * c["dk"], c["Tk"]).to(dt)
    s["bias"] = 0.5 * normal(c["H"], 2 * c["bias"] + 1) if c["bias"] else None
    s["dout"] = normal(c["B"], c["H"] * c["dk"], c["Tq"]).to(dt) if c["train"] else None
    whole = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    s["lengths"] = whole(_lengths(c, seed))
    s["docs"] = whole(_bounds(c, seed))
    s["prefix"] = whole([max(0, c["prefix"] - 3 * b) for b in range(c["B"])]) if c["prefix"] else None
    s["offset"] = s["lengths"] - c["Tq"] if c["ragged"] and c["Tq"] < c["Tk"] else None      # the newest Tq positions of each cache
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------

def _words(seed, n):
    """The counter-based generator's 64-bit words for counters 0..n-1, as int64."""
    shift = lambda z, k: (z >> k) & ((1 << (64 - k)) - 1)  # noqa: E731
    z = torch.arange(n, dtype=torch.int64, device=seed.device) * STEP + (seed + START)
    z = (z ^ shift(z, 30)) * MIX1
    z = (z ^ shift(z, 27)) * MIX2
    return z ^ shift(z, 31)


def _attention_keep(s):
    """Keep factors [B, H, Tq, Tk] of the attention dropout: four 16-bit fields of a word for four neighbouring keys."""
    c = s["case"]
    rows, groups = c["B"] * c["H"] * c["Tq"], (c["Tk"] + 3) // 4
    words = _words(s["seed"], rows * groups).view(rows, groups, 1)
    fields = (words >> torch.tensor([0, 16, 32, 48], device=words.device)) & 0xFFFF
    threshold = int(round(c["p"] * 65536))
    keep = fields.reshape(rows, groups * 4)[:, :c["Tk"]] >= threshold
    return (keep.float() * (1.0 / (1.0 - threshold / 65536.0))).view(c["B"], c["H"], c["Tq"], c["Tk"])


def _visible(s):
    """Which keys each query sees, [B, 1, Tq, Tk], and the distance of key and query, [B or 1, Tq, Tk]."""
    c, dev = s["case"], s["q"].device
    key = torch.arange(c["Tk"], device=dev)
    offset = s["offset"][:, None].long() if s["offset"] is not None else torch.full((c["B"], 1), c["Tk"] - c["Tq"], device=dev)
    at = (offset + torch.arange(c["Tq"], device=dev))[:, :, None]
    length = s["lengths"][:, None, None].long() if s["lengths"] is not None else c["Tk"]
    see = (key < length) & (at >= 0) & (at < length)
    if c["docs"]:
        inner = s["docs"][:, None, None, :].long()
        of_key, of_query = (inner <= key[:, None]).sum(-1), (inner <= at[..., None]).sum(-1)
        see = see & (of_key == of_query) & (of_query > 0) & (of_query <= c["docs"])
    if c["causal"]:
        ahead = key <= at
        see = see & (ahead | (key < s["prefix"][:, None, None]) if c["prefix"] else ahead)
    if c["window"]:
        see = see & ((key - at).abs() <= c["window"])
    return see[:, None], key - at


def _plain_attention(s):
    c = s["case"]
    B, H, G, dk, Tq, Tk = (c[k] for k in ("B", "H", "G", "dk", "Tq", "Tk"))
    scale = dk ** -0.5
    q = s["q"].float().view(B, H, dk, Tq)
    k = s["k"].float().view(B, G, dk, Tk)
    v = s["v"].float().view(B, G, dk, Tk)
    k, v = (x.repeat_interleave(H // G, 1) if G != H else x for x in (k, v))
    see, distance = _visible(s)
    a = torch.matmul(q.transpose(2, 3).contiguous(), k) * scale
    th = None
    if c["cap"]:
        th = torch.tanh(a / c["cap"])
        a = th * c["cap"]
    if c["bias"]:
        bin_of = distance.clamp(-c["bias"], c["bias"]) + c["bias"]          # [B, Tq, Tk]
        a = a + s["bias"][:, bin_of].transpose(0, 1)
    a = a.masked_fill(~see, -math.inf)
    top = a.amax(-1, keepdim=True)
    e = torch.exp(a - top.masked_fill(top == -math.inf, 0.0))
    total = e.sum(-1, keepdim=True)
    P = e / total.masked_fill(total == 0, 1.0)
    keep = _attention_keep(s) if c["p"] else None
    Pz = P * keep if c["p"] else P
    out = torch.matmul(v, Pz.transpose(2, 3).contiguous())
    dt = s["q"].dtype
    res = {"out": out.reshape(B, H * dk, Tq).to(dt)}
    if not c["train"]:
        return res
    do = s["dout"].float().view(B, H, dk, Tq)
    dv = torch.matmul(do, Pz)
    dP = torch.matmul(do.transpose(2, 3).contiguous(), v)
    if c["p"]:
        dP = dP * keep
    dS = P * (dP - (P * dP).sum(-1, keepdim=True))
    if c["bias"]:
        # rows from the last backwards, each one place further right than the one before: a column holds one distance
        flipped = torch.nn.functional.pad(dS.sum(0).flip(1), (0, Tq)).reshape(H, -1)[:, :Tq * (Tk + Tq - 1)]
        diagonal = flipped.view(H, Tq, Tk + Tq - 1).sum(1)                 # column j: s - t = j - (Tq - 1)
        W = c["bias"]
        at = (torch.arange(Tk + Tq - 1, device=dS.device) - (Tq - 1) - (Tk - Tq)).clamp(-W, W) + W
        res["dbias"] = torch.matmul(diagonal, (at[:, None] == torch.arange(2 * W + 1, device=dS.device)).float())
    if c["cap"]:
        dS = dS * (1 - th * th)
    dq = torch.matmul(k, dS.transpose(2, 3).contiguous()) * scale
    dk_ = torch.matmul(q, dS) * scale
    res["dq"] = dq.reshape(B, H * dk, Tq).to(dt)
    res["dk"], res["dv"] = (x.view(B, G, H // G, dk, Tk).sum(2).reshape(B, G * dk, Tk).to(dt) for x in (dk_, dv))
    return res


def _norm_keep(s):
    c = s["case"]
    u = ((_words(s["seed"], s["x"].numel()) >> 40) & 0xFFFFFF).float() * (1.0 / 16777216.0)
    return ((u >= c["p"]).float() / (1.0 - c["p"])).view(s["x"].shape)


def _plain_norm(s):
    c, dt = s["case"], s["x"].dtype
    keep = _norm_keep(s) if c["p"] else None
    x = s["x"].float() * keep if c["p"] else s["x"].float()
    h = s["r"].float() + x
    gamma, beta = s["gamma"][:, None], s["beta"][:, None]
    d = h - h.mean(1, keepdim=True)
    rs = torch.rsqrt((d * d).mean(1, keepdim=True) + 1e-5)
    xh = d * rs
    y = xh * gamma + beta
    if c["mask"]:
        y = y * s["mask"][:, None]
    res = {"y": y.to(dt)}
    if not c["train"]:
        return res
    dy = s["dy"].float() * s["mask"][:, None] if c["mask"] else s["dy"].float()
    g = dy * gamma
    dh = rs * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    res["dr"] = dh.to(dt)
    res["dx"] = (dh * keep).to(dt) if c["p"] else res["dr"]
    res["dgamma"], res["dbeta"] = (dy * xh).sum((0, 2)), dy.sum((0, 2))
    return res


# ---- the framework's calls ---------------------------------------------------------------------------------------------

def _engine():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "so-vits-svc_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import svc_autograd
    import svc_hip
    return svc_autograd, svc_hip


def _own_attention(s):
    A, S = _engine()
    c = s["case"]
    more = dict(bias=s["bias"], softcap=c["cap"], causal=c["causal"], window=c["window"] or None, prefix=s["prefix"], docs=s["docs"],
                lengths=s["lengths"], offset=s["offset"])
    if not c["train"]:
        return {"out": S.attention_scored(s["q"], s["k"], s["v"], c["H"], **more)}
    q, k, v = (s[n].detach().requires_grad_() for n in "qkv")
    leaves = [q, k, v]
    if c["bias"]:
        more["bias"] = s["bias"].detach().requires_grad_()
        leaves.append(more["bias"])
    out = A.attention_scored(q, k, v, c["H"], draw=S.HashDraw(s["seed"], SITE) if c["p"] else None, p_drop=c["p"], **more)
    grads = torch.autograd.grad(out, leaves, s["dout"])
    res = {"out": out.detach(), "dq": grads[0], "dk": grads[1], "dv": grads[2]}
    if c["bias"]:
        res["dbias"] = grads[3]
    return res


def _own_norm(s):
    A, S = _engine()
    c = s["case"]
    if not c["train"]:
        return {"y": S.dropout_add_layernorm(s["x"], s["r"], s["gamma"], s["beta"], mask=s["mask"])}
    x, r, gamma, beta = (s[n].detach().requires_grad_() for n in ("x", "r", "gamma", "beta"))
    y = A.dropout_add_layernorm(x, r, gamma, beta, draw=S.HashDraw(s["seed"], SITE) if c["p"] else None, p=c["p"], mask=s["mask"])
    dx, dr, dgamma, dbeta = torch.autograd.grad(y, (x, r, gamma, beta), s["dy"])
    return {"y": y.detach(), "dr": dr, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def run(state):
    if own:
        return _own_norm(state) if state["case"]["op"] == "norm" else _own_attention(state)
    with torch.no_grad():
        return _plain_norm(state) if state["case"]["op"] == "norm" else _plain_attention(state)


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def _pairs(c):
    """Visible (query, key) pairs of one head over the batch, and the keys that some query sees."""
    lengths = torch.tensor(_lengths(c) or [c["Tk"]] * c["B"])[:, None]
    first = lengths - c["Tq"] if c["ragged"] and c["Tq"] < c["Tk"] else torch.full((c["B"], 1), c["Tk"] - c["Tq"])
    at = first + torch.arange(c["Tq"])
    lo, hi = torch.zeros_like(at), lengths.expand_as(at).clone()
    inside = (at >= 0) & (at < lengths)
    if c["docs"]:
        bounds = torch.tensor(_bounds(c))
        n = torch.searchsorted(bounds, at, right=True)
        inside &= n <= c["docs"]
        n = n.clamp(1, c["docs"])
        lo, hi = torch.maximum(lo, bounds.gather(1, n - 1)), torch.minimum(hi, bounds.gather(1, n))
    if c["causal"]:
        ahead = torch.maximum(at + 1, torch.tensor([[max(0, c["prefix"] - 3 * b)] for b in range(c["B"])]))
        hi = torch.minimum(hi, ahead)
    if c["window"]:
        lo, hi = torch.maximum(lo, at - c["window"]), torch.minimum(hi, at + c["window"] + 1)
    n = ((hi - lo).clamp(min=0) * inside).sum().item()
    lo, hi = lo.masked_fill(~inside, c["Tk"]), hi.masked_fill(~inside, 0)
    return n, (hi.amax(1) - lo.amin(1)).clamp(min=0).sum().item()


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    if c["op"] == "norm":
        n = c["B"] * c["C"] * c["T"]
        # x, r in, y out; a training pass adds dy in and dr out, and dx where dropout makes it another tensor
        passes = 3 + ((3 if c["p"] else 2) if c["train"] else 0)
        return {"bytes": float(n * size * passes + c["C"] * 8), "flops": float(n * (24 if c["train"] else 9))}
    pairs, keys = _pairs(c)
    rows, kv = c["B"] * c["H"] * c["dk"] * c["Tq"], c["G"] * c["dk"] * keys
    moved = 2 * rows + 2 * kv
    flops = 4.0 * pairs * c["H"] * c["dk"]
    if c["train"]:
        moved += 2 * rows + 2 * kv
        flops += 10.0 * pairs * c["H"] * c["dk"]
    return {"bytes": float(moved * size + 4 * c["H"] * (2 * c["bias"] + 1)), "flops": flops}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def _uniform_words(state, counters):
    """The generator's words at the given counters by 32-bit halves (no 64-bit wrap-around arithmetic)."""
    M = 0xFFFFFFFF

    def times(hi, lo, k):
        kh, kl = (k >> 32) & M, k & M
        a, b = (lo & 0xFFFF) * kl, (lo >> 16) * kl
        low = a + ((b & 0xFFFF) << 16)
        carry = (low >> 32) + (b >> 16)
        high = (carry + ((hi & 0xFFFF) * kl + (((hi >> 16) * kl & 0xFFFF) << 16)) + ((lo & 0xFFFF) * kh + (((lo >> 16) * kh & 0xFFFF) << 16))) & M
        return high, low & M

    def xor_shift(hi, lo, k):
        return hi ^ (hi >> k), lo ^ (((lo >> k) | (hi << (32 - k))) & M)

    start = (int(state["seed"].item()) + (SITE + 1) * 0x9E3779B97F4A7C15) & 0xFFFFFFFFFFFFFFFF
    hi, lo = times(counters >> 32, counters & M, 0xD1B54A32D192ED03)
    lo = lo + (start & M)
    hi = (hi + (start >> 32) + (lo >> 32)) & M
    lo = lo & M
    hi, lo = times(*xor_shift(hi, lo, 30), 0xBF58476D1CE4E5B9)
    hi, lo = times(*xor_shift(hi, lo, 27), 0x94D049BB133111EB)
    return xor_shift(hi, lo, 31)


def _exact_head(s, b, h, q, k, v, bias):
    """One head of one item from the definition, in float64: out [dk, Tq]."""
    c, dev = s["case"], q.device
    first = int(s["offset"][b]) if s["offset"] is not None else c["Tk"] - c["Tq"]
    length = int(s["lengths"][b]) if s["lengths"] is not None else c["Tk"]
    p, t = torch.arange(c["Tq"], device=dev) + first, torch.arange(c["Tk"], device=dev)
    gap = t[None, :] - p[:, None]
    hidden = (t[None, :] >= length) | (p[:, None] < 0) | (p[:, None] >= length)
    if c["docs"]:
        number = torch.full((c["Tk"],), -1, device=dev)
        edges = s["docs"][b].tolist()
        for n in range(c["docs"]):
            number[edges[n]:edges[n + 1]] = n
        mine = number[p.clamp(0, c["Tk"] - 1)]
        hidden = hidden | (mine[:, None] != number[None, :]) | (mine[:, None] < 0)
    if c["causal"]:
        front = int(s["prefix"][b]) if c["prefix"] else 0
        hidden = hidden | ((gap > 0) & (t[None, :] >= front))
    if c["window"]:
        hidden = hidden | (gap > c["window"]) | (gap < -c["window"])
    score = q.t() @ k / math.sqrt(c["dk"])
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    if c["bias"]:
        W = c["bias"]
        score = score + bias[gap.clamp(-W, W) + W]
    none = hidden.all(1, keepdim=True)
    prob = torch.softmax(score.masked_fill(hidden & ~none, -math.inf), 1).masked_fill(none, 0.0)
    if c["p"]:
        groups = (c["Tk"] + 3) // 4
        row = (b * c["H"] + h) * c["Tq"] + torch.arange(c["Tq"], device=dev)
        hi, lo = _uniform_words(s, row[:, None] * groups + torch.arange(groups, device=dev))
        field = torch.stack([lo & 0xFFFF, lo >> 16, hi & 0xFFFF, hi >> 16], 2).view(c["Tq"], -1)[:, :c["Tk"]]
        cut = int(round(c["p"] * 65536))
        prob = torch.where(field >= cut, prob / (1 - cut / 65536), torch.zeros_like(prob))
    return v @ prob.t()


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "norm":
        x, r = (s[n].double().requires_grad_(c["train"]) for n in "xr")
        gamma, beta = (s[n].double().requires_grad_(c["train"]) for n in ("gamma", "beta"))
        dropped = x
        if c["p"]:
            hi, _ = _uniform_words(s, torch.arange(x.numel(), device=x.device))
            kept = (hi >> 8).double() / 16777216 >= float(torch.tensor(c["p"], dtype=torch.float32))
            dropped = torch.where(kept.view(x.shape), x / (1 - c["p"]), torch.zeros_like(x))
        y = torch.nn.functional.layer_norm((r + dropped).transpose(1, 2), (c["C"],), gamma, beta, 1e-5).transpose(1, 2)
        if c["mask"]:
            y = y * s["mask"].double()[:, None]
        if not c["train"]:
            return {"y": y}
        dx, dr, dgamma, dbeta = torch.autograd.grad(y, (x, r, gamma, beta), s["dy"].double())
        return {"y": y.detach(), "dr": dr, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}
    B, H, G, dk = c["B"], c["H"], c["G"], c["dk"]
    q, k, v = (s[n].double().view(B, m, dk, -1) for n, m in (("q", H), ("k", G), ("v", G)))
    bias = s["bias"].double() if c["bias"] else None
    out = torch.empty_like(q)
    dq, dk_, dv = (torch.zeros_like(x) for x in (q, k, v))
    dbias = torch.zeros_like(bias) if c["bias"] else None
    for b in range(B):
        for h in range(H):
            leaves = [x.detach().requires_grad_() for x in (q[b, h], k[b, h // (H // G)], v[b, h // (H // G)])]
            leaves += [bias[h].detach().requires_grad_()] if c["bias"] else []
            o = _exact_head(s, b, h, *leaves[:3], leaves[3] if c["bias"] else None)
            out[b, h] = o.detach()
            if c["train"]:
                g = torch.autograd.grad(o, leaves, s["dout"].double().view(B, H, dk, -1)[b, h])
                dq[b, h] = g[0]
                dk_[b, h // (H // G)] += g[1]
                dv[b, h // (H // G)] += g[2]
                if c["bias"]:
                    dbias[h] += g[3]
    res = {"out": out.view(s["q"].shape)}
    if c["train"]:
        res.update(dq=dq.view(s["q"].shape), dk=dk_.view(s["k"].shape), dv=dv.view(s["v"].shape))
        if c["bias"]:
            res["dbias"] = dbias
    return res
