"""float64 restatement of attention_scored and dropout_add_layernorm (forward and explicit gradients), with the companions that error bounds
are made of: for every output the same sum over absolute values."""
import math

import numpy as np
import torch

M64 = (1 << 64) - 1


def words(seed, site, counters):
    """svc_dropout_rng_f32's 64-bit word of (seed, site) at each counter (numpy uint64)."""
    with np.errstate(over="ignore"):
        c = counters.astype(np.uint64)
        z = np.uint64((int(seed) + (site + 1) * 0x9E3779B97F4A7C15) & M64) + c * np.uint64(0xD1B54A32D192ED03)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return z ^ (z >> np.uint64(31))


def attention_keep(seed, site, B, H, Tq, Tk, p):
    """Z [B, H, Tq, Tk]: 0 or 1 / (1 - theta)."""
    ng, cut = (Tk + 3) // 4, int(round(p * 65536))
    w = words(seed, site, np.arange(B * H * Tq * ng)).reshape(B * H * Tq, ng, 1)
    f = (w >> np.array([0, 16, 32, 48], dtype=np.uint64)) & np.uint64(0xFFFF)
    keep = (f.reshape(B * H * Tq, ng * 4)[:, :Tk] >= cut).astype(np.float64) / (1 - cut / 65536)
    return torch.from_numpy(keep).view(B, H, Tq, Tk)


def visible(B, Tq, Tk, causal=False, window=None, prefix=None, docs=None, lengths=None, offset=None):
    """[B, Tq, Tk] by the definition, entry by entry; and the query positions [B, Tq]."""
    see = torch.zeros(B, Tq, Tk, dtype=torch.bool)
    pos = torch.zeros(B, Tq, dtype=torch.long)
    for b in range(B):
        off = Tk - Tq if offset is None else int(offset[b]) if isinstance(offset, torch.Tensor) else offset
        n = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
        edge = None if docs is None else docs[b].tolist()
        for t in range(Tq):
            p = pos[b, t] = off + t
            if p < 0 or p >= n:
                continue
            lo, hi, start, front = 0, n, 0, 0 if prefix is None or docs is not None else int(prefix[b])
            if edge is not None:
                mine = [i for i in range(len(edge) - 1) if edge[i] <= p < edge[i + 1]]
                if not mine:
                    continue
                lo, hi, start = max(lo, edge[mine[0]]), min(hi, edge[mine[0] + 1]), edge[mine[0]]
                if prefix is not None:
                    front = int(prefix[b, mine[0]])
            for s in range(lo, hi):
                see[b, t, s] = (not causal or s <= p or s < start + front) and (window is None or abs(s - p) <= window)
    return see, pos


def visible_matrix(B, Tq, Tk, causal=False, window=None, prefix=None, docs=None, lengths=None, offset=None):
    """visible() by comparisons of whole matrices, for long sequences."""
    see, pos, s = torch.zeros(B, Tq, Tk, dtype=torch.bool), torch.zeros(B, Tq, dtype=torch.long), torch.arange(Tk)
    for b in range(B):
        off = Tk - Tq if offset is None else int(offset[b]) if isinstance(offset, torch.Tensor) else offset
        n = Tk if lengths is None else min(max(int(lengths[b]), 0), Tk)
        p = pos[b] = off + torch.arange(Tq)
        start, front = torch.zeros(Tq, dtype=torch.long), torch.full((Tq,), 0 if prefix is None or docs is not None else int(prefix[b]))
        ok = ((p >= 0) & (p < n))[:, None] & (s < n)
        if docs is not None:
            mine = torch.zeros_like(ok)
            for i, (lo, hi) in enumerate(zip(docs[b].tolist(), docs[b].tolist()[1:])):
                own = (lo <= p) & (p < hi)
                mine |= own[:, None] & (lo <= s) & (s < hi)
                start[own] = lo
                if prefix is not None:
                    front[own] = int(prefix[b, i])
            ok &= mine
        if causal:
            ok &= (s <= p[:, None]) | (s < (start + front)[:, None])
        if window is not None:
            ok &= (s - p[:, None]).abs() <= window
        see[b] = ok
    return see, pos


def attention(q, k, v, n_heads, dout=None, bias=None, softcap=0.0, scale=None, draw=None, p_drop=0.0, **mask):
    """-> dict of out (dq, dk, dv, dbias) and, under "mag_<name>", the sums of absolute values behind them; "score": the largest sum of |q||k| scale."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    B, Cq, Tq = q.shape
    H, dk, Tk = n_heads, Cq // n_heads, k.shape[2]
    G = k.shape[1] // dk
    scale = dk ** -0.5 if scale is None else scale
    mask = {n: x.cpu() if isinstance(x, torch.Tensor) else x for n, x in mask.items()}
    see, pos = visible(B, Tq, Tk, **mask)
    q4 = q.view(B, H, dk, Tq)
    k4, v4 = (x.view(B, G, dk, Tk).repeat_interleave(H // G, 1) for x in (k, v))
    k4, v4 = (torch.where(see.any(1)[:, None, None, :], x, torch.zeros_like(x)) for x in (k4, v4))      # unseen keys are not used
    a = torch.einsum("bhdt,bhds->bhts", q4, k4) * scale
    res = {"score": float((torch.einsum("bhdt,bhds->bhts", q4.abs(), k4.abs()) * abs(scale)).max()) if a.numel() else 0.0}
    res["Tk"] = Tk
    th = torch.zeros_like(a)
    if softcap:
        th = torch.tanh(a / softcap)
        a = softcap * th
    at = None
    if bias is not None:
        W = bias.shape[1] // 2
        at = (torch.arange(Tk) - pos[..., None]).clamp(-W, W) + W                                       # [B, Tq, Tk]
        tab = bias.detach().cpu().double().expand(H, -1)
        a = a + tab[:, at].transpose(0, 1)
    hide = (~see[:, None]).expand(B, H, Tq, Tk)
    if bias is not None:      # fp16's lowest value and below mask a distance
        hide = hide | (tab <= -65504)[:, at].transpose(0, 1)
        a = torch.where(hide, torch.zeros_like(a), a)
    none = hide.all(-1, keepdim=True)
    P = torch.softmax(a.masked_fill(hide & ~none, -math.inf), -1).masked_fill(hide, 0.0)
    Z = attention_keep(int(draw.seed.item()), draw.site, B, H, Tq, Tk, p_drop) if p_drop else torch.ones(())
    ZP = Z * P
    out = torch.einsum("bhts,bhds->bhdt", ZP, v4)
    res["out"], res["mag_out"] = out.reshape(q.shape), torch.einsum("bhts,bhds->bhdt", ZP, v4.abs()).reshape(q.shape)
    top = lambda x: float(x.abs().max()) if x.numel() else 0.0  # noqa: E731
    n = max(Tq, Tk) * (H // G)
    res["floor"] = {"out": n * 2.0 ** -33 * top(v4)}              # what fp16's subnormal operands may add (tests' docstring)
    if dout is None:
        return res
    do = dout.detach().cpu().double().view(B, H, dk, Tq)
    do = torch.where(none.squeeze(-1)[:, :, None, :], torch.zeros_like(do), do)
    fold = lambda x: x.reshape(B, G, H // G, dk, Tk).sum(2).reshape(k.shape)  # noqa: E731
    d = top(do)
    res["floor"].update(dv=n * 2.0 ** -33 * d, dq=n * 2.0 ** -25 * d * top(k4) * abs(scale), dk=n * 2.0 ** -25 * d * top(q4) * abs(scale),
                        dbias=n * 2.0 ** -33 * Tk * dk * d * top(v4))
    D = (do * out).sum(2)[..., None]
    dS = P * (Z * torch.einsum("bhdt,bhds->bhts", do, v4) - D)
    mag = P * (Z * torch.einsum("bhdt,bhds->bhts", do.abs(), v4.abs()) + (do.abs() * res["mag_out"].view(q4.shape)).sum(2)[..., None])
    res["dv"], res["mag_dv"] = fold(torch.einsum("bhts,bhdt->bhds", ZP, do)), fold(torch.einsum("bhts,bhdt->bhds", ZP, do.abs()))
    if bias is not None:
        bins = lambda x: torch.stack([torch.bincount(at.reshape(-1), x[:, h].reshape(-1), minlength=bias.shape[1]) for h in range(H)])  # noqa: E731
        res["dbias"], res["mag_dbias"] = bins(dS), bins(mag)
        if bias.shape[0] == 1:
            res["dbias"], res["mag_dbias"] = res["dbias"].sum(0, keepdim=True), res["mag_dbias"].sum(0, keepdim=True)
    dS = dS * (1 - th * th)
    q4 = torch.where(none.squeeze(-1)[:, :, None, :], torch.zeros_like(q4), q4)
    res["dq"], res["mag_dq"] = ((torch.einsum("bhts,bhds->bhdt", x, y) * scale).reshape(q.shape) for x, y in ((dS, k4), (mag, k4.abs())))
    res["dk"], res["mag_dk"] = (fold(torch.einsum("bhts,bhdt->bhds", x, y) * scale) for x, y in ((dS, q4), (mag, q4.abs())))
    return res


def junction(x, r, gamma, beta, dy=None, draw=None, p=0.0, mask=None, eps=1e-5):
    """LayerNorm_C(r + dropout(x)) * gamma + beta (* mask) and its gradients by their formulas -> dict, with "xh" and "rs"."""
    x, gamma, beta = (t.detach().cpu().double() for t in (x, gamma, beta))
    r = torch.zeros_like(x) if r is None else r.detach().cpu().double()
    Z = torch.ones(())
    if p:
        u = (words(int(draw.seed.item()), draw.site, np.arange(x.numel())) >> np.uint64(40)).astype(np.float64) / 16777216
        Z = torch.from_numpy((u >= float(np.float32(p))).astype(np.float64) / (1 - p)).view(x.shape)
    on = torch.ones(x.shape[0], 1, x.shape[2], dtype=torch.float64) if mask is None else mask.detach().cpu().double().view(x.shape[0], 1, -1)
    live = on != 0
    h = torch.where(live, r, torch.zeros_like(r)) + torch.where(live, x, torch.zeros_like(x)) * Z
    d = h - h.mean(1, keepdim=True)
    rs = 1 / torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    xh = d * rs
    res = {"y": (xh * gamma[:, None] + beta[:, None]) * on, "xh": xh, "rs": rs, "h": h}
    if dy is None:
        return res
    g0 = torch.where(live, dy.detach().cpu().double() * on, torch.zeros_like(h))
    g = g0 * gamma[:, None]
    dh = torch.where(live, rs * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True)), torch.zeros_like(h))
    res.update(dr=dh, dx=dh * Z, dgamma=(g0 * xh).sum((0, 2)), dbeta=g0.sum((0, 2)), g=g, mag_dgamma=(g0 * xh).abs().sum((0, 2)),
               mag_dbeta=g0.abs().sum((0, 2)))
    return res
