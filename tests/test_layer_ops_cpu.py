"""attention_scored and dropout_add_layernorm on the host: refusals at the C entry and in the binding (nothing is launched), struct layouts, and the
float64 oracle's explicit gradients against central differences."""
import ctypes
import os
import re
import subprocess

import pytest
import torch

from oracle import layer_oracle as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Draw:
    def __init__(self, seed, site):
        self.seed, self.site = torch.tensor([seed]), site


def test_struct_layouts_match_the_header(tmp_path):
    import shutil
    import svc_hip as S
    if shutil.which("gcc") is None:
        pytest.skip("no C compiler on this host")
    pairs = {"svc_attn_scored_t": S.AttnScored, "svc_dropout_add_layernorm_t": S.DropoutAddLayernorm}
    header = os.path.join(ROOT, "include", "svc_hip.h")
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {"]
    for c, cls in pairs.items():
        lines.append(f'  printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'  printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "l.c").write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True, capture_output=True)
    got = dict(x.split() for x in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.splitlines())
    for c, cls in pairs.items():
        assert int(got[c]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(cls, f).offset, (c, f)


def _attn(**kw):
    """Arguments that pass the checks, with made-up addresses, then `kw`: every use here is refused or empty, so nothing is read."""
    import svc_hip as S
    a = S.AttnScored()
    for n in ("q", "k", "v", "out", "out32", "lse", "dout", "dq", "dk_", "dv", "ws"):
        setattr(a, n, 4096)
    a.ws_bytes = 1 << 40
    a.dtype, a.B, a.H, a.G, a.dk, a.Tq, a.Tk, a.window, a.scale = 1, 1, 4, 2, 64, 8, 8, -1, 0.125
    for n, v in kw.items():
        setattr(a, n, v)
    return a


BAD = [dict(dtype=3), dict(dtype=-1), dict(B=-1), dict(Tq=9), dict(Tq=-1), dict(Tk=1 << 30), dict(G=3), dict(G=0), dict(H=0), dict(dk=0), dict(dk=129),
       dict(offset=1), dict(offset=-1), dict(window=-2), dict(n_docs=2), dict(n_docs=-1), dict(prefix=4096), dict(prefix=4096, causal=1, window=3),
       dict(bias=4096, bias_heads=2), dict(bias=4096, bias_heads=4, bias_w=-1), dict(softcap=-1.0), dict(softcap=float("inf")),
       dict(softcap=float("nan")), dict(scale=float("nan")), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(seed=4096, p_drop=1.0), dict(seed=4096, p_drop=-0.1), dict(seed=4096, p_drop=float("nan")),
       dict(q=None), dict(k=None), dict(v=None), dict(B=1 << 30, Tk=1 << 20), dict(B=5 << 18, Tk=1, Tq=1), dict(bias=4096, bias_heads=1, bias_w=1 << 24),
       dict(bias=4096, bias_heads=65536, H=65536)]


@pytest.mark.parametrize("bad", BAD, ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_attention_refuses(bad):
    import svc_hip as S
    for fn in (S.lib().svc_attn_scored_fwd, S.lib().svc_attn_scored_bwd):
        assert fn(ctypes.byref(_attn(**bad)), None) == -1
        assert b"attn_scored" in S.lib().svc_last_error()


@pytest.mark.parametrize("bad", [dict(dout=None), dict(lse=None), dict(dq=None), dict(dk_=None), dict(dv=None), dict(out32=None), dict(dtype=0, out=None),
                                 dict(dbias=4096), dict(ws=None), dict(ws_bytes=8), dict(ws=4100)])
def test_attention_backward_refuses(bad):
    import svc_hip as S
    assert S.lib().svc_attn_scored_bwd(ctypes.byref(_attn(**bad)), None) == -1


def test_attention_null_and_empty():
    import svc_hip as S
    assert S.lib().svc_attn_scored_fwd(None, None) == -1
    assert S.lib().svc_attn_scored_ws_bytes(None, 1) == 0
    assert S.lib().svc_attn_scored_fwd(ctypes.byref(_attn(B=0)), None) == 0
    assert S.lib().svc_attn_scored_fwd(ctypes.byref(_attn(Tq=0)), None) == 0
    assert S.lib().svc_attn_scored_bwd(ctypes.byref(_attn(B=0)), None) == 0


def _junction(**kw):
    import svc_hip as S
    a = S.DropoutAddLayernorm()
    for n in ("x", "r", "gamma", "beta", "y", "mean", "rstd", "dy", "dx", "dr", "dgamma", "dbeta", "ws"):
        setattr(a, n, 4096)
    a.ws_bytes, a.dtype, a.B, a.C, a.T, a.eps = 1 << 40, 0, 2, 16, 8, 1e-5
    for n, v in kw.items():
        setattr(a, n, v)
    return a


@pytest.mark.parametrize("bad", [dict(dtype=3), dict(B=-1), dict(B=65536), dict(C=0), dict(T=-1), dict(C=1 << 25), dict(T=1 << 26), dict(eps=0.0), dict(eps=float("nan")), dict(x=None),
                                 dict(gamma=None), dict(beta=None), dict(seed=4096, p=1.0), dict(seed=4096, p=-0.5), dict(seed=4096, p=float("nan"))])
def test_junction_refuses(bad):
    import svc_hip as S
    for fn in (S.lib().svc_dropout_add_layernorm_fwd, S.lib().svc_dropout_add_layernorm_bwd):
        assert fn(ctypes.byref(_junction(**bad)), None) == -1
        assert b"dropout_add_layernorm" in S.lib().svc_last_error()


@pytest.mark.parametrize("bad", [dict(dy=None), dict(mean=None), dict(rstd=None), dict(dr=None, dx=None), dict(dgamma=None), dict(dbeta=None), dict(ws=None),
                                 dict(ws_bytes=4), dict(ws=4100), dict(B=0), dict(T=0)])
def test_junction_backward_refuses(bad):
    import svc_hip as S
    assert S.lib().svc_dropout_add_layernorm_bwd(ctypes.byref(_junction(**bad)), None) == -1


def test_junction_forward_refuses_one_statistic_and_takes_nothing():
    import svc_hip as S
    f = S.lib().svc_dropout_add_layernorm_fwd
    assert f(ctypes.byref(_junction(rstd=None)), None) == -1 and f(ctypes.byref(_junction(y=None)), None) == -1 and f(None, None) == -1
    assert f(ctypes.byref(_junction(B=0)), None) == 0 and f(ctypes.byref(_junction(T=0)), None) == 0


def test_binding_refuses_cpu_tensors_and_other_types():
    import svc_hip as S
    x = torch.zeros(1, 8, 4)
    with pytest.raises(S.SvcError, match="GPU"):
        S.attention_scored(x, x, x, 2)
    with pytest.raises(S.SvcError, match="GPU"):
        S.dropout_add_layernorm(x, x, torch.ones(8), torch.zeros(8))
    with pytest.raises(S.SvcError, match="fp32, bf16 or fp16"):
        S.attention_scored(x.double(), x.double(), x.double(), 2)


def test_draw_words_are_the_documented_ones():
    """splitmix64's published finaliser on one counter, by Python integers."""
    M = (1 << 64) - 1
    z = (12345 + 4 * 0x9E3779B97F4A7C15 + 77 * 0xD1B54A32D192ED03) & M
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
    assert int(O.words(12345, 3, torch.tensor([77]).numpy())[0]) == z ^ (z >> 31)


@pytest.mark.parametrize("kw", [dict(causal=True, softcap=2.0), dict(window=2, p_drop=0.3), dict(docs=torch.tensor([[0, 3, 3, 6], [1, 2, 5, 7]], dtype=torch.int32)),
                                dict(causal=True, prefix=torch.tensor([3, 0], dtype=torch.int32)), dict(lengths=torch.tensor([4, 7], dtype=torch.int32))])
@pytest.mark.parametrize("shared", [False, True])
def test_oracle_attention_gradients_against_differences(kw, shared):
    g = torch.Generator().manual_seed(4)
    B, H, G, dk, T = 2, 4, 2, 3, 7
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = {"q": r(B, H * dk, T), "k": r(B, G * dk, T), "v": r(B, G * dk, T), "bias": r(1 if shared else H, 5)}
    do = r(B, H * dk, T)
    kw = dict(kw, draw=Draw(99, 2))
    f = lambda: (O.attention(x["q"], x["k"], x["v"], H, bias=x["bias"], **kw)["out"] * do).sum().item()  # noqa: E731
    grads = O.attention(x["q"], x["k"], x["v"], H, dout=do, bias=x["bias"], **kw)
    for name, t in x.items():
        flat, got = t.view(-1), grads["d" + name].reshape(-1)
        for i in range(0, flat.numel(), max(1, flat.numel() // 12)):
            old, eps = flat[i].item(), 1e-5
            flat[i] = old + eps
            up = f()
            flat[i] = old - eps
            down = f()
            flat[i] = old
            # truncation ~ eps^2 f''' (some 1e-9), rounding ~ 1e-15 |f| / eps (some 1e-9)
            assert abs((up - down) / (2 * eps) - got[i].item()) < 1e-7 * max(1.0, abs(got[i].item())), (name, i)


@pytest.mark.parametrize("p,mask", [(0.0, None), (0.3, torch.tensor([[1., 1, 0, 1], [1, 0, 0, 0.5]]))])
def test_oracle_junction_gradients_against_differences(p, mask):
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = {"x": r(2, 6, 4), "r": r(2, 6, 4), "gamma": r(6), "beta": r(6)}
    dy, kw = r(2, 6, 4), dict(p=p, mask=mask, draw=Draw(7, 1))
    f = lambda: (O.junction(**x, **kw)["y"] * dy).sum().item()  # noqa: E731
    grads = O.junction(**x, dy=dy, **kw)
    for name, t in x.items():
        flat, got = t.view(-1), grads["d" + name].reshape(-1)
        for i in range(flat.numel()):
            old, eps = flat[i].item(), 1e-5
            flat[i] = old + eps
            up = f()
            flat[i] = old - eps
            down = f()
            flat[i] = old
            assert abs((up - down) / (2 * eps) - got[i].item()) < 1e-7 * max(1.0, abs(got[i].item())), (name, i)


def test_product_names_are_exported():
    header = open(os.path.join(ROOT, "include", "svc_hip.h")).read()
    import svc_hip as S
    for n in re.findall(r"\b(svc_(?:attn_scored|dropout_add_layernorm)_[a-z_]+)\(", header):
        assert n in S.EXPORTS
