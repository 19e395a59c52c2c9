"""The workspace queries of attention_scored and dropout_add_layernorm for arguments that the calls themselves refuse: 0, no division by 0 and no overflow."""
import ctypes
import subprocess
import sys

import pytest

from test_layer_ops_cpu import ROOT, _attn

CHILD = """
import ctypes, sys
sys.path[:0] = [{root!r}, {root!r} + "/so-vits-svc_amd"]
import svc_hip as S
a = S.AttnScored()
a.dtype, a.B, a.H, a.G, a.dk, a.Tq, a.Tk, a.window, a.scale = 1, 1, 4, 2, 64, 8, 8, -1, 0.125
for n, v in {kw!r}.items():
    setattr(a, n, v)
print(S.lib().svc_attn_scored_ws_bytes(ctypes.byref(a), {backward}))
"""


@pytest.mark.parametrize("backward", [0, 1])
@pytest.mark.parametrize("kw", [dict(H=1), dict(H=0), dict(H=3), dict(G=0), dict(H=-4), dict(G=-2), dict(B=-1), dict(B=0), dict(Tq=0), dict(Tq=-5), dict(Tq=9), dict(dk=0), dict(dk=129),
                                dict(B=1 << 30, H=1 << 30), dict(B=5 << 18, Tk=1, Tq=1), dict(Tk=1 << 30), dict(dtype=7), dict(bias_w=-1, bias=4096, bias_heads=1)],
                         ids=lambda d: ",".join(f"{k}={v}" for k, v in d.items()))
def test_attention_workspace_of_refused_arguments(kw, backward):
    r = subprocess.run([sys.executable, "-c", CHILD.format(root=ROOT, kw=kw, backward=backward)], capture_output=True, text=True)      # (a division by 0 ends the process)
    assert r.returncode == 0, (r.returncode, r.stderr[-300:])
    assert int(r.stdout.split()[-1]) == 0


def test_attention_workspace_of_ordinary_arguments():
    import svc_hip as S
    f = S.lib().svc_attn_scored_ws_bytes
    assert f(ctypes.byref(_attn()), 0) == 0                                               # 8 keys: one part
    assert f(ctypes.byref(_attn(Tq=1, Tk=8192)), 0) > 0 and f(ctypes.byref(_attn(Tq=1, Tk=8192)), 0) % 4 == 0
    # documented: rows, intervals and tiles of the queries, and with dbias B H ceil(Tq / 32) (2 W + 1) floats
    with_bias = _attn(Tq=64, Tk=64, bias=4096, bias_heads=4, bias_w=100, dbias=4096)
    assert f(ctypes.byref(with_bias), 1) - f(ctypes.byref(_attn(Tq=64, Tk=64)), 1) == -(-1 * 4 * 2 * 201 * 4 // 16) * 16


@pytest.mark.parametrize("B,C,T", [(0, 8, 8), (-1, 8, 8), (8, 0, 8), (8, 8, 0), (65536, 8, 8), (8, 1 << 25, 8), (65535, 8, 2 ** 31 - 1), (2 ** 31 - 1,) * 3, (2, 8, 1 << 26)])
def test_junction_workspace_of_refused_arguments(B, C, T):
    import svc_hip as S
    assert S.lib().svc_dropout_add_layernorm_ws_bytes(B, C, T) == 0


def test_junction_workspace_of_the_largest_arguments():
    import svc_hip as S
    assert S.lib().svc_dropout_add_layernorm_ws_bytes(8, 200, 5000) == 2 * 200 * 512 * 4
    assert S.lib().svc_dropout_add_layernorm_ws_bytes(65535, (1 << 25) - 1, 1) == 2 * ((1 << 25) - 1) * 65535 * 4


@pytest.mark.parametrize("bad", [dict(scale=3e38), dict(softcap=3e38), dict(softcap=1e-40), dict(scale=1e30, softcap=1e-10)], ids=str)
def test_factors_beyond_fp32_are_refused(bad):
    """Scores are worked out in units of log 2 from scale log2(e), cap log2(e) and 2 log2(e) scale / cap: an infinite one makes NaN of a score of 0."""
    import svc_hip as S
    for fn in (S.lib().svc_attn_scored_fwd, S.lib().svc_attn_scored_bwd):
        assert fn(ctypes.byref(_attn(**bad)), None) == -1
        assert b"scale" in S.lib().svc_last_error()


def test_no_kernel_source_records_a_memset():
    """What a caller may capture clears memory by a kernel (svc::zero)."""
    import os
    import re
    d = os.path.join(ROOT, "so-vits-svc_amd", "csrc")
    for f in sorted(os.listdir(d)):
        if f.endswith((".hip", ".h")):
            assert not re.search(r"hipMemset\w*\s*\(", open(os.path.join(d, f)).read()), f
