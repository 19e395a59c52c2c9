"""Gradients that kernels add up by atomics over cleared memory, captured and replayed: every replay starts from 0 (a memset recorded into a graph did not clear on
replays after the first)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _ops(S, dev):
    """name -> (inputs by seed, the call)."""
    g = lambda seed: torch.Generator().manual_seed(seed)  # noqa: E731
    r = lambda seed, *s: torch.randn(*s, generator=g(seed)).to(dev)  # noqa: E731

    def wgrad(a, b):
        db = torch.empty(a.shape[1], device=dev)
        return S.conv1d_wgrad(a, b, 3, 1, 1, out=torch.empty(a.shape[1], b.shape[1], 3, device=dev), dbias=db), db

    taps = torch.hann_window(12, periodic=False).tolist()
    u, v = torch.nn.functional.normalize(r(1, 40), dim=0), torch.nn.functional.normalize(r(2, 60), dim=0)
    sigma, win = torch.full((1,), 1.7, device=dev), torch.hann_window(64, device=dev)
    return {
        "conv1d_wgrad": (lambda s: (r(s, 2, 64, 90), r(s + 50, 2, 48, 90)), wgrad),
        "conv1d_wgrad_small": (lambda s: (r(s, 2, 16, 300), r(s + 50, 2, 24, 300)), wgrad),
        "gconv1d_wgrad": (lambda s: (r(s, 2, 64, 50), r(s + 50, 2, 16, 200)), lambda dy, x: S.gconv1d_wgrad(dy, x, 41, 4, 20, 4)),
        "snake_alias_bwd": (lambda s: (r(s, 2, 16, 400), r(s + 50, 2, 16, 400), 0.3 * r(s + 70, 16), 0.3 * r(s + 90, 16)),
                            lambda x, dy, a, b: S.snake_alias_bwd(x, dy, a, b, taps)),
        "nsf_linear_bwd": (lambda s: (r(s, 2, 3000, 9), torch.tanh(r(s + 50, 2, 1, 3000)), r(s + 70, 2, 1, 3000)), S.nsf_linear_bwd),
        "stft_frame_bwd": (lambda s: (r(s, 2, 30, 64),), lambda d: S.stft_frame_bwd(d, win, 500, 16, 24)),
        "spectral_norm_bwd": (lambda s: (r(s, 40, 60), r(s + 50, 40, 60)), lambda W, gr: S.spectral_norm_bwd(W, u, v, sigma, gr)),
    }


@pytest.mark.parametrize("name", ["conv1d_wgrad", "conv1d_wgrad_small", "gconv1d_wgrad", "snake_alias_bwd", "nsf_linear_bwd", "stft_frame_bwd", "spectral_norm_bwd"])
def test_every_replay_starts_from_zero(dev, name):
    import svc_hip as S
    make, call = _ops(S, dev)[name]
    flat = lambda x: list(x) if isinstance(x, tuple) else [x]  # noqa: E731
    want = {s: [t.clone() for t in flat(call(*make(s)))] for s in (1, 2, 3)}
    held = [t.clone() for t in make(1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(*held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        got = flat(call(*held))
    for s in (1, 2, 3, 1, 2):
        for h, t in zip(held, make(s)):
            h.copy_(t)
        gr.replay()
        torch.cuda.synchronize()
        torch.randn(500, 500, device=dev) @ torch.randn(500, 500, device=dev)
        for a, b in zip(got, want[s]):      # (sums of some thousand terms added in another order)
            assert torch.isfinite(a).all() and (a - b).abs().max() <= 1e-4 * b.abs().max(), (name, s)
