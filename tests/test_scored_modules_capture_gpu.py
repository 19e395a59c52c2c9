"""Modules with a proximal bias in captured graphs of several lengths, between eager calls of other lengths."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _fft(dev):
    from modules.attentions import FFT
    torch.manual_seed(7)
    return FFT(64, 128, 2, n_layers=2, kernel_size=3, proximal_bias=True).to(dev).eval()


def test_graphs_of_two_lengths_and_eager_calls_between_them(dev):
    """A graph captured at one length is replayed after calls at other lengths and allocations over what they freed; and an eager call at a length whose
    first call was recorded, before any replay."""
    fft = _fft(dev)
    x = {T: torch.randn(2, 64, T, device=dev) for T in (90, 150, 201)}
    m = {T: torch.ones(2, 1, T, device=dev) for T in x}
    with torch.no_grad():
        fresh = _fft(dev)
        want = {T: fresh(x[T], m[T]).clone() for T in x}
        fft(x[150], m[150])
        torch.cuda.synchronize()
        graphs, out = {}, {}
        for T in (90, 201):                                    # 90 and 201: first calls of these lengths
            graphs[T] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graphs[T]):
                out[T] = fft(x[T], m[T])
        assert torch.equal(fft(x[90], m[90]), want[90]) and torch.equal(fft(x[201], m[201]), want[201])
        for T in (90, 201, 90, 201):
            assert torch.equal(fft(x[150], m[150]), want[150])
            junk = [torch.full((n,), 1e4, device=dev) for n in range(100, 700, 20)]
            graphs[T].replay()
            torch.cuda.synchronize()
            assert torch.equal(out[T], want[T]) and len(junk) == 30
            del junk


def test_a_pass_on_another_stream_makes_its_own_table(dev):
    fft, x = _fft(dev), torch.randn(1, 64, 120, device=dev)
    m = torch.ones(1, 1, 120, device=dev)
    with torch.no_grad():
        want = fft(x, m).clone()
        torch.cuda.synchronize()
        outs = []
        for _ in range(3):
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                outs.append(fft(x, m))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_inference_mode_and_training_alternate(dev):
    fft, x = _fft(dev), torch.randn(1, 64, 77, device=dev)
    m = torch.ones(1, 1, 77, device=dev)
    with torch.inference_mode():
        a = fft(x, m).clone()
    fft.train()
    y = fft(x.clone().requires_grad_(), m)
    y.sum().backward()
    assert (y.detach() - a).abs().max() <= 2e-4 * a.abs().max()      # (the training path's own launches: tolerance of tests/test_scored_modules_gpu.py)
