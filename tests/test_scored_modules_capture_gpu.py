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


def test_padding_masks_with_holes(dev):
    """Refused on every route; in a captured graph, where the host cannot look, the frames that a sequence mask would have otherwise are NaN."""
    from modules.attentions import MASK_PADDING, MultiHeadAttention
    torch.manual_seed(2)
    mod = MultiHeadAttention(64, 64, 2, block_length=5).to(dev).eval()
    x = torch.randn(2, 64, 60, device=dev)
    good = (torch.arange(60, device=dev) < torch.tensor([[60], [37]], device=dev)).float()
    bad = good.clone()
    bad[0, 20] = 0
    with torch.no_grad():
        for kw in (dict(mask_mode=MASK_PADDING, mask_vec=bad), dict(attn_mask=(bad[:, None, :, None] * bad[:, None, None]))):
            with pytest.raises(NotImplementedError, match="sequence mask"):
                mod(x, x, **kw)
        with pytest.raises(NotImplementedError, match="sequence mask"):
            mod.forward_train(x, MASK_PADDING, bad)
        want = mod(x, x, mask_mode=MASK_PADDING, mask_vec=good).clone()
        assert torch.equal(mod(x, x, attn_mask=good[:, None, :, None] * good[:, None, None]), want)
        held = good.clone()
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = mod(x, x, mask_mode=MASK_PADDING, mask_vec=held)
        for m in (good, bad, good, bad):
            held.copy_(m)
            gr.replay()
            torch.cuda.synchronize()
            if m is good:
                assert torch.equal(out, want)
            else:           # first 0 at 20 by the search or 60: the frames that differ from the mask are marked, and no other item's
                assert torch.isnan(out[0]).any() and torch.equal(out[1], want[1])


def test_block_length_without_a_mask_cuts_nothing(dev):
    """(modules/attentions.py:223-229: the block is inside the mask's branch)"""
    from modules.attentions import MASK_NONE, MultiHeadAttention
    torch.manual_seed(4)
    mod, wide = (MultiHeadAttention(64, 64, 2, block_length=n).to(dev).eval() for n in (3, 100))
    wide.load_state_dict(mod.state_dict())
    x = torch.randn(2, 64, 50, device=dev)
    with torch.no_grad():
        everything = wide(x, x, mask_mode=MASK_NONE)
        assert torch.equal(mod(x, x), everything)
        cut = mod(x, x, attn_mask=torch.ones(1, 1, 50, 50, device=dev))
        assert torch.equal(cut, mod(x, x, mask_mode=MASK_NONE)) and not torch.equal(cut, everything)


def test_a_training_pass_in_a_graph_between_eager_passes_of_another_length(dev):
    """Forward and gradients of a stack captured at one length (its backward reads the pass's own table), replayed on new data between eager training passes
    and allocations.  Weight gradients are combined with atomics: equal up to their order."""
    from modules.attentions import FFT
    torch.manual_seed(9)
    fft, other = (FFT(64, 128, 2, n_layers=2, kernel_size=3, proximal_bias=True).to(dev).train() for _ in range(2))
    other.load_state_dict(fft.state_dict())
    params = [p for n, p in fft.named_parameters() if not n.endswith("conv_k.bias")]      # (whose gradient is rounding alone)
    twins = [p for n, p in other.named_parameters() if not n.endswith("conv_k.bias")]
    data = [torch.randn(2, 64, 90, device=dev) for _ in range(3)]
    m, way = {T: torch.ones(2, 1, T, device=dev) for T in (90, 130)}, {T: torch.randn(2, 64, T, device=dev) for T in (90, 130)}

    def step(net, ps, x):
        y = net(x, m[x.shape[2]])
        return [y, *torch.autograd.grad((y * way[x.shape[2]]).sum(), [x, *ps])]

    want = [[t.detach().clone() for t in step(other, twins, x.clone().requires_grad_())] for x in data]
    held = data[0].clone().requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fft, params, held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        got = step(fft, params, held)
    for i in (1, 2, 0, 1):
        step(other, twins, torch.randn(2, 64, 130, device=dev).requires_grad_())
        junk = [torch.full((n,), 1e4, device=dev) for n in range(100, 700, 20)]
        with torch.no_grad():
            held.copy_(data[i])
        gr.replay()
        torch.cuda.synchronize()
        assert len(junk) == 30
        for a, b in zip(got, want[i]):
            assert (a - b).abs().max() <= 1e-4 * b.abs().max().clamp(min=1e-6)
