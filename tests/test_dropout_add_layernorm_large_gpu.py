"""dropout_add_layernorm at the sizes of a training batch: 16 time steps a workgroup (from 256 such tiles on), every built number of channels a thread,
workgroups that walk several tiles with the parameters' sums in LDS — against the float64 definition with the bounds of
tests/test_dropout_add_layernorm_gpu.py.  The parameters' sums there are of at most 64 terms in order, tiles of one workgroup one after the other; here
a workgroup walks up to four tiles more, each adding one fp32 term."""
import pytest
import torch

from test_dropout_add_layernorm_gpu import TYPES, _mask, _run

pytestmark = pytest.mark.gpu

# channels of each built class (1, 2, 3, 4, 6, 8 a thread), a full one and a ragged one
CHANNELS = [100, 128, 192, 300, 512, 513, 768, 1001, 1024]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", CHANNELS)
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_tiles_of_sixteen_steps(dev, dt, C, p):
    """8 x 34 tiles, the last ragged."""
    _run(dev, TYPES[dt], 8, C, 531, p=p, mask=_mask(8, 531) if C % 2 or p else None)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("B,C,T", [(16, 130, 531), (16, 64, 1040), (33, 200, 257), (7, 770, 1500), (16, 1001, 600), (520, 33, 3), (1, 192, 9000)])
def test_several_tiles_a_workgroup(dev, dt, B, C, T):
    """More than 512 tiles: each of 512 workgroups takes the next of its XCD's run."""
    _run(dev, TYPES[dt], B, C, T, p=0.25, mask=_mask(B, T))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.3])
@pytest.mark.parametrize("B,C,T", [(2, 1000, 200), (1, 800, 77), (2, 513, 40), (1, 1024, 9)])
def test_tiles_of_eight_steps_with_many_channels(dev, dt, B, C, T, p):
    """Few columns: up to 1024 channels, four a thread."""
    _run(dev, TYPES[dt], B, C, T, p=p, mask=_mask(B, T) if T % 2 else None)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("C", [1025, 1280, 2100])
def test_more_channels_than_registers_hold(dev, dt, C):
    _run(dev, TYPES[dt], 5, C, 901, p=0.1, mask=_mask(5, 901))


@pytest.mark.parametrize("dt", TYPES)
def test_without_residual_and_without_mask(dev, dt):
    _run(dev, TYPES[dt], 16, 192, 531, p=0.1, with_r=False)
    _run(dev, TYPES[dt], 16, 192, 531, with_r=False)


def test_two_runs_of_a_large_batch_are_bit_equal_and_replays_too(dev):
    import svc_hip as S
    g = torch.Generator().manual_seed(3)
    x, r, dy = (torch.randn(16, 192, 790, generator=g).to(dev) for _ in range(3))
    gamma, beta = torch.randn(192, generator=g).to(dev), torch.randn(192, generator=g).to(dev)
    seed = torch.tensor([9], device=dev)
    draw = S.HashDraw(seed, 4)

    def step():
        y, (mu, rs) = S.dropout_add_layernorm(x, r, gamma, beta, draw=draw, p=0.1, stats=True)
        return (y, *S.dropout_add_layernorm_bwd(dy, x, r, gamma, beta, mu, rs, draw=draw, p=0.1))

    want = {}
    for s in (9, 10):
        seed.fill_(s)
        want[s] = [t.clone() for t in step()]
        assert all(torch.equal(a, b) for a, b in zip(step(), want[s]))
    gr = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        out = step()
    for s in (10, 9, 10):
        seed.fill_(s)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[s]))
        torch.randn(500, 500, device=dev).sum()


def test_saved_tensors_that_come_back_with_other_strides(dev):
    """Hooks may bring an equal tensor of any layout."""
    import svc_autograd as A
    g = torch.Generator().manual_seed(4)
    x, r, dy = (torch.randn(2, 48, 60, generator=g).to(dev).requires_grad_(i < 2) for i in range(3))
    gamma, beta = torch.ones(48, device=dev), torch.zeros(48, device=dev)
    want = torch.autograd.grad(A.dropout_add_layernorm(x, r, gamma, beta), (x, r), dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.transpose(1, 2).contiguous().transpose(1, 2) if t.shape == x.shape else t.clone()):
        y = A.dropout_add_layernorm(x, r, gamma, beta)
    for a, b in zip(want, torch.autograd.grad(y, (x, r), dy)):
        assert torch.equal(a, b)


def test_saved_statistics_that_come_back_at_the_same_address_with_other_strides(dev):
    import svc_autograd as A
    g = torch.Generator().manual_seed(4)
    x, r, dy = (torch.randn(2, 48, 60, generator=g).to(dev).requires_grad_(i < 2) for i in range(3))
    gamma, beta = torch.ones(48, device=dev), torch.zeros(48, device=dev)
    want = torch.autograd.grad(A.dropout_add_layernorm(x, r, gamma, beta), (x, r), dy)

    def unpack(t):
        if t.shape != (2, 2, 60):           # mean and rstd
            return t
        turned = t.transpose(0, 1).contiguous()
        t.view(-1).copy_(turned.view(-1))
        return t.view(-1).view(2, 2, 60).transpose(0, 1)

    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
        y = A.dropout_add_layernorm(x, r, gamma, beta)
    for a, b in zip(want, torch.autograd.grad(y, (x, r), dy)):
        assert torch.equal(a, b)
