"""The module options that run on attention_scored and dropout_add_layernorm — MultiHeadAttention(proximal_bias=True / block_length=n) and the FFT
stack built with proximal_bias — against the reference's formulas (modules/attentions.py:207-239,305-316,43-70) in float64 torch.

Tolerance 2e-4 of the largest value of a result for one attention module and 1e-3 for a stack's gradients: fp32 products over up to 192 channels and 60
keys leave some 1e-6 per layer, and each of the 2 x 5 layers between an input and a gradient can amplify by its gain (weights as the modules draw
them, a LayerNorm divides by the column's spread): measured bounds of the same stacks without these options (tests/test_train_ops_gpu.py) are 2e-5
per operator."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _ref_mha(m, x, mask, block=None, proximal=False, Z=None):
    B, C, T = x.shape
    H, dk = m["heads"], C // m["heads"]
    q, k, v = (F.conv1d(x, m[f"conv_{n}.weight"], m[f"conv_{n}.bias"]).view(B, H, dk, T).transpose(2, 3) for n in "qkv")
    s = q @ k.transpose(2, 3) / dk ** 0.5
    if proximal:
        r = torch.arange(T)
        s = s - torch.log1p((r[:, None] - r[None]).abs().double())
    s = s.masked_fill(mask == 0, -1e4)
    if block is not None:
        s = s.masked_fill(torch.ones(T, T).triu(-block).tril(block) == 0, -1e4)
    p = torch.softmax(s, -1)
    p = p if Z is None else p * Z
    return F.conv1d((p @ v).transpose(2, 3).reshape(B, C, T), m["conv_o.weight"], m["conv_o.bias"])


def _params(mod, heads):
    return {"heads": heads, **{n: p.detach().cpu().double().requires_grad_() for n, p in mod.named_parameters()}}


def _near(a, b, tol, what):
    a, b = a.detach().double().cpu(), b.detach()
    assert a.shape == b.shape and (a - b).abs().max() <= tol * b.abs().max().clamp(min=1e-6), (what, (a - b).abs().max().item(), b.abs().max().item())


@pytest.mark.parametrize("kind", ["proximal", "block", "both"])
@pytest.mark.parametrize("mask_mode", ["padding", "causal"])
def test_multi_head_attention(dev, kind, mask_mode):
    from modules.attentions import MASK_CAUSAL, MASK_PADDING, MultiHeadAttention
    torch.manual_seed(3)
    B, C, T, H = 2, 96, 60, 2
    block, prox = (7 if kind != "proximal" else None), kind != "block"
    mod = MultiHeadAttention(C, C, H, block_length=block, proximal_bias=prox).to(dev).eval()
    x = torch.randn(B, C, T)
    n = torch.tensor([T, 41])
    vec = (torch.arange(T) < n[:, None]).float()
    if mask_mode == "padding":
        mask, mode, mv = vec[:, None, :, None] * vec[:, None, None, :], MASK_PADDING, vec.to(dev)
    else:
        mask, mode, mv = torch.ones(T, T).tril()[None, None], MASK_CAUSAL, None
    valid = vec[:, None].double() if mask_mode == "padding" else torch.ones(B, 1, T, dtype=torch.double)
    ref = _params(mod, H)
    xr = x.double().requires_grad_()
    want = _ref_mha(ref, xr, mask, block, prox) * valid
    with torch.no_grad():
        xd = x.to(dev)
        got = mod(xd, xd, mask_mode=mode, mask_vec=mv)
    _near(got * valid.to(dev).float(), want, 2e-4, "inference")
    go = torch.randn(B, C, T)
    xt = x.to(dev).requires_grad_()
    y = mod.forward_train(xt, mode, mv)
    (y * (go.to(dev) * valid.to(dev).float())).sum().backward()
    (want * go.double()).sum().backward()
    _near(y * valid.to(dev).float(), want, 2e-4, "training forward")
    _near(xt.grad, xr.grad, 2e-4, "dx")
    for name, p in mod.named_parameters():
        if name != "conv_k.bias":                 # the softmax does not change when every key's score does: its gradient is rounding alone
            _near(p.grad, ref[name].grad, 2e-4, name)


def test_options_that_stay_refused():
    from modules.attentions import MultiHeadAttention
    for kw in (dict(heads_share=False), dict(proximal_bias=True, window_size=4), dict(block_length=3, window_size=4)):
        with pytest.raises(NotImplementedError):
            MultiHeadAttention(32, 32, 2, **kw)


def _ref_fft(fft, params, x, x_mask, H, T):
    causal = torch.ones(T, T).tril()[None, None]
    x = x * x_mask
    for i in range(fft.n_layers):
        pick = lambda pre: {"heads": H, **{n[len(pre):]: p for n, p in params.items() if n != "heads" and n.startswith(pre)}}  # noqa: E731
        norm = lambda y, pre: F.layer_norm(y.transpose(1, 2), (y.shape[1],), params[pre + "gamma"], params[pre + "beta"], 1e-5).transpose(1, 2)  # noqa: E731
        y = _ref_mha(pick(f"self_attn_layers.{i}."), x, causal, proximal=True)
        x = norm(x + y, f"norm_layers_0.{i}.")
        f = pick(f"ffn_layers.{i}.")
        k = fft.kernel_size
        h = torch.relu(F.conv1d(F.pad(x * x_mask, (k - 1, 0)), f["conv_1.weight"], f["conv_1.bias"]))
        h = F.conv1d(F.pad(h * x_mask, (k - 1, 0)), f["conv_2.weight"], f["conv_2.bias"]) * x_mask
        x = norm(x + h, f"norm_layers_1.{i}.")
    return x * x_mask


def test_stack_of_proximal_layers(dev):
    """Attention, junction, FFN, junction, five layers deep: the operators together as a model uses them, inference and training."""
    from modules.attentions import FFT
    torch.manual_seed(5)
    B, C, T, H = 2, 96, 50, 2
    fft = FFT(C, 2 * C, H, n_layers=5, kernel_size=3, p_dropout=0.0, proximal_bias=True, proximal_init=False).to(dev)
    x, m = torch.randn(B, C, T), (torch.arange(T) < torch.tensor([T, 37])[:, None]).float()[:, None]
    params = _params(fft, H)
    xr = x.double().requires_grad_()
    want = _ref_fft(fft, params, xr, m.double(), H, T)
    with torch.no_grad():
        _near(fft.eval()(x.to(dev), m.to(dev)), want, 2e-4, "inference")
    fft.train()
    xt = x.to(dev).requires_grad_()
    y = fft(xt, m.to(dev))
    go = torch.randn(B, C, T)
    (y * go.to(dev)).sum().backward()
    (want * go.double()).sum().backward()
    _near(y, want, 2e-4, "training forward")
    _near(xt.grad, xr.grad, 1e-3, "dx")
    for name, p in fft.named_parameters():
        if not name.endswith("conv_k.bias"):
            _near(p.grad, params[name].grad, 1e-3, name)


def test_stack_with_dropout_is_reproducible_and_differs_by_seed(dev):
    """Forward and backward of a site draw alike: a pass repeated from the same counter gives the same gradients, the next one others."""
    from modules.attentions import FFT, DropoutDraws
    torch.manual_seed(6)
    fft = FFT(64, 128, 2, n_layers=2, kernel_size=3, p_dropout=0.2, proximal_bias=True).to(dev).train()
    x, m = torch.randn(2, 64, 40, device=dev), torch.ones(2, 1, 40, device=dev)

    def step():
        fft.zero_grad()
        y = fft(x, m)
        (y * y).sum().backward()
        return [y.detach().clone()] + [p.grad.clone() for p in fft.parameters()]

    step()
    key = next(k for k in DropoutDraws._SEED if str(k).startswith("cuda"))
    start = DropoutDraws._SEED[key].clone()
    a = step()
    b = step()
    DropoutDraws._SEED[key].copy_(start)
    c = step()
    assert torch.equal(a[0], c[0]) and not torch.equal(a[0], b[0])
    for u, v in zip(a, c):          # (weight gradients are combined with atomics: equal up to their order)
        assert (u - v).abs().max() <= 1e-4 * u.abs().max().clamp(min=1e-6)


def test_earlier_stacks_do_not_take_the_new_path(dev):
    from modules.attentions import Encoder, FFT
    for mod in (Encoder(32, 64, 2, 1), FFT(32, 64, 2, 1)):
        layers = mod.attn_layers if hasattr(mod, "attn_layers") else mod.self_attn_layers
        assert not any(layer.scored for layer in layers)
