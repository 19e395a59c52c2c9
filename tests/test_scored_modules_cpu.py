"""What MultiHeadAttention(proximal_bias / block_length) hands to attention_scored, on the host: tables, lengths, windows and refusals (no launch)."""
import pytest
import torch

CPU = torch.device("cpu")


def _mha(**kw):
    from modules.attentions import MultiHeadAttention
    torch.manual_seed(1)
    return MultiHeadAttention(32, 32, 2, **kw)


def test_the_distance_table_belongs_to_its_call():
    """A table kept by the module and replaced at another length would leave a graph that was captured with it on freed memory; one made while a
    graph is recorded, or on another stream, would be read before it is written.  So a call's table is its own and the module holds none."""
    from modules.attentions import MASK_NONE
    mod = _mha(proximal_bias=True)
    a = mod._scored_options(MASK_NONE, None, 9, CPU)["bias"]
    b = mod._scored_options(MASK_NONE, None, 9, CPU)["bias"]
    mod._scored_options(MASK_NONE, None, 5, CPU)
    assert a.data_ptr() != b.data_ptr()
    want = -torch.log1p(torch.arange(-8, 9).abs().double())[None]
    for t in (a, b):
        assert t.shape == (1, 17) and t.dtype == torch.float32 and (t.double() - want).abs().max() <= 2 * 2.0 ** -24 * 3      # log1p(8) < 3
    held = [x for v in mod.__dict__.values() for x in (v if isinstance(v, tuple) else (v,)) if isinstance(x, torch.Tensor)]
    assert not held


def test_a_table_made_in_inference_mode_is_not_met_again_in_training():
    from modules.attentions import MASK_NONE
    mod = _mha(proximal_bias=True)
    with torch.inference_mode():
        mod._scored_options(MASK_NONE, None, 9, CPU)
    assert not mod._scored_options(MASK_NONE, None, 9, CPU)["bias"].is_inference()      # (it could not be saved for a backward)


@pytest.mark.parametrize("mask", [[[1, 1, 0, 1, 0]], [[0, 1, 1, 1, 1]], [[1, 1, 1, 1, 1], [1, 0, 1, 1, 0]], [[0, 0, 0, 0, 1]]])
def test_a_padding_mask_with_a_hole_is_refused_whatever_the_route(mask):
    """mask_mode=MASK_PADDING with a mask that is not ones, then zeros: its sum is not a length."""
    from modules.attentions import MASK_PADDING
    for mod in (_mha(proximal_bias=True), _mha(block_length=2)):
        with pytest.raises(NotImplementedError, match="sequence mask"):
            mod._scored_options(MASK_PADDING, torch.tensor(mask, dtype=torch.float32), 5, CPU)


@pytest.mark.parametrize("mask,want", [([[1, 1, 0, 0, 0], [1, 1, 1, 1, 1], [0, 0, 0, 0, 0]], [2, 5, 0]), ([[0.25, 3.0, 2.0, 0, 0]], [3]), ([[1.0]], [1]), ([[0.0]], [0])])
def test_lengths_count_the_places_that_are_not_zero(mask, want):
    """A place belongs to the item where the mask is not 0 (masked_fill(mask == 0)), whatever its value."""
    from modules.attentions import MASK_PADDING
    mod = _mha(block_length=2)
    got = mod._scored_options(MASK_PADDING, torch.tensor(mask, dtype=torch.float32), len(mask[0]), CPU)["lengths"]
    assert got.dtype == torch.int32 and got.tolist() == want and got.is_contiguous()


def test_block_length_goes_with_a_mask(monkeypatch):
    """modules/attentions.py:223-229: the block is cut out of the scores where a mask is given, not without one."""
    import modules.attentions as M
    mod = _mha(block_length=2).eval()
    seen = []
    monkeypatch.setattr(M.S, "conv1d", lambda x, *a, **kw: torch.zeros(x.shape[0], 96, x.shape[2]))
    monkeypatch.setattr(mod, "_qkv_packed", lambda: (None, None))
    monkeypatch.setattr(type(mod.conv_o), "run", lambda self, x: x)
    monkeypatch.setattr(M.S, "attention_scored", lambda q, k, v, n, **kw: seen.append(kw["window"]) or q)
    x = torch.zeros(1, 32, 6)
    with torch.no_grad():
        mod(x, x)
        mod(x, x, attn_mask=torch.ones(1, 1, 6, 6))
        mod(x, x, mask_mode=M.MASK_CAUSAL)
        mod(x, x, mask_mode=M.MASK_NONE)              # a caller's promise that its mask is all ones
    assert seen == [None, 2, 2, 2]
    seen.clear()
    monkeypatch.setattr(type(mod.conv_o), "forward_train", lambda self, x, **kw: x)
    monkeypatch.setattr(M.A, "attention_scored", lambda q, k, v, n, **kw: seen.append(kw["window"]) or q)
    y = x.requires_grad_()
    mod(y, y)
    mod(y, y, attn_mask=torch.ones(1, 1, 6, 6))
    assert seen == [None, 2]
