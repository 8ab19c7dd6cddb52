"""Fp8Linear and the 8-bit projections as modules: what a move, a copy or a gradient does to them (no GPU)."""
import copy

import pytest
import torch
import torch.nn as nn

from hierarchicalglobalattention_b200 import Fp8Linear


def _model():
    torch.manual_seed(0)
    return nn.Sequential(Fp8Linear.from_linear(nn.Linear(200, 136).bfloat16()), nn.Linear(136, 8).bfloat16())


@pytest.mark.parametrize("move", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.float(),
                                  lambda m: m.to(torch.float16), lambda m: m.to("cpu", torch.bfloat16),
                                  lambda m: m.type(torch.float32), lambda m: copy.deepcopy(m), lambda m: m.cpu()])
def test_a_move_to_another_type_leaves_weight_and_scales(move):
    m = _model()
    want = {k: v.clone() for k, v in m[0].state_dict().items()}
    m = move(m)
    lin = m[0]
    assert lin.weight.dtype == torch.float8_e4m3fn and lin.weight_scale_inv.dtype == torch.float32
    assert torch.equal(lin.weight.float(), want["weight"].float())
    assert torch.equal(lin.weight_scale_inv, want["weight_scale_inv"])
    assert lin.bias.dtype == m[1].weight.dtype         # the result's type follows the model
    assert set(lin.state_dict()) == {"weight", "weight_scale_inv", "bias"}


def test_meta_and_empty_moves():
    m = _model().to("meta")
    assert m[0].weight.is_meta and m[0].weight.dtype == torch.float8_e4m3fn and m[0].weight_scale_inv.is_meta
    m = m.to_empty(device="cpu").bfloat16()
    assert m[0].weight.device.type == "cpu" and m[0].weight.dtype == torch.float8_e4m3fn
    n = _model()
    m.load_state_dict(n.state_dict())
    assert torch.equal(m[0].weight.float(), n[0].weight.float())


def test_a_single_8bit_layer_is_used_where_it_is(monkeypatch):
    """o_proj of an FP8 checkpoint: the product reads the layer's own tensors and the wrapper keeps no copy."""
    import types
    import hierarchicalglobalattention_b200 as hga
    from hierarchicalglobalattention_b200 import ops
    from hierarchicalglobalattention_b200.fp8 import fp8_concat
    torch.manual_seed(1)
    o = Fp8Linear.from_linear(nn.Linear(128, 64).bfloat16())
    w, s, b = fp8_concat([o])
    assert w.data_ptr() == o.weight.data_ptr() and s.data_ptr() == o.weight_scale_inv.data_ptr()
    assert b.data_ptr() == o.bias.data_ptr()
    seen = []
    monkeypatch.setattr(ops, "fp8_linear", lambda x, w, s, bias=None: seen.append((w, s, bias)) or x)
    cfg = types.SimpleNamespace(num_attention_heads=2, num_key_value_heads=1, head_dim=64, hidden_size=64)
    orig = nn.Module()
    orig.o_proj = o
    layer = hga.QwenRoutedAttention(orig, cfg, fp8_projections=True)
    layer._o_proj(torch.zeros(1, 128, dtype=torch.bfloat16))
    assert seen[-1][0].data_ptr() == o.weight.data_ptr() and not layer._fp8_cache
    o.weight = torch.zeros(64, 128).to(torch.float8_e4m3fn)      # a replaced weight is seen, the old one let go
    layer._o_proj(torch.zeros(1, 128, dtype=torch.bfloat16))
    assert seen[-1][0].data_ptr() == o.weight.data_ptr()
