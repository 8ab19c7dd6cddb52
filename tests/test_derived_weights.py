"""Weights that the layers derive from their projections (concatenated, quantised) follow their sources."""
import copy
import gc
import pickle
import types

import numpy as np
import pytest
import torch
import torch.nn as nn

import hierarchicalglobalattention_b200 as hga
from hierarchicalglobalattention_b200 import ops
from hierarchicalglobalattention_b200.weights import WeightSources

IN = 64


def _linear(buf):
    """An nn.Linear over a caller's memory: two of them on one buffer have one address and version 0."""
    m = nn.Linear(IN, buf.shape[0], bias=False)
    m.weight = nn.Parameter(torch.from_numpy(buf), requires_grad=False)
    return m


def _wrapper(**kw):
    cfg = types.SimpleNamespace(num_attention_heads=2, num_key_value_heads=1, head_dim=64, hidden_size=IN)
    buf = {"q": np.ones((128, IN), np.float32), "k": np.ones((64, IN), np.float32), "v": np.ones((64, IN), np.float32),
           "o": np.ones((64, IN), np.float32)}
    orig = nn.Module()
    for n, b in buf.items():
        setattr(orig, n + "_proj", _linear(b))
    return hga.QwenRoutedAttention(orig, cfg, **kw), orig, buf


@pytest.fixture
def plain_fp8(monkeypatch):
    """ops.fp8_linear on the CPU: the dequantised product of the weight it is given."""
    def run(x, w, s, bias=None, **kw):
        n, k = w.shape
        wd = w.float() * s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        return x @ wd.T if bias is None else x @ wd.T + bias
    monkeypatch.setattr(ops, "fp8_linear", run)


def test_a_replaced_projection_at_the_same_address_is_seen_8bit(plain_fp8):
    w, orig, buf = _wrapper(fp8_projections=True)
    x = torch.ones(1, IN)
    assert (w._qkv(x) == IN).all() and (w._o_proj(x) == IN).all()
    for name in ("v", "o"):
        old = getattr(orig, name + "_proj").weight
        at, version = old.data_ptr(), old._version
        delattr(orig, name + "_proj")
        del old
        gc.collect()
        buf[name][:] = 2.0
        setattr(orig, name + "_proj", _linear(buf[name]))
        new = getattr(orig, name + "_proj").weight
        assert (new.data_ptr(), new._version) == (at, version)
    y = w._qkv(x)
    assert (y[:, :192] == IN).all() and (y[:, 192:] == 2 * IN).all()
    assert (w._o_proj(x) == 2 * IN).all()


def test_other_values_moved_to_the_same_address_are_seen_8bit(plain_fp8):
    """Offload and return: the parameter object stays, its storage is another one at the same address."""
    w, orig, buf = _wrapper(fp8_projections=True)
    x = torch.ones(1, IN)
    assert (w._o_proj(x) == IN).all()
    p = orig.o_proj.weight
    at, version = p.data_ptr(), p._version
    p.data = torch.empty(1)
    buf["o"][:] = 3.0
    p.data = torch.from_numpy(buf["o"])
    assert (p.data_ptr(), p._version) == (at, version)
    assert (w._o_proj(x) == 3 * IN).all()


def test_unchanged_sources_are_derived_once_and_data_writes_after_refresh_8bit(plain_fp8, monkeypatch):
    w, orig, buf = _wrapper(fp8_projections=True)
    calls = []
    real = ops.fp8_quantize_weight
    monkeypatch.setattr(ops, "fp8_quantize_weight", lambda t: calls.append(1) or real(t))
    x = torch.ones(1, IN)
    w._qkv(x)
    first = len(calls)
    for _ in range(3):
        w._qkv(x)
    assert first >= 3 and len(calls) == first
    with torch.no_grad():
        orig.k_proj.weight.mul_(2.0)
    assert (w._qkv(x)[:, 128:192] == 2 * IN).all()
    orig.k_proj.weight.data.mul_(2.0)      # not counted
    w.refresh_weights()
    assert (w._qkv(x)[:, 128:192] == 4 * IN).all()


def test_a_replaced_projection_at_the_same_address_is_seen_16bit():
    w, orig, buf = _wrapper()
    x = torch.ones(1, IN)
    mod = hga.HierarchicalGlobalAttentionRouted(d_model=IN, nhead=2, kv_heads=1, head_dim=64)
    mod.v_proj = _linear(buf["v"])
    assert (w._qkv(x) == IN).all() and (mod._fused_qkv()[0][192:] == 1).all()
    buf["v"][:] = 2.0                      # a fresh layer in the old one's memory
    for m in (orig, mod):
        at = m.v_proj.weight.data_ptr()
        del m.v_proj
        gc.collect()
        m.v_proj = _linear(buf["v"])
        assert m.v_proj.weight.data_ptr() == at and m.v_proj.weight._version == 0
    assert (w._qkv(x)[:, 192:] == 2 * IN).all() and (mod._fused_qkv()[0][192:] == 2).all()
    one = mod._fused_qkv()[0]
    assert mod._fused_qkv()[0] is one      # unchanged sources: nothing is made again
    mod.v_proj.weight.data.fill_(5.0)      # not counted
    mod.refresh_weights()
    assert (mod._fused_qkv()[0][192:] == 5).all()


def test_sources_are_not_kept_alive_and_survive_copies():
    t = torch.ones(4, 4)
    s = WeightSources((t, None))
    assert s.same((t, None)) and not s.same((t, t)) and not s.same((t,)) and not s.same((t.view(4, 4), None))
    assert not copy.deepcopy(s).same((t, None)) and not copy.copy(s).same((t, None))
    assert not pickle.loads(pickle.dumps(s)).same((t, None))
    t.add_(1)
    assert not s.same((t, None))
    import weakref
    r = weakref.ref(t)
    del t
    assert r() is None
