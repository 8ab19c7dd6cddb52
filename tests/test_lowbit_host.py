"""Host side of the 8-bit and 4-bit operators: refusals before any launch, weight quantisation, fake shapes."""
import ctypes

import pytest
import torch

from hierarchicalglobalattention_b200 import _lib, ops

ONE = ctypes.c_void_p(16)   # any aligned non-NULL pointer: validation fails before it is used


def test_fp8_entry_points_validate():
    h = _lib.lib()
    assert h.hga_fp8_quantize(4, 0, 1, ONE, 8, ONE, 8, ONE, None) == -1
    assert h.hga_fp8_quantize(0, 8, 1, None, 8, None, 8, None, None) == 0
    assert h.hga_fp8_quantize(4, 8, 3, ONE, 8, ONE, 8, ONE, None) == -1 and b"dtype" in h.hga_last_error()
    assert h.hga_fp8_quantize(4, 8, 1, ONE, 7, ONE, 8, ONE, None) == -1 and b"stride" in h.hga_last_error()
    assert h.hga_fp8_quantize(4, 8, 1, None, 8, ONE, 8, ONE, None) == -1 and b"NULL" in h.hga_last_error()
    lin = lambda m=4, n=8, k=256, xd=1, xs=None, xst=256, wst=256, wss=2, od=1, ost=8, ws=None, wsb=0: h.hga_fp8_linear(  # noqa: E731
        m, n, k, xd, ONE, xst, xs, ONE, wst, ONE, wss, None, od, ONE, ost, ws, wsb, None)
    assert lin(m=0) == 0
    assert lin(n=0) == -1 and lin(k=0, xst=0) == -1 and lin(m=-1) == -1
    assert lin(xd=4) == -1 and b"x_dtype" in h.hga_last_error()
    assert lin(od=3) == -1 and b"out_dtype" in h.hga_last_error()
    assert lin(xd=3) == -1 and b"x_scale" in h.hga_last_error()
    assert lin(wst=255) == -1 and lin(wss=1) == -1 and lin(ost=7) == -1 and b"stride" in h.hga_last_error()
    assert lin(m=2 ** 31) == -2
    need = h.hga_fp8_linear_workspace(4000, 4096, 4096, 1, ONE, 4096, ONE, 4096)
    assert need > 0
    rc = h.hga_fp8_linear(4000, 4096, 4096, 1, ONE, 4096, None, ONE, 4096, ONE, 32, None, 1, ONE, 4096, ONE, need - 1, None)
    assert rc == -1 and b"workspace" in h.hga_last_error()


def test_kv4_entry_points_validate():
    h = _lib.lib()
    pack = lambda dt=1, dh=128, heads=2, rows=16, cap=16, ucap=1, u0=0, k=ONE: h.hga_kv4_pack(  # noqa: E731
        dt, dh, heads, rows, k, ONE, cap, ONE, ONE, ucap, u0, None)
    assert pack(rows=0) == 0 and pack(heads=0) == 0
    assert pack(dt=3) == -1 and pack(dh=96) == -2 and pack(dh=320) == -2
    assert pack(cap=15) == -1 and b"kv_cap" in h.hga_last_error()
    assert pack(rows=17, cap=17) == -1 and b"capacity" in h.hga_last_error()
    assert pack(u0=1) == -1 and pack(u0=-1) == -1
    assert pack(k=ctypes.c_void_p(8)) == -1 and b"aligned" in h.hga_last_error()
    assert pack(k=None) == -1 and b"NULL" in h.hga_last_error()
    p = _lib.make_params(batch=1, nhead=4, kv_heads=2, head_dim=128, chunk_size=64, group_size=16, topk_chunks=4,
                         topk_groups=8, keep_first=1, keep_last=1, theta=1e4, dtype=torch.bfloat16)
    att = lambda L=1, kg=4, rec=ONE, q=ONE: h.hga_attend_decode_kv4(  # noqa: E731
        ctypes.byref(p), L, q, ONE, ONE, ONE, 192, rec, ONE, 64, ONE, ONE, kg, ONE, None)
    assert att(L=0) == -1 and att(L=65) == -1 and att(rec=None) == -1 and att(kg=-1) == -1
    assert att(q=ctypes.c_void_p(8)) == -1 and b"aligned" in h.hga_last_error()
    p.head_dim = 80
    assert att() == -2 and b"head_dim" in h.hga_last_error()
    p.head_dim, p.group_size = 128, 8
    assert att() == -2 and b"group_size" in h.hga_last_error()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 128)
    k = torch.zeros(1, 1, 16, 64)
    for call in (lambda: ops.fp8_quantize(x), lambda: ops.fp8_linear(x, x.to(torch.float8_e4m3fn), x),
                 lambda: ops.kv4_pack(k, k)):
        with pytest.raises(_lib.HgaError, match="CUDA"):
            call()


def test_weight_quantisation():
    """Every block's largest magnitude becomes 448, odd sizes keep their edges, a zero block has scale 1."""
    g = torch.Generator().manual_seed(0)
    w = torch.randn(300, 200, generator=g)
    w[128:256, :128] = 0
    q, s = ops.fp8_quantize_weight(w)
    assert q.shape == (300, 200) and s.shape == (3, 2) and q.dtype == torch.float8_e4m3fn
    assert s[1, 0] == 1 and (q[128:256, :128].float() == 0).all()
    for i in range(3):
        for j in range(2):
            blk, qb = w[128 * i:128 * i + 128, 128 * j:128 * j + 128], q[128 * i:128 * i + 128, 128 * j:128 * j + 128].float()
            if blk.abs().max() == 0:
                continue
            assert qb.abs().max() == 448
            # e4m3 has 4 significant bits: half a unit in the last place is 1/16 of a normal value
            assert ((qb * s[i, j] - blk).abs() <= blk.abs() / 16 + s[i, j] * 2.0 ** -10).all()
    with pytest.raises(_lib.HgaError):
        ops.fp8_quantize_weight(w[0])


def test_fp8_concat_lines_up_blocks():
    import torch.nn as nn
    from hierarchicalglobalattention_b200.fp8 import Fp8Linear, fp8_concat, fp8_weight_of
    torch.manual_seed(0)
    a, b, c = nn.Linear(200, 256, bias=False), nn.Linear(200, 128), nn.Linear(200, 30, bias=False)
    w, s, bias = fp8_concat([a, b, c])
    assert w.shape == (414, 200) and s.shape == (4, 2) and bias.shape == (414,)
    assert torch.equal(bias[256:384], b.bias) and (bias[:256] == 0).all() and (bias[384:] == 0).all()
    qa, sa = ops.fp8_quantize_weight(a.weight.detach())
    assert torch.equal(w[:256].float(), qa.float()) and torch.equal(s[:2], sa)
    assert fp8_concat([c, a]) is None                       # 30 features end inside a block
    assert fp8_concat([a, nn.ReLU()]) is None
    with pytest.raises(_lib.HgaError):
        fp8_concat([a, nn.Linear(100, 128)])
    m = Fp8Linear.from_linear(b)
    got = fp8_weight_of(m)
    assert torch.equal(got[0].float(), m.weight.float()) and torch.equal(got[2], b.bias)
    assert fp8_weight_of(a) is None and set(m.state_dict()) == {"weight", "weight_scale_inv", "bias"}


def test_low_bit_options_are_validated():
    import types
    import torch.nn as nn
    import hierarchicalglobalattention_b200 as hga
    with pytest.raises(ValueError, match="kv_bits"):
        hga.HierarchicalGlobalAttentionRouted(d_model=64, nhead=4, kv_heads=2, kv_bits=8)
    cfg = types.SimpleNamespace(num_attention_heads=4, num_key_value_heads=2, head_dim=64, hidden_size=64)
    with pytest.raises(ValueError, match="kv_bits"):
        hga.QwenRoutedAttention(nn.Identity(), cfg, kv_bits=2)
    with pytest.raises(ValueError, match="Dual Chunk"):
        hga.QwenRoutedAttention(nn.Identity(), cfg, kv_bits=4, dca_chunk=256)


def test_fake_shapes_of_the_dispatcher_ops():
    from hierarchicalglobalattention_b200 import torch_ops
    m = dict(device="meta", dtype=torch.bfloat16)
    x = torch.empty(3, 5, 300, **m)
    q, s = torch.ops.hga.fp8_quantize(x)
    assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and s.shape == (3, 5, 3) and s.dtype == torch.float32
    w, ws = torch.empty(200, 300, device="meta", dtype=torch.float8_e4m3fn), torch.empty(2, 3, device="meta")
    y = torch.ops.hga.fp8_linear(x, w, ws, None, None, None)
    assert y.shape == (3, 5, 200) and y.dtype == torch.bfloat16
    assert torch.ops.hga.fp8_linear(q, w, ws, None, s, torch.float32).dtype == torch.float32
    k = torch.empty(2, 4, 100, 128, **m)
    rk, rv = torch.ops.hga.kv4_pack(k, k)
    assert rk.shape == (2, 4, 7, 1280) and rv.dtype == torch.uint8
    assert torch.ops.hga.kv4_unpack(rk, rv, 100, torch.bfloat16)[0].shape == k.shape
    p = _lib.make_params(batch=2, nhead=8, kv_heads=4, head_dim=128, chunk_size=64, group_size=16, topk_chunks=4,
                         topk_groups=8, keep_first=1, keep_last=2, theta=1e4, dtype=torch.bfloat16)
    pi, pf = torch_ops.params_lists(p)
    qd = torch.empty(2, 8, 1, 128, **m)
    i32 = dict(device="meta", dtype=torch.int32)
    out = torch.ops.hga.attend_decode_kv4(pi, pf, qd, torch.empty(2, **i32), k, k, rk, rv, torch.empty(2, 8, 8, **i32),
                                          torch.empty(2, 8, 8, **i32))
    assert out.shape == qd.shape
