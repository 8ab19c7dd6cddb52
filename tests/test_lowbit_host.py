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
