"""The dispatcher operators' fake results have the strides of the real ones (contiguous), whatever the inputs' are."""
import torch

from hierarchicalglobalattention_b200 import _lib, torch_ops


def test_decode_operators_return_contiguous_rows():
    m = dict(device="meta", dtype=torch.bfloat16)
    i32 = dict(device="meta", dtype=torch.int32)
    p = _lib.make_params(batch=2, nhead=8, kv_heads=4, head_dim=128, chunk_size=64, group_size=16, topk_chunks=4,
                         topk_groups=8, keep_first=1, keep_last=2, theta=1e4, dtype=torch.bfloat16)
    pi, pf = torch_ops.params_lists(p)
    q = torch.empty(2, 5, 8, 128, **m).transpose(1, 2)              # token-major rows seen as [B,H,L,Dh]
    hot = torch.empty(2, 4, 256, 128, **m)
    rec = torch.empty(2, 4, 40, 1280, device="meta", dtype=torch.uint8)
    pos, gid = torch.empty(2, **i32), torch.empty(2, 8, 8, **i32)
    h = torch.ops.hga
    for out in (h.attend_decode_kv4(pi, pf, q, pos, hot, hot, rec, rec, gid, gid),
                h.attend_decode(pi, pf, q, pos, hot, hot, 0, hot, hot, gid, gid),
                h.attend_decode_dca(pi, pf, q, pos, hot, hot, 0, hot, hot, gid, gid, None, 128, 256, 1e4)):
        assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    t = torch.empty(8, 2, 8, **i32).transpose(0, 1)
    slots = torch.empty(2, 4, 16, **i32)
    out = h.gather_h2d(pi, pf, t, hot, hot, hot, hot, slots, slots, slots, 0, torch.empty(2, device="meta", dtype=torch.int64))
    assert out.shape == t.shape and out.is_contiguous()
