"""Ways into a 4-bit store besides a prefill, run on the CPU with a plain record and on the GPU with the real one."""
import gc

import torch
from torch.multiprocessing.reductions import StorageWeakRef

from hierarchicalglobalattention_b200 import ChunkPlacementPolicy, Kv4CacheStore, ops

C, GS, DH, KVH, B = 32, 16, 64, 2, 2


def store(dev, record):
    pol = ChunkPlacementPolicy(keep_first=1, keep_last=2, first_token_level=True)
    return Kv4CacheStore(record_device=record, compute_device=dev, policy=pol, kv_heads=KVH, head_dim=DH, chunk_size=C,
                         groups_per_chunk=C // GS, batch_size=B, dtype=torch.bfloat16, initial_capacity=4)


def rows(n, dev):
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(B, KVH, n, DH, generator=g).bfloat16().to(dev) for _ in range(2))
    return k, v


def _ingest(st, how, n, dev):
    """n chunks of fresh rows: a weak reference to their memory and what reading the record back has to give."""
    k, v = rows(n * C, dev)
    s = torch.zeros(B, KVH, n, DH, device=dev, dtype=torch.bfloat16)
    gsum = torch.zeros(B, KVH, n, C // GS, DH, device=dev, dtype=torch.bfloat16)
    if how == "bulk":
        st.seed_closed_chunks(0, s, gsum, gsum, k.view(B, KVH, n, C, DH), v.view(B, KVH, n, C, DH))
    else:
        for i in range(n):
            sl = slice(i * C, (i + 1) * C)
            st.append_closed_chunk(0, s[:, :, i], gsum[:, :, i], gsum[:, :, i], k[:, :, sl], v[:, :, sl])
    want = ops.kv4_unpack(*ops.kv4_pack(k, v), n * C, torch.bfloat16)
    return StorageWeakRef(k.untyped_storage()), want


def check_ingest(dev, record, how):
    """The rows are let go at once, and after_seed fills the windows from the record, as often as it is called."""
    st = store(dev, record)
    n = 7
    ref, (wk, wv) = _ingest(st, how, n, dev)
    gc.collect()
    assert ref.expired()
    for _ in range(2):
        st.after_seed(0, n * C)
    hk, hv = st.hot_buffers(0)
    for c, slot in ((0, 0), (5, 1 + 5 % 2), (6, 1 + 6 % 2)):
        a, b = slice(slot * C, (slot + 1) * C), slice(c * C, (c + 1) * C)
        assert torch.equal(hk[:, :, a], wk[:, :, b]) and torch.equal(hv[:, :, a], wv[:, :, b])
    # one sequence's windows of a shorter length, a ragged tail in the active chunk
    st.after_seed(0, 5 * C + 9, row=1)
    act = slice(3 * C, 3 * C + 9)
    tail = slice(5 * C, 5 * C + 9)
    assert torch.equal(hk[1, :, act], wk[1, :, tail]) and torch.equal(hv[1, :, act], wv[1, :, tail])
    assert torch.equal(hk[1, :, C:2 * C], wk[1, :, 4 * C:5 * C]) and torch.equal(hk[0, :, 2 * C:3 * C], wk[0, :, 5 * C:6 * C])


def check_prefill_windows_are_exact(dev, record):
    st = store(dev, record)
    n = 4 * C + 5
    k, v = rows(n, dev)
    st.ensure_capacity(0, 4, n)
    st.seed_tokens(0, k, v)
    ref = StorageWeakRef(k.untyped_storage())
    st.after_seed(0, n)
    hk, hv = st.hot_buffers(0)
    for c, slot in ((0, 0), (2, 1), (3, 2)):
        a, b = slice(slot * C, (slot + 1) * C), slice(c * C, (c + 1) * C)
        assert torch.equal(hk[:, :, a], k[:, :, b]) and torch.equal(hv[:, :, a], v[:, :, b])
    assert torch.equal(hk[:, :, 3 * C:3 * C + 5], k[:, :, 4 * C:])
    del k
    gc.collect()
    assert ref.expired()
