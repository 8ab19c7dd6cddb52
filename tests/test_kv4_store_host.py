"""Ways into the 4-bit store on the CPU: its kernels replaced by plain code over a record of the same size."""
import pytest
import torch

import kv4_store_cases as K
import lowbit_ref as R
from hierarchicalglobalattention_b200 import ops


def _pack(k, v, rec=None, unit0=0):
    B, KVH, S, Dh = k.shape
    units = -(-S // 16)
    if rec is None:
        rec = tuple(torch.zeros(B, KVH, unit0 + units, 10 * Dh, dtype=torch.uint8) for _ in range(2))
    for x, r in zip((k, v), rec):
        p = torch.zeros(B, KVH, units * 16, Dh, dtype=x.dtype)
        p[:, :, :S] = x
        n, s, m = R.kv4_codes(p)
        n = n.flatten(-2).to(torch.uint8).view(B, KVH, units, 16 * Dh)
        meta = torch.cat((s, m), -1).view(B, KVH, units, -1).view(torch.uint8)
        r[:, :, unit0:unit0 + units] = torch.cat((n[..., ::2] | n[..., 1::2] << 4, meta), -1)
    return rec


def _unpack(rk, rv, rows, dtype, unit0=0, device=None):
    out = []
    for r in (rk, rv):
        B, KVH, _, nb = r.shape
        Dh = nb // 10
        r = r[:, :, unit0:unit0 + -(-rows // 16)]
        c = r[..., :8 * Dh]
        n = torch.stack((c & 15, c >> 4), -1).flatten(-2).view(B, KVH, -1, Dh // 32, 32).float()
        meta = r[..., 8 * Dh:].contiguous().view(dtype).view(B, KVH, -1, Dh // 32, 2)
        out.append(R.kv4_value(n, meta[..., :1], meta[..., 1:], dtype)[:, :, :rows])
    return tuple(out)


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(ops, "kv4_pack", _pack)
    monkeypatch.setattr(ops, "kv4_unpack", _unpack)


@pytest.mark.parametrize("how", ["bulk", "one by one"])
def test_ingested_chunks(plain, how):
    K.check_ingest(torch.device("cpu"), "cuda", how)


def test_prefill_windows_are_exact(plain):
    K.check_prefill_windows_are_exact(torch.device("cpu"), "cuda")
