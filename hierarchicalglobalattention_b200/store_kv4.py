"""4-bit tier: the cold token record as 4-bit codes, windows and the active chunk in the model's type.

The layout of ``RamKVCacheStore`` with a record of 10 * head_dim bytes per 16 tokens and KV head instead of
32 * head_dim (bf16): codes with a 16-bit scale and minimum per token and 32 channels (``ops.kv4_pack``).  The
record is pinned host memory (``record_device="cpu"``, the RAM tier's place: 3.2 times fewer bytes cross the
host link per opened group) or HBM (``"cuda"``: 3.2 times the context in the same memory).  What is always
attended - the keep_first and keep_last windows and the active chunk - stays exact in HBM slots; a token is
read through its codes only once its chunk has left the windows and a group of it is opened.  Routing reads
the chunk and group summaries, which are built from the exact rows before they are packed.

The VRAM bank of the RAM tier works on packed groups unchanged (a group is a run of 16-byte pieces), so
``vram_cache_chunks`` holds 3.2 times the chunks in the same memory.

No counterpart in the reference, whose records hold the model dtype (ram_kv_cache_store.py:29-619).
"""
from __future__ import annotations

import copy
from typing import Dict, Optional, Tuple

import torch

from . import _lib, ops
from .store_ram import RamKVCacheStore


class Kv4CacheStore(RamKVCacheStore):
    """4-bit cold record with exact HBM windows (see module docstring)."""

    kv_bits = 4

    def __init__(self, *, record_device: str = "cpu", **kwargs) -> None:
        if record_device not in ("cpu", "cuda"):
            raise ValueError(f"record_device must be 'cpu' (pinned) or 'cuda'; got {record_device!r}")
        super().__init__(**kwargs)
        gs = self.C // self.M
        if gs % ops.KV4_UNIT or self.dh % 64 or self.dh > 256:
            raise ValueError("the 4-bit record needs a group_size that is a multiple of 16 and head_dim 64, 128, 192 or 256")
        self.record_device = record_device
        self.units_per_group = gs // ops.KV4_UNIT
        # exact rows of a prefill between seed_tokens and the filling of the windows (after_seed)
        self._seed_rows: Dict[int, Tuple[torch.Tensor, torch.Tensor]] = {}

    # -- buffers -----------------------------------------------------------------------------
    def _record(self, units: int) -> torch.Tensor:
        shape = (self.B, self.kvh, units, ops.kv4_unit_bytes(self.dh))
        if self.record_device == "cuda":
            return torch.zeros(shape, dtype=torch.uint8, device=self.compute_device)
        return torch.zeros(shape, dtype=torch.uint8).pin_memory()

    def ensure_capacity(self, layer: int, n_chunks: int, n_tokens: Optional[int] = None):
        n_tokens = n_chunks * self.C if n_tokens is None else n_tokens
        st = super().ensure_capacity(layer, n_chunks, 0)      # summaries and slots
        if n_tokens > st.tcap:
            cap = max(self._init_cap * self.C, 2 * st.tcap, n_tokens)
            cap = (cap + self.C - 1) // self.C * self.C
            rk, rv = self._record(cap // ops.KV4_UNIT), self._record(cap // ops.KV4_UNIT)
            if st.token_k is not None:
                if self.record_device == "cpu":
                    # packing kernels write the old record asynchronously
                    torch.cuda.current_stream(self.compute_device).synchronize()
                n = st.token_k.shape[2]
                rk[:, :, :n] = st.token_k
                rv[:, :, :n] = st.token_v
            st.token_k, st.token_v, st.tcap = rk, rv, cap
        return st

    def record(self, layer: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(rec_k, rec_v) uint8 [B,KVH,units,10*Dh] of the layer."""
        st = self.layer_buffers(layer)
        return st.token_k, st.token_v

    def cold_buffers(self, layer: int):
        # new rows enter the record when their chunk closes
        return None, None

    def adopt_tokens(self, layer, token_k, token_v) -> None:
        raise NotImplementedError("the 4-bit record is packed from its rows; write_tokens does that")

    def reset(self) -> None:
        self._seed_rows.clear()
        super().reset()

    # -- writing -----------------------------------------------------------------------------
    def write_tokens(self, layer: int, row0: int, token_k: torch.Tensor, token_v: torch.Tensor) -> None:
        """Pack rows [row0, row0 + L); row0 a multiple of 16."""
        if row0 % ops.KV4_UNIT:
            raise ValueError("rows enter the 4-bit record in whole 16-token units")
        ops.kv4_pack(token_k, token_v, self.record(layer), unit0=row0 // ops.KV4_UNIT)

    def seed_tokens(self, layer: int, token_k: torch.Tensor, token_v: torch.Tensor) -> None:
        """A prefill's rows: packed, and held until after_seed has filled the windows from them."""
        self.write_tokens(layer, 0, token_k, token_v)
        self._seed_rows[layer] = (token_k, token_v)

    def on_chunk_closed(self, layer: int, n: int, row: Optional[int] = None) -> None:
        """The completed active chunk is packed into the record and enters its window slots."""
        k_act, v_act = self.active_rows(layer, n)
        rk, rv = self.record(layer)
        b = slice(None) if row is None else slice(row, row + 1)
        ops.kv4_pack(k_act[b], v_act[b], (rk[b], rv[b]), unit0=n * self.C // ops.KV4_UNIT)
        super().on_chunk_closed(layer, n, row)

    def after_seed(self, layer: int, seq_len: int, row: Optional[int] = None) -> None:
        """Fill the window / active slots: from the prefill's exact rows where seed_tokens brought them, else with
        the record's values (RamKVCacheStore.after_seed reads its record)."""
        seed = self._seed_rows.get(layer)
        C, n = self.C, seq_len // self.C
        f_lo, f_hi = self.policy.hot_first_range(n)
        l_lo, l_hi = self.policy.hot_last_range(n)
        bs = slice(None) if row is None else slice(row, row + 1)

        def rows(r0: int, r1: int) -> Tuple[torch.Tensor, torch.Tensor]:
            if seed is not None:
                return seed[0][bs, :, r0:r1], seed[1][bs, :, r0:r1]
            self._sync_record()
            u0, u1 = r0 // ops.KV4_UNIT, -(-r1 // ops.KV4_UNIT)
            return self._unpacked(tuple(t[bs, :, u0:u1] for t in self.record(layer)), r1 - r0)

        for c in sorted(set(range(f_lo, f_hi)) | set(range(l_lo, l_hi))):
            self._to_slot(layer, c, *rows(c * C, (c + 1) * C), None if row is None else 0, row)
        rem = seq_len - n * C
        if rem:
            k_act, v_act = self.active_rows(layer, n)
            k, v = rows(n * C, seq_len)
            k_act[bs, :, :rem].copy_(k)
            v_act[bs, :, :rem].copy_(v)
        if row is None or row == self.B - 1:
            self._seed_rows.pop(layer, None)

    # -- the VRAM bank, on packed groups ---------------------------------------------------------
    def _group_bytes(self) -> int:
        return self.units_per_group * ops.kv4_unit_bytes(self.dh)

    def _effective_slots(self) -> int:
        if self._bank_slots is None:
            want = 0 if self.record_device == "cuda" else self.vram_cache_chunks * self.M
            if want > 0 and self.compute_device.type == "cuda":
                free, _ = torch.cuda.mem_get_info(self.compute_device)
                budget = free - self.vram_cache_reserve_gb * (1 << 30)
                per_slot = self.B * self.kvh * (2 * self._group_bytes() + 8)
                want = min(want, int(max(0, budget) // max(1, self.num_layers) // per_slot))
            self._bank_slots = max(0, want)
        return self._bank_slots

    def bank_for(self, layer: int, need_slots: int) -> Optional[dict]:
        slots = self._effective_slots()
        if slots <= 0 or slots < need_slots:
            return None
        gid_cap = self.layer_buffers(layer).tcap // (self.C // self.M)
        bk, dev = self._bank.get(layer), self.compute_device
        i32 = dict(dtype=torch.int32, device=dev)
        if bk is None:
            shape = (self.B, self.kvh, slots * self.units_per_group, ops.kv4_unit_bytes(self.dh))
            bk = {"k": torch.zeros(shape, dtype=torch.uint8, device=dev), "v": torch.zeros(shape, dtype=torch.uint8, device=dev),
                  "slot_gid": torch.full((self.B, self.kvh, slots), -1, **i32),
                  "slot_stamp": torch.full((self.B, self.kvh, slots), -1, **i32),
                  "gid_slot": torch.full((self.B, self.kvh, gid_cap), -1, **i32), "slots": slots, "stamp": 0}
            self._bank[layer] = bk
        elif bk["gid_slot"].shape[2] < gid_cap:
            g = torch.full((self.B, self.kvh, gid_cap), -1, **i32)
            g[:, :, :bk["gid_slot"].shape[2]] = bk["gid_slot"]
            bk["gid_slot"] = g
        return bk

    def bank_gather(self, layer: int, hp, open_gid: torch.Tensor):
        """One decode step's hga_gather_h2d on packed groups: (bank_k, bank_v, open_slot), or None."""
        H, Kg = open_gid.shape[1], open_gid.shape[2]
        bk = self.bank_for(layer, (H // self.kvh) * Kg)
        if bk is None or Kg == 0:
            return None
        # the gather copies a group's bytes: rows of 10 * Dh / 16 bytes seen as 16-bit values
        p = copy.copy(hp)
        p.head_dim, p.dtype = 10 * self.dh // 32, _lib.DTYPE_CODE[torch.bfloat16]
        rk, rv = (self._as_rows(t, p.head_dim) for t in self.record(layer))
        slot = ops.gather_h2d(p, open_gid, rk, rv, self._as_rows(bk["k"], p.head_dim), self._as_rows(bk["v"], p.head_dim),
                              bk["slot_gid"], bk["gid_slot"], bk["slot_stamp"], bk["stamp"], self._counters)
        bk["stamp"] += 1
        return bk["k"], bk["v"], slot

    @staticmethod
    def _as_rows(rec: torch.Tensor, width: int) -> torch.Tensor:
        return rec.view(torch.bfloat16).view(rec.shape[0], rec.shape[1], -1, width)

    # -- attention ---------------------------------------------------------------------------
    def attend_decode(self, layer: int, hp, q: torch.Tensor, seq_pos: torch.Tensor, open_gid: torch.Tensor,
                      open_t0: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of one routed decode block over the slots and the record (through the bank, if any)."""
        hot_k, hot_v = self.hot_buffers(layer)
        rk, rv = self.record(layer)
        banked = self.bank_gather(layer, hp, open_gid)
        if banked is not None:
            rk, rv, open_gid = banked
        return ops.attend_decode_kv4(hp, q, seq_pos, hot_k, hot_v, rk, rv, open_gid, open_t0, out=out)

    # -- reading back (KVCacheStore API): the record's values -----------------------------------
    def _unpacked(self, rec_units: Tuple[torch.Tensor, torch.Tensor], rows: int):
        rk, rv = (t.to(self.compute_device).contiguous() for t in rec_units)
        return ops.kv4_unpack(rk, rv, rows, self.dtype)

    def _sync_record(self) -> None:
        if self.record_device == "cpu":
            # indexing on the host: the packing kernels' writes have to have landed
            torch.cuda.current_stream(self.compute_device).synchronize()

    def gather_tokens(self, layer, chunk_idx, group_idx):
        self._sync_record()
        rk, rv = self.record(layer)
        gs, U = self.C // self.M, self.units_per_group
        cidx = chunk_idx.to(rk.device)
        unit = ((cidx * self.C + group_idx.to(rk.device) * gs) // ops.KV4_UNIT).unsqueeze(-1) + torch.arange(U, device=rk.device)
        b, kv = self._kvh_index(cidx)
        b, kv = b.to(rk.device).unsqueeze(-1), kv.to(rk.device).unsqueeze(-1)
        B, H, K = chunk_idx.shape
        units = tuple(t[b, kv, unit].reshape(B, H, K * U, -1) for t in (rk, rv))
        k, v = self._unpacked(units, K * gs)
        return k.view(B, H, K, gs, self.dh), v.view(B, H, K, gs, self.dh)

    def gather_chunk_tokens_kvh(self, layer, chunk_idx):
        self._sync_record()
        rk, rv = self.record(layer)
        B, KVH, K = chunk_idx.shape
        per = self.C // ops.KV4_UNIT
        unit = (chunk_idx.to(rk.device).unsqueeze(-1) * per + torch.arange(per, device=rk.device)).flatten(-2)
        idx = unit.unsqueeze(-1).expand(-1, -1, -1, rk.shape[-1])
        k, v = self._unpacked((rk.gather(2, idx), rv.gather(2, idx)), K * self.C)
        return k.view(B, KVH, K, self.C, self.dh), v.view(B, KVH, K, self.C, self.dh)

    def hot_tokens(self, layer, lo, hi):
        self._sync_record()
        rk, rv = self.record(layer)
        per = self.C // ops.KV4_UNIT
        k, v = self._unpacked((rk[:, :, lo * per:hi * per], rv[:, :, lo * per:hi * per]), (hi - lo) * self.C)
        shape = (self.B, self.kvh, hi - lo, self.C, self.dh)
        return k.view(shape), v.view(shape)


__all__ = ["Kv4CacheStore"]
