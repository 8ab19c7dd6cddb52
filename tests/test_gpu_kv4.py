"""The 4-bit KV record (pack, unpack) and the decode attention over it against plain implementations."""
import math

import pytest
import torch

import lowbit_ref as R

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
# largest relative error of one rounding to the type
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def _kv(g, B, KVH, S, Dh, dtype):
    gain = 1 + 5 * (torch.rand(KVH, 1, Dh, generator=g) > 0.95)
    return (torch.randn(B, KVH, S, Dh, generator=g) * gain).to(dtype), torch.randn(B, KVH, S, Dh, generator=g).to(dtype)


def _same(a, b):
    return torch.equal(torch.nan_to_num(a.float(), nan=123.0), torch.nan_to_num(b.float(), nan=123.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,KVH,S,Dh", [(1, 1, 1, 64), (2, 3, 15, 128), (1, 2, 16, 192), (3, 1, 17, 256), (2, 4, 64, 128),
                                        (1, 2, 333, 64)])
def test_pack_unpack_is_the_definition(cuda, dtype, B, KVH, S, Dh):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(S * 7 + Dh)
    k, v = _kv(g, B, KVH, S, Dh, dtype)
    k[..., 0, :32] = 0.75              # a block of equal values
    rk, rv = ops.kv4_pack(k.to(cuda), v.to(cuda))
    units = (S + 15) // 16
    assert rk.shape == (B, KVH, units, 10 * Dh) and rk.dtype == torch.uint8
    uk, uv = ops.kv4_unpack(rk, rv, S, dtype)
    for x, rec, u, is_v in ((k, rk, uk, False), (v, rv, uv, True)):
        n, s, m = R.kv4_codes(x)
        assert torch.equal(u.cpu(), R.kv4_value(n, s, m, dtype))
        codes = R.kv4_byte_codes(rec.cpu(), Dh, is_v).flatten(2, 3)
        assert torch.equal(codes[:, :, :S].float(), n.flatten(-2))
        assert (codes[:, :, S:] == 0).all()
        meta = rec.cpu()[..., 8 * Dh:].contiguous().view(R.META[dtype]).view(B, KVH, units * 16, Dh // 32, 2)
        assert torch.equal(meta[:, :, :S, :, :1], s) and torch.equal(meta[:, :, :S, :, 1:], m)
    assert torch.equal(uk[..., 0, :32].cpu(), torch.full((B, KVH, 32), 0.75, dtype=dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_pack_extremes(cuda, dtype):
    """Infinities and NaN cost their own block, large and tiny values keep their block's accuracy."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(5)
    k, v = _kv(g, 1, 1, 32, 128, dtype)
    k[0, 0, 3, 40] = math.inf
    v[0, 0, 17, 127] = math.nan
    k[0, 0, 5, :32] *= 1e3
    v[0, 0, 6, :32] *= 1e-4
    v[0, 0, 7, :] = 0
    out = ops.kv4_unpack(*ops.kv4_pack(k.to(cuda), v.to(cuda)), 32, dtype)
    for x, u in zip((k, v), out):
        n, s, m = R.kv4_codes(x)
        assert _same(u.cpu(), R.kv4_value(n, s, m, dtype))
        assert int(u.isnan().sum()) == 32
    assert (out[1][0, 0, 7] == 0).all()


def test_pack_places_and_layouts(cuda):
    """Units in the middle of a larger record, row-slices of a larger buffer, transposed rows, pinned host records."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(6)
    k, v = (t.to(cuda) for t in _kv(g, 2, 3, 96, 128, torch.bfloat16))
    want = ops.kv4_pack(k[:, :, 32:80], v[:, :, 32:80])
    for pinned in (False, True):
        rec = tuple(torch.full((2, 3, 9, 1280), 7, dtype=torch.uint8) for _ in range(2))
        rec = tuple(r.pin_memory() if pinned else r.to(cuda) for r in rec)
        ops.kv4_pack(k[:, :, 32:80], v[:, :, 32:80], rec, unit0=4)
        torch.cuda.synchronize()
        for r, w in zip(rec, want):
            assert torch.equal(r[:, :, 4:7].cpu(), w.cpu()) and (r[:, :, :4] == 7).all() and (r[:, :, 7:] == 7).all()
        back = ops.kv4_unpack(*rec, 48, torch.bfloat16, unit0=4, device=cuda)
        for a, b in zip(back, ops.kv4_unpack(*want, 48, torch.bfloat16)):
            assert torch.equal(a, b)
    tk, tv = k.transpose(1, 2).contiguous().transpose(1, 2), v.transpose(1, 2).contiguous().transpose(1, 2)
    for r, w in zip(ops.kv4_pack(tk, tv), ops.kv4_pack(k, v)):
        assert torch.equal(r, w)
    for r, w in zip(ops.kv4_pack(tk, v), ops.kv4_pack(k, v)):
        assert torch.equal(r, w)
    assert ops.kv4_pack(k[:, :, :0], v[:, :, :0])[0].shape == (2, 3, 0, 1280)


def _state(g, B, H, KVH, Dh, dtype, C, gs, kf, kl, pos, L, Kg, cuda, chunks=None, t0_max=None, opened=True):
    """A decode state with a record of random rows; opened groups random in the routed pool (-1 elsewhere)."""
    from hierarchicalglobalattention_b200 import _lib, ops
    n_chunks = (max(pos) // C + 1) if chunks is None else chunks
    k, v = _kv(g, B, KVH, n_chunks * C, Dh, dtype)
    rec = ops.kv4_pack(k.to(cuda), v.to(cuda))
    hk, hv = _kv(g, B, KVH, (kf + kl + 1) * C, Dh, dtype)
    q = torch.randn(B, H, L, Dh, generator=g).to(dtype)
    gid = torch.full((B, H, Kg), -1, dtype=torch.int32)
    t0 = torch.full((B, H, Kg), -1, dtype=torch.int32)
    M = C // gs
    for b in range(B):
        n = pos[b] // C
        f_hi = min(kf, n)
        l_lo = n if kl <= 0 else min(max(kf, n - kl), n)
        pool = max(0, l_lo - f_hi) * M
        for h in range(H):
            c = min(Kg, pool) if opened else 0
            if c and h % 3 == 2:
                c = int(torch.randint(0, c + 1, (1,), generator=g))
            ids = torch.randperm(pool, generator=g)[:c].sort().values + f_hi * M if c else torch.zeros(0)
            gid[b, h, :c] = ids.int()
            t0[b, h, :c] = torch.randint(0, L if t0_max is None else t0_max, (c,), generator=g).int()
    p = _lib.make_params(batch=B, nhead=H, kv_heads=KVH, head_dim=Dh, chunk_size=C, group_size=gs, topk_chunks=16,
                         topk_groups=64, keep_first=kf, keep_last=kl, theta=1e6, dtype=dtype)
    return dict(p=p, q=q, pos=torch.tensor(pos, dtype=torch.int32), hk=hk, hv=hv, rec=rec, gid=gid, t0=t0, C=C, gs=gs,
                kf=kf, kl=kl, rows=n_chunks * C)


def _run(st, cuda, rec=None):
    from hierarchicalglobalattention_b200 import ops
    rk, rv = st["rec"] if rec is None else rec
    return ops.attend_decode_kv4(st["p"], st["q"].to(cuda), st["pos"].to(cuda), st["hk"].to(cuda), st["hv"].to(cuda), rk,
                                 rv, st["gid"].to(cuda), st["t0"].to(cuda))


def _want(st):
    from hierarchicalglobalattention_b200 import ops
    # the record's values in fp32 (scale * code + min, unrounded)
    dt = st["q"].dtype
    mt = R.META[dt]
    vals = []
    for rec, is_v in zip(st["rec"], (False, True)):
        Dh = rec.shape[-1] // 10
        n = R.kv4_byte_codes(rec.cpu(), Dh, is_v).double()
        meta = rec.cpu()[..., 8 * Dh:].contiguous().view(mt).view(*rec.shape[:3], 16, Dh // 32, 2).double()
        x = n.unflatten(-1, (-1, 32)) * meta[..., :1] + meta[..., 1:]
        vals.append(x.flatten(-2).flatten(2, 3))
    assert ops.KV4_UNIT == 16
    return R.attend(st["q"], st["pos"], st["hk"], st["hv"], vals[0], vals[1], st["gid"], st["t0"], st["C"], st["gs"],
                    st["kf"], st["kl"])


def _check(out, st):
    ref, mag = _want(st)
    dt = st["q"].dtype
    # the result's rounding; the weights (times the record's scale) enter the products in 16 bits for the
    # 16-bit types: half an ulp of bf16 each; fp32 elsewhere
    tol = HALF_ULP[dt] * 1.01 * ref.abs() + (2.0 ** -8 if dt != torch.float32 else 2.0 ** -15) * mag + 1e-6
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} of the tolerance"


CASES = [
    # B, H, KVH, Dh, C, gs, kf, kl, pos, L, Kg
    (1, 1, 1, 64, 64, 16, 0, 0, [0], 1, 0),
    (1, 4, 1, 128, 64, 16, 1, 1, [1], 1, 8),
    (2, 8, 1, 128, 64, 16, 2, 2, [63, 64], 1, 8),
    (2, 8, 2, 128, 64, 16, 1, 2, [700, 65], 1, 16),
    (1, 8, 1, 64, 64, 16, 0, 0, [1000], 1, 32),
    (2, 6, 2, 128, 64, 16, 2, 1, [900, 383], 1, 20),
    (1, 16, 1, 128, 64, 16, 1, 1, [640], 1, 12),
    (1, 40, 2, 64, 64, 16, 0, 1, [500], 1, 9),
    (1, 8, 2, 128, 32, 16, 1, 3, [499], 2, 10),
    (1, 8, 1, 128, 128, 32, 1, 1, [1000], 3, 6),
    (2, 4, 2, 192, 64, 32, 0, 2, [600, 122], 5, 8),
    (1, 2, 1, 256, 64, 16, 1, 1, [300], 7, 8),
    (1, 8, 1, 128, 64, 16, 1, 2, [640], 64, 24),
    (1, 8, 2, 64, 64, 16, 0, 1, [459], 33, 16),
    (2, 3, 1, 128, 64, 16, 2, 0, [512, 0], 12, 16),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_attend(cuda, case, dtype):
    B, H, KVH, Dh, C, gs, kf, kl, pos, L, Kg = case
    g = torch.Generator().manual_seed(H * 100 + L * 10 + Kg)
    st = _state(g, B, H, KVH, Dh, dtype, C, gs, kf, kl, pos, L, Kg, cuda)
    _check(_run(st, cuda), st)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 6])
def test_unseen_rows_may_hold_anything(cuda, dtype, L):
    """NaN and infinities in rows that no (or not this) query row sees: window slots of chunks that do not exist
    yet, the active chunk's later rows, groups of other heads, groups that later rows open."""
    g = torch.Generator().manual_seed(11)
    st = _state(g, 2, 8, 1, 128, dtype, 64, 16, 2, 3, [200, 1030], L, 6, cuda)
    clean = _run(st, cuda)
    C, kf = 64, 2
    for b, pos in enumerate((200, 1030)):
        st["hk"][b, :, 5 * C + pos % C + L:] = math.nan
        st["hv"][b, :, 5 * C + pos % C + L:] = math.inf
    # sequence 0 has chunks 0..2 closed: chunk 2 sits in ring slot 2 + 2 % 3, the ring's others are empty
    for slot in (2 + 0, 2 + 1):
        st["hk"][0, :, slot * C:(slot + 1) * C] = math.inf
        st["hv"][0, :, slot * C:(slot + 1) * C] = math.nan
    assert torch.equal(_run(st, cuda), clean)
    # a group that only head 0 opens reads back as NaN: only head 0's rows from its t0 on are NaN
    used = set(st["gid"][1].flatten().tolist())
    lone = next(i for i in range(kf * 4, 13 * 4) if i not in used)
    st["gid"][1, 0, 0], st["t0"][1, 0, 0] = lone, L - 1
    clean = _run(st, cuda)
    rec = tuple(r.clone() for r in st["rec"])
    meta = rec[1].view(R.META[dtype]) if dtype != torch.float32 else rec[1].view(torch.bfloat16)
    meta[1, 0, lone, 4 * 128:] = math.nan
    bad = _run(st, cuda, rec)
    assert bad[1, 0, L - 1].isnan().all() and not clean.isnan().any()
    bad[1, 0, L - 1] = clean[1, 0, L - 1]
    assert torch.equal(bad, clean)


@pytest.mark.parametrize("L", [2, 9, 64])
def test_a_later_token_that_is_not_finite_leaves_the_earlier_rows_alone(cuda, L):
    g = torch.Generator().manual_seed(12)
    st = _state(g, 1, 8, 2, 128, torch.bfloat16, 64, 16, 1, 1, [512], L, 6, cuda)
    clean = _run(st, cuda)
    st["hv"][0, 1, 2 * 64 + L - 1, 7] = math.inf
    bad = _run(st, cuda)
    assert torch.equal(bad[:, :, :-1], clean[:, :, :-1]) and torch.equal(bad[:, :4], clean[:, :4])
    assert bad[0, 4:, -1, 7].isinf().all()


def test_gaps_in_the_lists(cuda):
    """-1 anywhere in a list and entries that no row sees are skipped."""
    g = torch.Generator().manual_seed(13)
    st = _state(g, 1, 8, 1, 128, torch.bfloat16, 64, 16, 1, 1, [1500], 1, 24, cuda)
    st["gid"][0, :, ::5] = -1
    st["t0"][0, 1, 3] = -1
    out = _run(st, cuda)
    st["gid"][0, 1, 3] = -1
    _check(out, st)


def test_every_group_opened_is_dense_attention(cuda):
    """All of the pool opened by every head: attention over the whole context; the shared heads agree with single ones."""
    g = torch.Generator().manual_seed(14)
    st = _state(g, 1, 8, 1, 128, torch.bfloat16, 64, 16, 1, 2, [64 * 30 + 5], 1, 27 * 4, cuda)
    st["gid"][:] = torch.arange(4, 28 * 4, dtype=torch.int32)
    st["t0"][:] = 0
    _check(_run(st, cuda), st)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_pinned_record_streams_and_graphs_give_the_same_bits(cuda, dtype):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(15)
    st = _state(g, 3, 16, 2, 128, dtype, 64, 16, 1, 2, [1999, 70, 3000], 1, 16, cuda)
    want = _run(st, cuda)
    host = tuple(r.cpu().pin_memory() for r in st["rec"])
    assert torch.equal(_run(st, cuda, host), want) and torch.equal(_run(st, cuda), want)
    args = [st["q"].to(cuda), st["pos"].to(cuda), st["hk"].to(cuda), st["hv"].to(cuda), *st["rec"], st["gid"].to(cuda),
            st["t0"].to(cuda)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = ops.attend_decode_kv4(st["p"], *args)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            b = ops.attend_decode_kv4(st["p"], *args)
        gr.replay()
    s.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


def test_long_record_offsets(cuda):
    """Unit offsets past 2^32 bytes: the same groups at the end of a 5 GB record and in a small one."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(16)
    st = _state(g, 1, 8, 2, 128, torch.bfloat16, 64, 16, 1, 1, [64 * 20], 1, 8, cuda)
    want = _run(st, cuda)
    units, small = 2 ** 21, st["rec"][0].shape[2]
    big = tuple(torch.zeros(1, 2, units, 1280, dtype=torch.uint8, device=cuda) for _ in range(2))
    for b, r in zip(big, st["rec"]):
        b[:, :, units - small:] = r
    st["gid"] += (st["gid"] >= 0).int() * (units - small)
    assert torch.equal(_run(st, cuda, big), want)
    k = torch.randn(1, 2, 64, 128, generator=g).bfloat16().to(cuda)
    ops.kv4_pack(k, k, big, unit0=units - 4)
    back = ops.kv4_unpack(*big, 64, torch.bfloat16, unit0=units - 4)
    for a, b in zip(back, ops.kv4_unpack(*ops.kv4_pack(k, k), 64, torch.bfloat16)):
        assert torch.equal(a, b)


def test_bounds_are_reported_not_read(cuda):
    """A group past the record is skipped, a position outside its slots gives zeros; both set the error word."""
    from hierarchicalglobalattention_b200 import _lib
    g = torch.Generator().manual_seed(17)
    st = _state(g, 2, 8, 1, 128, torch.bfloat16, 64, 16, 1, 1, [700, 640], 1, 8, cuda)
    _lib.device_status()
    clean = _run(st, cuda)
    assert _lib.device_status() == 0
    st["gid"][0, 2, 0] = 4 * 11 + 3 + 1000
    out = _run(st, cuda)
    assert _lib.device_status() == 0x104
    assert torch.equal(out[1], clean[1]) and out.isfinite().all()
    st["pos"][0] = -3
    out = _run(st, cuda)
    assert _lib.device_status() == 0x104 and (out[0] == 0).all() and torch.equal(out[1], clean[1])
    assert _lib.device_status() == 0


@pytest.mark.parametrize("Dh,dtype", [(128, torch.bfloat16), (64, torch.float16), (128, torch.float32)])
def test_scores_of_minus_infinity(cuda, Dh, dtype):
    """A key of -infinity against every query has weight 0, also where it is all that a unit shows."""
    g = torch.Generator().manual_seed(19)
    st = _state(g, 1, 8, 2, Dh, dtype, 64, 16, 1, 1, [640], 1, 6, cuda)
    st["q"][..., 5] = 1.0
    st["hk"][:, :, 2 * 64, 5] = -math.inf
    _check(_run(st, cuda), st)


def test_largest_group_number_is_out_of_bounds(cuda):
    from hierarchicalglobalattention_b200 import _lib
    g = torch.Generator().manual_seed(20)
    for dtype in (torch.bfloat16, torch.float32):
        st = _state(g, 1, 8, 1, 128, dtype, 64, 16, 1, 1, [700], 1, 8, cuda)
        _lib.device_status()
        st["gid"][0, 2, 0] = 2 ** 31 - 1
        out = _run(st, cuda)
        assert _lib.device_status() == 0x104
        st["gid"][0, 2, 0] = -1
        assert torch.equal(_run(st, cuda), out)


@pytest.mark.parametrize("B", [1, 2])
@pytest.mark.parametrize("S", [1, 40])
def test_pack_one_kv_head_of_token_major_rows(cuda, B, S):
    """[B,S,1,Dh] rows seen as [B,1,S,Dh]: contiguous, with free strides in the dimensions of size one."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(21)
    k, v = (t.to(cuda) for t in _kv(g, B, 1, 2 * S, 128, torch.bfloat16))
    want = ops.kv4_pack(k[:, :, :S].contiguous(), v[:, :, :S].contiguous())
    tk, tv = k[:, 0, :S].unsqueeze(2).contiguous().transpose(1, 2), v[:, 0, :S, None].transpose(1, 2)
    for a, b in ((tk, tv), (tk, tk), (k[:, :, :S], tv), (k[:, :, :S], v[:, :, :S])):
        got = ops.kv4_pack(a, b)
        assert torch.equal(got[0], want[0]) and (b is tk or torch.equal(got[1], want[1]))


def test_strided_positions(cuda):
    g = torch.Generator().manual_seed(22)
    st = _state(g, 2, 8, 1, 128, torch.bfloat16, 64, 16, 1, 1, [700, 300], 1, 8, cuda)
    want = _run(st, cuda)
    st["pos"] = torch.tensor([[700, 0], [300, 0]], dtype=torch.int32, device=cuda)[:, 0]
    assert torch.equal(_run(st, cuda), want)


def test_refusals(cuda):
    from hierarchicalglobalattention_b200 import _lib, ops
    g = torch.Generator().manual_seed(18)
    st = _state(g, 1, 4, 2, 128, torch.bfloat16, 64, 16, 1, 1, [300], 1, 4, cuda)
    E = _lib.HgaError
    k = torch.zeros(1, 2, 16, 128, device=cuda)
    with pytest.raises(E, match="one shape and type"):
        ops.kv4_pack(k, k.half())
    with pytest.raises(E, match="head_dim"):
        ops.kv4_pack(k[..., :96].contiguous(), k[..., :96].contiguous())
    with pytest.raises(E, match="capacity"):
        ops.kv4_pack(k, k, ops.kv4_pack(k, k), unit0=1)
    with pytest.raises(E, match="uint8"):
        ops.kv4_pack(k, k, (k, k))
    with pytest.raises(E, match="pinned"):
        ops.kv4_pack(k, k, tuple(r.cpu() for r in ops.kv4_pack(k, k)))
    with pytest.raises(E, match="capacity"):
        ops.kv4_unpack(*ops.kv4_pack(k, k), 17, torch.float32)
    with pytest.raises(E, match="fit the layer"):
        ops.attend_decode_kv4(
            st["p"], st["q"].half().to(cuda), st["pos"].to(cuda), st["hk"].to(cuda), st["hv"].to(cuda), *st["rec"],
            st["gid"].to(cuda), st["t0"].to(cuda))
    for name in ("hk", "hv"):      # the slots of too few sequences, of another width
        for bad in (st[name][:0], st[name][..., :64].contiguous()):
            with pytest.raises(E, match="one layout"):
                _run({**st, name: bad}, cuda)
            with pytest.raises(E, match="one layout"):
                _run({**st, "hk": bad, "hv": bad}, cuda)
    with pytest.raises(E, match="slots"):
        _run({**st, "hk": st["hk"][:, :, 1:], "hv": st["hv"][:, :, 1:]}, cuda)
    dev = (st["q"].to(cuda), st["pos"].to(cuda), st["hk"].to(cuda), st["hv"].to(cuda), *st["rec"], st["gid"].to(cuda),
           st["t0"].to(cuda))
    with pytest.raises(E, match="out must be"):
        ops.attend_decode_kv4(st["p"], *dev, out=torch.empty_like(st["q"]))
    st["gid"] = st["gid"].long()
    with pytest.raises(E, match="int32"):
        _run(st, cuda)
    st["gid"] = st["gid"].int()
    st["p"].group_size = 8
    with pytest.raises(E, match="group_size"):
        _run(st, cuda)
