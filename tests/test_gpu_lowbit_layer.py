"""The 8-bit projections and the 4-bit store in the framework's own paths: router decode, graphs, mixed lengths, the
VRAM bank, and the Qwen3 wrapper that runs them together."""
import types

import pytest
import torch

import cases
import lowbit_ref as R
from test_gpu_store_bank import SPEC, _inputs, _store

pytestmark = pytest.mark.gpu


def _kv4(dev, B, device="cpu", bank_chunks=0, dtype=torch.bfloat16):
    from hierarchicalglobalattention_b200 import ChunkPlacementPolicy, ChunkRouter, Kv4CacheStore, RouterConfig
    s = SPEC
    cfg = RouterConfig(nhead=s["H"], kv_heads=s["KVH"], head_dim=s["Dh"], chunk_size=s["C"], group_size=s["gs"],
                       topk_chunks=s["Kc"], topk_groups=s["Kg"], theta=1e4)
    pol = ChunkPlacementPolicy(keep_first=s["kf"], keep_last=s["kl"], first_token_level=True)
    return ChunkRouter(cfg, Kv4CacheStore(record_device=device, compute_device=dev, policy=pol, kv_heads=s["KVH"],
                                          head_dim=s["Dh"], chunk_size=s["C"], groups_per_chunk=s["C"] // s["gs"],
                                          batch_size=B, dtype=dtype, vram_cache_chunks=bank_chunks))


def _decode(router, g, S0, steps, look=()):
    """Outputs, routing lists, and at the steps of `look` the (out, want, sum of weight * |v|) of the block."""
    router.seed(0, g["k_rope"][:, :, :S0], g["k_raw"][:, :, :S0], g["v"][:, :, :S0])
    outs, routes, seen = [], [], []
    for i in range(steps):
        p = S0 + i
        sl = slice(p, p + 1)
        q = g["q"][:, :, sl]
        rk = router.decode_block(0, q, g["k_rope"][:, :, sl], g["k_raw"][:, :, sl], g["v"][:, :, sl], p)
        routes.append({k: t.clone() for k, t in rk.routing.items()})
        if i in look:
            store = router.store
            torch.cuda.synchronize()
            hk, hv = (t.cpu() for t in store.hot_buffers(0))
            vals = []
            for rec, is_v in zip(store.record(0), (False, True)):
                n = R.kv4_byte_codes(rec.cpu(), SPEC["Dh"], is_v).double()
                meta = rec.cpu()[..., 8 * SPEC["Dh"]:].contiguous().view(q.dtype).view(*rec.shape[:3], 16, -1, 2).double()
                vals.append((n.unflatten(-1, (-1, 32)) * meta[..., :1] + meta[..., 1:]).flatten(-2).flatten(2, 3))
            want = R.attend(q.cpu(), [p] * q.shape[0], hk, hv, *vals, rk.routing["open_gid"].cpu(),
                            rk.routing["open_t0"].cpu(), SPEC["C"], SPEC["gs"], SPEC["kf"], SPEC["kl"])
        outs.append(rk.attend(q))
        if i in look:
            seen.append((outs[-1].cpu().double(), *want))
    return torch.cat(outs, 2), routes, seen


def test_decode_through_the_4bit_store(cuda):
    """Routing is that of the exact store; every block attends its windows exactly and its opened groups through
    their codes, before and after chunks close; pinned record, HBM record and bank give the same bits."""
    B, S0, steps = 1, 700, 90
    g = _inputs(cuda, B, S0 + steps)
    ref = _store(cuda, B, "vram")
    ref.seed(0, g["k_rope"][:, :, :S0], g["k_raw"][:, :, :S0], g["v"][:, :, :S0])
    out, routes, seen = _decode(_kv4(cuda, B), g, S0, steps, look=(0, 3, 4, 67, 68, 89))
    for i in range(steps):
        p = S0 + i
        sl = slice(p, p + 1)
        rk = ref.decode_block(0, g["q"][:, :, sl], g["k_rope"][:, :, sl], g["k_raw"][:, :, sl], g["v"][:, :, sl], p)
        assert all(torch.equal(rk.routing[k], routes[i][k]) for k in rk.routing)
        rk.attend(g["q"][:, :, sl])
    for o, want, mag in seen:
        tol = 2.0 ** -8 * 1.01 * want.abs() + 2.0 ** -8 * mag + 1e-6
        assert ((o - want).abs() <= tol).all()
    for other in (_kv4(cuda, B, "cuda"), _kv4(cuda, B, "cpu", bank_chunks=32)):
        got, r2, _ = _decode(other, g, S0, steps)
        assert torch.equal(got, out) and all(torch.equal(a[k], b[k]) for a, b in zip(r2, routes) for k in a)
    assert other.store.cache_hits > 0 and other.store.cache_misses > 0


def test_a_seeded_store_lets_go_of_the_exact_rows(cuda):
    import weakref
    g = _inputs(cuda, 2, 300)
    for mixed in (False, True):
        router = _kv4(cuda, 2)
        k, v = g["k_rope"][:, :, :300].clone(), g["v"][:, :, :300].clone()
        refs = weakref.ref(k), weakref.ref(v)
        if mixed:
            router.seed_mixed(0, k, g["k_raw"][:, :, :300], v, [300, 130])
        else:
            router.seed(0, k, g["k_raw"][:, :, :300], v)
        del k, v
        assert refs[0]() is None and refs[1]() is None


def test_graph_and_reset_equal_eager(cuda):
    from hierarchicalglobalattention_b200.decode_graph import DecodeStepGraph
    B, S0, steps = 2, 500, 70
    g = _inputs(cuda, B, S0 + steps)
    eager = _kv4(cuda, B, "cuda")
    for _ in range(2):   # a store reused for a second sequence gives what a fresh one gives
        eager.reset()
        want, _, _ = _decode(eager, g, S0, steps)
    r = _kv4(cuda, B, "cuda")
    r.seed(0, g["k_rope"][:, :, :S0], g["k_raw"][:, :, :S0], g["v"][:, :, :S0])
    gr = DecodeStepGraph(r, [0], [S0] * B, S0 + steps + 1)
    outs = []
    for i in range(steps):
        sl = slice(S0 + i, S0 + i + 1)
        gr.q[0].copy_(g["q"][:, :, sl])
        for name in ("k_rope", "k_raw", "v"):
            getattr(gr, name)[0].copy_(g[name][:, :, sl])
        outs.append(gr.step()[0].clone())
    got = torch.cat(outs, 2)
    # the graph's lists are padded to the largest pool it can meet: the same sets
    torch.testing.assert_close(got.float(), want.float(), atol=2e-2, rtol=2e-2)


def test_mixed_lengths(cuda):
    B, lens = 2, [700, 333]
    g = _inputs(cuda, B, 800)
    r = _kv4(cuda, B)
    r.seed_mixed(0, g["k_rope"][:, :, :700], g["k_raw"][:, :, :700], g["v"][:, :, :700], lens)
    pos, steps = list(lens), 60
    outs = []
    for _ in range(steps):
        x = {k: torch.stack([g[k][b, :, pos[b]:pos[b] + 1] for b in range(B)]).contiguous() for k in ("q", "k_rope", "k_raw", "v")}
        sp = torch.tensor(pos, dtype=torch.int32, device=cuda)
        outs.append(r.decode_step(0, x["q"], x["k_rope"], x["k_raw"], x["v"], sp, pos).attend(x["q"]))
        pos = [p + 1 for p in pos]
    out = torch.cat(outs, 2)
    for b in range(B):
        one = {k: t[b:b + 1] for k, t in g.items()}
        want, _, _ = _decode(_kv4(cuda, 1), one, lens[b], steps)
        torch.testing.assert_close(out[b:b + 1].float(), want.float(), atol=2e-2, rtol=2e-2)


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_reading_the_record_back(cuda, device):
    from hierarchicalglobalattention_b200 import ops
    g = _inputs(cuda, 2, 640)
    r = _kv4(cuda, 2, device)
    r.seed(0, g["k_rope"], g["k_raw"], g["v"])
    uk, uv = ops.kv4_unpack(*ops.kv4_pack(g["k_rope"], g["v"]), 640, torch.bfloat16)
    st = r.store
    hk, hv = st.hot_tokens(0, 2, 5)
    assert torch.equal(hk.flatten(2, 3), uk[:, :, 128:320]) and torch.equal(hv.flatten(2, 3), uv[:, :, 128:320])
    chunk = torch.tensor([[[0, 7], [3, 9]], [[1, 1], [8, 2]]], device=cuda)
    ck, cv = st.gather_chunk_tokens_kvh(0, chunk)
    tk, tv = st.gather_tokens(0, chunk[:, torch.arange(8) // 4], torch.ones(2, 8, 2, dtype=torch.long, device=cuda))
    for b in range(2):
        for kv in range(2):
            for j in range(2):
                c = int(chunk[b, kv, j])
                assert torch.equal(ck[b, kv, j], uk[b, kv, c * 64:c * 64 + 64])
                assert torch.equal(cv[b, kv, j], uv[b, kv, c * 64:c * 64 + 64])
                assert torch.equal(tk[b, kv * 4 + 1, j], uk[b, kv, c * 64 + 16:c * 64 + 32])
                assert torch.equal(tv[b, kv * 4 + 2, j], uv[b, kv, c * 64 + 16:c * 64 + 32])


def test_store_refusals(cuda):
    from hierarchicalglobalattention_b200 import Kv4CacheStore
    with pytest.raises(ValueError, match="record_device"):
        _kv4(cuda, 1, "disk")
    pol = _kv4(cuda, 1).store.policy
    with pytest.raises(ValueError, match="head_dim"):
        Kv4CacheStore(compute_device=cuda, policy=pol, kv_heads=1, head_dim=80, chunk_size=64, groups_per_chunk=4, batch_size=1)
    r = _kv4(cuda, 1)
    r.store.ensure_capacity(0, 2)
    with pytest.raises(ValueError, match="16-token"):
        r.store.write_tokens(0, 8, torch.zeros(1, 2, 16, 128, device=cuda, dtype=torch.bfloat16),
                             torch.zeros(1, 2, 16, 128, device=cuda, dtype=torch.bfloat16))


# ---- the Qwen3 wrapper with both ---------------------------------------------------------------------
def _hf_layer(dev, seed=0):
    from transformers import Qwen3MoeConfig
    from transformers.models.qwen3_moe.modeling_qwen3_moe import Qwen3MoeAttention, Qwen3MoeRotaryEmbedding
    torch.manual_seed(seed)
    cfg = Qwen3MoeConfig(hidden_size=512, num_attention_heads=8, num_key_value_heads=2, head_dim=128, num_hidden_layers=1,
                         num_experts=4, num_experts_per_tok=2, rms_norm_eps=1e-6)
    attn = Qwen3MoeAttention(cfg, layer_idx=0).to(device=dev, dtype=torch.bfloat16).eval()
    return cfg, attn, Qwen3MoeRotaryEmbedding(cfg).to(dev)


def _wrapper_run(w, rot, x, cuts):
    S = x.shape[1]
    pos = torch.arange(S, device=x.device).unsqueeze(0)
    cos, sin = rot(x, pos)
    pkv, outs = types.SimpleNamespace(), []
    with torch.no_grad():
        for lo, hi in cuts:
            outs.append(w(x[:, lo:hi], position_embeddings=(cos[:, lo:hi], sin[:, lo:hi]), past_key_values=pkv,
                          position_ids=pos[:, lo:hi])[0])
    return torch.cat(outs, 1)


@pytest.mark.parametrize("tier", ["vram", "ram"])
def test_wrapper_with_8bit_projections_and_4bit_record(cuda, tier):
    """Prefill, a block over resident context, then single tokens: within the formats' accuracy of the 16-bit
    wrapper; an FP8 layer's own weights are used as they are."""
    from hierarchicalglobalattention_b200 import Fp8Linear, QwenRoutedAttention
    cfg, attn, rot = _hf_layer(cuda)
    x = torch.randn(2, 900, 512, device=cuda).bfloat16()
    cuts = [(0, 700), (700, 832)] + [(i, i + 1) for i in range(832, 900)]
    kw = dict(keep_first=1, keep_last=2, topk_chunks=4, topk_groups=16, cache_location=tier, vram_cache_chunks=4)
    full = _wrapper_run(QwenRoutedAttention(attn, cfg, **kw), rot, x, cuts)
    low = _wrapper_run(QwenRoutedAttention(attn, cfg, kv_bits=4, fp8_projections=True, **kw), rot, x, cuts)
    rel = (low.float() - full.float()).norm() / full.float().norm()
    # e4m3 operands (relative error 2^-4 / sqrt(3) each, two products in a row) and 4-bit records
    assert low.isfinite().all() and 0 < rel < 0.2
    for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
        setattr(attn, name, Fp8Linear.from_linear(getattr(attn, name)))
    w = QwenRoutedAttention(attn, cfg, kv_bits=4, fp8_projections=True, **kw)
    assert torch.equal(_wrapper_run(w, rot, x, cuts), low)
    attn.q_proj.weight_scale_inv.mul_(2.0)        # a changed weight is seen
    assert not torch.equal(_wrapper_run(w, rot, x, [(0, 700)]), low[:, :700])


def test_module_with_4bit_record(cuda):
    from hierarchicalglobalattention_b200 import HierarchicalGlobalAttentionRouted, Kv4CacheStore
    torch.manual_seed(1)
    kw = dict(d_model=256, nhead=4, kv_heads=2, head_dim=64, topk_chunks=4, topk_groups=8, keep_first=1, keep_last=2)
    a = HierarchicalGlobalAttentionRouted(**kw).to(cuda).bfloat16()
    b = HierarchicalGlobalAttentionRouted(**kw, kv_bits=4, cache_location="ram").to(cuda).bfloat16()
    b.load_state_dict(a.state_dict())
    x = torch.randn(1, 700, 256, device=cuda).bfloat16()
    with torch.no_grad():
        for lo, hi in ((0, 640), (640, 641), (641, 700)):
            cp = torch.arange(lo, hi, device=cuda)
            ya, yb = a(x[:, lo:hi], cache_position=cp)[0], b(x[:, lo:hi], cache_position=cp)[0]
            if lo == 0:
                assert torch.equal(ya, yb)        # the prefill attends the exact rows
            else:
                assert (ya - yb).float().norm() / ya.float().norm() < 0.1
    assert isinstance(b._kv_router.store, Kv4CacheStore)


def test_fp8_linear_module(cuda):
    from hierarchicalglobalattention_b200 import Fp8Linear, ops
    torch.manual_seed(2)
    lin = torch.nn.Linear(384, 200).to(cuda).bfloat16()
    m = Fp8Linear.from_linear(lin)
    x = torch.randn(3, 5, 384, device=cuda).bfloat16()
    y = m(x)
    assert y.shape == (3, 5, 200)
    assert (y - lin(x)).float().norm() / lin(x).float().norm() < 0.1
    n = Fp8Linear(384, 200, bias=True).to(cuda)
    n.load_state_dict(m.state_dict())
    assert torch.equal(n(x), y)
    assert torch.equal(torch.ops.hga.fp8_linear(x, m.weight, m.weight_scale_inv, m.bias, None, None), y)
    q, s = torch.ops.hga.fp8_quantize(x)
    assert torch.equal(ops.fp8_linear(q, m.weight, m.weight_scale_inv, bias=m.bias, x_scale=s), y)
