"""Plain implementations of the 8-bit and 4-bit operators on the CPU, in 64 bits where values are computed."""
import math

import torch

META = {torch.bfloat16: torch.bfloat16, torch.float16: torch.float16, torch.float32: torch.bfloat16}


def fp8_quantize(x):
    """e4m3 values and fp32 scales of rows x [M, K] (fp32 IEEE divisions: the operator's definition)."""
    M, K = x.shape
    kb = -(-K // 128)
    f = torch.zeros(M, kb * 128)
    f[:, :K] = x.float()
    f = f.view(M, kb, 128)
    amax = f.abs().amax(-1)
    s = torch.where(amax <= 1e-30, torch.ones(()), amax / torch.full_like(amax, 448.0))
    return (f / s[..., None]).view(M, kb * 128)[:, :K].to(torch.float8_e4m3fn), s


def fp8_product(xq, xs, w, ws, bias):
    """(y, sum of the magnitudes of its terms) in 64 bits."""
    K = w.shape[1]
    xd = xq.double() * xs.double().repeat_interleave(128, 1)[:, :K]
    wd = w.double() * ws.double().repeat_interleave(128, 0)[:w.shape[0]].repeat_interleave(128, 1)[:, :K]
    y, mag = xd @ wd.T, xd.abs() @ wd.abs().T
    return (y + bias.double(), mag + bias.double().abs()) if bias is not None else (y, mag)


def kv4_codes(x):
    """Codes, scale and minimum of x [..., Dh] by 32 channels (fp32 arithmetic: the definition)."""
    mt = META[x.dtype]
    f = x.float().unflatten(-1, (-1, 32))
    lo, hi = f.amin(-1, keepdim=True), f.amax(-1, keepdim=True)
    s = ((hi - lo) * torch.tensor(1.0) .div(15.0)).to(mt)
    m = lo.to(mt)
    bad = ~torch.isfinite(f).all(-1, keepdim=True)
    s, m = torch.where(bad, torch.full_like(s, math.nan), s), torch.where(bad, torch.full_like(m, math.nan), m)
    sf = s.float()
    n = torch.clamp(torch.round((f - m.float()) / sf), 0, 15)
    n = torch.where((sf > 0) & torch.isfinite(sf), n, torch.zeros(()))
    return n, s, m


def kv4_value(n, s, m, dtype):
    return (n * s.float() + m.float()).flatten(-2).to(dtype)


def kv4_byte_codes(rec, dh, is_v):
    """Codes [..., 16, dh] of units' bytes [..., 10 * dh], looked up one by one from the documented layout."""
    out = torch.zeros(*rec.shape[:-1], 16, dh, dtype=torch.int64)
    for tok in range(16):
        for ch in range(dh):
            t = ch // 16
            r, c = (ch % 16, tok) if is_v else (tok, ch % 16)
            lane = 4 * (r % 8) + (c % 8) // 2
            byte = ((t // 4) * 32 + lane) * 16 + (t % 4) * 4
            nib = r // 8 + 2 * (c // 8) + 4 * (c % 2)
            out[..., tok, ch] = (rec[..., byte + nib // 2].long() >> (4 * (nib % 2))) & 15
    return out


def attend(q, seq_pos, hot_k, hot_v, dk, dv, gid, t0, C, gs, kf, kl, scale=None):
    """(out, sum of weight * |v|) [B,H,L,Dh] in 64 bits; dk / dv [B,KVH,groups*gs,Dh]: the record's values."""
    B, H, L, Dh = q.shape
    KVH = hot_k.shape[1]
    scale = Dh ** -0.5 if scale is None else scale
    out, mag = torch.zeros(B, H, L, Dh, dtype=torch.float64), torch.zeros(B, H, L, Dh, dtype=torch.float64)
    for b in range(B):
        pos = int(seq_pos[b])
        n, c0 = pos // C, pos % C
        f_hi = min(kf, n)
        l_lo = n if kl <= 0 else min(max(kf, n - kl), n)
        for h in range(H):
            g = h // (H // KVH)
            rows = [(hot_k[b, g, c * C + u], hot_v[b, g, c * C + u], 0) for c in range(f_hi) for u in range(C)]
            rows += [(hot_k[b, g, (kf + c % kl) * C + u], hot_v[b, g, (kf + c % kl) * C + u], 0)
                     for c in range(l_lo, n) for u in range(C)]
            for j in range(gid.shape[-1]):
                if gid[b, h, j] < 0:
                    continue
                r0 = int(gid[b, h, j]) * gs
                rows += [(dk[b, g, r0 + u], dv[b, g, r0 + u], int(t0[b, h, j])) for u in range(gs)]
            rows += [(hot_k[b, g, (kf + kl) * C + u], hot_v[b, g, (kf + kl) * C + u], u - c0) for u in range(c0 + L)]
            kk = torch.stack([r[0] for r in rows]).double()
            vv = torch.stack([r[1] for r in rows]).double()
            first = torch.tensor([r[2] for r in rows])
            for t in range(L):
                see = first <= t
                w = torch.softmax(kk[see] @ q[b, h, t].double() * scale, 0)
                out[b, h, t] = w @ vv[see]
                mag[b, h, t] = w @ vv[see].abs()
    return out, mag
