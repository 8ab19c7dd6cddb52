"""Attention over the 4-bit record where its parts meet: results joined across the CTAs of a cluster, weights that
cancel, caches of every type."""
import math

import pytest
import torch

from test_gpu_kv4 import HALF_ULP, TYPES, _run, _state, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 5])
def test_a_nan_score_is_not_lost_behind_a_far_larger_one(cuda, dtype, L):
    """A visible key whose score is NaN makes its rows NaN, however small its CTA's other scores are beside
    another CTA's (a factor that underflows to 0)."""
    g = torch.Generator().manual_seed(31)
    # 24 units of slots over the CTAs of one cluster: the first window's and the last one's are in different CTAs
    st = _state(g, 1, 2, 1, 128, dtype, 64, 16, 2, 3, [64 * 9 + 30], L, 0, cuda)
    st["q"][..., 7] = 4.0
    st["hk"][..., 7] = 0.0
    st["hk"][0, 0, 4 * 64 + 9, 7] = 1000.0       # 4 * 1000 / sqrt(128) = 354 above the others: e^-354 underflows
    clean = _run(st, cuda)
    assert clean.isfinite().all()
    st["hk"][0, 0, 3, 20] = math.nan             # first window, visible to every row
    assert _run(st, cuda).isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("L", [1, 4])
def test_a_visible_value_of_infinity_stays_one(cuda, dtype, L):
    g = torch.Generator().manual_seed(33)
    st = _state(g, 1, 8, 2, 128, dtype, 64, 16, 1, 2, [64 * 6 + 10], L, 6, cuda)
    st["hv"][0, 1, 5, 11] = math.inf             # first window
    st["hv"][0, 1, 3 * 64 + 2, 12] = -math.inf   # active chunk, before the block
    out = _run(st, cuda)[0, 4:]
    assert (out[..., 11] == math.inf).all() and (out[..., 12] == -math.inf).all()
    assert int(out.isfinite().logical_not().sum()) == 2 * 4 * L


# A weight's error: 2^-15 of it from its two 16-bit terms; a score's error of 2^-13 (fp32 sums of products, the
# record's blocks with 128 in place of 8 among them, the exponential) enters weight and sum once each.
WEIGHT_ERR = 2.0 ** -15 + 2 * 2.0 ** -13


def _check_weights(out, st):
    ref, mag = _want(st)
    dt = st["q"].dtype
    tol = HALF_ULP[dt] * 1.01 * ref.abs() + WEIGHT_ERR * mag + 1e-6
    err = (out.cpu().double() - ref).abs()
    assert (err <= tol).all(), f"worst {float((err / tol).max()):.2f} of the tolerance"


def _cancel(st, slot_row):
    """Sets a value row so that each channel's weighted sum is 0 but for the row's own rounding: what is left of the
    result shows the weights' errors, not its own rounding."""
    st["hv"][0, 0, slot_row] = 0.0
    ref, _ = _want(st)
    probe = st["hv"].clone()
    st["hv"][0, 0, slot_row] = 1.0
    one, _ = _want(st)
    st["hv"] = probe
    st["hv"][0, 0, slot_row] = (-ref[0, 0, 0] / (one - ref)[0, 0, 0]).to(st["hv"].dtype)
    assert st["hv"][0, 0, slot_row].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Dh", [64, 128, 256])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_weights_of_the_windows_keep_their_bits(cuda, dtype, Dh, seed):
    """Exact rows: results that cancel are as accurate as their terms."""
    g = torch.Generator().manual_seed(seed)
    st = _state(g, 1, 1, 1, Dh, dtype, 64, 16, 0, 0, [4 + seed], 1, 0, cuda)
    _cancel(st, 4 + seed)
    _check_weights(_run(st, cuda), st)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Dh", [64, 128, 256])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_weights_of_the_record_keep_their_bits(cuda, dtype, Dh, seed):
    """An opened group against an exact row that cancels it."""
    g = torch.Generator().manual_seed(100 + seed)
    st = _state(g, 1, 1, 1, Dh, dtype, 64, 16, 0, 0, [64 + seed], 1, 1, cuda)
    assert (st["gid"] >= 0).all()
    st["q"] *= 0.25            # many keys count
    _cancel(st, seed)
    _check_weights(_run(st, cuda), st)


def test_queries_off_the_16_byte_grid(cuda):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(41)
    st = _state(g, 2, 8, 2, 128, torch.bfloat16, 64, 16, 1, 1, [700, 300], 3, 8, cuda)
    want = _run(st, cuda)
    flat = torch.zeros(st["q"].numel() + 8, dtype=torch.bfloat16, device=cuda)
    for off in (1, 3, 8):
        q = flat[off:off + st["q"].numel()].view(st["q"].shape)
        q.copy_(st["q"])
        out = ops.attend_decode_kv4(st["p"], q, st["pos"].to(cuda), st["hk"].to(cuda), st["hv"].to(cuda), *st["rec"],
                                    st["gid"].to(cuda), st["t0"].to(cuda))
        assert torch.equal(out, want)
