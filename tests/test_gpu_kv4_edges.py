"""Attention over the 4-bit record where its parts meet: results joined across the CTAs of a cluster, weights that
cancel, caches of every type."""
import math

import pytest
import torch

from test_gpu_kv4 import TYPES, _run, _state

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
