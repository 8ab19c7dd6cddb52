"""The 4-bit store over both records: ways into it besides a prefill, decode steps in the 16-bit types."""
import pytest
import torch

import kv4_store_cases as K
from test_gpu_kv4 import HALF_ULP
from test_gpu_kv4_edges import WEIGHT_ERR
from test_gpu_lowbit_layer import _decode, _kv4
from test_gpu_store_bank import _inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("record", ["cpu", "cuda"])
@pytest.mark.parametrize("how", ["bulk", "one by one"])
def test_ingested_chunks(cuda, record, how):
    K.check_ingest(cuda, record, how)


@pytest.mark.parametrize("record", ["cpu", "cuda"])
def test_prefill_windows_are_exact(cuda, record):
    K.check_prefill_windows_are_exact(cuda, record)


# ---- decode through the store, at the accuracy of its arithmetic ---------------------------------------
# one rounding to the type and the weights' error (two 16-bit terms, scores: see test_gpu_kv4_edges.py)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("record", ["cpu", "cuda"])
def test_decode_keeps_the_accuracy_of_the_type(cuda, dtype, record):
    B, S0, steps = 2, 380, 70
    g = {k: t.to(dtype) for k, t in _inputs(cuda, B, S0 + steps).items()}
    _, _, seen = _decode(_kv4(cuda, B, record, dtype=dtype), g, S0, steps, look=(0, 3, 4, 69))
    for out, want, mag in seen:
        tol = HALF_ULP[dtype] * 1.01 * want.abs() + WEIGHT_ERR * mag + 1e-6
        assert ((out - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_graph_equals_eager_within_two_roundings(cuda, dtype):
    """The graph's lists are padded to the largest pool it can meet: the same sets in another order."""
    from hierarchicalglobalattention_b200.decode_graph import DecodeStepGraph
    B, S0, steps = 2, 500, 70
    g = {k: t.to(dtype) for k, t in _inputs(cuda, B, S0 + steps).items()}
    want, _, _ = _decode(_kv4(cuda, B, "cuda", dtype=dtype), g, S0, steps)
    r = _kv4(cuda, B, "cuda", dtype=dtype)
    r.seed(0, g["k_rope"][:, :, :S0], g["k_raw"][:, :, :S0], g["v"][:, :, :S0])
    gr = DecodeStepGraph(r, [0], [S0] * B, S0 + steps + 1, dtype=dtype)
    outs = []
    for i in range(steps):
        sl = slice(S0 + i, S0 + i + 1)
        gr.q[0].copy_(g["q"][:, :, sl])
        for name in ("k_rope", "k_raw", "v"):
            getattr(gr, name)[0].copy_(g[name][:, :, sl])
        outs.append(gr.step()[0].clone())
    a, b = torch.cat(outs, 2).double(), want.double()
    vmax = float(g["v"].abs().max())           # no sum of weights times |v| is larger
    assert ((a - b).abs() <= 2 * HALF_ULP[dtype] * 1.01 * b.abs() + 2 * WEIGHT_ERR * vmax).all()
