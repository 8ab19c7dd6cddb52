"""The low-bit operators launch on their tensors' device, whichever is current (no GPU: fake tensors, a recorded
library)."""
import contextlib

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from hierarchicalglobalattention_b200 import _lib, ops


class _Library:
    """Stands for the loaded library: notes the device that is current when an entry point is called."""

    def __init__(self, state):
        self.state, self.calls = state, []

    def __getattr__(self, name):
        return lambda *a: self.calls.append((name, self.state["device"])) or 0


@pytest.fixture
def recorded(monkeypatch):
    state = {"device": 0}

    @contextlib.contextmanager
    def device(d):
        old, state["device"] = state["device"], d if isinstance(d, int) else torch.device(d).index
        yield
        state["device"] = old

    h = _Library(state)
    monkeypatch.setattr(ops, "lib", lambda: h)
    monkeypatch.setattr(ops, "stream_ptr", lambda d: 0)
    monkeypatch.setattr(ops, "_current_device", lambda: state["device"])
    monkeypatch.setattr(torch.cuda, "device", device)
    return h, state


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
@pytest.mark.parametrize("at", [0, 1])
def test_launches_go_to_the_tensors_device(recorded, at):
    h, state = recorded
    dev = f"cuda:{at}"
    with FakeTensorMode():
        x = torch.empty(3, 256, device=dev, dtype=torch.bfloat16)
        w = torch.empty(128, 256, device=dev, dtype=torch.float8_e4m3fn)
        ws = torch.empty(1, 2, device=dev)
        q, s = ops.fp8_quantize(x)
        assert q.device == s.device == x.device
        for m in (3, 40):
            assert ops.fp8_linear(torch.empty(m, 256, device=dev), w, ws).device == x.device
        k = torch.empty(1, 2, 64, 128, device=dev, dtype=torch.bfloat16)
        rec = ops.kv4_pack(k, k)
        assert rec[0].device == x.device and ops.kv4_unpack(*rec, 64, k.dtype)[0].device == x.device
        p = _lib.make_params(batch=1, nhead=4, kv_heads=2, head_dim=128, chunk_size=64, group_size=16, topk_chunks=4,
                             topk_groups=8, keep_first=0, keep_last=0, theta=1e4, dtype=torch.bfloat16)
        i32 = dict(device=dev, dtype=torch.int32)
        lst = torch.empty(1, 4, 2, **i32)
        out = ops.attend_decode_kv4(p, torch.empty(1, 4, 1, 128, device=dev, dtype=torch.bfloat16), torch.empty(1, **i32), k, k,
                                    *rec, lst, lst)
        assert out.device == x.device
    names = {n for n, _ in h.calls}
    assert {"hga_fp8_quantize", "hga_fp8_linear", "hga_kv4_pack", "hga_kv4_unpack", "hga_attend_decode_kv4"} <= names
    assert {d for _, d in h.calls} == {at} and state["device"] == 0
