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


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
@pytest.mark.parametrize("codes,want", [([0], 1), ([_lib.E_WORKSPACE, 0], 2), ([-3], 1), ([_lib.E_WORKSPACE, -3], 2)])
def test_only_a_missing_workspace_is_asked_for_again(recorded, monkeypatch, codes, want):
    """A product of few rows is first called without a workspace; any other error is raised as it is, once."""
    calls = []

    class Library:
        def hga_fp8_linear(self, *a):
            calls.append(a[15:17])
            return codes[len(calls) - 1]

        def hga_fp8_linear_workspace(self, *a):
            return 1024

        def hga_last_error(self):
            return b"text of the library"

    monkeypatch.setattr(ops, "lib", Library)
    monkeypatch.setattr(_lib, "lib", Library)
    with FakeTensorMode():
        x = torch.empty(3, 256, device="cuda:0", dtype=torch.bfloat16)
        w = torch.empty(128, 256, device="cuda:0", dtype=torch.float8_e4m3fn)
        ws = torch.empty(1, 2, device="cuda:0")
        if codes[-1]:
            with pytest.raises(_lib.HgaError, match="text of the library"):
                ops.fp8_linear(x, w, ws)
        else:
            ops.fp8_linear(x, w, ws)
    assert len(calls) == want and calls[0] == (None, 0)


def test_a_missing_workspace_has_its_own_code():
    import ctypes
    one = ctypes.c_void_p(16)
    h = _lib.lib()
    args = (4000, 4096, 4096, 1, one, 4096, None, one, 4096, one, 32, None, 1, one, 4096)
    assert h.hga_fp8_linear(*args, None, 0, None) == _lib.E_WORKSPACE and b"workspace" in h.hga_last_error()
    assert h.hga_fp8_linear(*args, one, 16, None) == -1


@pytest.mark.filterwarnings("ignore:Accessing the data pointer")
def test_strides_of_dimensions_of_size_one_are_free(recorded):
    """One block of channels, or one channel: a transposed row is a column as good as any."""
    h, _ = recorded
    with FakeTensorMode():
        for K in (1, 100):
            x = torch.empty(40, K, device="cuda:0", dtype=torch.bfloat16)
            w = torch.empty(K, 300, device="cuda:0", dtype=torch.float8_e4m3fn).t()
            w = w if K == 1 else torch.empty(300, K, device="cuda:0", dtype=torch.float8_e4m3fn)
            ws = torch.empty(1, 3, device="cuda:0").t()
            assert ws.stride(1) != 1
            assert ops.fp8_linear(x, w, ws).shape == (40, 300)
        with pytest.raises(_lib.HgaError, match="w_scale"):
            ops.fp8_linear(torch.empty(4, 200, device="cuda:0"), torch.empty(300, 200, device="cuda:0", dtype=w.dtype),
                           torch.empty(2, 3, device="cuda:0").t())
