"""The 8-bit operators beside autograd."""
import pytest
import torch

from hierarchicalglobalattention_b200 import Fp8Linear, _lib, ops

pytestmark = pytest.mark.gpu


def test_a_gradient_is_refused_not_left_out(cuda):
    """Forward gives the same values; backward raises, as through torch.ops.hga.fp8_linear."""
    torch.manual_seed(3)
    m = Fp8Linear.from_linear(torch.nn.Linear(256, 136).to(cuda).bfloat16())
    for rows in (4, 300):
        x = torch.randn(rows, 256, device=cuda).bfloat16()
        want = m(x)
        assert not want.requires_grad
        xg = x.clone().requires_grad_()
        with torch.no_grad():
            assert not m(xg).requires_grad
        y = m(xg)
        assert torch.equal(y, want) and y.requires_grad
        with pytest.raises(_lib.HgaError, match="no backward"):
            y.float().sum().backward()
        bias = m.bias.clone().requires_grad_()
        y = ops.fp8_linear(x, m.weight, m.weight_scale_inv, bias=bias)
        assert torch.equal(y, want)
        with pytest.raises(_lib.HgaError, match="no backward"):
            y.float().sum().backward()
        q, s = ops.fp8_quantize(xg)
        q0, s0 = ops.fp8_quantize(x)
        assert torch.equal(q.float(), q0.float()) and torch.equal(s, s0)
        with pytest.raises(_lib.HgaError, match="no backward"):
            s.sum().backward()
        out = torch.empty_like(want)
        with pytest.raises(_lib.HgaError, match="out goes with"):
            ops.fp8_linear(xg, m.weight, m.weight_scale_inv, bias=m.bias, out=out)
        with torch.no_grad():
            assert torch.equal(ops.fp8_linear(xg, m.weight, m.weight_scale_inv, bias=m.bias, out=out), want)
