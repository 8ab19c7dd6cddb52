"""8-bit products whose CTAs take several output tiles with one or two channel blocks each: a tile's results are staged
while the last tile's stores may still be on their way."""
import pytest
import torch

import lowbit_ref as R
from test_gpu_fp8 import _check, _weight, _x

pytestmark = pytest.mark.gpu

# M, N, K: about 290 tiles of 128 x 128 on 148 SMs, whole and ragged; as many of 256 x 256 as there are CTA pairs, and
# more; pairs with 64 or fewer columns in the last tile
SHAPES = [(2432, 1920, 64), (2432, 1920, 128), (2432, 1920, 256), (2432, 1904, 128), (2304 + 9, 1920, 64),
          (2048, 2048, 64), (2048, 2048, 128), (1024, 4096, 256), (512, 5120, 128), (4096, 2048 + 64, 128),
          (10240, 320, 64), (10240, 320, 256), (20480, 264, 128)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_second_tiles(cuda, M, N, K, dtype):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M + N + K)
    x = _x(g, M, K, dtype)
    w, ws = _weight(g, N, K)
    xq, xs = R.fp8_quantize(x)
    q, s, wd, wsd = xq.to(cuda), xs.to(cuda), w.to(cuda), ws.to(cuda)
    y = ops.fp8_linear(q, wd, wsd, x_scale=s, out_dtype=dtype)
    rows = torch.cat([torch.arange(0, M, 97), torch.arange(M - 130, M)])     # every tile row, the last ones whole
    _check(y[rows.to(cuda)], xq[rows], xs[rows], w, ws, None, dtype)
    out = torch.empty_like(y)
    for _ in range(50):
        out.fill_(float("nan"))
        ops.fp8_linear(q, wd, wsd, x_scale=s, out_dtype=dtype, out=out)
        assert torch.equal(out, y)
