"""hga_fp8_quantize and hga_fp8_linear against plain implementations (64-bit sums) on the same values."""
import math

import pytest
import torch

import lowbit_ref as R

pytestmark = pytest.mark.gpu

# largest relative error of one rounding to the type
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}


def _x(g, M, K, dtype):
    return (torch.randn(M, K, generator=g) * (1 + 20 * (torch.rand(K, generator=g) > 0.98))).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (1, 128), (5, 129), (17, 1000), (64, 2048), (301, 260)])
def test_quantize_is_the_definition(cuda, dtype, M, K):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M * 1000 + K)
    x = _x(g, M, K, dtype)
    x[M // 2, : K // 2] = 0
    if M > 2:
        x[1] = 0
    q, s = ops.fp8_quantize(x.to(cuda))
    rq, rs = R.fp8_quantize(x)
    assert q.dtype == torch.float8_e4m3fn and torch.equal(s.cpu(), rs)
    assert torch.equal(q.cpu().float(), rq.float())


def test_quantize_views_and_shapes(cuda):
    """Rows that start off the 16-byte grid, padded rows, transposed inputs and leading dimensions."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(0)
    base = _x(g, 24, 515, torch.bfloat16).to(cuda)
    for v in (base[:, 3:400], base[:, :256], base[5:6, 1:], base.t()[:40], base.view(2, 3, 4, 515)):
        q, s = ops.fp8_quantize(v)
        rq, rs = R.fp8_quantize(v.reshape(-1, v.shape[-1]).cpu())
        assert q.shape == v.shape and s.shape == (*v.shape[:-1], rs.shape[1])
        assert torch.equal(s.cpu().reshape(rs.shape), rs)
        assert torch.equal(q.cpu().float().reshape(rq.shape), rq.float())
    q, s = ops.fp8_quantize(base[:0])
    assert q.shape == (0, 515) and s.shape == (0, 5)


def test_quantize_extremes(cuda):
    """The type's largest values, tiny blocks, infinities and NaN: only their own block is touched."""
    from hierarchicalglobalattention_b200 import ops
    x = torch.ones(6, 384)
    x[0, :128] = 3.3e38
    x[1, 128:256] = 1e-31
    x[2, 130] = math.inf
    x[3, 383] = math.nan
    x[4, :128] = -1e-38
    q, s = ops.fp8_quantize(x.to(cuda))
    v = q.cpu().float() * s.cpu().repeat_interleave(128, 1)
    torch.testing.assert_close(v[0], x[0], rtol=1e-6, atol=0)
    assert (v[1, 128:256] == 0).all() and (v[4, :128] == 0).all()
    assert v[2, 128:256].isnan().any() and not v[2, :128].isnan().any() and not v[2, 256:].isnan().any()
    assert s[3, 2].isnan() and not v[3, :256].isnan().any()
    assert torch.equal(v[5], x[5])


def _check(y, xq, xs, w, ws, bias, dtype):
    ref, mag = R.fp8_product(xq, xs, w, ws, bias)
    # one rounding to the result's type and K roundings of an fp32 sum
    tol = HALF_ULP[dtype] * ref.abs() * 1.001 + (w.shape[1] + 4) * 2.0 ** -24 * mag + 1e-30
    err = (y.cpu().double() - ref).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol).max()):.2f} of the tolerance"


def _weight(g, N, K):
    from hierarchicalglobalattention_b200 import ops
    return ops.fp8_quantize_weight(torch.randn(N, K, generator=g) * K ** -0.5)


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 5120, 256), (1, 640, 2048), (15, 129, 100), (16, 256, 512), (17, 1000, 1056),
          (31, 8, 4000), (33, 384, 136), (64, 127, 2048), (65, 1024, 1040), (127, 255, 129), (128, 128, 640),
          (129, 513, 384), (200, 2048, 1536), (257, 300, 1000), (700, 1100, 272), (1500, 896, 256)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_linear(cuda, M, N, K, dtype):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M + 7 * N + 13 * K)
    x = _x(g, M, K, dtype)
    w, ws = _weight(g, N, K)
    bias = torch.randn(N, generator=g).to(dtype) if (M + N) % 2 else None
    y = ops.fp8_linear(x.to(cuda), w.to(cuda), ws.to(cuda), bias=None if bias is None else bias.to(cuda))
    assert y.dtype == dtype and y.shape == (M, N)
    xq, xs = R.fp8_quantize(x)
    _check(y, xq, xs, w, ws, bias, dtype)


@pytest.mark.parametrize("M,N,K,dtype", [(2500, 2000, 300, torch.bfloat16), (4900, 1024, 64, torch.float16),
                                         (5001, 1111, 1000, torch.bfloat16), (9500, 512, 640, torch.float32),
                                         (257, 19000, 272, torch.bfloat16), (20000, 300, 128, torch.float16)])
def test_linear_many_tiles(cuda, M, N, K, dtype):
    """Products that fill the GPU with tiles, whole and ragged in every direction."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M)
    x = _x(g, M, K, dtype)
    w, ws = _weight(g, N, K)
    bias = torch.randn(N, generator=g).to(dtype) if N % 2 else None
    y = ops.fp8_linear(x.to(cuda), w.to(cuda), ws.to(cuda), bias=None if bias is None else bias.to(cuda))
    xq, xs = R.fp8_quantize(x)
    _check(y, xq, xs, w, ws, bias, dtype)


@pytest.mark.parametrize("M", [1, 9, 40, 300])
def test_linear_quantised_input(cuda, M):
    """8-bit rows with their scales give what the same rows give when they are quantised on the way in."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M)
    x = _x(g, M, 776, torch.bfloat16).to(cuda)
    w, ws = (t.to(cuda) for t in _weight(g, 384, 776))
    q, s = ops.fp8_quantize(x)
    y = ops.fp8_linear(q, w, ws, x_scale=s)
    assert y.dtype == torch.bfloat16
    _check(y, q.cpu(), s.cpu(), w.cpu(), ws.cpu(), None, torch.bfloat16)
    y32 = ops.fp8_linear(q, w, ws, x_scale=s, out_dtype=torch.float32)
    _check(y32, q.cpu(), s.cpu(), w.cpu(), ws.cpu(), None, torch.float32)


@pytest.mark.parametrize("M", [1, 20, 130, 1400])
def test_linear_strides_and_alignment(cuda, M):
    """x and w as slices with other strides and starts, leading dimensions, a caller's out, a sub-block of a
    larger scale table."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M)
    N, K = 200, 400
    wide = _x(g, M, K + 37, torch.float16).to(cuda)
    w, ws = _weight(g, N, K)
    store = torch.zeros(N, K + 11, dtype=torch.float8_e4m3fn, device=cuda)
    for off in (0, 5):
        wv = store[:, off:off + K]
        wv.copy_(w)
        table = torch.zeros(2, 9, device=cuda)
        table[:, 3:7] = ws.to(cuda)
        for x in (wide[:, 3:3 + K], wide[:, :K], wide[:, 8:8 + K]):
            out = torch.full((M, N), 7.0, dtype=torch.float16, device=cuda)
            y = ops.fp8_linear(x, wv, table[:, 3:7], out=out)
            assert y is out
            xq, xs = R.fp8_quantize(x.cpu())
            _check(y, xq, xs, w, ws, None, torch.float16)
    y3 = ops.fp8_linear(wide[:, :K].reshape(1, M, K), w.to(cuda), ws.to(cuda))
    assert y3.shape == (1, M, N) and torch.equal(y3[0], ops.fp8_linear(wide[:, :K], w.to(cuda), ws.to(cuda)))
    assert ops.fp8_linear(wide[:0, :K], w.to(cuda), ws.to(cuda)).shape == (0, N)


@pytest.mark.parametrize("M", [4, 100, 900])
def test_linear_non_finite_rows_stay_in_their_rows(cuda, M):
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(3)
    x = _x(g, M, 512, torch.bfloat16)
    w, ws = (t.to(cuda) for t in _weight(g, 320, 512))
    clean = ops.fp8_linear(x.to(cuda), w, ws)
    x[1, 200] = math.nan
    x[M - 1, 5] = math.inf
    y = ops.fp8_linear(x.to(cuda), w, ws)
    assert y[1].isnan().all() and y[M - 1].isnan().all()
    keep = [i for i in range(M) if i not in (1, M - 1)]
    assert torch.equal(y[keep], clean[keep])


@pytest.mark.parametrize("M", [1, 16, 48, 333, 2000])
def test_linear_is_reproducible_and_rows_are_independent(cuda, M):
    """The same call twice gives the same bits; so does another stream, and a call captured in a graph."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(M)
    x = _x(g, M, 1024, torch.bfloat16).to(cuda)
    w, ws = (t.to(cuda) for t in _weight(g, 1280, 1024))
    y = ops.fp8_linear(x, w, ws)
    assert torch.equal(y, ops.fp8_linear(x, w, ws))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y2 = ops.fp8_linear(x, w, ws)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            y3 = ops.fp8_linear(x, w, ws)
        gr.replay()
    s.synchronize()
    assert torch.equal(y, y2) and torch.equal(y, y3)


def test_linear_against_differences_of_its_rows(cuda):
    """Linearity where it holds exactly: a power of two on a row scales its result by it."""
    from hierarchicalglobalattention_b200 import ops
    g = torch.Generator().manual_seed(1)
    x = _x(g, 70, 640, torch.float32).to(cuda)
    w, ws = (t.to(cuda) for t in _weight(g, 256, 640))
    y = ops.fp8_linear(x, w, ws)
    assert torch.equal(ops.fp8_linear(x * 8, w, ws), y * 8)
    assert torch.equal(ops.fp8_linear(-x, w, ws), -y)


def test_refusals(cuda):
    from hierarchicalglobalattention_b200 import _lib, ops
    g = torch.Generator().manual_seed(1)
    w, ws = (t.to(cuda) for t in _weight(g, 256, 384))
    x = torch.zeros(4, 384, device=cuda, dtype=torch.bfloat16)
    E = _lib.HgaError
    with pytest.raises(E, match="does not fit"):
        ops.fp8_linear(x[:, :300], w, ws)
    with pytest.raises(E, match="e4m3"):
        ops.fp8_linear(x, w.float(), ws)
    with pytest.raises(E, match="w_scale"):
        ops.fp8_linear(x, w, ws[:1])
    with pytest.raises(E, match="w_scale"):
        ops.fp8_linear(x, w, ws.half())
    with pytest.raises(E, match="x_scale"):
        ops.fp8_linear(ops.fp8_quantize(x)[0], w, ws)
    with pytest.raises(E, match="x_scale"):
        ops.fp8_linear(x, w, ws, x_scale=ws)
    with pytest.raises(E, match="bias"):
        ops.fp8_linear(x, w, ws, bias=torch.zeros(256, device=cuda))
    with pytest.raises(E, match="out"):
        ops.fp8_linear(x, w, ws, out=torch.zeros(4, 255, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(E, match="overlap"):
        ops.fp8_linear(x, w[:1].expand(256, 384), ws)
    with pytest.raises(E, match="overlap"):
        ops.fp8_linear(x, w, ws[:1].expand(2, 3))
    one = ops.fp8_linear(x + 1, w[:1].expand(1, 384), ws[:1].expand(1, 3))
    assert torch.equal(one, ops.fp8_linear(x + 1, w[:1].clone(), ws[:1].clone()))
    with pytest.raises(E, match="CUDA"):
        ops.fp8_linear(x.cpu(), w, ws)
    with pytest.raises(E, match="x must be"):
        ops.fp8_linear(x.long(), w, ws)
    with pytest.raises(E, match="rows"):
        ops.fp8_quantize(x.long())
