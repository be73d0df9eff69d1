"""Root-mean-square norm with an 8-bit output against the definition in 64 bits."""
import math

import pytest
import torch

from inductor_x_b200 import ops
from oracle import window_layer as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1), (3, 7), (16, 4096), (5, 128), (9, 129), (4, 1537), (130, 64), (7, 127), (2, 3, 264), (33, 2048), (3, 20000),
          (2, 16384), (300, 136), (1000, 96), (5, 8200), (2, 70001)]


def verify(got, x, w, eps, residual, group, return_residual=True):
    h, y, scales, wide = ref.rmsnorm_quantised(x, w, eps, residual, group)
    q, s = got[:2]
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.dtype == torch.float32 and s.shape == scales.shape
    if residual is not None and return_residual:
        assert torch.equal(got[2], h)
    # the mean of n squares in 32 bits, in at most 2^10 partial sums of at most 2^7 terms each, is off by (2^7 + 10) 2^-24 at
    # most, its root by half of that; the root, two products and the scale's division round once each
    rel = 2.0 ** -24 * (138 / 2 + 8)
    assert bool(((s.double() - scales).abs() <= rel * scales + 2.0 ** -149).all())
    # e4m3: half a step is 2^-4 of a value at most, 2^-10 where the step is fixed (below 2^-6)
    t = q.double()
    ratio = y / torch.where(wide > 0, wide, 1.0)
    assert bool(((t - ratio).abs() <= 2.0 ** -4 * ratio.abs() * (1 + 4 * rel) + 2.0 ** -10 + 4 * rel * ratio.abs()).all())
    # and to the nearest, wherever that is beyond the arithmetic's own error
    nearest = ratio.float().to(torch.float8_e4m3fn).double()
    lo, hi = ((ratio * (1 - 4 * rel)).float().to(torch.float8_e4m3fn).double(), (ratio * (1 + 4 * rel)).float().to(torch.float8_e4m3fn).double())
    assert bool(((t == nearest) | (t == lo) | (t == hi)).all())
    assert float((t != nearest).double().mean()) <= 0.001 + 2 / t.numel()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("group", [0, 128])
def test_against_64_bits(cuda, dtype, shape, group):
    gen = torch.Generator(device=cuda).manual_seed(shape[-1])
    x, r = (torch.randn(*shape, generator=gen, device=cuda).to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(shape[-1], generator=gen, device=cuda)).to(dtype)
    verify(ops.rmsnorm_quantised(x, w, 1e-6, group=group), x, w, 1e-6, None, group)
    verify(ops.rmsnorm_quantised(x, w, 1e-5, residual=r, group=group), x, w, 1e-5, r, group, False)
    verify(ops.rmsnorm_quantised(x, w, 1e-5, residual=r, return_residual=True, group=group), x, w, 1e-5, r, group)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [256, 1000, 1537])
def test_views_off_a_boundary(cuda, dtype, cols):
    for start in (1, 2, 3, 4, 8):
        flat = torch.randn(2, 10 * cols + 16, device=cuda).to(dtype)
        x, r = (f[start:start + 10 * cols].view(10, cols) for f in flat)
        w = torch.randn(cols + 16, device=cuda).to(dtype)[start:start + cols]
        for group in (0, 128):
            verify(ops.rmsnorm_quantised(x, w, residual=r, return_residual=True, group=group), x, w, 1e-6, r, group)
        verify(ops.rmsnorm_quantised(x, w), x, w, 1e-6, None, 0)


@pytest.mark.parametrize("cols", [300, 1024])
def test_zeros_tiny_and_huge_rows(cuda, cols):
    """Rows of nothing, of values whose scale is below the smallest normal number, and near the largest."""
    x = torch.randn(6, cols, device=cuda)
    x[0] = 0
    x[1] *= 1e-30
    x[2] *= 1e15
    x[3, 128:] = 0
    x[4] = 0
    x[4, 5] = 3e-39
    w = torch.randn(cols, device=cuda)
    for group in (0, 128):
        verify(ops.rmsnorm_quantised(x, w, 1e-6, group=group), x, w, 1e-6, None, group)
        q, s = ops.rmsnorm_quantised(x, torch.zeros_like(w), 1e-6, group=group)
        assert not s.any() and not q.float().any()
        # scales below the smallest normal number still make values that fill the range
        small = w * 1e-37
        q, s = ops.rmsnorm_quantised(x[5:], small, 1e-6, group=group)
        assert bool((q.float().abs().max() >= 400)) and bool((s > 0).all())


@pytest.mark.parametrize("cols", [72, 77, 260, 1537])
def test_rows_whose_root_is_infinite(cuda, cols):
    """Without eps the squares of tiny values are zero: what lies beside a row's end must not come in."""
    x = torch.full((9, cols), 1e-30, device=cuda)
    for group in (0, 128):
        q, s = ops.rmsnorm_quantised(x, torch.ones(cols, device=cuda), 0.0, group=group)
        assert bool(torch.isinf(s).all()) and bool(torch.isnan(q.float()).all())


def test_values_that_are_not_finite(cuda):
    x = torch.randn(4, 512, device=cuda)
    x[1, 200] = math.nan
    x[2, 300] = math.inf
    w = torch.ones(512, device=cuda)
    q, s = ops.rmsnorm_quantised(x, w, group=0)
    assert bool(torch.isnan(s[1:3]).all()) and bool(torch.isnan(q[1:3].float()).all())
    assert bool(torch.isfinite(s[[0, 3]]).all()) and bool(torch.isfinite(q[[0, 3]].float()).all())
    q, s = ops.rmsnorm_quantised(x, w, group=128)
    assert bool(torch.isnan(s[1]).all()) and bool(torch.isnan(q[1].float()).all())
    # an infinity makes the others of its row zeros and itself NaN
    assert bool(torch.isnan(s[2, 2])) and bool(torch.isnan(q[2, 256:384].float()).all())
    assert not s[2, [0, 1, 3]].any() and not q[2, :256].float().any()
    w[7] = math.inf
    q, s = ops.rmsnorm_quantised(x, w, group=0)
    assert bool(torch.isinf(s[0])) and bool(torch.isnan(q[0, 7].float())) and not q[0, 8:].float().any()


def test_streams_and_graphs(cuda):
    x, r = (torch.randn(40, 4096, device=cuda).bfloat16() for _ in range(2))
    w = torch.ones(4096, device=cuda).bfloat16()
    call = lambda: ops.rmsnorm_quantised(x, w, residual=r, return_residual=True, group=128)  # noqa: E731
    expected = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured = call()
        graph.replay()
    side.synchronize()
    for a, b, c in zip(expected, got, captured):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)) and torch.equal(a.view(torch.uint8), c.view(torch.uint8))
    q, s = ops.rmsnorm_quantised(x[:0], w, group=128)
    assert q.shape == (0, 4096) and s.shape == (0, 32)
