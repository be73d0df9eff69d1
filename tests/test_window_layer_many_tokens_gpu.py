"""Rotary positions and the norm with an 8-bit output at sizes that run their kernels' loops: several tokens a block, a second
round of heads, a second row of a team."""
import pytest
import torch

import test_axial_rotary_gpu as rotary
import test_norm_quantised_gpu as norm
from inductor_x_b200 import ops
from kernels_taken import kernels, sm_count
from oracle import window_layer as ref

pytestmark = pytest.mark.gpu

TOKENS = [
    # B, H, HK, S, D, sections
    (3, 4, 2, 701, 128, [16, 24, 24]),        # the ends of sequences inside blocks, a last block in part
    (3, 2, 1, 701, 64, [16, 16]),
    (3, 5, 3, 1369, 80, [20, 20]),
    (2, 3, 2, 901, 96, [16, 16]),             # the last 32 are copied
    (1500, 2, 2, 3, 64, [8, 24]),             # several sequences in a block
    (2, 1, 1, 20011, 16, [8]),                # as many tokens as threads
    (5, 32, 8, 700, 128, [22, 21, 21]),
    (2, 1, 0, 5003, 128, [64]),
]


@pytest.mark.parametrize("dtype", rotary.DTYPES)
@pytest.mark.parametrize("shape", TOKENS)
@pytest.mark.parametrize("storage", ["bshd", "bhsd"])
def test_several_tokens_a_block(cuda, dtype, shape, storage):
    *sizes, sections = shape
    B, H, HK, S, D = sizes
    assert B * S >= 4 * sm_count()  # (two blocks an SM, two tokens a block)
    q, k, positions = rotary.inputs(cuda, dtype, *sizes, len(sections), storage, far=20000, seed=S)
    for pairing, inverse in (("halves", False), ("neighbours", True)):
        call = ops.axial_rotary_backward if inverse else ops.axial_rotary
        got = call(q, k, positions, sections, pairing=pairing)
        for x, y in zip((q, k), got if k is not None else (got,)):
            ref.check(y, ref.axial_rotary(x, positions, sections, pairing=pairing, inverse=inverse), pairing)
    pairs, vector = sum(sections), 16 // q.element_size()
    taken = kernels(lambda: ops.axial_rotary(q, k, positions, sections))
    assert len(taken) == 1 and ("rotary_vector_kernel" in taken.pop()) == (pairs % vector == 0)


@pytest.mark.parametrize("dtype", rotary.DTYPES)
@pytest.mark.parametrize("storage", ["bshd", "bhsd"])
def test_more_heads_than_are_in_flight(cuda, dtype, storage):
    q, k, positions = rotary.inputs(cuda, dtype, 2, 64, 64, 331, 128, 1, storage, far=5000)
    for pairing in ops.PAIRINGS:
        for x, y in zip((q, k), ops.axial_rotary(q, k, positions, [64], pairing=pairing)):
            ref.check(y, ref.axial_rotary(x, positions, [64], pairing=pairing), pairing)


ROWS = [(40009, 77), (12007, 301), (20003, 161), (9001, 1537), (4001, 2501), (3001, 4097), (1500, 8193), (700, 20001)]


@pytest.mark.parametrize("dtype", norm.DTYPES)
@pytest.mark.parametrize("rows,cols", ROWS)
@pytest.mark.parametrize("group", [0, 128])
def test_rows_off_a_boundary_one_behind_the_other(cuda, dtype, rows, cols, group):
    gen = torch.Generator(device=cuda).manual_seed(cols)
    x, r = (torch.randn(rows, cols, generator=gen, device=cuda).to(dtype) for _ in range(2))
    # rows that a team takes in turn are of very different sizes, and some are zeros
    x *= (2.0 ** (torch.arange(rows, device=cuda) % 9 - 4))[:, None].to(dtype)
    x[::7] = 0
    w = (1 + 0.2 * torch.randn(cols, generator=gen, device=cuda)).to(dtype)
    norm.verify(ops.rmsnorm_quantised(x, w, 1e-6, group=group), x, w, 1e-6, None, group)
    norm.verify(ops.rmsnorm_quantised(x, w, 1e-5, residual=r, return_residual=True, group=group), x, w, 1e-5, r, group)
    taken = kernels(lambda: ops.rmsnorm_quantised(x, w, 1e-6, group=group))
    assert len(taken) == 1 and "norm_quantised_shifted_kernel" in taken.pop()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_rows_of_whole_vectors_and_of_views_off_a_boundary(cuda, dtype):
    gen = torch.Generator(device=cuda).manual_seed(5)
    flat = torch.randn(5000 * 1000 + 3, generator=gen, device=cuda).to(dtype)
    w = torch.randn(1000, generator=gen, device=cuda).to(dtype)
    for start, form in ((0, "norm_quantised_kernel"), (3, "norm_quantised_long_kernel")):
        x = flat[start:start + 5000 * 1000].view(5000, 1000)
        for group in (0, 128):
            norm.verify(ops.rmsnorm_quantised(x, w, 1e-6, group=group), x, w, 1e-6, None, group)
        assert all(form in n for n in kernels(lambda: ops.rmsnorm_quantised(x, w, 1e-6)))
