"""Rotary positions with several axes against the definition in 64 bits."""
import pytest
import torch

from inductor_x_b200 import ops
from oracle import window_layer as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]

SHAPES = [
    # B, H, HK, S, D, sections
    (1, 1, 1, 1, 2, [1]),
    (2, 4, 2, 33, 128, [16, 24, 24]),
    (3, 5, 1, 7, 80, [20, 20]),
    (1, 3, 3, 130, 64, [10, 11, 11]),
    (2, 2, 2, 19, 96, [16, 16]),               # the last 32 are copied
    (1, 2, 1, 11, 37, [3, 0, 5]),              # odd heads, an axis without pairs
    (1, 9, 3, 257, 256, [128]),
    (2, 32, 8, 5, 128, [22, 21, 21]),
    (16, 32, 8, 1, 128, [64]),
    (1, 1, 0, 100, 128, [16, 16, 16, 16]),     # no k
    (1, 2, 2, 50, 24, [4, 4, 4]),
]


def inputs(dev, dtype, B, H, HK, S, D, axes, storage, wide=True, far=1000, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def new(h):
        shape = (B, S, h, D) if storage == "bshd" else (B, h, S, D)
        t = torch.randn(*shape, generator=gen, device=dev).to(dtype)
        return t.transpose(1, 2) if storage == "bshd" else t

    positions = torch.randint(0, far, (axes, B, S), generator=gen, device=dev)
    return new(H), new(HK) if HK else None, positions if wide else positions.int()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("pairing", ops.PAIRINGS)
def test_against_64_bits(cuda, dtype, shape, pairing):
    *sizes, sections = shape
    storage, ladder = ("bshd", "own") if sum(sizes) % 2 else ("bhsd", "shared")
    q, k, positions = inputs(cuda, dtype, *sizes, len(sections), storage, wide=sizes[0] % 2 == 0, far=100000)
    for name, inverse in (("axial_rotary", False), ("axial_rotary_backward", True)):
        got = getattr(ops, name)(q, k, positions, sections, pairing=pairing, ladder=ladder)
        for x, y in zip((q, k), got if k is not None else (got,)):
            assert y.dtype == x.dtype and (x.numel() == 1 or y.stride() == x.stride() or 1 in x.shape)
            ref.check(y, ref.axial_rotary(x, positions, sections, pairing=pairing, ladder=ladder, inverse=inverse), name)


def test_far_positions(cuda):
    """The fraction of a turn survives at positions that 32 bits cannot tell apart."""
    q, _, _ = inputs(cuda, torch.float32, 1, 2, 0, 64, 128, 1, "bhsd")
    positions = (2 ** 31 - 64 + torch.arange(64, device=cuda))[None, None]
    for p in (positions, positions.int(), -positions):
        ref.check(ops.axial_rotary(q, None, p, [64]), ref.axial_rotary(q, p, [64]), "far")
    positions = 2 ** 40 + positions
    ref.check(ops.axial_rotary(q, None, positions, [64]), ref.axial_rotary(q, positions, [64]), "farther")


def test_frequencies_base_and_one_row_of_positions_for_all(cuda):
    q, k, _ = inputs(cuda, torch.bfloat16, 3, 4, 2, 21, 64, 2, "bshd")
    positions = torch.randint(0, 50, (2, 21), device=cuda)
    f = [0.7 ** i for i in range(20)]
    got = ops.axial_rotary(q, k, positions, [12, 8], frequencies=f)
    spread = positions[:, None].expand(2, 3, 21)
    for x, y in zip((q, k), got):
        ref.check(y, ref.axial_rotary(x, spread, [12, 8], frequencies=f), "frequencies")
    again = ops.axial_rotary(q, k, spread, [12, 8], frequencies=f)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    ref.check(ops.axial_rotary(q, None, positions, [32, 0], base=5e5), ref.axial_rotary(q, spread, [32, 0], base=5e5), "base")


@pytest.mark.parametrize("dtype", DTYPES)
def test_slices_off_a_boundary_and_expanded_inputs(cuda, dtype):
    """Heads of a fused projection that start anywhere, rows of odd pitch, and one head expanded to several."""
    fused = torch.randn(2, 9, 7 * 64 + 3, device=cuda).to(dtype)
    positions = torch.randint(0, 500, (2, 2, 9), device=cuda)
    for start in (0, 1, 2, 3):
        x = fused[..., start:start + 6 * 64].unflatten(-1, (6, 64)).transpose(1, 2)
        for pairing in ops.PAIRINGS:
            ref.check(ops.axial_rotary(x, None, positions, [16, 16], pairing=pairing),
                      ref.axial_rotary(x, positions, [16, 16], pairing=pairing), f"from {start}")
    one = torch.randn(2, 1, 9, 64, device=cuda).to(dtype).expand(2, 5, 9, 64)
    ref.check(ops.axial_rotary(one, None, positions, [16, 16]), ref.axial_rotary(one, positions, [16, 16]), "expanded")


def test_there_and_back_and_the_gradient_is_the_transpose(cuda):
    q, k, positions = inputs(cuda, torch.float32, 2, 3, 1, 40, 128, 3, "bshd", far=30000)
    how = dict(sections=[16, 24, 24], base=1e6)
    turned = ops.axial_rotary(q, k, positions, **how)
    back = ops.axial_rotary_backward(*turned, positions, **how)
    for x, t, y in zip((q, k), turned, back):
        # two turns, each off by 6 roundings of |u| + |w|, which the pair's length bounds by sqrt(2) of itself
        assert float((x - y).abs().max()) <= 20 * 2.0 ** -24 * float(x.abs().max())
        g = torch.randn_like(x)
        dx = ops.axial_rotary_backward(g, None, positions, **how)
        assert abs(float((t.double() * g.double()).sum() - (x.double() * dx.double()).sum())) <= \
            12 * 2.0 ** -24 * float((x.double().abs() * g.double().abs()).sum()) * 2


def test_streams_graphs_and_nothing_to_do(cuda):
    q, k, positions = inputs(cuda, torch.bfloat16, 2, 8, 2, 60, 128, 3, "bshd")
    call = lambda: ops.axial_rotary(q, k, positions, [16, 24, 24])  # noqa: E731
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
        assert torch.equal(a, b) and torch.equal(a, c)
    none, _ = ops.axial_rotary(q[:, :, :0], k[:, :, :0], positions[:, :, :0], [16, 24, 24])
    assert none.shape == (2, 8, 0, 128)


@pytest.mark.parametrize("strides", [(1000, 300, 1, 1), (2000, 1, 10, 1), (1, 1, 1, 1), (32, 64, 5, 1)])
def test_views_whose_rows_overlap(cuda, strides):
    """(the memory order of such a view is no order for a result)"""
    q = torch.randn(5000, device=cuda).as_strided((2, 3, 5, 64), strides)
    k = torch.randn(2, 1, 5, 64, device=cuda)
    positions = torch.randint(0, 500, (1, 2, 5), device=cuda)
    for f in (ops.axial_rotary, ops.axial_rotary_backward):
        got = f(q, k, positions, [32])
        assert got[0].stride(3) == 1
        for a, b in zip(got, f(q.contiguous(), k, positions, [32])):
            assert torch.equal(a, b)
    assert torch.equal(ops.axial_rotary(k, q[:, :1], positions, [32])[1], ops.axial_rotary(q[:, :1].contiguous(), None, positions, [32]))
