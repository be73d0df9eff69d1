"""Rotary positions, the norm with an 8-bit output and windowed attention on tensors of more than 2^31 elements, and at the longest
rows and caches: what lies at the ends, against the definition in 64 bits."""
import pytest
import torch

import test_norm_quantised_gpu as norm
from inductor_x_b200 import ops
from oracle import window_layer as ref

pytestmark = pytest.mark.gpu


def filled(dev, *shape, dtype=torch.bfloat16):
    """A short random stretch over and over: quick to make at any size."""
    t = torch.empty(*shape, dtype=dtype, device=dev)
    flat, some = t.view(-1), torch.randn(1000003, generator=torch.Generator(device=dev).manual_seed(1), device=dev).to(dtype)
    whole = flat.numel() // some.numel() * some.numel()
    flat[:whole].view(-1, some.numel()).copy_(some)
    flat[whole:].copy_(some[:flat.numel() - whole])
    return t


@pytest.mark.parametrize("cols,off", [(8192, 0), (8191, 0), (8192, 1)])
def test_norm(cuda, cols, off):
    rows = (2 ** 31 + 2 ** 24) // cols
    x = filled(cuda, rows * cols + off)[off:].view(rows, cols)
    w = filled(cuda, cols)
    for group in (0, 128):
        q, s, h = ops.rmsnorm_quantised(x, w, 1e-5, residual=x, return_residual=True, group=group)
        for part in (slice(0, 3), slice(2 ** 31 // cols - 2, 2 ** 31 // cols + 2), slice(rows - 3, rows)):
            norm.verify((q[part], s[part], h[part]), x[part], w, 1e-5, x[part], group)
        del q, s, h


@pytest.mark.parametrize("cols", [2 ** 20, 2 ** 20 - 1, 130000])
def test_the_longest_rows(cuda, cols):
    x, w = filled(cuda, 3, cols, dtype=torch.float16), filled(cuda, cols, dtype=torch.float16)
    for group in (0, 128):
        q, s = ops.rmsnorm_quantised(x, w, group=group)
        h, y, scales, wide = ref.rmsnorm_quantised(x, w, 1e-6, None, group)
        # a mean of 2^20 squares in partial sums of at most 2^10 + 2^5 terms
        rel = 2.0 ** -24 * ((2 ** 10 + 2 ** 5 + 10) / 2 + 8)
        assert bool(((s.double() - scales).abs() <= rel * scales).all())
        ratio = y / torch.where(wide > 0, wide, 1.0)
        assert bool(((q.double() - ratio).abs() <= (2.0 ** -4 + 2 * rel) * ratio.abs() + 2.0 ** -10).all())


@pytest.mark.parametrize("D,sections,pairing", [(128, [16, 24, 24], "halves"), (126, [63], "neighbours")])
@pytest.mark.parametrize("storage", ["bshd", "bhsd"])
def test_rotary(cuda, D, sections, pairing, storage):
    H, S = 32, (2 ** 31 + 2 ** 24) // (32 * D)
    q = filled(cuda, 1, S, H, D).transpose(1, 2) if storage == "bshd" else filled(cuda, 1, H, S, D)
    positions = torch.arange(S, device=cuda).expand(len(sections), 1, S)
    got = ops.axial_rotary(q, None, positions, sections, pairing=pairing)
    for part in (slice(0, 4), slice(S - 4, S)):
        ref.check(got[:, :, part], ref.axial_rotary(q[:, :, part], positions[:, :, part], sections, pairing=pairing), f"{part}")


def test_attention_over_a_long_cache(cuda):
    """One key head's cache of 2^24 keys and more, 2^31 elements: windows at its end and all over it."""
    n = 2 ** 24 + 300
    k, v = filled(cuda, 1, 1, n, 128), filled(cuda, 1, 1, n, 128).neg_()
    for queries in (1, 3, 300):
        q = filled(cuda, 1, 2, queries, 128)
        for length in (n, n - 131):
            out, lse = ops.window_attention(q, k, v, 0.09, window=500, sinks=5, return_lse=True, check=True,
                                            kv_lengths=torch.tensor([length], dtype=torch.int32, device=cuda))
            # the keys that are seen, as a short cache of their own: the first five in front of the last 900
            first = length - 900
            near = lambda t: torch.cat([t[:, :, :5], t[:, :, first:length]], 2)  # noqa: E731
            expected = ref.window_attention(q, near(k), near(v), 0.09, window=500, sinks=5)
            ref.check(out, expected["out"], "out")
            ref.check(lse, expected["lse"], "lse")
    q = filled(cuda, 1, 1, 1, 128)
    out = ops.window_attention(q, k, torch.ones_like(v), 0.001, window=n, check=True)
    # a mean of ones, rounded once: the weights' 16-bit roundings, 2^-9 each at most, are what it may be off by
    assert bool(((out.float() - 1).abs() <= 2.0 ** -8 + 2.0 ** -9).all())
