"""Windowed attention with more work items than the GPU has SMs: two tiles of rows in an item of the forward, the two with different
windows or one left over, items that a running block takes over (forward, dK/dV, dQ), heads that leave the last group of
the dispatch order short, and the form of every kernel.  Against the definition in 64 bits."""
import pytest
import torch

import test_window_attention_gpu as window
from inductor_x_b200 import ops
from kernels_taken import kernels, sm_count

pytestmark = pytest.mark.gpu


def tiles_of_rows(H, HK, Sq):
    """Tiles of 128 rows that a key head has: R rows of each of 128 / R of its query heads."""
    R = min(128, max(8, 1 << (Sq - 1).bit_length()))
    return -(-Sq // 128) * -(-(H // HK) // (128 // R))


MANY = [
    # B, H, HK, Sq, Sk, window, sinks, lengths of the queries, of the keys
    (2, 16, 4, 700, 700, 200, 5, None, None),
    (2, 15, 5, 640, 900, 200, 7, None, None),                                          # 15 tiles: one is left over
    (3, 37, 37, 400, 400, 130, 4, None, None),                                         # two tiles of an item, tile 0 in one's window only
    (4, 20, 10, 500, 900, 150, 33, [500, 0, 129, 257], [900, 640, 0, 200]),            # nothing to do in many; a long step of first tokens
    (2, 30, 6, 300, 1000, 100, 128, None, [1000, 333]),
    (5, 64, 8, 60, 700, 200, 9, None, [700, 60, 61, 0, 300]),                          # tiles of two heads' rows
    (6, 56, 8, 40, 500, 150, 40, [40, 1, 39, 40, 17, 40], [500, 500, 128, 129, 0, 41]),  # and one of a single head
    (2, 48, 48, 260, 260, 1000, 0, None, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", MANY)
def test_more_tiles_than_sms(cuda, dtype, case):
    B, H, HK, Sq, Sk = case[:5]
    assert tiles_of_rows(H, HK, Sq) * B * HK > sm_count()  # two tiles an item
    window.both(cuda, dtype, *case, storage="bshd" if H % 2 else "bhsd", seed=Sq)


@pytest.mark.parametrize("case,rounds", [(MANY[2], 1), (MANY[3], 1), ((5, 48, 24, 380, 380, 90, 2, None, [380, 100, 0, 380, 379]), 2)])
def test_items_taken_over(cuda, case, rounds):
    """More items of each kernel than the GPU runs at a time."""
    B, H, HK, Sq, Sk = case[:5]
    sms = sm_count()
    assert -(-tiles_of_rows(H, HK, Sq) // 2) * B * HK > rounds * sms                   # forward
    assert -(-Sk // 128) * B * HK > rounds * sms and -(-Sq // 128) * B * H > rounds * sms  # dK/dV, dQ
    window.both(cuda, torch.bfloat16, *case, seed=1)


def test_a_few_heads_alone_have_the_same_bits(cuda):
    """Whoever works on an item, its arithmetic is the same: tiles and gradients of three key heads, in items of their own."""
    B, H, HK, Sq, Sk, w, sinks = 2, 60, 30, 520, 520, 150, 4
    q, k, v, g, _, _ = window.make(cuda, torch.bfloat16, B, H, HK, Sq, Sk, seed=9)
    how = dict(window=w, sinks=sinks)
    out, lse = ops.window_attention(q, k, v, 0.09, return_lse=True, **how)
    grads = ops.window_attention_backward(q, k, v, out, lse, g, 0.09, **how)
    few = [t[1:, -(6 * t.shape[1] // H):].contiguous() for t in (q, k, v)]
    fewer = [t[1:, -6:].contiguous() for t in (out, lse, g)]
    alone = ops.window_attention_backward(*few, *fewer, 0.09, **how)
    for a, b in zip(grads, alone):
        assert torch.equal(a[1:, -b.shape[1]:], b)


KERNELS = [
    # the kernel, and B, H, HK, Sq, Sk, window, sinks, lengths of the keys
    ("fa_window_fwd_kernel<{}>", (2, 8, 8, 300, 600, 100, 4, None)),
    ("fa_window_fwd_kernel<{}>", (3, 40, 40, 300, 600, 200, 4, [600, 300, 0])),
    ("window_split_kernel<{}, 1>", (3, 16, 8, 130, 1300, 1200, 3, [1300, 1153, 700])),
    ("window_split_kernel<{}, 2>", (3, 8, 4, 200, 1500, 1300, 4, None)),
    ("window_split_kernel<{}, 4>", (1, 8, 2, 512, 4096, 2048, 4, None)),
    ("window_split_kernel<{}, 8>", (2, 5, 1, 60, 3100, 3000, 0, [3100, 2944])),
    ("window_decode_kernel<{}, 1, 1>", (25, 16, 8, 1, 700, 500, 4, [700 - 29 * i for i in range(25)])),
    ("window_decode_kernel<{}, 1, 2>", (16, 16, 8, 2, 400, 300, 4, [400 - 27 * i for i in range(15)] + [0])),
    ("window_decode_kernel<{}, 1, 4>", (5, 24, 8, 2, 900, 500, 5, [900, 0, 2, 503, 700])),
    ("window_decode_kernel<{}, 1, 8>", (2, 14, 2, 1, 3000, 1000, 128, [3000, 1])),
    ("window_decode_kernel<{}, 2, 1>", (24, 96, 8, 1, 300, 200, 7, [300 - 13 * i for i in range(24)])),
    ("window_decode_kernel<{}, 2, 2>", (5, 64, 8, 4, 500, 300, 5, [500, 3, 301, 299, 0])),
    ("window_decode_kernel<{}, 2, 4>", (4, 64, 8, 4, 500, 300, 0, [500, 3, 301, 77])),
    ("window_decode_kernel<{}, 2, 8>", (2, 48, 2, 4, 1000, 500, 5, [1000, 100])),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kernel,case", KERNELS)
def test_every_kernel_is_taken_and_right(cuda, dtype, kernel, case):
    """Which kernel takes a call goes by what each promises: a constant that moves must not leave one without a test."""
    B, H, HK, Sq, Sk, w, sinks, lengths = case
    q, k, v, _, _, kl = window.make(cuda, dtype, B, H, HK, Sq, Sk, kv_lengths=lengths)
    call = lambda: ops.window_attention(q, k, v, 0.1, window=w, sinks=sinks, kv_lengths=kl)  # noqa: E731
    call()
    assert kernels(call) == {kernel.format("true" if dtype == torch.bfloat16 else "false")}
    window.both(cuda, dtype, B, H, HK, Sq, Sk, w, sinks, None, lengths, backward=False, seed=Sk)


def test_as_many_tiles_as_sms(cuda):
    """One tile of rows for each SM, and one more."""
    sms = sm_count()
    for heads in (sms, sms + 1):
        assert tiles_of_rows(heads, heads, 128) * heads == heads
        window.both(cuda, torch.float16, 1, heads, heads, 128, 700, 600, 3, None, [690], backward=False, seed=heads)
        window.both(cuda, torch.bfloat16, 1, heads, heads, 128, 300, 100, 3, seed=heads)


def test_kernels_of_the_backward(cuda):
    q, k, v, g, _, _ = window.make(cuda, torch.bfloat16, 2, 4, 2, 300, 300)
    out, lse = ops.window_attention(q, k, v, 0.1, window=70, sinks=3, return_lse=True)
    for sinks, more in ((0, set()), (3, {"window_sinks_kernel<true>"})):
        names = kernels(lambda: ops.window_attention_backward(q, k, v, out, lse, g, 0.1, window=70, sinks=sinks))
        assert names == {"window_delta_kernel<true>", "window_dkv_kernel<true>", "window_dq_kernel<true>"} | more
