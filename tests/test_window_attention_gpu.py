"""Attention with a sliding window and first tokens that stay visible: output, log-sum-exp and gradients against the
definition in 64 bits, at the sizes, masks and layouts where they can go wrong."""
import math

import pytest
import torch

from inductor_x_b200 import ops
from oracle import window_layer as ref

pytestmark = pytest.mark.gpu


def make(dev, dtype, B, H, HK, Sq, Sk, storage="bhsd", seed=0, q_lengths=None, kv_lengths=None, junk=float("nan")):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def new(h, s):
        shape = (B, s, h, 128) if storage == "bshd" else (B, h, s, 128)
        t = torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dtype)
        return t.transpose(1, 2) if storage == "bshd" else t

    q, k, v, g = new(H, Sq), new(HK, Sk), new(HK, Sk), new(H, Sq)
    lengths = [torch.tensor(n, dtype=torch.int32, device=dev) if n is not None else None for n in (q_lengths, kv_lengths)]
    # nothing behind a length may reach a result, whatever it is
    for n, ts in zip((q_lengths, kv_lengths), ((q, g), (k, v))):
        for b, m in enumerate(n or []):
            for t in ts:
                t[b, :, max(0, m):] = junk
    return q, k, v, g, *lengths


def both(dev, dtype, B, H, HK, Sq, Sk, window, sinks, q_lengths=None, kv_lengths=None, scale=128 ** -0.5, backward=True, **how):
    q, k, v, g, ql, kl = make(dev, dtype, B, H, HK, Sq, Sk, q_lengths=q_lengths, kv_lengths=kv_lengths, **how)
    mask = dict(window=window, sinks=sinks, q_lengths=ql, kv_lengths=kl)
    out, lse = ops.window_attention(q, k, v, scale, return_lse=True, check=True, **mask)
    expected = ref.window_attention(q, k, v, scale, window=window, sinks=sinks, q_lengths=q_lengths, kv_lengths=kv_lengths,
                                    dout=g if backward else None)
    ref.check(out, expected["out"], "out")
    ref.check(lse, expected["lse"], "lse")
    again = ops.window_attention(q, k, v, scale, **mask)
    assert torch.equal(again, out)
    if backward:
        grads = ops.window_attention_backward(q, k, v, out, lse, g, scale, check=True, **mask)
        for name, d in zip(("dq", "dk", "dv"), grads):
            ref.check(d, expected[name], name)
        for a, b in zip(grads, ops.window_attention_backward(q, k, v, out, lse, g, scale, **mask)):
            assert torch.equal(a, b)


SIZES = [
    # B, H, HK, Sq, Sk, window, sinks
    (1, 1, 1, 1, 1, 1, 0),
    (1, 2, 1, 2, 2, 1, 1),
    (2, 4, 2, 130, 130, 1, 0),
    (2, 6, 2, 129, 129, 64, 0),
    (1, 4, 4, 257, 700, 128, 16),
    (1, 3, 3, 200, 50, 40, 3),        # fewer keys than queries: the first ones see nothing
    (1, 5, 1, 300, 300, 127, 128),
    (1, 2, 2, 640, 640, 256, 4),
    (1, 4, 2, 513, 1025, 200, 7),
    (1, 8, 2, 384, 384, 1000, 0),     # the window is longer than the sequence
    (1, 2, 1, 200, 900, 100, 128),
    (2, 7, 7, 65, 1000, 33, 1),
    (1, 2, 2, 1, 129, 128, 0),
    (1, 4, 1, 900, 900, 129, 64),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", SIZES)
def test_against_64_bits(cuda, dtype, sizes):
    both(cuda, dtype, *sizes, storage="bshd" if sizes[1] % 2 else "bhsd", seed=sum(sizes))


RAGGED = [
    # B, H, HK, Sq, Sk, window, sinks, lengths of the queries, of the keys
    (4, 4, 2, 150, 333, 90, 7, [150, 1, 0, 77], [333, 1, 200, 64]),
    (3, 2, 1, 256, 256, 100, 4, [256, 128, 129], [256, 128, 129]),
    (3, 4, 4, 129, 129, 30, 0, None, [0, 1, 128]),
    (2, 6, 3, 260, 400, 500, 3, [260, 200], None),
    (2, 2, 2, 140, 500, 64, 9, [300, -3], [9999, -1]),          # out of range: the nearest length counts
    (2, 4, 2, 400, 400, 60, 130 - 2, [400, 390], [399, 300]),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", RAGGED)
def test_padded_batches(cuda, dtype, case):
    both(cuda, dtype, *case, storage="bshd" if case[1] == 4 else "bhsd", seed=case[3])


DECODE = [
    # B, H, HK, Sq, Sk, window, sinks, lengths of the keys
    (1, 8, 2, 1, 3000, 512, 4, None),
    (4, 16, 2, 1, 5000, 1024, 4, [5000, 1, 0, 1029]),
    (3, 5, 1, 1, 700, 300, 0, [700, 299, 301]),
    (2, 14, 2, 2, 2000, 257, 33, [2000, 261]),
    (5, 8, 8, 4, 300, 64, 64, [300, 3, 64, 65, 200]),
    (2, 32, 1, 3, 900, 100000, 0, [900, 2]),
    (1, 4, 4, 1, 20000, 8192, 128, None),
    (64, 2, 1, 1, 200, 128, 1, None),
    (2, 48, 2, 4, 1000, 500, 5, [1000, 100]),
    (1, 1, 1, 1, 40000, 50000, 0, None),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", DECODE)
def test_few_queries_over_a_cache(cuda, dtype, case):
    *sizes, lengths = case
    both(cuda, dtype, *sizes, None, lengths, backward=False, seed=sizes[4])


@pytest.mark.parametrize("Sq", [1, 3, 16, 17, 128, 129, 300])
@pytest.mark.parametrize("share", [1, 2, 3, 8])
def test_any_number_of_queries_and_shared_heads(cuda, Sq, share):
    both(cuda, torch.bfloat16, 2, 2 * share, 2, Sq, 400, 150, 5, None, [400, 260], backward=False, seed=Sq + share)


def test_large_scores_and_one_sided_rows(cuda):
    """Scores of some hundreds: the running maximum moves by far more than a rescale's threshold, both ways."""
    q, k, v, _, _, _ = make(cuda, torch.float16, 1, 2, 1, 300, 600, seed=5)
    for order in (False, True):
        ramp = torch.linspace(-3, 3, 600, device=cuda, dtype=torch.float16)[:, None]
        kk = k + (ramp.flip(0) if order else ramp)
        out, lse = ops.window_attention(q, kk, v, 0.5, window=400, sinks=4, return_lse=True)
        expected = ref.window_attention(q, kk, v, 0.5, window=400, sinks=4)
        # the exponent's argument, up to some hundreds, is 2^-24 of itself off: 2^-14 of a probability, with the products' sum
        value, bound = expected["out"]
        ref.check(out, (value, bound + 2.0 ** -13 * v.abs().max().double()), "out")
        ref.check(lse, (expected["lse"][0], expected["lse"][1] * 4), "lse")


def test_strides_of_a_fused_projection_and_of_single_entries(cuda):
    """q, k and v as slices of one projection; axes of one entry with strides that say nothing."""
    B, S, H, HK = 2, 200, 4, 2
    fused = torch.randn(B, S, (H + 2 * HK) * 128, device=cuda, dtype=torch.float32).to(torch.bfloat16)
    q, k, v = (t.unflatten(-1, (-1, 128)).transpose(1, 2) for t in fused.split([H * 128, HK * 128, HK * 128], -1))
    out, lse = ops.window_attention(q, k, v, 0.1, window=50, sinks=2, return_lse=True)
    g = torch.randn_like(out)
    grads = ops.window_attention_backward(q, k, v, out, lse, g, 0.1, window=50, sinks=2)
    expected = ref.window_attention(q, k, v, 0.1, window=50, sinks=2, dout=g)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        ref.check(t, expected[name], name)
    one = torch.randn(1, 1, 1, 128, device=cuda).half().as_strided((1, 1, 1, 128), (3, 5, 7, 1))
    out = ops.window_attention(one, one, one, 0.1, window=1)
    assert torch.equal(out, one)


def test_no_keys_and_no_queries(cuda):
    q, k = torch.randn(2, 2, 3, 128, device=cuda).half(), torch.empty(2, 1, 0, 128, device=cuda).half()
    out, lse = ops.window_attention(q, k, k, 0.1, window=4, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())
    dq, dk, dv = ops.window_attention_backward(q, k, k, out, lse, q, 0.1, window=4)
    assert not dq.any() and dk.shape == k.shape and dv.shape == k.shape
    none = q[:, :, :0]
    kk = torch.randn(2, 1, 5, 128, device=cuda).half()
    out, lse = ops.window_attention(none, kk, kk, 0.1, window=4, return_lse=True)
    assert out.shape == none.shape and lse.shape == (2, 2, 0)
    dq, dk, dv = ops.window_attention_backward(none, kk, kk, out, lse, none, 0.1, window=4)
    assert dq.shape == none.shape and not dk.any() and not dv.any()
    empty = q[:0]
    assert ops.window_attention(empty, kk[:0], kk[:0], 0.1, window=4).shape == empty.shape


def test_no_heads(cuda):
    q, k = torch.empty(2, 0, 3, 128, device=cuda).half(), torch.randn(2, 2, 5, 128, device=cuda).half()
    out, lse = ops.window_attention(q, k, k, 0.1, window=4, return_lse=True)
    dq, dk, dv = ops.window_attention_backward(q, k, k, out, lse, out, 0.1, window=4)
    assert out.shape == q.shape and dq.shape == q.shape and not dk.any() and not dv.any()


def test_gradients_off_a_boundary_are_taken(cuda):
    """An incoming gradient may start and step anywhere."""
    q, k, v, g, _, _ = make(cuda, torch.bfloat16, 2, 2, 1, 70, 90, seed=4)
    out, lse = ops.window_attention(q, k, v, 0.1, window=30, return_lse=True)
    expected = ops.window_attention_backward(q, k, v, out, lse, g, 0.1, window=30)
    off = torch.empty(g.numel() + 1, device=cuda, dtype=g.dtype)[1:].view(g.shape).copy_(g)
    wide = torch.empty(2, 2, 70, 131, device=cuda, dtype=g.dtype)[..., :128].copy_(g)
    other = g.transpose(2, 3).contiguous().transpose(2, 3)
    for d in (off, wide, other):
        for a, b in zip(expected, ops.window_attention_backward(q, k, v, out, lse, d, 0.1, window=30)):
            assert torch.equal(a, b)


def test_offsets_beyond_32_bits(cuda):
    """A cache, queries and gradients whose batches lie more than 2^31 elements apart."""
    far = 2 ** 31 + 4096
    memory = torch.zeros(far + (1 << 20), dtype=torch.float16, device=cuda)
    gen = torch.Generator(device=cuda).manual_seed(8)

    def view(heads, s, at):
        t = memory.as_strided((2, heads, s, 128), (far, s * 128, 128, 1), at)
        return t.copy_(torch.randn(2, heads, s, 128, generator=gen, device=cuda))

    k, v, q, g = view(2, 600, 0), view(2, 600, 200000), view(4, 150, 400000), view(4, 150, 500000)
    lengths = torch.tensor([600, 333], dtype=torch.int32, device=cuda)
    how = dict(window=100, sinks=5, kv_lengths=lengths)
    out, lse = ops.window_attention(q, k, v, 0.09, return_lse=True, **how)
    expected = ref.window_attention(q, k, v, 0.09, dout=g, **how)
    grads = ops.window_attention_backward(q, k, v, out, lse, g, 0.09, **how)
    for name, t in zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)):
        ref.check(t, expected[name], name)
    one = q[:, :, :1]
    ref.check(ops.window_attention(one, k, v, 0.09, **how), ref.window_attention(one, k, v, 0.09, **how)["out"], "decode")


def test_many_first_tokens_and_a_short_window_over_a_long_sequence(cuda):
    """The first tokens' later queries make more items than are kept apart."""
    both(cuda, torch.bfloat16, 1, 1, 1, 18000, 18000, 16, 128, seed=6)


def test_gradients_against_differences(cuda):
    """Along a random direction, by the definition's own differences in 64 bits."""
    q, k, v, g, _, _ = make(cuda, torch.float16, 1, 4, 2, 150, 150, seed=3)
    how = dict(window=40, sinks=3)
    out, lse = ops.window_attention(q, k, v, 0.09, return_lse=True, **how)
    grads = ops.window_attention_backward(q, k, v, out, lse, g, 0.09, **how)
    for i, (t, d) in enumerate(zip((q, k, v), grads)):
        step = torch.randn(t.shape, device=cuda, dtype=torch.float64)
        moved = []
        for sign in (1, -1):
            args = [x.double() for x in (q, k, v)]
            args[i] = args[i] + sign * 1e-5 * step
            o = _plain(*args, 0.09, **how)
            moved.append((o * g.double()).sum())
        slope = (moved[0] - moved[1]) / 2e-5
        value, bound = ref.window_attention(q, k, v, 0.09, dout=g, **how)[("dq", "dk", "dv")[i]]
        # differences of a smooth sum: 1e-10 of the third derivative, next to nothing
        assert abs(float((d.double() * step).sum() - slope)) <= float((bound * step.abs()).sum()) + 1e-4 * abs(float(slope))
        assert abs(float((value * step).sum() - slope)) <= 1e-5 * float((value * step).abs().sum())


def _plain(q, k, v, scale, window, sinks):
    share = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(share, 1), v.repeat_interleave(share, 1)
    i = torch.arange(q.shape[2], device=q.device)[:, None] + k.shape[2] - q.shape[2]
    j = torch.arange(k.shape[2], device=q.device)
    s = (q @ k.transpose(-1, -2) * scale).masked_fill((j > i) | ((j <= i - window) & (j >= sinks)), -math.inf)
    return torch.softmax(s, -1) @ v


def test_other_streams_and_graphs(cuda):
    q, k, v, g, ql, kl = make(cuda, torch.bfloat16, 2, 8, 2, 200, 300, q_lengths=[200, 90], kv_lengths=[300, 120])
    dec = q[:, :, :1].contiguous()
    how = dict(window=70, sinks=4, q_lengths=ql, kv_lengths=kl)

    def all_of_it():
        out, lse = ops.window_attention(q, k, v, 0.1, return_lse=True, **how)
        one = ops.window_attention(dec, k, v, 0.1, window=70, sinks=4, kv_lengths=kl)
        return (out, lse, one, *ops.window_attention_backward(q, k, v, out, lse, g, 0.1, **how))

    expected = all_of_it()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = all_of_it()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                captured = all_of_it()
            graphs.append((graph, captured))
        for graph, captured in graphs:
            for t in captured:
                t.zero_()
            graph.replay()
        for graph, _ in graphs:
            graph.replay()
    side.synchronize()
    for captured in [got] + [c for _, c in graphs]:
        assert all(torch.equal(a, b) for a, b in zip(expected, captured))


def test_lengths_are_read_when_the_kernel_runs(cuda):
    """A captured decoding step serves a cache that grows."""
    q, k, v, _, _, kl = make(cuda, torch.bfloat16, 2, 4, 2, 1, 500, kv_lengths=[500, 500])
    kl.fill_(100)
    ops.window_attention(q, k, v, 0.1, window=64, sinks=2, kv_lengths=kl)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.window_attention(q, k, v, 0.1, window=64, sinks=2, kv_lengths=kl)
    for n in (1, 63, 64, 66, 499):
        kl.fill_(n)
        graph.replay()
        torch.cuda.synchronize()
        ref.check(out, ref.window_attention(q, k, v, 0.1, window=64, sinks=2, kv_lengths=[n, n])["out"], "out")


FEW_TILES = [
    # B, H, HK, Sq, Sk, window, sinks, lengths of the queries, of the keys: few tiles of rows over many keys
    (1, 4, 2, 200, 1500, 600, 4, None, None),
    (1, 8, 2, 512, 4096, 2048, 4, None, None),
    (2, 4, 1, 300, 2500, 5000, 0, [300, 129], [2500, 129]),
    (1, 2, 2, 140, 9000, 8000, 128, None, None),
    (1, 1, 1, 1024, 1024, 4096, 0, None, None),
    (3, 3, 1, 140, 1300, 1100, 9, [140, 1, 77], [1300, 1153, 0]),       # a first token's tile, a last tile of one key
    (4, 2, 2, 260, 1200, 700, 1, [260, 128, 129, 5], [1200, 128, 100, 1025]),
    (1, 6, 1, 100, 2000, 1900, 128, [100], [1999]),                     # (a tile holds rows of one head, heads of it are missing)
    (2, 5, 1, 60, 3100, 3000, 0, [60, 59], [3100, 2944]),
    (1, 7, 1, 130, 700, 1, 1, None, None),
    (3, 16, 8, 130, 1300, 1200, 3, None, [1300, 1153, 700]),             # as many tiles as SMs: one block a tile
    (3, 8, 4, 200, 1500, 1300, 4, [200, 128, 0], None),                  # two
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("case", FEW_TILES)
def test_few_tiles_over_many_keys(cuda, dtype, case):
    both(cuda, dtype, *case, storage="bshd" if case[1] % 2 else "bhsd", seed=case[3])


def test_few_tiles_on_two_streams_and_in_a_graph(cuda):
    calls = [make(cuda, torch.bfloat16, 1, 4, 2, s, 2000, seed=s)[:3] for s in (256, 400)]
    run = lambda i: ops.window_attention(*calls[i], 0.09, window=1500, sinks=4)
    expected = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, run(i)))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        captured = [(i, run(i)) for i in (0, 1)]
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, expected[i]) for i, o in got + captured)
