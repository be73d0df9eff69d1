"""The operators of a windowed decoder layer as PyTorch operators, and a run of them together."""
import math

import pytest
import torch
import torch.nn.functional as F

import inductor_x_b200  # noqa: F401
from inductor_x_b200 import llama_layer, ops
from inductor_x_b200 import window_ops  # noqa: F401
from oracle import window_layer as ref

G = torch.ops.b200_graph


def test_shapes_without_memory():
    m = lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="meta")  # noqa: E731
    q, k = m(2, 8, 33, 128).transpose(1, 2).contiguous().transpose(1, 2), m(2, 2, 77, 128)
    out, lse = G.b200_window_attention(q, k, k, 0.1, 16, 2)
    assert out.shape == q.shape and out.is_contiguous() and lse.shape == (2, 8, 33) and lse.dtype == torch.float32
    assert [t.shape for t in G.b200_window_attention_backward(q, k, k, out, lse, out, 0.1, 16)] == [q.shape, k.shape, k.shape]
    a, b = G.b200_axial_rotary(q, k[:, :, :33], m(3, 2, 33, dtype=torch.int64), [16, 24, 24])
    assert a.shape == q.shape and a.stride() == q.stride() and b.shape == (2, 2, 33, 128)
    for group, scales in ((0, (2, 5)), (128, (2, 5, 3))):
        x = m(2, 5, 300)
        q8, s, h = G.b200_rmsnorm_quantised(x, m(300), 1e-6, x, group)
        assert q8.dtype == torch.float8_e4m3fn and q8.shape == x.shape and s.shape == scales and h.shape == x.shape
        assert G.b200_rmsnorm_quantised(x, m(300), 1e-6, None, group)[2].numel() == 0


def weights(dev, dtype, hidden, heads, kv_heads, D=128):
    gen = torch.Generator(device=dev).manual_seed(1)
    new = lambda o, i: (torch.randn(o, i, generator=gen, device=dev) / math.sqrt(i)).to(dtype)  # noqa: E731
    return {"norm1": (1 + 0.1 * torch.randn(hidden, generator=gen, device=dev)).to(dtype), "wq": new(heads * D, hidden),
            "wk": new(kv_heads * D, hidden), "wv": new(kv_heads * D, hidden), "wo": new(hidden, heads * D)}


SHAPE = dict(heads=6, kv_heads=2, sections=(16, 24, 24))


def layer_inputs(dev, dtype=torch.bfloat16, B=2, S=150, hidden=256):
    gen = torch.Generator(device=dev).manual_seed(0)
    x = torch.randn(B, S, hidden, generator=gen, device=dev).to(dtype)
    positions = torch.stack([torch.arange(S, device=dev).expand(B, S) + 1000, torch.randint(0, 30, (B, S), generator=gen, device=dev),
                             torch.randint(0, 30, (B, S), generator=gen, device=dev)])
    return x, positions, weights(dev, dtype, hidden, SHAPE["heads"], SHAPE["kv_heads"])


@pytest.mark.gpu
def test_gradients_of_the_operators_are_those_of_the_functions(cuda):
    B, S = 2, 130
    q = torch.randn(B, S, 6, 128, device=cuda).bfloat16().transpose(1, 2).requires_grad_()
    k, v = (torch.randn(B, S, 2, 128, device=cuda).bfloat16().transpose(1, 2).requires_grad_() for _ in range(2))
    lengths = torch.tensor([130, 70], dtype=torch.int32, device=cuda)
    positions = torch.randint(0, 5000, (3, B, S), device=cuda)
    tq, tk = G.b200_axial_rotary(q, k, positions, [16, 24, 24])
    out, lse = G.b200_window_attention(tq, tk, v, 0.09, 40, 3, lengths, lengths)
    assert not lse.requires_grad
    g = torch.randn_like(out)
    grads = torch.autograd.grad(out, (q, k, v), g)
    how = dict(window=40, sinks=3, q_lengths=lengths, kv_lengths=lengths)
    o, l = ops.window_attention(tq.detach(), tk.detach(), v.detach(), 0.09, return_lse=True, **how)
    assert torch.equal(o, out) and torch.equal(l, lse)
    dtq, dtk, dv = ops.window_attention_backward(tq.detach(), tk.detach(), v.detach(), o, l, g, 0.09, **how)
    dq, dk = ops.axial_rotary_backward(dtq, dtk, positions, [16, 24, 24])
    for a, b in zip(grads, (dq, dk, dv)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_gradients_without_strides_and_unused_results(cuda):
    """The gradient of a sum is one value seen everywhere; an unused result has none."""
    q, k = (torch.randn(1, 2, 9, 64, device=cuda, requires_grad=True) for _ in range(2))
    positions = torch.randint(0, 500, (1, 9), device=cuda)
    a, b = G.b200_axial_rotary(q, k, positions, [32])
    a.sum().backward()
    expected, bound = ref.axial_rotary(torch.ones_like(q), positions[:, None].expand(1, 1, 9), [32], inverse=True)
    ref.check(q.grad, (expected, bound), "dq")
    assert not k.grad.any()
    x = torch.randn(1, 2, 9, 128, device=cuda).half().requires_grad_()
    out, _ = G.b200_window_attention(x, x, x, 0.1, 4)
    out.sum().backward()
    e = ref.window_attention(x.detach(), x.detach(), x.detach(), 0.1, window=4, dout=torch.ones_like(x))
    total = sum(e[n][0] for n in ("dq", "dk", "dv"))
    # the sum of three, rounded to 16 bits twice
    bound = sum(e[n][1] for n in ("dq", "dk", "dv")) + 2.0 ** -11 * 2 * sum(e[n][0].abs() for n in ("dq", "dk", "dv")) * 1.01
    ref.check(x.grad, (total, bound), "all of it")


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [False, True])
def test_training_half(cuda, compiled):
    """Forward and gradients of the whole half against a plain form in 64 bits, in fp16: within what 16-bit tensors between its
    steps can be off."""
    x, positions, w = layer_inputs(cuda, torch.float16)
    lengths = torch.tensor([150, 91], dtype=torch.int32, device=cuda)
    how = dict(window=40, sinks=4, lengths=lengths, **SHAPE)
    f = torch.compile(llama_layer.window_attention_half, fullgraph=True) if compiled else llama_layer.window_attention_half
    leaves = [x.clone().requires_grad_()] + [w[n].clone().requires_grad_() for n in ("norm1", "wq", "wk", "wv", "wo")]
    y = f(leaves[0], dict(zip(("norm1", "wq", "wk", "wv", "wo"), leaves[1:])), positions, **how)
    live = (torch.arange(150, device=cuda) < lengths[:, None])[..., None]
    g = torch.randn_like(y) * live
    grads = torch.autograd.grad(y, leaves, g)

    exact = [t.detach().double().requires_grad_() for t in leaves]
    z = _half_in_64_bits(exact[0], dict(zip(("norm1", "wq", "wk", "wv", "wo"), exact[1:])), positions, how)
    expected = torch.autograd.grad(z, exact, g.double())
    # A result is a chain of at most twelve 16-bit tensors (norm, projections, turned, attention's and back again), each off by half
    # a step of its values at most, 2^-11, independent of one another: sums over hundreds of them are off by about that share of
    # their norm.  Norms are compared, 4 times twelve half steps.
    for a, b, name in zip((y, *grads), (z, *expected), ("y", "dx", "dnorm", "dwq", "dwk", "dwv", "dwo")):
        a, b = (t.double() * live if name == "y" else t.double() for t in (a, b))
        assert float((a - b).norm()) <= 48 * 2.0 ** -11 * float(b.norm()), name


def _half_in_64_bits(x, w, positions, how):
    B, S, _ = x.shape
    H, K, D = how["heads"], how["kv_heads"], 128
    h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w["norm1"]
    split = lambda t, n: t.view(B, S, n, D).transpose(1, 2)  # noqa: E731
    q, k, v = split(F.linear(h, w["wq"]), H), split(F.linear(h, w["wk"]), K), split(F.linear(h, w["wv"]), K)
    axis = torch.tensor([a for a, n in enumerate(how["sections"]) for _ in range(n)], device=x.device)
    angle = positions[axis].double().permute(1, 2, 0)[:, None] * 10000.0 ** (-torch.arange(64, device=x.device, dtype=torch.float64) / 64)
    turn = lambda t: torch.cat([t[..., :64] * angle.cos() - t[..., 64:] * angle.sin(),  # noqa: E731
                                t[..., :64] * angle.sin() + t[..., 64:] * angle.cos()], -1)
    q, k = turn(q), turn(k).repeat_interleave(H // K, 1)
    v = v.repeat_interleave(H // K, 1)
    i = torch.arange(S, device=x.device)
    seen = (i[None] <= i[:, None]) & ((i[None] > i[:, None] - how["window"]) | (i[None] < how["sinks"]))
    s = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(~seen, -math.inf)
    a = torch.softmax(s, -1) @ v
    live = (i < how["lengths"][:, None])[:, None, :, None]
    a = torch.where(live, a, 0.0)
    return x + F.linear(a.transpose(1, 2).reshape(B, S, H * D), w["wo"])


@pytest.mark.gpu
def test_serving_steps_over_a_cache(cuda):
    """Three tokens of each sequence: every operator of a step against its definition on what it was given, and what the steps
    leave in the cache against a prefill over the same keys."""
    B, hidden, H, K, D, capacity = 3, 512, 6, 2, 128, 300
    dtype = torch.bfloat16
    w = weights(cuda, dtype, hidden, H, K)
    w8 = {"norm1": w["norm1"], "wqkv": llama_layer.quantise_rows(torch.cat([w["wq"], w["wk"], w["wv"]])), "wo": w["wo"]}
    gen = torch.Generator(device=cuda).manual_seed(2)
    before = torch.tensor([0, 70, 290], dtype=torch.int32, device=cuda)
    cache_k, cache_v = (torch.full((B, K, capacity, D), float("nan"), device=cuda, dtype=dtype) for _ in range(2))
    for b, n in enumerate(before.tolist()):
        for c in (cache_k, cache_v):
            c[b, :, :n] = torch.randn(K, n, D, generator=gen, device=cuda).to(dtype)
    lengths, how = before.clone(), dict(window=64, sinks=4)
    seen = []
    originals = ops.rmsnorm_quantised, ops.axial_rotary, ops.window_attention

    def watched(f, name):
        def call(*args, **kw):
            args = [a.clone() if isinstance(a, torch.Tensor) and a.dim() != 4 else a for a in args]
            r = f(*args, **kw)
            seen.append((name, args, {k: v.clone() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}, r))
            return r
        return call

    try:
        ops.rmsnorm_quantised, ops.axial_rotary, ops.window_attention = (
            watched(f, n) for f, n in zip(originals, ("norm", "rotary", "attention")))
        x, residual = (torch.randn(B, hidden, generator=gen, device=cuda).to(dtype) for _ in range(2))
        for step in range(3):
            positions = torch.stack([lengths.long(), lengths.long() // 8, lengths.long() % 8])[:, :, None]
            x, residual = llama_layer.window_attention_step(x, residual, w8, positions, cache_k, cache_v, lengths, heads=H, kv_heads=K,
                                                            sections=(16, 24, 24), **how)
            name, args, kw, (q8, scales, h) = seen[-3]
            expected_h, y, expected_s, wide = ref.rmsnorm_quantised(args[0], args[1], args[2], kw["residual"])
            assert name == "norm" and torch.equal(h, expected_h)
            assert bool(((q8.double() * scales[:, None].double() - y).abs() <= 2.0 ** -4 * y.abs() * 1.001 + 2.0 ** -10 * wide).all())
            name, args, kw, turned = seen[-2]
            for a, t in zip(args[:2], turned):
                ref.check(t, ref.axial_rotary(a, positions, (16, 24, 24)), name)
            name, (q, ck, cv, scale), kw, out = seen[-1]
            assert lengths.tolist() == [n + step + 1 for n in before.tolist()]
            ref.check(out, ref.window_attention(q, ck, cv, scale, kv_lengths=lengths, **how)["out"], name)
    finally:
        ops.rmsnorm_quantised, ops.axial_rotary, ops.window_attention = originals
    # the three queries at once over the same cache: each within its bound of the definition
    q = torch.cat([s[1][0] for s in seen if s[0] == "attention"], 2)
    steps = torch.cat([s[3] for s in seen if s[0] == "attention"], 2)
    together = ops.window_attention(q, cache_k, cache_v, 1 / math.sqrt(D), kv_lengths=lengths, **how)
    value, bound = ref.window_attention(q, cache_k, cache_v, 1 / math.sqrt(D), kv_lengths=lengths, **how)["out"]
    ref.check(together, (value, bound), "at once")
    ref.check(steps, (value, bound), "one by one")


@pytest.mark.gpu
def test_a_serving_step_without_room(cuda):
    """A full cache, and a length that is none, stay as they are; the others are served as they are without them."""
    B, hidden, H, K, D, capacity = 4, 256, 4, 2, 128, 20
    w = weights(cuda, torch.bfloat16, hidden, H, K)
    w8 = {"norm1": w["norm1"], "wqkv": llama_layer.quantise_rows(torch.cat([w["wq"], w["wk"], w["wv"]])), "wo": w["wo"]}
    gen = torch.Generator(device=cuda).manual_seed(3)
    new = lambda *shape: torch.randn(*shape, generator=gen, device=cuda).bfloat16()  # noqa: E731
    caches, x, residual = [new(B, K, capacity, D) for _ in range(2)], new(B, hidden), new(B, hidden)
    how = dict(heads=H, kv_heads=K, sections=(64,), window=8, sinks=2)

    def step(lengths):
        lengths, here = torch.tensor(lengths, dtype=torch.int32, device=cuda), [c.clone() for c in caches]
        y, _ = llama_layer.window_attention_step(x, residual, w8, lengths.clamp(min=0).long()[None, :, None], *here, lengths, **how)
        return y, here, lengths.tolist()

    y, here, lengths = step([20, 19, -1, 5])
    expected, there, _ = step([3, 19, 4, 5])
    assert lengths == [20, 20, -1, 6]
    assert bool(y[[0, 2]].isnan().all()) and torch.equal(y[[1, 3]], expected[[1, 3]])
    for c, a, b in zip(caches, here, there):
        assert torch.equal(a[[0, 2]], c[[0, 2]]) and torch.equal(a[[1, 3]], b[[1, 3]])
