"""The registered operators of a windowed decoder layer take what the functions take: eager, with gradients and compiled."""
import pytest
import torch

import inductor_x_b200  # noqa: F401
from inductor_x_b200 import llama_layer, ops
from inductor_x_b200 import window_ops  # noqa: F401
from oracle import window_layer as ref

G = torch.ops.b200_graph
FREQUENCIES = [0.9 * 0.6 ** i for i in range(20)]


def test_frequencies_without_memory():
    q = torch.empty(2, 3, 9, 64, dtype=torch.bfloat16, device="meta")
    a, b = G.b200_axial_rotary(q, q[:, :1], torch.empty(2, 2, 9, dtype=torch.int64, device="meta"), [12, 8], frequencies=FREQUENCIES)
    assert a.shape == q.shape and b.shape == (2, 1, 9, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("pairing", ops.PAIRINGS)
def test_frequencies(cuda, compiled, pairing):
    gen = torch.Generator(device=cuda).manual_seed(0)
    q, k = (torch.randn(2, 9, h, 64, generator=gen, device=cuda).half().transpose(1, 2).requires_grad_() for h in (3, 1))
    positions = torch.randint(0, 3000, (2, 2, 9), generator=gen, device=cuda)
    f = lambda q, k: G.b200_axial_rotary(q, k, positions, [12, 8], 10000.0, pairing, frequencies=FREQUENCIES)  # noqa: E731
    torch._dynamo.reset()
    turned = (torch.compile(f, fullgraph=True) if compiled else f)(q, k)
    g = [torch.randn(t.shape, generator=gen, device=cuda).half() for t in turned]
    grads = torch.autograd.grad(turned, (q, k), g)
    how = dict(pairing=pairing, frequencies=FREQUENCIES)
    for x, y, dy, dx in zip((q, k), turned, g, grads):
        ref.check(y.detach(), ref.axial_rotary(x.detach(), positions, [12, 8], **how), "turned")
        ref.check(dx, ref.axial_rotary(dy, positions, [12, 8], inverse=True, **how), "gradient")


LAYOUTS = {
    "expanded heads": lambda t: t[:, :1].expand_as(t),
    "expanded batch": lambda t: t[:1].expand_as(t),
    "a slice at an odd offset": lambda t: torch.cat([t[..., :4], t], -1)[..., 4:],
    "an odd pitch": lambda t: torch.cat([t, t[..., :3]], -1)[..., :128],
    "off a boundary": lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape),
    "the head dimension apart": lambda t: t.transpose(2, 3).contiguous().transpose(2, 3),
}


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("layout", LAYOUTS)
def test_attention_of_operands_in_any_layout(cuda, layout, compiled):
    """As of dense copies, bit for bit, and so are the gradients; those of an expanded operand are summed."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    base = [torch.randn(2, h, s, 128, generator=gen, device=cuda).bfloat16() for h, s in ((4, 70), (2, 90), (2, 90))]
    lengths = torch.tensor([90, 33], dtype=torch.int32, device=cuda)
    g = torch.randn(2, 4, 70, 128, generator=gen, device=cuda).bfloat16()

    def run(change, compiled):
        leaves = [t.clone().requires_grad_() for t in base]
        f = lambda q, k, v: G.b200_window_attention(q, k, v, 0.1, 30, 3, None, lengths)  # noqa: E731
        torch._dynamo.reset()
        f = torch.compile(f, fullgraph=True) if compiled else f
        operands = [change(t) for t in leaves]
        out, lse = f(*operands)
        return operands, out, lse, torch.autograd.grad(out, operands, g)

    operands, out, lse, grads = run(LAYOUTS[layout], compiled)
    assert not any(ops._operand_fits(t) for t in operands)
    dense = [t.detach().clone(memory_format=torch.contiguous_format) for t in operands]
    how = dict(window=30, sinks=3, kv_lengths=lengths)
    expected, e_lse = ops.window_attention(*dense, 0.1, return_lse=True, **how)
    assert torch.equal(out, expected) and torch.equal(lse, e_lse)
    for a, b in zip(grads, ops.window_attention_backward(*dense, expected, e_lse, g, 0.1, **how)):
        assert torch.equal(a, b)
    direct = torch.ops.b200_graph.b200_window_attention_backward(*operands, LAYOUTS[layout](out), lse, g, 0.1, 30, 3, None, lengths)
    assert [t.shape for t in direct] == [t.shape for t in operands]


@pytest.mark.gpu
@pytest.mark.parametrize("compiled", [False, True])
@pytest.mark.parametrize("group", [0, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_norm(cuda, compiled, group, dtype):
    """What the function gives, bit for bit, beside compiled arithmetic on its inputs and results."""
    gen = torch.Generator(device=cuda).manual_seed(2)
    x, r = (torch.randn(2, 5, 300, generator=gen, device=cuda).to(dtype) for _ in range(2))
    w = (1 + 0.2 * torch.randn(300, generator=gen, device=cuda)).to(dtype)

    def with_residual(x, w, r):
        q, s, h = G.b200_rmsnorm_quantised(x + 0.0, w, 1e-5, r, group)
        return q, s, h, q.float() * 2.0, s * 3.0, h + 1.0

    def without(x, w):
        q, s, none = G.b200_rmsnorm_quantised(x, w, 1e-5, None, group)
        return q, s * 1.0, none

    def same(a, b):
        return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))

    torch._dynamo.reset()
    make = (lambda f: torch.compile(f, fullgraph=True)) if compiled else (lambda f: f)
    q, s, h, q2, s3, h1 = make(with_residual)(x, w, r)
    e = ops.rmsnorm_quantised(x, w, 1e-5, residual=r, return_residual=True, group=group)
    assert all(same(a, b) for a, b in zip((q, s, h), e))
    assert same(q2, e[0].float() * 2.0) and same(s3, e[1] * 3.0) and same(h1, e[2] + 1.0)
    q, s, none = make(without)(x, w)
    e = ops.rmsnorm_quantised(x, w, 1e-5, group=group)
    assert same(q, e[0]) and same(s, e[1]) and none.shape == (0,) and none.dtype == dtype


EIGHT_BITS = {
    "to 32 bits": lambda q, s, h: q.float() * s[:, None],
    "to 16 bits": lambda q, s, h: q.to(torch.bfloat16) + h,
    "from 16 bits": lambda q, s, h: (h * 2).to(torch.float8_e4m3fn),
    "and back": lambda q, s, h: (h * 2).to(torch.float8_e5m2).float() + 1,
    "the other way round": lambda q, s, h: q.t().contiguous(),
    "a slice": lambda q, s, h: q[1:3].clone(),
    "two": lambda q, s, h: torch.cat([q, q[:2]]),
    "into another": lambda q, s, h: torch.zeros_like(q).copy_(q),
    "another shape": lambda q, s, h: q.view(2, 3, 512).transpose(0, 1),
}


@pytest.mark.gpu
@pytest.mark.parametrize("then", EIGHT_BITS)
def test_what_a_compiled_graph_does_with_8_bits(cuda, then):
    gen = torch.Generator(device=cuda).manual_seed(3)
    x, r = (torch.randn(6, 512, generator=gen, device=cuda).bfloat16() for _ in range(2))
    w = torch.ones(512, device=cuda).bfloat16()
    f = lambda x, r: EIGHT_BITS[then](*G.b200_rmsnorm_quantised(x, w, 1e-5, r, 0))  # noqa: E731
    torch._dynamo.reset()
    a, b = torch.compile(f, fullgraph=True)(x, r), f(x, r)
    assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.gpu
def test_a_compiled_norm_before_a_product_of_8_bits(cuda):
    gen = torch.Generator(device=cuda).manual_seed(4)
    x, r = (torch.randn(6, 512, generator=gen, device=cuda).bfloat16() for _ in range(2))
    w = torch.ones(512, device=cuda).bfloat16()
    w8, w_scales = llama_layer.quantise_rows(torch.randn(256, 512, generator=gen, device=cuda).bfloat16())

    def f(x, r):
        q, s, h = G.b200_rmsnorm_quantised(x, w, 1e-5, r, 0)
        return torch._scaled_mm(q, w8.t(), scale_a=s[:, None], scale_b=w_scales.t(), out_dtype=torch.bfloat16), h

    torch._dynamo.reset()
    for a, b in zip(torch.compile(f, fullgraph=True)(x, r), f(x, r)):
        assert torch.equal(a, b)
