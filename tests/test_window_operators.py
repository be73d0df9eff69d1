"""The registered operators of a windowed decoder layer take what the functions take: eager, with gradients and compiled."""
import pytest
import torch

import inductor_x_b200  # noqa: F401
from inductor_x_b200 import ops
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
