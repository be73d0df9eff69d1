"""The windowed layer's operators in captured graphs: as a process' first call, as a serving step whose cache grows from replay to
replay, and as a training step."""
import os
import subprocess
import sys

import pytest
import torch

import test_window_layer as layer
import test_window_serving as serving
from inductor_x_b200 import llama_layer

pytestmark = pytest.mark.gpu

FIRST = {
    "decode": "q, k = new(2, 8, 1, 128), new(2, 2, 3000, 128); call = lambda: ops.window_attention(q, k, k, 0.1, window=1000, sinks=4)",
    "split": "q, k = new(1, 8, 512, 128), new(1, 2, 4096, 128); call = lambda: ops.window_attention(q, k, k, 0.1, window=2048, sinks=4)",
    "prefill": "q, k = new(2, 16, 700, 128), new(2, 4, 700, 128); call = lambda: ops.window_attention(q, k, k, 0.1, window=200, sinks=5)",
    "backward": "q, k, l = new(2, 4, 300, 128), new(2, 2, 300, 128), torch.zeros(2, 4, 300, device='cuda') + 9; "
                "call = lambda: torch.cat([t.flatten() for t in ops.window_attention_backward(q, k, k, q, l, q, 0.1, window=50, sinks=3)])",
    "rotary": "q, p = new(2, 4, 900, 64), torch.arange(900, device='cuda')[None]; call = lambda: ops.axial_rotary(q, None, p, [32])",
    "norm": "x, w = new(300, 1024), new(1024); call = lambda: ops.rmsnorm_quantised(x, w)[0].view(torch.uint8)",
    "odd norm": "x, w = new(9000, 1537), new(1537); call = lambda: ops.rmsnorm_quantised(x, w, group=128)[0].view(torch.uint8)",
}


def test_the_first_calls_of_a_process_may_be_captured(cuda):
    """What a kernel asks of the device at its first call it may ask while a stream is being captured."""
    code = "import torch; from inductor_x_b200 import ops; torch.manual_seed(0); new = lambda *s: torch.randn(*s, device='cuda').half()\n"
    for name, line in FIRST.items():
        code += (f"{line}; torch.cuda.synchronize(); g = torch.cuda.CUDAGraph()\n"
                 "with torch.cuda.graph(g):\n    out = call()\n"
                 f"out.zero_(); g.replay(); torch.cuda.synchronize(); assert torch.equal(out, call()) and bool(out.any()); print('{name}')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    child = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert child.stdout.splitlines() == list(FIRST), child.stderr[-2000:]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_captured_serving_step(cuda, dtype):
    B = 3
    gen = torch.Generator(device=cuda).manual_seed(6)
    w = serving.weights(cuda, dtype, gen)
    new = lambda *shape: torch.randn(*shape, generator=gen, device=cuda).to(dtype)  # noqa: E731
    x, residual, caches = new(B, serving.HIDDEN), new(B, serving.HIDDEN), [new(B, serving.K, 60, serving.D) for _ in range(2)]
    before = torch.tensor([0, 41, 58], dtype=torch.int32, device=cuda)

    def steps(run, lengths, here):
        got = []
        for i in range(4):                                   # (the last sequence is full after two)
            y, r = run()
            got += [y.clone(), r.clone(), lengths.clone(), *(c.clone() for c in here)]
        return got

    def prepared():
        lengths, here = before.clone(), [c.clone() for c in caches]
        step = lambda: llama_layer.window_attention_step(  # noqa: E731
            x, residual, w, torch.stack([lengths.long(), lengths.long() // 8, lengths.long() % 8])[:, :, None], *here, lengths, **serving.HOW)
        return step, lengths, here

    step, lengths, here = prepared()
    expected = steps(step, lengths, here)
    step, lengths, here = prepared()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                                               # (the product's workspace)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            results = step()
        lengths.copy_(before)
        for c, was in zip(here, caches):
            c.copy_(was)

        def replay():
            graph.replay()
            return results

        got = steps(replay, lengths, here)
    side.synchronize()
    for a, b in zip(got, expected):
        assert torch.equal(a.nan_to_num(), b.nan_to_num()) and torch.equal(a.isnan(), b.isnan())


def test_a_captured_training_step(cuda):
    """Forward and gradients through the registered operators.  (No graph of the leaves that ran eagerly on another stream may live
    while theirs is captured: PyTorch refuses that for its own operators too.)"""
    x, positions, w = layer.layer_inputs(cuda, torch.float16)
    names = ("norm1", "wq", "wk", "wv", "wo")
    leaves = [x.requires_grad_()] + [w[n].requires_grad_() for n in names]
    how = dict(window=40, sinks=4, lengths=torch.tensor([150, 91], dtype=torch.int32, device=cuda), **layer.SHAPE)
    g = torch.randn_like(x)
    forward = lambda: llama_layer.window_attention_half(leaves[0], dict(zip(names, leaves[1:])), positions, **how)  # noqa: E731
    alive = forward()
    expected = [alive.detach().clone(), *torch.autograd.grad(alive, leaves, g)]
    del alive
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = forward()
        torch.autograd.grad(y, leaves, g)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = forward()
            captured = [y.detach(), *torch.autograd.grad(y, leaves, g)]
        for t in captured:
            t.zero_()
        graph.replay()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(captured, expected))
