"""The serving step of a windowed decoder layer: its projections against the definition in 64 bits, in both 16-bit types."""
import math

import pytest
import torch

from inductor_x_b200 import llama_layer, ops
from oracle import window_layer as ref

H, K, D, HIDDEN = 6, 2, 128, 512
HOW = dict(heads=H, kv_heads=K, sections=(16, 24, 24), window=40, sinks=3)


def weights(dev, dtype, gen):
    new = lambda o, i: (torch.randn(o, i, generator=gen, device=dev) / math.sqrt(i)).to(dtype)  # noqa: E731
    return {"norm1": (1 + 0.1 * torch.randn(HIDDEN, generator=gen, device=dev)).to(dtype),
            "wqkv": llama_layer.quantise_rows(new((H + 2 * K) * D, HIDDEN)), "wo": new(HIDDEN, H * D)}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B", [1, 5, 33])
def test_step(cuda, monkeypatch, dtype, B):
    gen = torch.Generator(device=cuda).manual_seed(B)
    w = weights(cuda, dtype, gen)
    new = lambda *shape: torch.randn(*shape, generator=gen, device=cuda).to(dtype)  # noqa: E731
    x, residual, cache_k, cache_v = new(B, HIDDEN), new(B, HIDDEN), new(B, K, 90, D), new(B, K, 90, D)
    lengths = torch.randint(0, 89, (B,), generator=gen, device=cuda, dtype=torch.int32)
    positions = torch.stack([lengths.long(), lengths.long() // 8, lengths.long() % 8])[:, :, None]
    places, seen = lengths.long(), {}

    def watch(name):
        f = getattr(ops, name)

        def call(*args, **kw):
            seen[name] = args, f(*args, **kw)
            return seen[name][1]
        monkeypatch.setattr(ops, name, call)

    for name in ("rmsnorm_quantised", "axial_rotary", "window_attention"):
        watch(name)
    y, _ = llama_layer.window_attention_step(x, residual, w, positions, cache_k, cache_v, lengths, **HOW)

    h8, scales, _ = seen["rmsnorm_quantised"][1]
    a, b = h8.double() * scales[:, None].double(), w["wqkv"][0].double() * w["wqkv"][1].double()
    # sums of HIDDEN products in 32 bits, each sum off by 2^-24 of their magnitudes, two scales, one rounding to 16 bits
    half = torch.finfo(dtype).eps / 2
    z, bound = a @ b.t(), (HIDDEN + 3) * 2.0 ** -24 * (a.abs() @ b.abs().t())
    bound = bound * (1 + half) + half * z.abs() + ref._floor(dtype)
    (q, k, *_), _ = seen["axial_rotary"]
    got = torch.cat([t.transpose(1, 2).reshape(B, -1) for t in (q, k)] + [cache_v[torch.arange(B, device=cuda), :, places].reshape(B, -1)], 1)
    ref.check(got, (z, bound), "q, k, v")
    # the output projection of what the attention gave, H * D products
    a, b = seen["window_attention"][1].reshape(B, -1).double(), w["wo"].double()
    z, bound = a @ b.t(), (H * D + 1) * 2.0 ** -24 * (a.abs() @ b.abs().t())
    ref.check(y, (z, bound * (1 + half) + half * z.abs() + ref._floor(dtype)), "y")
    assert bool(torch.isfinite(y).all())
