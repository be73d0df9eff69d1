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


def _refused(**other):
    """A step on host memory that has to be refused before anything is computed (there are no weights)."""
    cache = lambda: torch.zeros(3, K, 20, D, dtype=torch.float16)  # noqa: E731
    a = dict(x=torch.zeros(3, HIDDEN, dtype=torch.float16), cache_k=cache(), cache_v=cache(), lengths=torch.full((3,), 4, dtype=torch.int32)) | HOW | other
    with pytest.raises(ValueError):
        llama_layer.window_attention_step(a.pop("x"), None, {}, None, a.pop("cache_k"), a.pop("cache_v"), a.pop("lengths"), **a)


@pytest.mark.parametrize("other", [
    dict(lengths=torch.full((3,), 4)), dict(lengths=torch.full((2,), 4, dtype=torch.int32)), dict(window=0), dict(sinks=129), dict(kv_heads=1),
    dict(heads=5), dict(cache_k=torch.zeros(3, K, 20, D)), dict(cache_v=torch.zeros(3, K, 21, D, dtype=torch.float16)),
    dict(cache_k=torch.zeros(2, K, 20, D, dtype=torch.float16), cache_v=torch.zeros(2, K, 20, D, dtype=torch.float16)),
    dict(x=torch.zeros(3, HIDDEN)), dict(cache_k=torch.zeros(3, K, 20, D + 4, dtype=torch.float16)[..., :D]),
    dict(cache_k=torch.zeros(3, K, 0, D, dtype=torch.float16), cache_v=torch.zeros(3, K, 0, D, dtype=torch.float16)),
    dict(cache_v=torch.zeros(1, K, 20, D, dtype=torch.float16).expand(3, K, 20, D))])
def test_refusals_come_before_anything_is_computed(monkeypatch, other):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(ops, "rmsnorm_quantised", lambda *a, **k: pytest.fail("a call that had to be refused was made"))
    _refused(**other)


@pytest.mark.gpu
@pytest.mark.parametrize("wrong", [dict(window=0), dict(sinks=129), dict(kind=torch.int64), dict(pitch=4)])
def test_what_is_refused_changes_nothing(cuda, wrong):
    gen = torch.Generator(device=cuda).manual_seed(7)
    w = weights(cuda, torch.bfloat16, gen)
    caches = [torch.randn(2, K, 30, D + wrong.get("pitch", 0), generator=gen, device=cuda).bfloat16()[..., :D] for _ in range(2)]
    x = torch.randn(2, HIDDEN, generator=gen, device=cuda).bfloat16()
    lengths = torch.tensor([3, 29], device=cuda, dtype=wrong.get("kind", torch.int32))
    before = [t.clone() for t in (*caches, lengths)]
    with pytest.raises(ValueError):
        llama_layer.window_attention_step(x, x, w, torch.zeros(3, 2, 1, dtype=torch.int64, device=cuda), *caches, lengths,
                                          **(HOW | {n: v for n, v in wrong.items() if n in HOW}))
    assert all(torch.equal(a, b) for a, b in zip(before, (*caches, lengths)))
