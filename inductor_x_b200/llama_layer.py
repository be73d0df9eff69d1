"""The Llama-style decoder layer of benchmark configuration 5, written as the plain PyTorch
graph a user would hand to ``torch.compile``: RMSNorm, QKV projections, rotary embedding,
causal attention, output projection, residual, RMSNorm, SwiGLU feed-forward, residual.
It exists so that tests and the benchmark compile the same graph; it is not a model zoo.

The attention half of a layer with a sliding window, shared key heads and positions with several axes stands beside it: for
training (``window_attention_half``) and for serving over a cache with 8-bit projections (``window_attention_step``)."""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def rms_norm(x: torch.Tensor, w: torch.Tensor, eps: float) -> torch.Tensor:
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)).to(x.dtype) * w


def apply_rope(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    d = x.shape[-1] // 2
    rot = torch.cat([-x[..., d:], x[..., :d]], dim=-1)
    return (x.float() * cos + rot.float() * sin).to(x.dtype)


def decoder_layer(x, w, cos, sin, heads: int = 32, eps: float = 1e-6):
    """x [B, S, hidden]; w: dict of weights as produced by the benchmark's input generator;
    cos / sin [S, head_dim] fp32 tables."""
    B, S, Hd = x.shape
    D = Hd // heads
    h1 = rms_norm(x, w["norm1"], eps)
    q = F.linear(h1, w["wq"]).view(B, S, heads, D).transpose(1, 2)
    k = F.linear(h1, w["wk"]).view(B, S, heads, D).transpose(1, 2)
    v = F.linear(h1, w["wv"]).view(B, S, heads, D).transpose(1, 2)
    q, k = apply_rope(q, cos, sin), apply_rope(k, cos, sin)
    a = F.scaled_dot_product_attention(q, k, v, is_causal=True, scale=1.0 / math.sqrt(D))
    a = a.transpose(1, 2).reshape(B, S, Hd)
    h = x + F.linear(a, w["wo"])
    h2 = rms_norm(h, w["norm2"], eps)
    ff = F.linear(F.silu(F.linear(h2, w["w_gate"])) * F.linear(h2, w["w_up"]), w["w_down"])
    return h + ff


def window_attention_half(x, w, positions, *, heads: int, kv_heads: int, sections, window: int, sinks: int = 0,
                          lengths=None, base: float = 10000.0, eps: float = 1e-6):
    """``x`` plus the attention of its norm: RMSNorm, projections, rotary positions, windowed attention, output projection.
    x [B, S, hidden]; w: dict with norm1, wq, wk, wv, wo; positions [axes, B, S]; lengths int32 [B] of a padded batch.
    Differentiable in x and w."""
    from . import window_ops  # noqa: F401  (registers the operators)

    B, S, Hd = x.shape
    D = w["wq"].shape[0] // heads
    h = rms_norm(x, w["norm1"], eps)
    split = lambda t, n: t.view(B, S, n, D).transpose(1, 2)  # noqa: E731
    q, k, v = split(F.linear(h, w["wq"]), heads), split(F.linear(h, w["wk"]), kv_heads), split(F.linear(h, w["wv"]), kv_heads)
    q, k = torch.ops.b200_graph.b200_axial_rotary(q, k, positions, sections, base)
    a, _ = torch.ops.b200_graph.b200_window_attention(q, k, v, 1.0 / math.sqrt(D), window, sinks, lengths, lengths)
    return x + F.linear(a.transpose(1, 2).reshape(B, S, heads * D), w["wo"])


def quantise_rows(weight: torch.Tensor):
    """A projection's weight [out, in] in 8 bits with a scale for each row, as ``window_attention_step`` takes it."""
    scales = weight.float().abs().amax(1, keepdim=True).clamp(min=1e-12) / 448.0
    return (weight.float() / scales).to(torch.float8_e4m3fn), scales


def _scaled_product(h8, scales, weight, dtype):
    """``(h8 * scales) @ (w8 * w_scales)^T`` in ``dtype``: a plain library product of 8-bit values whose results take a row's and
    a column's scale.  With those scales the library rounds to bf16 only (asked for fp16 it returns values that are off by as much
    as the largest); for fp16 its unscaled 32-bit sums are scaled here and rounded once."""
    w8, w_scales = weight
    if dtype == torch.bfloat16:
        return torch._scaled_mm(h8, w8.t(), scale_a=scales[:, None], scale_b=w_scales.t(), out_dtype=dtype)
    one = scales.new_ones(())
    sums = torch._scaled_mm(h8, w8.t(), scale_a=one, scale_b=one, out_dtype=torch.float32)
    return (sums * scales[:, None] * w_scales.t()).to(dtype)


def window_attention_step(x, residual, w, positions, cache_k, cache_v, lengths, *, heads: int, kv_heads: int, sections,
                          window: int, sinks: int = 0, base: float = 10000.0, eps: float = 1e-6):
    """One token of each sequence: the residual is added and normalised to 8 bits, projected, turned and written to the
    cache at ``lengths`` (int32 [B], which it then advances), and attends to what its window leaves of the cache.
    x, residual [B, hidden], bf16 or fp16; w: dict with norm1 and, from :func:`quantise_rows`, wqkv, and wo; positions [axes, B, 1];
    cache_k, cache_v [B, kv_heads, capacity, D], as :func:`ops.window_attention` takes them.  Returns the output projection and the
    new residual.  A sequence whose cache has no room (nothing waits for the device to say so) keeps its cache and its length, and
    its projection is NaN."""
    from . import ops

    # a call that is refused leaves the cache and the lengths as they are
    B, D = x.shape[0], cache_k.shape[-1]
    ops._window_arguments(x.new_empty(B, heads, 0, D), cache_k, cache_v, window, sinks, None, lengths)
    if cache_k.shape[1] != kv_heads or cache_k.shape[2] == 0 or not (ops._operand_fits(cache_k) and ops._operand_fits(cache_v)):
        raise ValueError("the caches must be [B, kv_heads, capacity, D] with strides of whole 16 bytes")
    h8, scales, residual = ops.rmsnorm_quantised(x, w["norm1"], eps, residual=residual, return_residual=True)
    qkv = _scaled_product(h8, scales, w["wqkv"], x.dtype)
    q, k, v = (t.view(B, 1, -1, D).transpose(1, 2) for t in qkv.split([heads * D, kv_heads * D, kv_heads * D], dim=1))
    q, k = ops.axial_rotary(q, k, positions, sections, base=base)
    # a sequence without room writes back what its last place holds
    rows, room = torch.arange(B, device=x.device), (lengths >= 0) & (lengths < cache_k.shape[2])
    place = lengths.clamp(0, cache_k.shape[2] - 1).long()
    for cache, new in ((cache_k, k), (cache_v, v)):
        cache[rows, :, place] = torch.where(room[:, None, None], new[:, :, 0], cache[rows, :, place])
    lengths += room
    a = ops.window_attention(q, cache_k, cache_v, 1.0 / math.sqrt(D), window=window, sinks=sinks, kv_lengths=lengths)
    return F.linear(a.view(B, heads * D), w["wo"]).masked_fill(~room[:, None], math.nan), residual
