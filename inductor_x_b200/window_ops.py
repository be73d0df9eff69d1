"""The operators of a decoder layer with a sliding window as PyTorch operators, for eager models, ``torch.compile`` and
autograd:

* ``b200_graph::b200_window_attention`` - :func:`ops.window_attention`, output and log-sum-exp, with its gradient. The log-sum-exp
  itself is not differentiated through: it does not require a gradient, and a loss that adds a term of it gets none for that term;
* ``b200_graph::b200_axial_rotary`` - :func:`ops.axial_rotary`, with its gradient;
* ``b200_graph::b200_rmsnorm_quantised`` - :func:`ops.rmsnorm_quantised` (a serving operator: no gradient).

They sit beside ``b200_sdpa`` of the fused-attention pass, in its namespace and with its conventions: a CUDA
implementation, a Meta implementation for tracing, ``register_autograd``.  The windows stand where the reference's operator
takes ``pre_tockens`` and ``next_tockens`` (``inductor_x/npu_fusion_attention_graph.py:13-18``); it has no counterpart to the
other two."""
from __future__ import annotations

import torch

from . import ops
from .fusion_attention_graph import b200_cuda, b200_def, b200_meta

b200_def.define("b200_window_attention(Tensor query, Tensor key, Tensor value, float scale, int window, int sinks=0, "
                "Tensor? q_lengths=None, Tensor? kv_lengths=None) -> (Tensor, Tensor)")
b200_def.define("b200_window_attention_backward(Tensor query, Tensor key, Tensor value, Tensor out, Tensor lse, Tensor dout, "
                "float scale, int window, int sinks=0, Tensor? q_lengths=None, Tensor? kv_lengths=None) "
                "-> (Tensor, Tensor, Tensor)")
b200_def.define("b200_axial_rotary(Tensor query, Tensor key, Tensor positions, int[] sections, float base=10000., "
                "str pairing='halves', str ladder='shared', bool inverse=False, float[]? frequencies=None) -> (Tensor, Tensor)")
b200_def.define("b200_rmsnorm_quantised(Tensor x, Tensor weight, float eps, Tensor? residual=None, int group=0) "
                "-> (Tensor, Tensor, Tensor)")


# ---- windowed attention ----------------------------------------------------------------------------
def _fit(t):
    """As it is where the kernels take it so, else dense (an expanded or oddly sliced operand; the functions refuse those)."""
    return t if t.dim() != 4 or ops._operand_fits(t) else t.clone(memory_format=torch.contiguous_format)


def _window_attention(query, key, value, scale, window, sinks=0, q_lengths=None, kv_lengths=None):
    return ops.window_attention(_fit(query), _fit(key), _fit(value), scale, window=window, sinks=sinks, q_lengths=q_lengths,
                                kv_lengths=kv_lengths, return_lse=True)


def _window_attention_meta(query, key, value, scale, window, sinks=0, q_lengths=None, kv_lengths=None):
    b, h, s, d = query.shape
    return query.new_empty((b, h, s, d)), query.new_empty((b, h, s), dtype=torch.float32)


def _window_attention_backward(query, key, value, out, lse, dout, scale, window, sinks=0, q_lengths=None, kv_lengths=None):
    return ops.window_attention_backward(_fit(query), _fit(key), _fit(value), _fit(out), lse, dout, scale, window=window, sinks=sinks,
                                         q_lengths=q_lengths, kv_lengths=kv_lengths)


def _window_attention_backward_meta(query, key, value, out, lse, dout, scale, window, sinks=0, q_lengths=None,
                                    kv_lengths=None):
    return query.new_empty(query.shape), key.new_empty(key.shape), value.new_empty(value.shape)


def _window_setup(ctx, inputs, output):
    query, key, value, ctx.scale, ctx.window, ctx.sinks, q_lengths, kv_lengths = inputs
    out, lse = output
    ctx.save_for_backward(query, key, value, out, lse, q_lengths, kv_lengths)
    ctx.mark_non_differentiable(lse)
    ctx.set_materialize_grads(False)


def _window_gradient(ctx, dout, _):
    query, key, value, out, lse, q_lengths, kv_lengths = ctx.saved_tensors
    if dout is None:
        return (None,) * 8
    dq, dk, dv = torch.ops.b200_graph.b200_window_attention_backward(
        query, key, value, out, lse, dout, ctx.scale, ctx.window, ctx.sinks, q_lengths, kv_lengths)
    return dq, dk, dv, None, None, None, None, None


# ---- rotary positions --------------------------------------------------------------------------------
def _axial_rotary(query, key, positions, sections, base=10000.0, pairing="halves", ladder="shared", inverse=False,
                  frequencies=None):
    turn = ops.axial_rotary_backward if inverse else ops.axial_rotary
    return turn(query, key, positions, sections, base=base, pairing=pairing, ladder=ladder, frequencies=frequencies)


def _axial_rotary_meta(query, key, positions, sections, base=10000.0, pairing="halves", ladder="shared", inverse=False,
                       frequencies=None):
    return ops._rotary_result(query), ops._rotary_result(key)


def _rotary_setup(ctx, inputs, output):
    _, _, positions, ctx.sections, ctx.base, ctx.pairing, ctx.ladder, ctx.inverse, ctx.frequencies = inputs
    ctx.save_for_backward(positions)


def _rotary_gradient(ctx, dq, dk):
    (positions,) = ctx.saved_tensors
    dense = lambda t: t if t.stride(3) == 1 or t.numel() == 0 else t.contiguous()  # noqa: E731  (the gradient of a sum has no strides)
    dq, dk = torch.ops.b200_graph.b200_axial_rotary(dense(dq), dense(dk), positions, ctx.sections, ctx.base, ctx.pairing,
                                                    ctx.ladder, not ctx.inverse, ctx.frequencies)
    return dq, dk, None, None, None, None, None, None, None


# ---- norm with an 8-bit output -----------------------------------------------------------------------
def _rmsnorm_quantised(x, weight, eps, residual=None, group=0):
    if residual is None:
        q, scales = ops.rmsnorm_quantised(x, weight, eps, group=group)
        return q, scales, x.new_empty(0)
    return ops.rmsnorm_quantised(x, weight, eps, residual=residual, return_residual=True, group=group)


def _rmsnorm_quantised_meta(x, weight, eps, residual=None, group=0):
    scales = tuple(x.shape[:-1]) + ((-(-x.shape[-1] // group),) if group else ())
    return (x.new_empty(x.shape, dtype=torch.float8_e4m3fn), x.new_empty(scales, dtype=torch.float32),
            x.new_empty(x.shape if residual is not None else (0,)))


for _name, _cuda, _meta in (("b200_window_attention", _window_attention, _window_attention_meta),
                            ("b200_window_attention_backward", _window_attention_backward, _window_attention_backward_meta),
                            ("b200_axial_rotary", _axial_rotary, _axial_rotary_meta),
                            ("b200_rmsnorm_quantised", _rmsnorm_quantised, _rmsnorm_quantised_meta)):
    b200_cuda.impl(_name, _cuda)
    b200_meta.impl(_name, _meta)

torch.library.register_autograd("b200_graph::b200_window_attention", _window_gradient, setup_context=_window_setup,
                                lib=b200_def)
torch.library.register_autograd("b200_graph::b200_axial_rotary", _rotary_gradient, setup_context=_rotary_setup, lib=b200_def)
