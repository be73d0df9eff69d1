"""Tensor-level entry points over the C ABI: one function per prebuilt kernel family.

These are what the generated wrapper code, the tests and ``bench.py`` call.  Each takes
CUDA tensors, validates layout, allocates the output with torch (plumbing only) and
enqueues exactly the native kernels on the current stream.  A CPU tensor is rejected:
there is no host path.
"""
from __future__ import annotations

import ctypes
import functools
import operator
from typing import Optional, Sequence, Tuple

import torch

from . import _ixb_host
from . import runtime as rt


def launch_count() -> int:
    """Calls made into the kernel library's launching entry points so far (each enqueues one
    kernel; a split outer reduction two)."""
    return rt.native_calls


def _native(fn: str, done):
    """What a native entry point (``csrc/host_launch.cpp``) returned: None for a call it leaves to
    Python, the status of one that failed, else the result."""
    if done is None:
        return None
    if type(done) is int:
        rt.check(fn, done)
    rt.native_calls += 1
    return done


def _need_cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("inductor_x_b200 kernels take CUDA tensors only (no CPU path)")


def _cfg_ref(cfg):
    c = rt.make_cfg(cfg)
    return (ctypes.byref(c) if c is not None else None), c


def affine_gelu_rowsum(x: torch.Tensor, w: torch.Tensor, b: torch.Tensor, *, out=None, cfg=None):
    """``sum(gelu(x * w + b), dim=-1)`` for fp32 ``x[rows, cols]``, ``w[cols]``, ``b[cols]``."""
    _need_cuda(x, w, b)
    if x.dtype != torch.float32 or x.dim() != 2 or not x.is_contiguous():
        raise ValueError("x must be a contiguous fp32 matrix")
    rows, cols = x.shape
    if w.shape != (cols,) or b.shape != (cols,) or w.dtype != x.dtype or b.dtype != x.dtype:
        raise ValueError("w and b must be fp32 vectors of length cols")
    w, b = w.contiguous(), b.contiguous()
    if out is None:
        out = torch.empty(rows, dtype=x.dtype, device=x.device)
    ref, keep = _cfg_ref(cfg)
    rt.check("ixb_affine_gelu_rowsum_f32", rt.load().ixb_affine_gelu_rowsum_f32(
        x.data_ptr(), w.data_ptr(), b.data_ptr(), out.data_ptr(), rows, cols, ref,
        rt.raw_stream(x.device)))
    return out


def softmax_layernorm(x, g, gamma, beta, eps: float = 1e-5, *, out=None, cfg=None):
    """``layer_norm(softmax(x, -1) * g + x, [cols], gamma, beta, eps)`` in one pass."""
    _need_cuda(x, g, gamma, beta)
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported dtype {x.dtype}")
    if not x.is_contiguous() or x.dim() < 1:
        raise ValueError("x must be contiguous")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    for name, v in (("g", g), ("gamma", gamma), ("beta", beta)):
        if v.shape != (cols,) or v.dtype != x.dtype:
            raise ValueError(f"{name} must have shape ({cols},) and dtype {x.dtype}")
    g, gamma, beta = g.contiguous(), gamma.contiguous(), beta.contiguous()
    if out is None:
        out = torch.empty_like(x)
    ref, keep = _cfg_ref(cfg)
    rt.check("ixb_softmax_layernorm", rt.load().ixb_softmax_layernorm(
        rt.DTYPE_CODE[x.dtype], x.data_ptr(), g.data_ptr(), gamma.data_ptr(), beta.data_ptr(),
        out.data_ptr(), rows, cols, float(eps), ref, rt.raw_stream(x.device)))
    return out


def rmsnorm(x, w, eps: float = 1e-6, *, residual=None, return_residual: bool = False, cfg=None):
    """RMSNorm over the last axis with an optional fused residual add.

    Returns ``y`` or ``(y, h)`` where ``h = x + residual`` (rounded to the storage dtype)."""
    if cfg is None:
        done = _native("ixb_rmsnorm", _ixb_host.rms_norm(x, w, eps, residual, return_residual))
        if done is not None:
            return done
    _need_cuda(x, w, residual)
    if not x.is_contiguous():
        raise ValueError("x must be contiguous")
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    if w.shape != (cols,) or w.dtype != x.dtype:
        raise ValueError("w must be a vector of length cols in x's dtype")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or not residual.is_contiguous()):
        raise ValueError("residual must match x")
    y = torch.empty_like(x)
    h = torch.empty_like(x) if (residual is not None and return_residual) else None
    ref, keep = _cfg_ref(cfg)
    rt.check("ixb_rmsnorm", rt.load().ixb_rmsnorm(
        rt.DTYPE_CODE[x.dtype], x.data_ptr(), rt.ptr(residual), w.contiguous().data_ptr(),
        y.data_ptr(), rt.ptr(h), rows, cols, float(eps), ref, rt.raw_stream(x.device)))
    return (y, h) if h is not None else y


def row_reduce(x: torch.Tensor, kind: str, *, correction: float = 1.0, cfg=None):
    """Reduce the last axis of contiguous ``x``.  ``kind``: sum, mean, amax, amin, argmax,
    argmin or var_mean (returns ``(var, mean)``)."""
    _need_cuda(x)
    if not x.is_contiguous() or x.dim() < 1:
        raise ValueError("x must be contiguous")
    code = rt.REDUCE_CODE[kind]
    cols = x.shape[-1]
    rows = x.numel() // cols if cols else 0
    lead = x.shape[:-1]
    out_dtype = torch.int64 if code in (rt.IXB_ARGMAX, rt.IXB_ARGMIN) else x.dtype
    out = torch.empty(lead, dtype=out_dtype, device=x.device)
    out2 = torch.empty(lead, dtype=x.dtype, device=x.device) if code == rt.IXB_VAR_MEAN else None
    ref, keep = _cfg_ref(cfg)
    rt.check("ixb_row_reduce", rt.load().ixb_row_reduce(
        rt.DTYPE_CODE[x.dtype], code, x.data_ptr(), out.data_ptr(), rt.ptr(out2), rows, cols,
        float(correction), ref, rt.raw_stream(x.device)))
    return (out, out2) if out2 is not None else out


def outer_reduce(x: torch.Tensor, kind: str, *, rsplit: int = 0, scratch: Optional[torch.Tensor] = None):
    """Reduce the middle axis of contiguous ``x[outer, R, inner]`` -> ``[outer, inner]``.

    ``rsplit`` > 1 forces a split of the reduced axis (0 = library's choice); the fp32
    scratch it needs is taken from ``scratch`` or allocated here with torch."""
    _need_cuda(x, scratch)
    if x.dim() != 3 or not x.is_contiguous():
        raise ValueError("x must be a contiguous [outer, R, inner] tensor")
    outer, R, inner = x.shape
    code = rt.REDUCE_CODE[kind]
    lib = rt.load()
    if rsplit <= 0 and outer and inner:
        rsplit = rt.choose_config(rt.IXB_FAM_OUTER, x.dtype, outer, R, inner).rsplit
    need = lib.ixb_outer_reduce_scratch_bytes(outer, inner, rsplit)
    if need and (scratch is None or scratch.numel() * scratch.element_size() < need):
        scratch = torch.empty(need // 4, dtype=torch.float32, device=x.device)
    out = torch.empty((outer, inner), dtype=x.dtype, device=x.device)
    cfg = rt.IxbCfg(rsplit=max(rsplit, 1))
    sbytes = scratch.numel() * scratch.element_size() if scratch is not None else 0
    rt.check("ixb_outer_reduce", lib.ixb_outer_reduce(
        rt.DTYPE_CODE[x.dtype], code, x.data_ptr(), out.data_ptr(), outer, R, inner, rt.ptr(scratch),
        sbytes, ctypes.byref(cfg), rt.raw_stream(x.device)))
    return out


def short_row_reduce(x: torch.Tensor, kind: str, out_strides: Sequence[int],
                     out: Optional[torch.Tensor] = None):
    """Reduce the short stride-1 axis of contiguous ``x[A, B, C, L]`` and store result
    ``(a, b, c)`` at element offset ``a*sa + b*sb + c*sc`` of ``out``."""
    _need_cuda(x, out)
    if x.dim() != 4 or not x.is_contiguous():
        raise ValueError("x must be a contiguous [A, B, C, L] tensor")
    A, B, C, L = x.shape
    sa, sb, sc = (int(s) for s in out_strides)
    if out is None:
        out = torch.empty(A * B * C, dtype=x.dtype, device=x.device)
    rt.check("ixb_short_row_reduce", rt.load().ixb_short_row_reduce(
        rt.DTYPE_CODE[x.dtype], rt.REDUCE_CODE[kind], x.data_ptr(), out.data_ptr(), A, B, C, L,
        sa, sb, sc, rt.raw_stream(x.device)))
    return out


def index_select_rows(table: torch.Tensor, idx: torch.Tensor, *, wrap_negative: bool = False,
                      check_bounds: bool = True):
    """``table.index_select(0, idx)`` for a 2-D+ table whose rows are contiguous.

    With ``check_bounds`` an out-of-range index raises ``IndexError`` (this reads a device
    status word back, i.e. synchronises; pass False inside latency-critical code)."""
    _need_cuda(table, idx)
    if table.dim() < 1 or idx.dim() != 1 or idx.dtype not in (torch.int64, torch.int32):
        raise ValueError("table must have >= 1 dim, idx must be a 1-D int32/int64 tensor")
    n_rows = table.shape[0]
    row_shape = table.shape[1:]
    if table.dim() > 1 and not table[0].is_contiguous():
        raise ValueError("rows of table must be contiguous")
    row_elems = 1
    for s in row_shape:
        row_elems *= s
    row_bytes = row_elems * table.element_size()
    pitch = (table.stride(0) if table.dim() > 1 else 1) * table.element_size()
    if n_rows <= 1:
        pitch = max(pitch, row_bytes)
    idx = idx.contiguous()
    m = idx.numel()
    out = torch.empty((m, *row_shape), dtype=table.dtype, device=table.device)
    status = torch.zeros(2, dtype=torch.int32, device=table.device) if check_bounds else None
    rt.check("ixb_index_select_rows", rt.load().ixb_index_select_rows(
        table.data_ptr(), idx.data_ptr(), out.data_ptr(), n_rows, m, row_bytes, pitch,
        rt.DTYPE_CODE[idx.dtype], int(wrap_negative), rt.ptr(status), rt.raw_stream(table.device)))
    if status is not None:
        flag, pos = status.tolist()
        if flag:
            raise IndexError(f"index_select_rows: index out of range at position {pos}")
    return out


_I64x3 = ctypes.c_int64 * 3


def _bhs_strides(t: torch.Tensor):
    b, h, s, _ = t.stride()
    return _I64x3(b, h, s)


def fused_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, *,
                    causal: bool = False, return_lse: bool = False, check: bool = False):
    """``softmax(q @ k^T * scale [+ causal mask]) @ v`` for ``[B, H, S, D]`` tensors
    (any batch/head/sequence strides, ``D`` contiguous, ``D == 128``, fp16 or bf16).

    Returns ``out`` (contiguous ``[B, H, Sq, D]``) or ``(out, lse)`` with ``lse`` the fp32
    log-sum-exp of the scaled scores ``[B, H, Sq]``.  ``check=True`` reads the kernel's
    status word back (synchronises) and raises if an internal wait gave up."""
    if not check:
        done = _native("ixb_fa_fwd", _ixb_host.fused_attention(q, k, v, scale, causal, return_lse))
        if done is not None:
            return done
    _need_cuda(q, k, v)
    if q.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("expected q[B,H,Sq,D], k[B,H,Sk,D], v[B,H,Sk,D]")
    if q.dtype not in (torch.float16, torch.bfloat16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k, v must share dtype float16 or bfloat16")
    for t in (q, k, v):
        if t.stride(3) != 1:
            raise ValueError("the head dimension must be contiguous")
    B, H, Sq, D = q.shape
    Sk = k.shape[2]
    out = torch.empty((B, H, Sq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    status = torch.zeros(1, dtype=torch.int32, device=q.device) if check else None
    rt.check("ixb_fa_fwd", rt.load().ixb_fa_fwd(
        rt.DTYPE_CODE[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rt.ptr(lse),
        B, H, Sq, Sk, D, _bhs_strides(q), _bhs_strides(k), _bhs_strides(v), _bhs_strides(out),
        float(scale), int(causal), rt.ptr(status), rt.raw_stream(q.device)))
    if status is not None and int(status.item()) != 0:
        raise RuntimeError("ixb_fa_fwd: an internal pipeline wait gave up; output is undefined")
    return (out, lse) if return_lse else out


#: bytes of dS the attention backward keeps at most between its two products (see ixb_fa_bwd_scratch):
#: what 4 x 32 heads of 4096 causal keys need in one go, 1/70 of the memory of a B200.  The same heads
#: in three launches with 1 GiB: 1700 us a call against 1625, the GPU drains after each
SCORE_GRADIENT_BYTES = 5 << 29


#: a request that fails makes the caching allocator give back all it holds, so a device that could not
#: give what was asked for is asked for less in this many calls
SCORE_GRADIENT_RETRY = 1000
_score_gradient_limits: dict = {}      # device index -> (bytes at most, calls left)


@functools.lru_cache(maxsize=1024)
def _score_gradient_room(B, H, Sq, Sk, causal, limit):
    return rt.load().ixb_fa_bwd_scratch_bytes(B, H, Sq, Sk, int(causal), limit)


def _score_gradient_limit(device: int) -> int:
    limit, left = _score_gradient_limits.get(device, (SCORE_GRADIENT_BYTES, 0))
    if left > 1:
        _score_gradient_limits[device] = (limit, left - 1)
    else:
        _score_gradient_limits.pop(device, None)
    return min(limit, SCORE_GRADIENT_BYTES)


def _backward_scratch(B, H, Sq, Sk, causal, device, limit, refused=False):
    """(one allocation, its bytes for dS ahead of the B * H * Sq floats of delta).  Where the memory
    is not to be had (``refused``: it was asked for already) the backward does with half of it, in more
    launches, and so on down to one head; without dS it computes the probabilities twice."""
    room = _score_gradient_room(B, H, Sq, Sk, causal, limit)
    while room:
        if not refused:
            try:
                return torch.empty(room + 4 * B * H * Sq, dtype=torch.uint8, device=device), room
            except torch.cuda.OutOfMemoryError:
                pass
        refused, less = False, room // 2
        _score_gradient_limits[device.index] = (less, SCORE_GRADIENT_RETRY)
        room = _score_gradient_room(B, H, Sq, Sk, causal, less)
    return torch.empty(4 * B * H * Sq, dtype=torch.uint8, device=device), 0


def fused_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                             lse: torch.Tensor, dout: torch.Tensor, scale: float, *, causal: bool = False,
                             check: bool = False):
    """Gradients ``(dq, dk, dv)`` of :func:`fused_attention` from its inputs, its output
    ``out``, its log-sum-exp ``lse`` (``return_lse=True``) and the incoming gradient ``dout``
    (tcgen05 kernels behind ``ixb_fa_bwd``; deterministic, no atomics)."""
    limit = SCORE_GRADIENT_BYTES if not _score_gradient_limits else _score_gradient_limit(q.device.index)
    refused = False
    if not check:
        done = _ixb_host.fused_attention_backward(q, k, v, out, lse, dout, scale, causal, limit)
        refused = done is False
        done = None if refused else _native("ixb_fa_bwd", done)
        if done is not None:
            return done
    _need_cuda(q, k, v, out, dout, lse)
    if q.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("expected q[B,H,Sq,D], k[B,H,Sk,D], v[B,H,Sk,D]")
    if out.shape != q.shape or dout.shape != q.shape:
        raise ValueError("out and dout must have the shape of q")
    if q.dtype not in (torch.float16, torch.bfloat16) or any(t.dtype != q.dtype for t in (k, v, out, dout)):
        raise ValueError("q, k, v, out, dout must share dtype float16 or bfloat16")
    B, H, Sq, D = q.shape
    Sk = k.shape[2]
    if lse.shape != (B, H, Sq) or lse.dtype != torch.float32:
        raise ValueError("lse must be float32 [B, H, Sq]")
    lse = lse.contiguous()
    if dout.stride(3) != 1 or any(st % 8 for st in dout.stride()[:3]):
        dout = dout.contiguous()
    for t in (q, k, v, out, dout):
        if t.stride(3) != 1:
            raise ValueError("the head dimension must be contiguous")
    dq = torch.empty((B, H, Sq, D), dtype=q.dtype, device=q.device)
    dk = torch.empty((B, H, Sk, D), dtype=q.dtype, device=q.device)
    dv = torch.empty((B, H, Sk, D), dtype=q.dtype, device=q.device)
    scratch, room = _backward_scratch(B, H, Sq, Sk, causal, q.device, limit, refused)
    status = torch.zeros(1, dtype=torch.int32, device=q.device) if check else None
    q_like, kv_like = _bhs_strides(dq), _bhs_strides(dk)
    rt.check("ixb_fa_bwd", rt.load().ixb_fa_bwd_scratch(
        rt.DTYPE_CODE[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(),
        lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), scratch.data_ptr() + room,
        scratch.data_ptr() if room else None, room,
        B, H, Sq, Sk, D,
        _bhs_strides(q), _bhs_strides(k), _bhs_strides(v), _bhs_strides(out), _bhs_strides(dout),
        q_like, kv_like, kv_like, float(scale), int(causal), rt.ptr(status), rt.raw_stream(q.device)))
    if status is not None and int(status.item()) != 0:
        raise RuntimeError("ixb_fa_bwd: an internal pipeline wait gave up; gradients are undefined")
    return dq, dk, dv


# ---- a decoder layer with a sliding window -----------------------------------------------
def rmsnorm_quantised(x, w, eps: float = 1e-6, *, residual=None, return_residual: bool = False, group: int = 0):
    """RMSNorm over the last axis with an optional residual added first, and an 8-bit result.

    Returns ``(q, scales)`` or ``(q, scales, h)``: ``h = x + residual`` rounded to the storage dtype, ``q``
    (``torch.float8_e4m3fn``, the shape of ``x``) times ``scales`` (float32) the norm of ``h``.  ``group=0``: a scale
    for each row, ``scales`` of shape ``x.shape[:-1]``; ``group=128``: one for each 128 values, ``[..., ceil(cols /
    128)]`` and contiguous (a product that wants the rows' axis innermost takes ``scales.t().contiguous().t()``).  A scale is the
    largest magnitude / 448; the norm is rounded once, to 8 bits.  A NaN of the norm makes its scale and all that the scale
    covers NaN, an infinity makes its scale infinite, itself NaN and the finite values beside it 0."""
    done = _native("ixb_rmsnorm_quantised", _ixb_host.rms_norm_quantised(x, w, eps, residual, return_residual, group))
    if done is not None:
        return done
    _need_cuda(x, w, residual)
    if x.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"unsupported dtype {x.dtype}")
    if group not in (0, 128):
        raise ValueError("group must be 0 (a scale a row) or 128")
    if not x.is_contiguous() or x.dim() < 1:
        raise ValueError("x must be contiguous")
    cols = x.shape[-1]
    if cols == 0:
        raise ValueError("a row must have a value")
    rows = x.numel() // cols
    if w.shape != (cols,) or w.dtype != x.dtype:
        raise ValueError("w must be a vector of length cols in x's dtype")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype
                                 or not residual.is_contiguous()):
        raise ValueError("residual must match x")
    _one_device(x, w, residual)
    w = w.contiguous()
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scales = torch.empty(x.shape[:-1] + ((-(-cols // group),) if group else ()), dtype=torch.float32, device=x.device)
    h = torch.empty_like(x) if residual is not None and return_residual else None
    if rows:
        with torch.cuda.device(x.device):
            rt.check("ixb_rmsnorm_quantised", rt.load().ixb_rmsnorm_quantised(
                rt.DTYPE_CODE[x.dtype], x.data_ptr(), rt.ptr(residual), w.data_ptr(), q.data_ptr(), scales.data_ptr(),
                rt.ptr(h), rows, cols, group, float(eps), rt.raw_stream(x.device)))
    return (q, scales) if h is None else (q, scales, h)


def _one_device(first: torch.Tensor, *others: Optional[torch.Tensor]) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError("all tensors must be on one device")


def _fits_32_bits(*ts: Optional[torch.Tensor]) -> None:
    """The entries take an axis as a 32-bit number (views of few bytes may have longer ones)."""
    if any(t is not None and any(n > 2 ** 31 - 1 for n in t.shape) for t in ts):
        raise ValueError("an axis may not have more than 2^31 - 1 entries")


def _operand_strides(t: torch.Tensor):
    """Strides of the (batch, head, sequence) axes; an axis of one entry, whose stride says nothing, counts as dense."""
    B, H, S, D = t.shape
    b, h, s, _ = t.stride()
    s = s if S > 1 else D
    h = h if H > 1 else S * D
    return _I64x3(b if B > 1 else H * S * D, h, s)


def _operand_fits(t: torch.Tensor) -> bool:
    """Whether the attention kernels take a tensor as it lies: ``D`` contiguous, other strides positive multiples of 8 elements, rows
    on 16-byte boundaries."""
    return t.numel() == 0 or (t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(st > 0 and st % 8 == 0 for st in _operand_strides(t)))


def _window_arguments(q, k, v, window, sinks, q_lengths, kv_lengths):
    _need_cuda(q, k, v, q_lengths, kv_lengths)
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise ValueError("expected q[B,H,Sq,D], k[B,HK,Sk,D], v[B,HK,Sk,D]")
    if k.shape[1] == 0 or q.shape[1] % k.shape[1]:
        raise ValueError("the query heads must be a multiple of the key heads")
    if q.shape[3] != 128:
        raise ValueError("the head dimension must be 128")
    _fits_32_bits(q, k)
    if q.dtype not in (torch.float16, torch.bfloat16) or any(t.dtype != q.dtype for t in (k, v)):
        raise ValueError("q, k, v must share dtype float16 or bfloat16")
    window, sinks = operator.index(window), operator.index(sinks)
    if not 1 <= window:
        raise ValueError("window must be at least 1")
    if not 0 <= sinks <= 128:
        raise ValueError("sinks must be between 0 and 128")
    for n in (q_lengths, kv_lengths):
        if n is not None and (n.dtype != torch.int32 or n.shape != q.shape[:1]):
            raise ValueError("lengths must be int32 [B]")
    for t in (q, k, v):
        if t.numel() and t.stride(3) != 1:
            raise ValueError("the head dimension must be contiguous")
    _one_device(q, k, v, q_lengths, kv_lengths)
    most = 2 ** 31 - 1
    return (min(window, most), sinks, q_lengths.contiguous() if q_lengths is not None else None,
            kv_lengths.contiguous() if kv_lengths is not None else None)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, *, window: int, sinks: int = 0,
                     q_lengths: Optional[torch.Tensor] = None, kv_lengths: Optional[torch.Tensor] = None,
                     return_lse: bool = False, check: bool = False):
    """Causal attention of ``q[B, H, Sq, D]`` over ``k``, ``v`` ``[B, HK, Sk, D]`` (``H`` a multiple of ``HK``, ``D`` contiguous,
    ``D == 128``, fp16 or bf16, batch/head/sequence strides that are positive multiples of 8 elements, the first element on a
    16-byte boundary; other operands are refused, and made dense by ``b200_graph::b200_window_attention``) in which a query
    sees the last ``window`` keys up to its own position and the first ``sinks`` (at most 128) of the sequence.

    ``q_lengths`` and ``kv_lengths`` (int32 ``[B]`` on the device; all of ``Sq`` and ``Sk`` without) are the lengths of
    a padded batch or of what a cache holds: query ``i`` stands at position ``kv_lengths[b] - q_lengths[b] + i``, the
    last query at the last key.  A query that sees nothing, and any behind ``q_lengths[b]``, gets zeros and a
    log-sum-exp of ``-inf``.  What lies behind the lengths may be anything; values of ``v`` before them have to be finite (a NaN
    or an infinity may reach queries that do not see its key, as a weight of 0 times it).  One to a few queries over a long
    cache are a decoding step: only the keys they see are read.

    Returns ``out`` (contiguous ``[B, H, Sq, D]``) or ``(out, lse)``; ``check=True`` as in :func:`fused_attention`."""
    if not check:
        done = _native("ixb_window_attention", _ixb_host.window_attention(q, k, v, scale, window, sinks, q_lengths, kv_lengths, return_lse))
        if done is not None:
            return done
    window, sinks, q_lengths, kv_lengths = _window_arguments(q, k, v, window, sinks, q_lengths, kv_lengths)
    B, H, Sq, D = q.shape
    HK, Sk = k.shape[1], k.shape[2]
    out = torch.empty((B, H, Sq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, H, Sq), dtype=torch.float32, device=q.device) if return_lse else None
    if Sk == 0:  # nothing to see
        out.zero_()
        return (out, lse.fill_(float("-inf"))) if return_lse else out
    status = torch.zeros(1, dtype=torch.int32, device=q.device) if check else None
    with torch.cuda.device(q.device):
        rt.check("ixb_window_attention", rt.load().ixb_window_attention(
            rt.DTYPE_CODE[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), rt.ptr(lse), B, H, HK, Sq, Sk, D, _operand_strides(q), _operand_strides(k), _operand_strides(v), _operand_strides(out),
            rt.ptr(q_lengths), rt.ptr(kv_lengths), float(scale), window, sinks, rt.ptr(status), rt.raw_stream(q.device)))
    if status is not None and int(status.item()) != 0:
        raise RuntimeError("ixb_window_attention: an internal pipeline wait gave up; output is undefined")
    return (out, lse) if return_lse else out


def window_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor, lse: torch.Tensor,
                              dout: torch.Tensor, scale: float, *, window: int, sinks: int = 0,
                              q_lengths: Optional[torch.Tensor] = None, kv_lengths: Optional[torch.Tensor] = None,
                              check: bool = False):
    """Gradients ``(dq, dk, dv)`` of :func:`window_attention` from its inputs, its output ``out``, its log-sum-exp
    ``lse`` (``return_lse=True``) and the incoming gradient ``dout`` (any strides; the others' as there); ``dk`` and ``dv`` are
    sums over the query heads that share a key head, and zero where no query sees the key.  Deterministic, no atomics."""
    if not check:
        done = _native("ixb_window_attention_bwd", _ixb_host.window_attention_backward(
            q, k, v, out, lse, dout, scale, window, sinks, q_lengths, kv_lengths))
        if done is not None:
            return done
    window, sinks, q_lengths, kv_lengths = _window_arguments(q, k, v, window, sinks, q_lengths, kv_lengths)
    _need_cuda(out, lse, dout)
    if out.shape != q.shape or dout.shape != q.shape or out.dtype != q.dtype or dout.dtype != q.dtype:
        raise ValueError("out and dout must have the shape and dtype of q")
    B, H, Sq, D = q.shape
    HK, Sk = k.shape[1], k.shape[2]
    if lse.shape != (B, H, Sq) or lse.dtype != torch.float32:
        raise ValueError("lse must be float32 [B, H, Sq]")
    _one_device(q, out, lse, dout)
    lse = lse.contiguous()
    if not _operand_fits(dout):
        dout = dout.clone(memory_format=torch.contiguous_format)
    if out.numel() and out.stride(3) != 1:
        raise ValueError("the head dimension must be contiguous")
    dq = torch.empty((B, H, Sq, D), dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty((B, HK, Sk, D), dtype=q.dtype, device=q.device) for _ in range(2))
    if q.numel() == 0 or k.numel() == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    status = torch.zeros(1, dtype=torch.int32, device=q.device) if check else None
    lib = rt.load()
    room = lib.ixb_window_attention_bwd_scratch_bytes(B, H, HK, Sq, Sk, window, sinks)
    scratch = torch.empty(room, dtype=torch.uint8, device=q.device)
    like_q, like_k = _operand_strides(dq), _operand_strides(dk)
    with torch.cuda.device(q.device):
        rt.check("ixb_window_attention_bwd", lib.ixb_window_attention_bwd(
            rt.DTYPE_CODE[q.dtype], q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), dout.data_ptr(), lse.data_ptr(),
            dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), scratch.data_ptr(), room, B, H, HK, Sq, Sk, D, _operand_strides(q),
            _operand_strides(k), _operand_strides(v), _operand_strides(out), _operand_strides(dout), like_q, like_k, like_k,
            rt.ptr(q_lengths), rt.ptr(kv_lengths), float(scale), window, sinks, rt.ptr(status), rt.raw_stream(q.device)))
    if status is not None and int(status.item()) != 0:
        raise RuntimeError("ixb_window_attention_bwd: an internal pipeline wait gave up; gradients are undefined")
    return dq, dk, dv


PAIRINGS, LADDERS = ("halves", "neighbours"), ("shared", "own")


# (kept by value: whole numbers and floats only, so that no entry holds a caller's tensor)
@functools.lru_cache(maxsize=256)
def _rotary_plan(sections: tuple, base: float, ladder: str, frequencies: Optional[tuple]):
    """(pairs, axes, ctypes sections, ctypes frequencies in radians a position, their addresses)."""
    pairs = sum(sections)
    if not sections or any(n < 0 for n in sections) or not 1 <= pairs <= 128:
        raise ValueError("sections must be one count of pairs for each axis, 1 to 128 together")
    if frequencies is None:
        if not base > 0:
            raise ValueError("base must be positive")
        powers = [j / n for n in sections for j in range(n)] if ladder == "own" else [i / pairs for i in range(pairs)]
        frequencies = tuple(base ** -p for p in powers)
    if len(frequencies) != pairs:
        raise ValueError("frequencies must be one number for each pair")
    c_sections, c_frequencies = (ctypes.c_int32 * len(sections))(*sections), (ctypes.c_double * pairs)(*frequencies)
    return (pairs, len(sections), c_sections, c_frequencies, ctypes.addressof(c_sections), ctypes.addressof(c_frequencies))


def _rotary_result(t: torch.Tensor) -> torch.Tensor:
    """In the memory order of the input; an expanded or overlapping input's is a dense tensor of its own."""
    like = torch.empty_like(t) if all(t.stride()) else t.new_empty(t.shape)
    return like if t.dim() != 4 or like.stride(3) == 1 else t.new_empty(t.shape)


def _rotary(q, k, positions, sections, base, pairing, ladder, frequencies, inverse):
    if pairing not in PAIRINGS or ladder not in LADDERS:
        raise ValueError(f"pairing must be one of {PAIRINGS}, ladder one of {LADDERS}")
    pairs, axes, c_sections, c_frequencies, *addresses = _rotary_plan(
        tuple(map(operator.index, sections)), float(base), ladder, tuple(map(float, frequencies)) if frequencies is not None else None)
    done = _native("ixb_axial_rotary", _ixb_host.axial_rotary(q, k, positions, pairs, axes, *addresses, pairing == "neighbours", inverse))
    if done is not None:
        return done
    _need_cuda(q, k, positions)
    if q.dtype not in (torch.float32, torch.float16, torch.bfloat16) or (k is not None and k.dtype != q.dtype):
        raise ValueError("q and k must share dtype float32, float16 or bfloat16")
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[2:] != q.shape[2:])):
        raise ValueError("expected q[B,H,S,D], k[B,HK,S,D]")
    B, H, S, D = q.shape
    _fits_32_bits(q, k)
    if 2 * pairs > D:
        raise ValueError("the sections turn more than the head dimension has")
    if positions.dtype not in (torch.int64, torch.int32) or positions.shape not in ((axes, B, S), (axes, S)):
        raise ValueError("positions must be int32 or int64 [axes, B, S] or [axes, S]")
    if any(t is not None and t.numel() and t.stride(3) != 1 for t in (q, k)):
        raise ValueError("the head dimension must be contiguous")
    _one_device(q, k, positions)
    at = positions.stride() if positions.dim() == 3 else (positions.stride(0), 0, positions.stride(1))
    q_out, k_out = _rotary_result(q), None if k is None else _rotary_result(k)
    strides = lambda t: _I64x3(*t.stride()[:3]) if t is not None else None  # noqa: E731
    if q.numel() or (k is not None and k.numel()):
        with torch.cuda.device(q.device):
            rt.check("ixb_axial_rotary", rt.load().ixb_axial_rotary(
                rt.DTYPE_CODE[q.dtype], q.data_ptr(), q_out.data_ptr(), strides(q), strides(q_out), H, rt.ptr(k), rt.ptr(k_out),
                strides(k), strides(k_out), k.shape[1] if k is not None else 0, positions.data_ptr(),
                rt.DTYPE_CODE[positions.dtype], _I64x3(*at), B, S, D, axes, c_sections, c_frequencies,
                int(pairing == "neighbours"), int(inverse), rt.raw_stream(q.device)))
    return q_out if k is None else (q_out, k_out)


def axial_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, sections: Sequence[int], *,
                 base: float = 10000.0, pairing: str = "halves", ladder: str = "shared",
                 frequencies: Optional[Sequence[float]] = None):
    """Rotary positions with one or several axes (time, height, width) on ``q[B, H, S, D]`` and ``k[B, HK, S, D]`` (any
    batch/head/sequence strides, ``D`` contiguous; fp32, fp16 or bf16; ``k`` may be None).

    ``positions`` (int32 or int64) is ``[axes, B, S]`` or, the same for every sequence, ``[axes, S]``;
    ``sections`` says how many pairs each axis turns, in order.  Pair ``i`` is turned by its axis' position times its
    frequency: ``base ** -(i / pairs)`` along one ladder over all pairs (``ladder="shared"``), ``base ** -(j / n)`` for
    pair ``j`` of an axis of ``n`` (``"own"``), or ``frequencies[i]``.  ``pairing="halves"`` pairs ``i`` with ``i +
    pairs``, ``"neighbours"`` ``2 i`` with ``2 i + 1``.  What lies behind the pairs is copied.  Angles are formed in 64
    bits, so that far positions keep their fraction of a turn.

    Returns the turned ``(q, k)``, or ``q`` alone where ``k`` is None, in the memory order of the inputs."""
    return _rotary(q, k, positions, sections, base, pairing, ladder, frequencies, False)


def axial_rotary_backward(dq: torch.Tensor, dk: Optional[torch.Tensor], positions: torch.Tensor, sections: Sequence[int], *,
                          base: float = 10000.0, pairing: str = "halves", ladder: str = "shared",
                          frequencies: Optional[Sequence[float]] = None):
    """Gradients of :func:`axial_rotary` for its ``q`` and ``k`` from those of its results: the same turns the other
    way."""
    return _rotary(dq, dk, positions, sections, base, pairing, ladder, frequencies, True)


# ---- context-parallel attention merge ----------------------------------------------------
def _stat_nstride(t: torch.Tensor, S: int) -> int:
    """Element stride of the N axis of a ``[B, N, S, 8]`` statistics tensor whose last two
    axes are dense and whose B axis is ``N`` times the N stride (a slice along S of a longer
    buffer qualifies)."""
    B, N = t.shape[0], t.shape[1]
    if t.stride(3) != 1 or t.stride(2) != 8 or (B > 1 and t.stride(0) != N * t.stride(1)):
        raise ValueError("statistics must be [B, N, S, 8] with dense trailing axes")
    return t.stride(1) if N > 1 else S * 8


def forward_update(prev_attn_out: torch.Tensor, prev_softmax_max: torch.Tensor,
                   prev_softmax_sum: torch.Tensor, cur_attn_out: torch.Tensor,
                   cur_softmax_max: torch.Tensor, cur_softmax_sum: torch.Tensor):
    """Merge the attention result of one ring step into the running result, (max, sum) form.
    Same name, arguments and return value ``(attn_out, softmax_max, softmax_sum)`` as the
    reference's ``forward_update`` / ``forward_update_triton``
    (``test/npu_indexing/attn_cp_test.py:36-59``,
    ``test/npu_indexing/written/attn_cp_triton_kernel_3d.py:85-140``): attention outputs are
    ``[S, B, H]``, statistics ``[B, N, S, 8]`` fp32."""
    _need_cuda(prev_attn_out, prev_softmax_max, prev_softmax_sum, cur_attn_out, cur_softmax_max, cur_softmax_sum)
    S, B, H = cur_attn_out.shape
    N = cur_softmax_max.shape[1]
    if prev_attn_out.shape != cur_attn_out.shape or prev_attn_out.dtype != cur_attn_out.dtype:
        raise ValueError("prev and cur attention outputs must share shape and dtype")
    if H % N != 0:
        raise ValueError("hidden size must be a multiple of the number of heads")
    for t in (prev_softmax_max, prev_softmax_sum, cur_softmax_max, cur_softmax_sum):
        if t.dtype != torch.float32 or tuple(t.shape) != (B, N, S, 8):
            raise ValueError("statistics must be fp32 [B, N, S, 8]")
    if not (prev_attn_out.is_contiguous() and cur_attn_out.is_contiguous()):
        raise ValueError("attention outputs must be contiguous [S, B, H]")
    pns, cns = _stat_nstride(prev_softmax_max, S), _stat_nstride(cur_softmax_max, S)
    if _stat_nstride(prev_softmax_sum, S) != pns or _stat_nstride(cur_softmax_sum, S) != cns:
        raise ValueError("max and sum of one side must share their layout")
    attn_out = torch.empty_like(cur_attn_out)
    out_max = torch.empty((B, N, S, 8), dtype=torch.float32, device=cur_attn_out.device)
    out_sum = torch.empty_like(out_max)
    rt.check("ixb_cp_forward_update", rt.load().ixb_cp_forward_update(
        rt.DTYPE_CODE[cur_attn_out.dtype], prev_attn_out.data_ptr(), prev_softmax_max.data_ptr(),
        prev_softmax_sum.data_ptr(), cur_attn_out.data_ptr(), cur_softmax_max.data_ptr(),
        cur_softmax_sum.data_ptr(), attn_out.data_ptr(), out_max.data_ptr(), out_sum.data_ptr(),
        S, B, N, H // N, pns, cns, S * 8, rt.raw_stream(cur_attn_out.device)))
    return attn_out, out_max, out_sum


def forward_update_la(prev_attn_out: torch.Tensor, prev_softmax_log_max_sum: torch.Tensor,
                      cur_attn_out: torch.Tensor, cur_softmax_log_max_sum: torch.Tensor) -> None:
    """Log-sum-exp form of the ring merge, in place on ``prev_attn_out`` ``[B, N, S, D]`` fp32
    and ``prev_softmax_log_max_sum`` ``[B, N, S]`` fp32 (the reference's
    ``forward_update_triton`` of ``test/npu_indexing/written/attn_cp_triton_kernel_3d_la.py:58-96``)."""
    _need_cuda(prev_attn_out, prev_softmax_log_max_sum, cur_attn_out, cur_softmax_log_max_sum)
    B, N, S, D = cur_attn_out.shape
    for a in (prev_attn_out, cur_attn_out):
        if a.dtype != torch.float32 or tuple(a.shape) != (B, N, S, D) or a.stride(3) != 1 or a.stride(2) != D \
                or (B > 1 and a.stride(0) != N * a.stride(1)):
            raise ValueError("attention outputs must be fp32 [B, N, S, D] with dense trailing axes")
    for l in (prev_softmax_log_max_sum, cur_softmax_log_max_sum):
        if l.dtype != torch.float32 or tuple(l.shape) != (B, N, S) or l.stride(2) != 1 \
                or (B > 1 and l.stride(0) != N * l.stride(1)):
            raise ValueError("log-sum-exp tensors must be fp32 [B, N, S] with a dense S axis")
    ns = lambda t, dense: t.stride(1) if N > 1 else dense
    rt.check("ixb_cp_forward_update_lse", rt.load().ixb_cp_forward_update_lse(
        prev_attn_out.data_ptr(), prev_softmax_log_max_sum.data_ptr(), cur_attn_out.data_ptr(),
        cur_softmax_log_max_sum.data_ptr(), B, N, S, D, ns(prev_attn_out, S * D),
        ns(prev_softmax_log_max_sum, S), ns(cur_attn_out, S * D), ns(cur_softmax_log_max_sum, S),
        rt.raw_stream(cur_attn_out.device)))


def grad_accumulate(acc: torch.Tensor, cur: torch.Tensor) -> torch.Tensor:
    """``acc.add_(cur.view(acc.shape))`` for dense tensors: the gradient accumulation steps of
    the reference's ring backward (``backward_update``,
    ``test/npu_indexing/written/test_attn_cp.py:267-287``)."""
    _need_cuda(acc, cur)
    if acc.dtype != cur.dtype or acc.numel() != cur.numel() or not (acc.is_contiguous() and cur.is_contiguous()):
        raise ValueError("acc and cur must be dense tensors of one dtype and size")
    rt.check("ixb_cp_accumulate", rt.load().ixb_cp_accumulate(
        rt.DTYPE_CODE[acc.dtype], acc.data_ptr(), cur.data_ptr(), acc.numel(), rt.raw_stream(acc.device)))
    return acc
