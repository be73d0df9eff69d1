"""64-bit definitions of the operators of a decoder layer with a sliding window, and how far results in fewer bits
may be from them.

A bound counts roundings: one to a type of 16 bits is off by at most half a step, ``finfo.eps / 2`` of the value
(2^-25 of nothing smaller in fp16, where values below 2^-14 have a fixed step), and whatever is computed in 32 bits
is given ``SLACK`` of the magnitudes that were summed."""
import math

import torch

#: of sums in 32 bits: the exponent of a probability is off by 2^-24 of arguments up to 50 and by the exponential's own
#: 2^-22, and a sum of n terms by at most n 2^-24 of their magnitudes, n up to 2^6 times a tensor core's blocks
SLACK = 2.0 ** -16


def _lengths(lengths, b, default):
    return default if lengths is None else min(max(int(lengths[b]), 0), default)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _floor(dtype):
    """Half the fixed step of the smallest values."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def window_attention(q, k, v, scale, *, window, sinks=0, q_lengths=None, kv_lengths=None, dout=None):
    """``{"out", "lse"}`` and, with ``dout``, ``{"dq", "dk", "dv"}``: each a pair (value in 64 bits, bound of the error of
    a result in the type of ``q``)."""
    B, H, Sq, D = q.shape
    HK, Sk = k.shape[1], k.shape[2]
    dtype, half, tiny = q.dtype, _half_step(q.dtype), _floor(q.dtype)
    zero = lambda t: torch.zeros(t.shape, dtype=torch.float64, device=t.device)  # noqa: E731
    out, out_e, dq, dq_e = (zero(q) for _ in range(4))
    dk, dk_e, dv, dv_e = (zero(k) for _ in range(4))
    lse = torch.full((B, H, Sq), -math.inf, dtype=torch.float64, device=q.device)
    for b in range(B):
        nq, nk = _lengths(q_lengths, b, Sq), _lengths(kv_lengths, b, Sk)
        if nq == 0 or nk == 0:
            continue
        at = torch.arange(nq, device=q.device)[:, None] + nk - nq
        j = torch.arange(nk, device=q.device)[None]
        seen = (j <= at) & ((j > at - window) | (j < sinks))
        for h in range(H):
            g = h // (H // HK)
            Q, K, V = q[b, h, :nq].double(), k[b, g, :nk].double(), v[b, g, :nk].double()
            S = torch.where(seen, scale * (Q @ K.T), -math.inf)
            L = torch.logsumexp(S, 1)
            some = seen.any(1)
            P = torch.where(seen, torch.exp(S - torch.where(some, L, 0.0)[:, None]), 0.0)
            O = P @ V
            out[b, h, :nq], lse[b, h, :nq] = O, torch.where(some, L, -math.inf)
            # a rounded probability (relative to a maximum that is at most 1, so the sum is at least one half), the result's
            pv = P @ V.abs()
            o_e = half * O.abs() + (half + SLACK) * pv + 2 * tiny * (seen.double() @ V.abs()) + tiny
            out_e[b, h, :nq] = o_e
            if dout is None:
                continue
            G = dout[b, h, :nq].double()
            dP = G @ V.T
            delta = (G * O).sum(1, keepdim=True)
            T = P * (dP - delta)                                     # dS before the scale
            # P and dP in 32 bits; delta from the rounded out; then T is rounded
            d_e = (G.abs() * (o_e + SLACK * O.abs())).sum(1, keepdim=True)
            T_e = half * T.abs() + P * (d_e * (1 + half) + SLACK * (G.abs() @ V.abs().T + delta.abs())) + SLACK * T.abs() + tiny * seen
            dq[b, h, :nq] = scale * (T @ K)
            dq_e[b, h, :nq] = scale * (T_e @ K.abs() + SLACK * (T.abs() @ K.abs()))
            dk[b, g, :nk] += scale * (T.T @ Q)
            dk_e[b, g, :nk] += scale * (T_e.T @ Q.abs() + SLACK * (T.abs().T @ Q.abs()))
            dv[b, g, :nk] += P.T @ G
            dv_e[b, g, :nk] += (half + SLACK) * (P.T @ G.abs()) + tiny * (seen.double().T @ G.abs())
    last = lambda e, x: e * (1 + half) + half * x.abs() + tiny  # noqa: E731  (the result's own rounding)
    lse_e = 2.0 ** -18 * (1 + lse.abs().nan_to_num(posinf=0.0))
    got = {"out": (out, out_e + tiny), "lse": (lse, lse_e)}
    if dout is not None:
        got |= {"dq": (dq, last(dq_e, dq)), "dk": (dk, last(dk_e, dk)), "dv": (dv, last(dv_e, dv))}
    return got


def check(got, expected, name):
    value, bound = expected
    got = got.double()
    same = (got == value)                                            # (infinities)
    far = torch.where(same, 0.0, (got - value).abs()) / torch.where(bound > 0, bound, 1e-300)
    assert not torch.isnan(got).any(), f"{name}: NaN"
    worst = float(far.max()) if far.numel() else 0.0
    assert worst <= 1.0, f"{name}: {worst:.3g} times the bound at {[int(i) for i in (far == far.max()).nonzero()[0]]}"
    return worst


def axial_rotary(x, positions, sections, *, base=10000.0, pairing="halves", ladder="shared", frequencies=None, inverse=False):
    """(value in 64 bits, bound)."""
    pairs = sum(sections)
    y, e = x.double(), torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    i = 0
    for a, n in enumerate(sections):
        for j in range(n):
            f = frequencies[i] if frequencies is not None else base ** -(j / n if ladder == "own" else i / pairs)
            angle = positions[a].double() * f * (-1 if inverse else 1)
            c, s = angle.cos(), angle.sin()
            while c.dim() < 2:
                c, s = c[None], s[None]
            c, s = c[:, None], s[:, None]
            lo, hi = (i, i + pairs) if pairing == "halves" else (2 * i, 2 * i + 1)
            u, w = x[..., lo].double(), x[..., hi].double()
            y[..., lo], y[..., hi] = u * c - w * s, u * s + w * c
            # sine and cosine in 32 bits are 2 steps off at most, products and sum round once each; the angle itself, in
            # 64 bits, is 2^-52 of its size off
            err = (u.abs() + w.abs()) * (6 * 2.0 ** -24 + 2.0 ** -50 * (1 + angle.abs())[:, None])
            e[..., lo] = e[..., hi] = err
            i += 1
    return y, e * 1.01 + _half_step(x.dtype) * y.abs() + _floor(x.dtype)


def rmsnorm_quantised(x, w, eps, residual=None, group=0):
    """``(h, y, scales, rounded)``: the row that is normalised, its norm and the scales in 64 bits."""
    h = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    d = h.double()
    y = d * torch.rsqrt(d.square().mean(-1, keepdim=True) + eps) * w.double()
    cols = y.shape[-1]
    parts = y.split(group or cols, dim=-1)
    scales = torch.stack([p.abs().amax(-1) / 448 for p in parts], -1)
    wide = torch.cat([s[..., None].expand(p.shape) for s, p in zip(scales.unbind(-1), parts)], -1)
    return h, y, scales if group else scales[..., 0], wide
