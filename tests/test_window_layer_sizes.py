"""Sizes beyond what the entries of the windowed decoder layer's operators count in: refused, without a GPU."""
import ctypes

import pytest
import torch

from inductor_x_b200 import ops
from inductor_x_b200 import runtime as rt


@pytest.fixture
def no_device(monkeypatch):
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(rt, "check", lambda *a: pytest.fail("a call that had to be refused was made"))


def view(*shape, dtype=torch.float16):
    """One value seen everywhere."""
    return torch.empty(1, dtype=dtype, device="meta").expand(*shape)


LONG = 2 ** 32 + 1  # one, in 32 bits


@pytest.mark.parametrize("shape", [(1, 1, LONG, 2), (1, LONG, 1, 2), (LONG, 1, 1, 2), (1, 1, 1, LONG)])
def test_rotary_axes(no_device, shape):
    q, p = view(*shape[:3], 1).expand(shape).as_strided(shape, (0, 0, 0, 1)), view(1, shape[0], shape[2], dtype=torch.int64)
    with pytest.raises(ValueError, match="entries"):
        ops.axial_rotary(q, None, p, [1])
    if shape[1] != 1:
        with pytest.raises(ValueError, match="entries"):
            ops.axial_rotary(q[:, :1], q, p, [1])


def test_attention_axes(no_device):
    q, k = view(1, 1, 4, 128).as_strided((1, 1, 4, 128), (512, 512, 128, 1)), view(1, 1, LONG, 128).as_strided((1, 1, LONG, 128), (8, 8, 8, 1))
    with pytest.raises(ValueError, match="entries"):
        ops.window_attention(q, k, k, 0.1, window=4)
    with pytest.raises(ValueError, match="entries"):
        ops.window_attention(k, q, q, 0.1, window=4)


@pytest.mark.parametrize("heads,k_heads,D,status", [
    (1 << 20, 0, 4096, rt.IXB_ERR_SHAPE), (1, 1 << 22, 1024, rt.IXB_ERR_SHAPE), ((1 << 31) - 1, (1 << 31) - 1, 2, rt.IXB_ERR_SHAPE),
    ((1 << 29) + 1, 0, 2, rt.IXB_ERR_SHAPE), (0, 0, 2, rt.IXB_OK)])
def test_values_of_a_token(heads, k_heads, D, status):
    S = (ctypes.c_int64 * 3)(0, 0, 0)
    assert rt.load().ixb_axial_rotary(rt.IXB_F16, 16, 16, S, S, heads, 16, 16, S, S, k_heads, 16, rt.IXB_I64, S, 1, 1, D, 1,
                                      (ctypes.c_int32 * 1)(1), (ctypes.c_double * 1)(1.0), 0, 0, None) == status
