"""What the operators of a decoder layer with a sliding window refuse, without a GPU: meta tensors with the look of CUDA
ones, and the C entries with arguments that are wrong before any device is asked."""
import ctypes

import pytest
import torch

from inductor_x_b200 import ops
from inductor_x_b200 import runtime as rt


@pytest.fixture
def no_device(monkeypatch):
    """Every tensor passes for one of the device; no call may get as far as the library."""
    monkeypatch.setattr(ops, "_need_cuda", lambda *ts: None)
    monkeypatch.setattr(rt, "check", lambda *a: pytest.fail("a call that had to be refused was made"))
    monkeypatch.setattr(rt, "load", lambda: pytest.fail("a call that had to be refused was made"))


def t(*shape, dtype=torch.float16):
    return torch.empty(*shape, dtype=dtype)


Q, K = t(2, 4, 8, 128), t(2, 2, 16, 128)
N = torch.zeros(2, dtype=torch.int32)
WRONG_ATTENTION = [
    dict(q=t(2, 4, 8)),
    dict(q=t(3, 4, 8, 128)),
    dict(q=t(2, 3, 8, 128)),                                 # 3 query heads, 2 key heads
    dict(q=t(2, 4, 8, 64), k=t(2, 2, 16, 64), v=t(2, 2, 16, 64)),
    dict(k=t(2, 2, 17, 128)),
    dict(k=t(2, 0, 16, 128), v=t(2, 0, 16, 128)),
    dict(q=Q.float(), k=K.float(), v=K.float()),
    dict(v=K.bfloat16()),
    dict(q=t(2, 4, 128, 8).transpose(2, 3)),
    dict(window=0),
    dict(window=4.5),
    dict(sinks=1.0),
    dict(window=-5),
    dict(sinks=-1),
    dict(sinks=129),
    dict(q_lengths=N.long()),
    dict(kv_lengths=N[:1]),
    dict(kv_lengths=N[None]),
]


@pytest.mark.parametrize("wrong", WRONG_ATTENTION)
def test_attention(no_device, wrong):
    args = dict(q=Q, k=K, v=K, scale=0.1, window=4) | wrong
    with pytest.raises((ValueError, TypeError)):
        ops.window_attention(**args)
    q = args["q"]
    with pytest.raises((ValueError, TypeError)):
        ops.window_attention_backward(out=torch.empty_like(q), lse=t(*q.shape[:3], dtype=torch.float32),
                                      dout=torch.empty_like(q), **args)


@pytest.mark.parametrize("wrong", [dict(out=t(2, 4, 7, 128)), dict(dout=Q.bfloat16()), dict(lse=t(2, 4, 8)),
                                   dict(lse=t(2, 4, 8, 1, dtype=torch.float32)), dict(out=t(2, 4, 128, 8).transpose(2, 3))])
def test_attention_backward(no_device, wrong):
    args = dict(out=Q, lse=t(2, 4, 8, dtype=torch.float32), dout=Q) | wrong
    with pytest.raises(ValueError):
        ops.window_attention_backward(Q, K, K, scale=0.1, window=4, **args)


P = torch.zeros(2, 2, 8, dtype=torch.int64)
WRONG_ROTARY = [
    dict(sections=[]), dict(sections=[0, 0]), dict(sections=[65, 0]), dict(sections=[-1, 3]), dict(sections=[32]),
    dict(sections=[100, 29]), dict(positions=P.float()), dict(positions=P[:, :1]), dict(positions=P[0]),
    dict(pairing="thirds"), dict(ladder="rope"), dict(base=0.0), dict(frequencies=[1.0]), dict(q=t(2, 4, 8)),
    dict(k=t(2, 2, 9, 128)), dict(k=K[:, :, :8].float()), dict(q=Q.double()), dict(q=t(2, 4, 128, 8).transpose(2, 3)),
]


@pytest.mark.parametrize("wrong", WRONG_ROTARY)
def test_rotary(no_device, wrong):
    args = dict(q=Q, k=K[:, :, :8], positions=P, sections=[32, 32]) | wrong
    with pytest.raises(ValueError):
        ops.axial_rotary(**args)
    args["dq"], args["dk"] = args.pop("q"), args.pop("k")
    with pytest.raises(ValueError):
        ops.axial_rotary_backward(**args)


X = t(4, 256)
WRONG_NORM = [dict(group=64), dict(group=-1), dict(x=X.double()), dict(x=X.t()), dict(w=t(255)), dict(w=t(256, dtype=torch.float32)),
              dict(residual=t(4, 255)), dict(residual=X.float()), dict(residual=t(256, 4).t())]


@pytest.mark.parametrize("wrong", WRONG_NORM)
def test_norm(no_device, wrong):
    args = dict(x=X, w=t(256)) | wrong
    with pytest.raises(ValueError):
        ops.rmsnorm_quantised(**args)


def test_host_memory():
    with pytest.raises(ValueError):
        ops.window_attention(Q, K, K, 0.1, window=4)
    with pytest.raises(ValueError):
        ops.axial_rotary(Q, None, P, [32, 32])
    with pytest.raises(ValueError):
        ops.rmsnorm_quantised(X, t(256))


def attention_status(**other):
    S = ctypes.c_int64 * 3
    a = dict(dtype=rt.IXB_F16, q=1 << 20, k=1 << 20, v=1 << 20, o=1 << 20, B=1, H=4, HK=2, Sq=8, Sk=16, D=128, strides=S(8192, 1024, 128),
             scale=0.1, window=4, sinks=0) | other
    s = a["strides"]
    return rt.load().ixb_window_attention(a["dtype"], a["q"], a["k"], a["v"], a["o"], None, a["B"], a["H"], a["HK"], a["Sq"],
                                          a["Sk"], a["D"], s, s, s, s, None, None, a["scale"], a["window"], a["sinks"], None, None)


@pytest.mark.parametrize("status,other", [
    (rt.IXB_ERR_ARG, dict(q=None)), (rt.IXB_ERR_ARG, dict(o=None)), (rt.IXB_ERR_ARG, dict(B=-1)), (rt.IXB_ERR_ARG, dict(window=0)),
    (rt.IXB_ERR_ARG, dict(sinks=-1)), (rt.IXB_ERR_ARG, dict(scale=0.0)), (rt.IXB_ERR_ARG, dict(scale=float("nan"))),
    (rt.IXB_ERR_ARG, dict(scale=float("inf"))), (rt.IXB_ERR_DTYPE, dict(dtype=rt.IXB_F32)), (rt.IXB_ERR_SHAPE, dict(D=64)),
    (rt.IXB_ERR_SHAPE, dict(HK=3)), (rt.IXB_ERR_SHAPE, dict(sinks=129)), (rt.IXB_ERR_SHAPE, dict(Sk=0)),
    (rt.IXB_ERR_ALIGN, dict(k=(1 << 20) + 8)), (rt.IXB_ERR_ALIGN, dict(strides=(ctypes.c_int64 * 3)(8192, 1024, 132))),
    (rt.IXB_ERR_ALIGN, dict(strides=(ctypes.c_int64 * 3)(8192, 0, 128))), (rt.IXB_OK, dict(B=0)), (rt.IXB_OK, dict(Sq=0)),
])
def test_attention_entry(status, other):
    assert attention_status(**other) == status


def test_other_entries():
    lib = rt.load()
    S = (ctypes.c_int64 * 3)(8192, 1024, 128)
    back = lambda scratch, room, Sk=16: lib.ixb_window_attention_bwd(  # noqa: E731
        rt.IXB_F16, *[1 << 20] * 5, 1 << 20, *[1 << 20] * 3, scratch, room, 1, 4, 2, 8, Sk, 128, S, S, S, S, S, S, S, S, None, None,
        0.1, 4, 0, None, None)
    need = lib.ixb_window_attention_bwd_scratch_bytes(1, 4, 2, 8, 16, 4, 0)
    assert need > 0 and back(None, need) == rt.IXB_ERR_SCRATCH and back(1 << 20, need - 1) == rt.IXB_ERR_SCRATCH
    assert back((1 << 20) + 4, need) == rt.IXB_ERR_ALIGN and back(1 << 20, need, 0) == rt.IXB_ERR_SHAPE
    assert lib.ixb_window_attention_bwd_scratch_bytes(0, 4, 2, 8, 16, 4, 0) == 0
    turn = lambda dtype, sections, D=128, positions=1, kind=rt.IXB_I64, q=1: lib.ixb_axial_rotary(  # noqa: E731
        dtype, q, 1, S, S, 4, None, None, None, None, 0, positions, kind, S, 1, 8, D, len(sections), (ctypes.c_int32 * len(sections))(*sections),
        (ctypes.c_double * 256)(), 0, 0, None)
    assert turn(rt.IXB_F16, [65]) == rt.IXB_ERR_SHAPE and turn(rt.IXB_F16, [100, 100], 512) == rt.IXB_ERR_SHAPE
    assert turn(rt.IXB_F16, [-1]) == rt.IXB_ERR_ARG and turn(rt.IXB_I64, [64]) == rt.IXB_ERR_DTYPE
    assert turn(rt.IXB_F16, [64], positions=None) == rt.IXB_ERR_ARG and turn(rt.IXB_F16, [64], kind=rt.IXB_F32) == rt.IXB_ERR_DTYPE
    assert turn(rt.IXB_F16, [64], q=None) == rt.IXB_ERR_ARG
    norm = lambda dtype=rt.IXB_F16, x=1, res=None, h=None, rows=4, cols=256, group=0: lib.ixb_rmsnorm_quantised(  # noqa: E731
        dtype, x, res, 1, 1, 1, h, rows, cols, group, 1e-6, None)
    assert norm(x=None) == rt.IXB_ERR_ARG and norm(h=1) == rt.IXB_ERR_ARG and norm(group=64) == rt.IXB_ERR_ARG
    assert norm(rows=-1) == rt.IXB_ERR_ARG and norm(cols=0) == rt.IXB_ERR_ARG and norm(rows=0, x=None) == rt.IXB_OK
    assert norm(cols=1 << 21) == rt.IXB_ERR_SHAPE and norm(dtype=rt.IXB_I64) == rt.IXB_ERR_DTYPE


@pytest.mark.parametrize("group", [0, 128])
def test_norm_of_rows_without_values(no_device, group):
    with pytest.raises(ValueError):
        ops.rmsnorm_quantised(t(4, 0), t(0), group=group)
