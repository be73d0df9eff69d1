"""The operators of a windowed decoder layer called from native code (csrc/host_launch.cpp): the same results and errors as
the Python functions they stand in for, which take every call that is out of the ordinary."""
import types

import pytest
import torch

from inductor_x_b200 import _ixb_host, ops
from inductor_x_b200 import runtime as rt

NAMES = ("rms_norm_quantised", "axial_rotary", "window_attention", "window_attention_backward")


def test_what_is_out_of_the_ordinary_is_left_to_python():
    rt.load()
    x, w = torch.ones(4, 256), torch.ones(256)
    assert _ixb_host.rms_norm_quantised(x, w, 1e-6, None, False, 0) is None                 # host memory
    assert _ixb_host.rms_norm_quantised(x, w, 1e-6, None, False) is None
    assert _ixb_host.rms_norm_quantised(None, w, 1e-6, None, False, 1 << 80) is None
    m = torch.empty(2, 2, 4, 128, device="meta", dtype=torch.float16)                       # no memory
    assert _ixb_host.window_attention(m, m, m, 1.0, 4, 0, None, None, True) is None
    assert _ixb_host.window_attention(m, m, m, 1.0, -4, 1 << 70, None, None, True) is None
    assert _ixb_host.window_attention_backward(m, m, m, m, m, m, 1.0, 4, 0, None, None) is None
    assert _ixb_host.axial_rotary(m, None, m, 64, 1, 0, 0, False, False) is None
    assert _ixb_host.axial_rotary(m, None, m, 64, 1, -1, "x", False, False) is None
    with pytest.raises(TypeError):
        _ixb_host.bind_library(1, 2, 3, 4)


def _both(monkeypatch, call):
    """Results of the native route (which is checked to be the one taken) and of the Python route."""
    counts = rt.native_calls
    with monkeypatch.context() as m:
        m.setattr(rt, "check", lambda *a: pytest.fail("the Python route was taken"))
        native = call()
    assert rt.native_calls == counts + 1
    with monkeypatch.context() as m:
        m.setattr(ops, "_ixb_host", types.SimpleNamespace(**{n: lambda *a: None for n in NAMES}))
        python = call()
    assert rt.native_calls == counts + 2
    native, python = (r if isinstance(r, tuple) else (r,) for r in (native, python))
    assert len(native) == len(python)
    for a, b in zip(native, python):
        assert a.shape == b.shape and a.stride() == b.stride() and a.dtype == b.dtype and not a.requires_grad
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(16, 4096), (3, 161), (2, 3, 64)])
def test_norm(cuda, monkeypatch, dtype, shape):
    rt.load()
    x, r = (torch.randn(*shape, device=cuda).to(dtype) for _ in range(2))
    w = torch.nn.Parameter(torch.randn(shape[-1], device=cuda).to(dtype))
    for group in (0, 128):
        _both(monkeypatch, lambda: ops.rmsnorm_quantised(x, w, 1e-5, group=group))
        _both(monkeypatch, lambda: ops.rmsnorm_quantised(x, w, 1e-5, residual=r, group=group))
        _both(monkeypatch, lambda: ops.rmsnorm_quantised(x, w, 1e-5, residual=r, return_residual=True, group=group))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rotary(cuda, monkeypatch, dtype):
    rt.load()
    q, k = (torch.randn(2, 9, h, 64, device=cuda).to(dtype).transpose(1, 2) for h in (4, 2))
    for positions in (torch.randint(0, 99, (2, 2, 9), device=cuda), torch.randint(0, 99, (2, 9), device=cuda).int()):
        for call in (ops.axial_rotary, ops.axial_rotary_backward):
            _both(monkeypatch, lambda: call(q, k, positions, [10, 22]))
            _both(monkeypatch, lambda: call(q, None, positions, (16, 8), pairing="neighbours", ladder="own", base=5e5))


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [1, 70])
def test_attention(cuda, monkeypatch, queries):
    rt.load()
    make = lambda s, h: torch.randn(2, s, h, 128, device=cuda).half().transpose(1, 2)  # noqa: E731
    q, k, v, g = make(queries, 4), make(200, 2), make(200, 2), make(queries, 4)
    ql, kl = (torch.tensor(n, dtype=torch.int32, device=cuda) for n in ([queries, 1], [200, 77]))
    for how in (dict(window=40), dict(window=1 << 40, sinks=3, kv_lengths=kl), dict(window=30, sinks=7, q_lengths=ql, kv_lengths=kl)):
        _both(monkeypatch, lambda: ops.window_attention(q, k, v, 0.1, **how))
        _both(monkeypatch, lambda: ops.window_attention(q, k, v, 0.1, return_lse=True, **how))
        out, lse = ops.window_attention(q, k, v, 0.1, return_lse=True, **how)
        _both(monkeypatch, lambda: ops.window_attention_backward(q, k, v, out, lse, g, 0.1, **how))


@pytest.mark.gpu
def test_errors_of_the_library_are_raised(cuda):
    rt.load()
    q = torch.randn(1, 2, 8, 128, device=cuda).half()
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(rt.IxbError):
            ops.window_attention(q, q, q, scale, window=4)
    off = torch.randn(2 * 8 * 128 + 4, device=cuda).half()[4:].view(1, 2, 8, 128)
    with pytest.raises(rt.IxbError):
        ops.window_attention(q, off, q, 0.1, window=4)
    with pytest.raises(rt.IxbError):
        ops.window_attention(q.expand(3, 2, 8, 128), q.expand(3, 2, 8, 128), q.expand(3, 2, 8, 128), 0.1, window=4)
    with pytest.raises(rt.IxbError):
        ops.axial_rotary(q, None, torch.zeros(1, 8, dtype=torch.int64, device=cuda), [64], frequencies=[float("nan")] * 64)
