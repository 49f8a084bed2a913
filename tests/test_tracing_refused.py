"""Tracing records torch's own operators only, so a traced call of these would be lost: each
entry point refuses it before its kernel is called (no GPU is needed for that)."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import checkers_amd as ck
from checkers_amd import kv


class _Gpu:
    """Calls that pass their checks up to the stream's handle on CPU tensors."""
    n_tokens, n_heads, head_dim, _device = 5, 2, 8, -1
    _p = _streams = k_scale = None


@pytest.fixture
def calls(monkeypatch):
    def called(*a):
        raise AssertionError("a kernel was called")

    class Lib:
        def __getattr__(self, name):
            return called
    monkeypatch.setattr(kv, "lib", lambda: Lib())
    monkeypatch.setattr(kv, "_rows", lambda t, *a: t.stride()[:2])
    monkeypatch.setattr(kv, "_row_stride", lambda t, *a: t.stride(0))
    monkeypatch.setattr(kv, "_new", lambda shape, dtype, device, stream: torch.empty(shape, dtype=dtype))
    _Gpu.k = torch.zeros(1)
    rot = object.__new__(ck.Rotary)
    rot._device, rot._streams = -1, ()
    plan = object.__new__(ck.KvAttention)
    plan.n_heads, plan._streams = 2, ()
    at = torch.zeros(5, dtype=torch.int32)
    return {
        "rotary": lambda x: ck.rotary(rot, at, x),
        "gradient": lambda x: torch.autograd.grad(ck.rotary(rot, at, x.detach().requires_grad_()).sum(), x),
        "kv_write": lambda x: ck.kv_write(_Gpu, _Gpu, x, x),
        "kv_append": lambda x: ck.kv_append(_Gpu, _Gpu, None, x, x, q=x),
        "kv_read": lambda x: ck.kv_read(_Gpu, _Gpu, ck.F32, out=(x, x)),
        "attention": lambda x: plan.run(_Gpu, _Gpu, x),
    }


NAMES = ("rotary", "gradient", "kv_write", "kv_append", "kv_read", "attention")


@pytest.mark.parametrize("name", NAMES)
def test_refused(calls, name):
    x = torch.randn(5, 2, 8)
    with pytest.raises(ck.CkrError, match="tracing"):
        torch.jit.trace(calls[name], x, check_trace=False)
    with pytest.raises(ck.CkrError, match="tracing"):
        make_fx(calls[name])(x)
    with pytest.raises(ck.CkrError, match="tracing"):
        make_fx(calls[name], pre_dispatch=True)(x)


def test_a_norm_is_refused_too(calls, monkeypatch):
    w = torch.ones(8)
    monkeypatch.setattr(torch.Tensor, "is_cuda", True)
    with pytest.raises(ck.CkrError, match="tracing"):
        torch.jit.trace(lambda x: ck.add_rms_norm(x, None, w)[0], torch.randn(5, 8), check_trace=False)


def test_modes_that_record_nothing_are_no_tracing(calls):
    """A mode that only looks on (here: counts operations) leaves calls alone."""
    from torch.utils.flop_counter import FlopCounterMode
    class Stream:
        cuda_stream = 7
    with FlopCounterMode(display=False):
        assert kv._stream_of(Stream, None) == 7
    with torch.device("cpu"):
        assert kv._stream_of(Stream, None) == 7
        with pytest.raises(ck.CkrError, match="tracing"):
            make_fx(lambda x: kv._stream_of(Stream, None) + x, pre_dispatch=True)(torch.zeros(1))
    assert kv._stream_of(Stream, None) == 7
