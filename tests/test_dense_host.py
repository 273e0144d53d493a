"""Host side of the dense operators and the router's gate: what is refused before any device is touched."""

import ctypes

import pytest
import torch

import cudnn_frontend_b200 as cf
from cudnn_frontend_b200 import _lib


def _args(**kw):
    a = dict(x=4096, w0=4096, w1=4096, y=4096, dy=4096, pre0=4096, pre1=4096, m=4, n=24, k=64, ld_x=64, ld_w0=64, ld_w1=64, ld_dy=24, ld_y=24, ld_pre0=24,
             ld_pre1=24, act=_lib.ACT_SWIGLU)  # fmt: skip
    a.update(kw)
    return ctypes.byref(_lib.DenseArgs(**a))


GATED, LINEAR = ("b200moe_gated_ffn", "b200moe_gated_ffn_backward"), ("b200moe_linear", "b200moe_linear_backward")


@pytest.mark.parametrize("fn", GATED + LINEAR)
@pytest.mark.parametrize(
    "bad,code",
    [
        (dict(k=60), _lib.E_SHAPE),
        (dict(n=0), _lib.E_SHAPE),
        (dict(m=-1), _lib.E_SHAPE),
        (dict(k=0), _lib.E_SHAPE),
        (dict(dtype=_lib.DTYPE_F32), _lib.E_UNSUPPORTED),
        (dict(act=17), _lib.E_UNSUPPORTED),
        (dict(wait_limit_ms=-1), _lib.E_SHAPE),
        (dict(w0=None), _lib.E_NULL),
        (dict(x=None), _lib.E_NULL),
        (dict(x=4104), _lib.E_ALIGN),
        (dict(w0=4098), _lib.E_ALIGN),
        (dict(ld_x=68), _lib.E_ALIGN),
        (dict(ld_x=56), _lib.E_SHAPE),
        (dict(ld_w0=0), _lib.E_SHAPE),
    ],
)
def test_c_abi_refuses_bad_dense_arguments(fn, bad, code):
    if "act" not in bad and fn in LINEAR:
        bad = dict(bad, act=_lib.ACT_SILU)
    assert getattr(_lib.load(), fn)(_args(**bad), None) == code
    assert fn.removeprefix("b200moe_") in _lib.last_error()


def test_c_abi_refuses_bad_router_arguments():
    lib = _lib.load()

    def call(dtype=_lib.DTYPE_F32, rows=4, experts=16, ld=16, topk=2, score=0, logits=4096, weights=4096):
        return lib.b200moe_router_topk(logits, dtype, rows, experts, ld, None, topk, score, 1, 1.0, weights, 4096, None)

    assert call(rows=0) == 0  # nothing to do
    assert call(experts=1025, ld=1025) == call(ld=15) == call(topk=0) == call(topk=17) == call(rows=-1) == _lib.E_SHAPE
    assert call(experts=64, ld=64, topk=33) == _lib.E_SHAPE
    assert call(dtype=_lib.DTYPE_E4M3) == call(score=2) == _lib.E_UNSUPPORTED
    assert call(logits=None) == call(weights=None) == _lib.E_NULL
    back = lib.b200moe_router_topk_backward
    assert back(4096, 4096, _lib.DTYPE_F32, None, 4, 16, 16, 2, 0, 1, 1.0, 4096, None) == _lib.E_NULL
    assert back(4096, 4096, _lib.DTYPE_F32, 4096, 4, 16, 16, 2, 0, 1, 1.0, 4100, None) == _lib.E_ALIGN


def test_workspace_of_the_backward_passes():
    need = _lib.load().b200moe_dense_workspace_bytes
    assert need(0, 100, 1) == need(0, 100, 0) == 0
    assert need(3, 100, 1) == 2 * 768  # two [3, 104] 16-bit buffers, each rounded up to 256 bytes
    assert need(3, 100, 0) >= 768 + 400  # one, and the column sums
    assert need(1 << 20, 1 << 14, 1) == 2 * (1 << 35)  # beyond 32 bits


def test_workspace_holds_the_scale_of_float16_gradients():
    need = _lib.load().b200moe_dense_workspace_bytes
    assert need(3, 100, 1 | _lib.DENSE_WORKSPACE_F16) == 2 * 768 + 256
    assert need(3, 100, _lib.DENSE_WORKSPACE_F16) == need(3, 100, 0) >= 768 + 400 + 256
    assert need(0, 100, 1 | _lib.DENSE_WORKSPACE_F16) == 0


def test_cpu_tensors_and_unknown_names_are_refused():
    x, w = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((24, 64), dtype=torch.bfloat16)
    for call in (
        lambda: cf.gated_ffn(x, w, w),
        lambda: cf.linear(x, w),
        lambda: cf.gated_ffn_backward(x, x, w, w, x, x),
        lambda: cf.linear_backward(x, x, w),
        lambda: cf.router_topk(torch.zeros((4, 8)), 2),
        lambda: cf.router_topk_backward(torch.zeros((4, 2)), torch.zeros((4, 8)), torch.zeros((4, 2), dtype=torch.int32)),
    ):
        with pytest.raises(ValueError):
            call()


def test_new_names_are_public():
    for name in ("gated_ffn", "gated_ffn_backward", "linear", "linear_backward", "router_topk", "router_topk_backward"):
        assert callable(getattr(cf, name)) and name in dir(cf)


def test_an_older_library_of_the_same_version_asks_to_be_rebuilt(monkeypatch):
    """Entry points were added within an ABI version: a library that lacks one is refused by name, before it is called."""

    class Older:
        def __init__(self, path):
            for name in _lib.EXPORTED_SYMBOLS:
                if "gated_ffn" not in name:
                    setattr(self, name, lambda *args: _lib.ABI_VERSION)

    monkeypatch.setattr(_lib, "_lib", None)
    monkeypatch.setattr(_lib.ctypes, "CDLL", Older)
    with pytest.raises(RuntimeError, match="b200moe_gated_ffn.*rebuild the library"):
        _lib.load()


def test_a_stream_of_another_device_is_refused(monkeypatch):
    from cudnn_frontend_b200 import ops

    class Stream:
        device = torch.device("cuda", 1)

    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    with pytest.raises(ValueError, match="stream belongs to cuda:1, the tensors live on cuda:0"):
        ops.call_on(torch.device("cuda", 0), Stream(), lambda s: s)
