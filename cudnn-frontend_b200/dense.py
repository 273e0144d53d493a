"""Dense 16-bit operators that stand next to the grouped GEMMs of an MoE layer.

``gated_ffn`` is the block of a shared (or dense) expert, the counterpart of the grouped FC1
(:mod:`.grouped_gemm_glu`) for weights that every token passes: both projections, the activation and the
product in one kernel.  ``linear`` is the projection behind it or the router's, with bias, activation and
residual in its epilogue.  Both have their backward pass.  The reference has no counterpart.

All functions take bf16 or fp16 tensors ``[rows, cols]`` with contiguous rows (any pitch that is a multiple
of 8 elements, 16-byte aligned, for what a tensor map reads: ``x`` and the weights) and sum in float32.  The forward
functions round their results once; the backward functions round twice, the gradient operand that both products share and
the results.  They allocate their outputs and launch on ``stream`` (default: the current stream of the tensors' device); when
another stream is passed, outputs and workspace belong to that stream, and inputs must stay alive until it has passed the
call.  They are not recorded by autograd: the backward functions are called explicitly, as with the grouped GEMMs.
While ``torch.compile`` traces, the forward functions go through custom ops (``torch.ops.b200moe.gated_ffn`` and ``linear``),
so the graph sees one opaque op per launch.
"""

from __future__ import annotations

import ctypes
from typing import List, Optional, Tuple

import torch

from . import _lib
from .ops import _ptr, call_on

_TYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
_GLU = {"swiglu": _lib.ACT_SWIGLU, "geglu": _lib.ACT_GEGLU}
_ACT = {None: _lib.ACT_NONE, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU, "gelu": _lib.ACT_GELU}


def _check_x(x: torch.Tensor) -> Tuple[int, int]:
    if not x.is_cuda:
        raise ValueError("all tensors must live on a CUDA device")
    if x.dtype not in _TYPES:
        raise NotImplementedError(f"x dtype {x.dtype} is not built (bf16 and fp16 are)")
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"x must be a 2-D tensor [tokens, k], got shape {tuple(shape)}")
    return shape


def _pitch(name: str, t: torch.Tensor, shape, dtype, device) -> int:
    """Row pitch of a ``shape`` tensor with contiguous rows."""
    if t.dtype is dtype and t.shape == shape and t.device == device and t.is_contiguous():  # (the usual case, in few steps)
        return shape[1] if shape[0] > 1 else (shape[1] + 7) // 8 * 8
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} lives on {t.device}, x on {device}")
    rows, cols = shape
    pitch, step = t.stride()
    if step != 1 and cols > 1 and rows > 0:
        raise ValueError(f"{name} must have contiguous rows")
    # the pitch of a single row is free: the next multiple of 8
    return pitch if rows > 1 else (cols + 7) // 8 * 8


def _like(t: torch.Tensor) -> torch.Tensor:
    """A dense tensor of t's shape and type."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _weight(name: str, w: torch.Tensor, k: int, x: torch.Tensor) -> int:
    shape = w.shape
    if len(shape) != 2 or shape[1] != k:
        raise ValueError(f"{name} must have shape [n, {k}], got {tuple(shape)}")
    return _pitch(name, w, shape, x.dtype, x.device)


def _eager_stream_only(stream) -> None:
    if stream is not None:
        raise NotImplementedError("stream is an eager-only launch option")


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, act_func: str = "swiglu", return_preact: bool = False, stream=None):
    """``act(x w_gate^T) * (x w_up^T)``: ``x [tokens, k]``, weights ``[n, k]`` -> ``h [tokens, n]``, and with
    ``return_preact`` also ``gate`` and ``up`` (what :func:`gated_ffn_backward` reads).

    ``act_func`` as in the grouped FC1: ``"swiglu"`` = ``gate * sigmoid(gate) * up``, ``"geglu"`` = the reference's
    GeGLU, ``gate <= 7``, ``-7 <= up <= 7``, ``(up + 1) * gate * sigmoid(1.702 * gate)`` (gate and up are returned
    without the limits)."""
    if torch.compiler.is_compiling():
        _eager_stream_only(stream)
        out = torch.ops.b200moe.gated_ffn(x, w_gate, w_up, act_func, return_preact)
        return tuple(out) if return_preact else out[0]
    m, k = _check_x(x)
    if act_func not in _GLU:
        raise ValueError(f"act_func must be 'swiglu' or 'geglu', got {act_func!r}")
    ld_x = _pitch("x", x, (m, k), x.dtype, x.device)
    ld_g, ld_u = _weight("w_gate", w_gate, k, x), _weight("w_up", w_up, k, x)
    if w_up.shape != w_gate.shape:
        raise ValueError("w_gate and w_up must have equal shapes")
    n = w_gate.shape[0]

    def launch(s):
        h = x.new_empty((m, n))
        gate, up = (torch.empty_like(h), torch.empty_like(h)) if return_preact else (None, None)
        t = _TYPES[x.dtype]
        args = _lib.DenseArgs(x=x.data_ptr(), w0=w_gate.data_ptr(), w1=w_up.data_ptr(), y=h.data_ptr(), m=m, n=n, k=k, ld_x=ld_x, ld_w0=ld_g, ld_w1=ld_u,
                              ld_y=n, ld_pre0=n, ld_pre1=n, dtype=t, y_dtype=t, act=_GLU[act_func])  # fmt: skip
        if return_preact:
            args.pre0, args.pre1 = gate.data_ptr(), up.data_ptr()
        _lib.check(_lib.load().b200moe_gated_ffn(ctypes.byref(args), s))
        return (h, gate, up) if return_preact else h

    return call_on(x.device, stream, launch)


def gated_ffn_backward(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, gate: torch.Tensor, up: torch.Tensor,
                       act_func: str = "swiglu", input_grad: bool = True, weight_grad: bool = True, stream=None):  # fmt: skip
    """Backward pass of :func:`gated_ffn` from ``dh [tokens, n]`` and the saved ``gate`` and ``up``: returns
    ``(dx, dw_gate, dw_up)``, with ``None`` for what ``input_grad`` or ``weight_grad`` leaves out.  A value that GeGLU limits has
    no gradient.  The gradients of gate and up are rounded to x's type before the products; in fp16 they are scaled by a power of two
    over the call, so they may lie outside its range (what is below 2^-28 of their largest loses bits)."""
    m, k = _check_x(x)
    if act_func not in _GLU:
        raise ValueError(f"act_func must be 'swiglu' or 'geglu', got {act_func!r}")
    ld_x = _pitch("x", x, (m, k), x.dtype, x.device)
    ld_g, ld_u = _weight("w_gate", w_gate, k, x), _weight("w_up", w_up, k, x)
    if w_up.shape != w_gate.shape:
        raise ValueError("w_gate and w_up must have equal shapes")
    n = w_gate.shape[0]
    lds = [_pitch(name, v, (m, n), x.dtype, x.device) for name, v in (("dh", dh), ("gate", gate), ("up", up))]

    def launch(s):
        lib = _lib.load()
        dx = _like(x) if input_grad else None
        dw_gate, dw_up = (_like(w_gate), _like(w_up)) if weight_grad else (None, None)
        need = lib.b200moe_dense_workspace_bytes(m, n, 1 | (_lib.DENSE_WORKSPACE_F16 if x.dtype == torch.float16 else 0))
        work = x.new_empty((need,), dtype=torch.uint8)
        t = _TYPES[x.dtype]
        args = _lib.DenseArgs(
            x=x.data_ptr(), w0=w_gate.data_ptr(), w1=w_up.data_ptr(), dy=dh.data_ptr(), pre0=gate.data_ptr(), pre1=up.data_ptr(),
            dx=_ptr(dx), dw0=_ptr(dw_gate), dw1=_ptr(dw_up), workspace=work.data_ptr(), workspace_bytes=need, m=m, n=n, k=k, ld_x=ld_x, ld_w0=ld_g,
            ld_w1=ld_u, ld_dy=lds[0], ld_pre0=lds[1], ld_pre1=lds[2], dtype=t, y_dtype=t, act=_GLU[act_func])  # fmt: skip
        _lib.check(lib.b200moe_gated_ffn_backward(ctypes.byref(args), s))
        return dx, dw_gate, dw_up

    return call_on(x.device, stream, launch)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, act_func: Optional[str] = None,
           residual: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None, return_preact: bool = False, stream=None):  # fmt: skip
    """``act(x weight^T + bias) + residual``: ``x [tokens, k]``, ``weight [n, k]``, ``bias [n]`` (x's type or float32),
    ``residual [tokens, n]`` (x's type; a pitch of 0, one row for every token, included) -> ``[tokens, n]`` of
    ``out_dtype`` (x's type, or float32).  ``act_func``: ``None``, ``"relu"``, ``"silu"`` or ``"gelu"`` (the error-function form).
    A float32 result is not exact to its rounding: the tensor cores truncate within 512 elements of k (4e-7 of the terms' size
    at most in the mean), SiLU and GELU are good to about 1e-6 and in their negative tails to 8e-6 relative, and SiLU is 0 below -87.  With ``return_preact`` the result is ``(y, x weight^T + bias)``,
    the second in x's type, for :func:`linear_backward`."""
    if torch.compiler.is_compiling():
        _eager_stream_only(stream)
        out = torch.ops.b200moe.linear(x, weight, bias, act_func, residual, out_dtype, return_preact)
        return tuple(out) if return_preact else out[0]
    m, k = _check_x(x)
    if act_func not in _ACT:
        raise ValueError(f"act_func must be None, 'relu', 'silu' or 'gelu', got {act_func!r}")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in (x.dtype, torch.float32):
        raise NotImplementedError(f"out_dtype {out_dtype} is not built for {x.dtype} inputs (their own type and float32 are)")
    ld_x = _pitch("x", x, (m, k), x.dtype, x.device)
    ld_w = _weight("weight", weight, k, x)
    n = weight.shape[0]
    if bias is not None:
        if tuple(bias.shape) != (n,) or bias.device != x.device or (n > 1 and bias.stride(0) != 1):
            raise ValueError(f"bias must be a contiguous [{n}] tensor on {x.device}")
        if bias.dtype not in (x.dtype, torch.float32):
            raise NotImplementedError(f"bias dtype {bias.dtype} is not built for {x.dtype} inputs (their own type and float32 are)")
    ld_r = 0 if residual is None else _pitch("residual", residual, (m, n), x.dtype, x.device)

    def launch(s):
        y = x.new_empty((m, n), dtype=out_dtype)
        t = _TYPES[x.dtype]
        args = _lib.DenseArgs(x=x.data_ptr(), w0=weight.data_ptr(), y=y.data_ptr(), m=m, n=n, k=k, ld_x=ld_x, ld_w0=ld_w, ld_residual=ld_r, ld_y=n, ld_pre0=n,
                              dtype=t, y_dtype=_lib.DTYPE_F32 if out_dtype == torch.float32 else t, bias_dtype=t, act=_ACT[act_func])  # fmt: skip
        if bias is not None:
            args.bias, args.bias_dtype = bias.data_ptr(), t if bias.dtype == x.dtype else _lib.DTYPE_F32
        if residual is not None:
            args.residual = residual.data_ptr()
        z = None
        if return_preact:
            z = torch.empty_like(y) if out_dtype is x.dtype else x.new_empty((m, n))
            args.pre0 = z.data_ptr()
        _lib.check(_lib.load().b200moe_linear(ctypes.byref(args), s))
        return (y, z) if return_preact else y

    return call_on(x.device, stream, launch)


def linear_backward(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor, preact: Optional[torch.Tensor] = None, act_func: Optional[str] = None,
                    bias_grad: bool = False, input_grad: bool = True, weight_grad: bool = True, stream=None):  # fmt: skip
    """Backward pass of :func:`linear` from ``dy [tokens, n]`` (x's type or float32): returns ``(dx, dweight, dbias)``,
    ``dbias`` float32, with ``None`` for what is not asked for.  ``preact`` is the saved pre-activation (needed with an
    activation).  The residual's gradient is ``dy`` itself (of a residual row that every token shares: its column sums).

    ``dy act'(preact)`` is rounded to x's type before the products (``dbias`` is summed before that).  In fp16 it is scaled by a
    power of two over the call, so a float32 ``dy`` may lie outside fp16's range; what is below 2^-28 of its largest value loses
    bits."""
    m, k = _check_x(x)
    if act_func not in _ACT:
        raise ValueError(f"act_func must be None, 'relu', 'silu' or 'gelu', got {act_func!r}")
    ld_x = _pitch("x", x, (m, k), x.dtype, x.device)
    ld_w = _weight("weight", weight, k, x)
    n = weight.shape[0]
    if dy.dtype not in (x.dtype, torch.float32):
        raise NotImplementedError(f"dy dtype {dy.dtype} is not built for {x.dtype} inputs (their own type and float32 are)")
    ld_dy = _pitch("dy", dy, (m, n), dy.dtype, x.device)
    ld_z = 0
    if act_func is not None:
        if preact is None:
            raise ValueError("preact is required with an activation")
        ld_z = _pitch("preact", preact, (m, n), x.dtype, x.device)

    def launch(s):
        lib = _lib.load()
        dx, dw = _like(x) if input_grad else None, _like(weight) if weight_grad else None
        db = x.new_empty((n,), dtype=torch.float32) if bias_grad else None
        need = lib.b200moe_dense_workspace_bytes(m, n, 0)
        work = x.new_empty((need,), dtype=torch.uint8)
        t = _TYPES[x.dtype]
        args = _lib.DenseArgs(
            x=x.data_ptr(), w0=weight.data_ptr(), dy=dy.data_ptr(), pre0=None if act_func is None else preact.data_ptr(),
            dx=_ptr(dx), dw0=_ptr(dw), dbias=_ptr(db), workspace=work.data_ptr(), workspace_bytes=need, m=m, n=n, k=k, ld_x=ld_x,
            ld_w0=ld_w, ld_dy=ld_dy, ld_pre0=ld_z, dtype=t, y_dtype=_lib.DTYPE_F32 if dy.dtype == torch.float32 else t, act=_ACT[act_func])  # fmt: skip
        _lib.check(lib.b200moe_linear_backward(ctypes.byref(args), s))
        return dx, dw, db

    return call_on(x.device, stream, launch)


# ---------------------------------------------------------------------------------------------
# torch custom ops
# ---------------------------------------------------------------------------------------------
@torch.library.custom_op("b200moe::gated_ffn", mutates_args=(), device_types="cuda")
def _gated_ffn_op(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, act_func: str, return_preact: bool) -> List[torch.Tensor]:
    out = gated_ffn(x, w_gate, w_up, act_func, return_preact)
    return list(out) if return_preact else [out]


@_gated_ffn_op.register_fake
def _(x, w_gate, w_up, act_func, return_preact):
    return [x.new_empty((x.shape[0], w_gate.shape[0])) for _ in range(3 if return_preact else 1)]


@torch.library.custom_op("b200moe::linear", mutates_args=(), device_types="cuda")
def _linear_op(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor], act_func: Optional[str], residual: Optional[torch.Tensor],
               out_dtype: Optional[torch.dtype], return_preact: bool) -> List[torch.Tensor]:  # fmt: skip
    out = linear(x, weight, bias, act_func, residual, out_dtype, return_preact)
    return list(out) if return_preact else [out]


@_linear_op.register_fake
def _(x, weight, bias, act_func, residual, out_dtype, return_preact):
    shape = (x.shape[0], weight.shape[0])
    return [x.new_empty(shape, dtype=out_dtype or x.dtype)] + ([x.new_empty(shape)] if return_preact else [])
