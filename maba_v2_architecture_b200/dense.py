"""Dense operators of the model's blocks: the linear map with its epilogue and the gated
feed-forward block, with their gradients (maba_linear*, maba_gated_ffn* of the C ABI).

    b200_linear      out = residual + scale * act(x weight^T + bias)
    b200_gated_ffn   out = act(x w_gate^T) * (x w_up^T)

The reference computes these with torch modules and autograd: SwiGLUFFN (maba_sparse/model.py:
28-37), the gated residual adds (:107-108, :126-127) and the layers' projections.

Inputs are float32, float16 or bfloat16 CUDA tensors of one type with any strides; leading
dimensions of ``x`` are rows.  Sums are float32 and a result is rounded once; results do not
depend on the order in which the GPU runs the work.  16-bit products run on the tensor cores,
float32 ones on the CUDA cores.  Inputs are never written, except that ``out`` may be ``residual``.
Autocast does not reach these functions: operands are multiplied in the type they have
(``layers.SwiGLUFFN`` casts its own).

Work is enqueued on the current stream of the tensors' device.  Scratch memory comes from torch's
allocator for each call (not from the per-stream buffer that the other ops keep): two captured
graphs, or a graph and an eager call, then never share it.

With gradients enabled and an input that requires one, both functions record themselves for
autograd (first derivatives, reverse mode; dual tensors are refused).  ``*_backward`` are the same
gradients as plain calls, for training loops that keep their own tape or are captured into a CUDA
graph.  (Autograd's own backward pass is to be captured only while no eager graph of the same
leaves lives: torch accumulates their gradients on the eager graph's stream.)
"""
from __future__ import annotations

from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable
from torch.autograd.graph import increment_version  # what a kernel writes in place, autograd cannot see

from . import _native as N
from ._native import pack_matrix, pack_vector

ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}
DENSE_DTYPES = (torch.float32, torch.float16, torch.bfloat16)


# ---------------------------------------------------------------------------
# argument checks
# ---------------------------------------------------------------------------
def _check_device(t: torch.Tensor, name: str, x: torch.Tensor) -> None:
    if t.device != x.device:
        raise RuntimeError(
            f"Expected all tensors to be on the same device, but got {x.device} and {t.device} for {name}"
        )


def _check_weight(w: torch.Tensor, name: str, x: torch.Tensor, n: int, k: int) -> None:
    if w.device == x.device and w.dtype is x.dtype and w.shape == (n, k):
        return
    _check_device(w, name, x)
    if w.dtype is not x.dtype:
        raise TypeError(f"Tensor dtypes must match, but got {x.dtype} for x and {w.dtype} for {name}")
    raise ValueError(f"{name} shape {list(w.shape)} must be [{n}, {k}]")


def _check_x(x: torch.Tensor, w: torch.Tensor, name: str) -> Tuple[int, int]:
    """Output and input features."""
    dt, shape = w.dtype, w.shape
    if x.dtype is dt and dt in DENSE_DTYPES and len(shape) == 2 and x.device == w.device:
        n, k = shape
        if n and k and x.dim() and x.shape[-1] == k:
            return n, k
    if x.dtype not in DENSE_DTYPES:
        raise TypeError(f"Unsupported dtype {x.dtype}. Supported: {DENSE_DTYPES}")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    k = x.shape[-1]
    _check_weight(w, name, x, shape[0] if w.dim() else 0, k)
    raise ValueError(f"no features: x {list(x.shape)}, {name} {list(shape)}")


def _check_side(t: torch.Tensor, name: str, x: torch.Tensor, shape: Sequence[int], f32: bool = True) -> None:
    if t.device == x.device and t.shape == shape and (t.dtype is x.dtype or (f32 and t.dtype is torch.float32)):
        return
    _check_device(t, name, x)
    if t.dtype is not x.dtype and not (f32 and t.dtype is torch.float32):
        raise TypeError(f"{name} must be {x.dtype}{' or torch.float32' if f32 else ''}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} shape {list(t.shape)} must be {list(shape)}")


def _activation(name: str, plain: bool) -> int:
    code = ACTIVATIONS.get(name)
    if code is None or (code == 0 and not plain):
        names = [a for a, c in ACTIVATIONS.items() if plain or c]
        raise ValueError(f"Unknown activation {name!r}. Supported: {names}")
    return code


def _no_tangents(op: str, *ts: Optional[torch.Tensor]) -> None:
    """Refuses dual tensors, whose tangents the kernels would drop; called inside a dual level."""
    for t in ts:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"{op}: forward-mode derivatives are not supported")


def _span(t: torch.Tensor) -> Tuple[int, int]:
    last = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _check_out(out: torch.Tensor, x: torch.Tensor, shape, inputs, residual) -> None:
    _check_side(out, "out", x, shape)
    if not out.is_contiguous() and (out.dim() != 2 or out.stride(1) != 1 or out.stride(0) < out.shape[1]):
        raise ValueError(f"out must be contiguous or have contiguous rows, got strides {list(out.stride())}")
    if out.numel() == 0:
        return
    lo, hi = _span(out)
    for name, t in inputs:
        if t is not None and t.numel() > 0:
            a, b = _span(t)
            if a < hi and lo < b:
                raise ValueError(f"out shares memory with {name}")
    if residual is not None:
        a, b = _span(residual)
        same = (a == lo and residual.dtype == out.dtype and residual.stride() == out.stride())
        if a < hi and lo < b and not same:
            raise ValueError("out overlaps residual without being the same tensor")


_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream without its Stream object
_current_device = torch._C._cuda_getDevice


def _call(fn, size, x: torch.Tensor, head, size_args) -> None:
    """Runs one entry on x's device (made current where it is not: the C entries launch on the current
    device) with scratch memory of the size it asks for."""
    index = x.get_device()
    if index != _current_device():
        with torch.cuda.device(index):
            return _call(fn, size, x, head, size_args)
    nbytes = size(*size_args)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    rc = fn(*head, ws.data_ptr() if nbytes else None, nbytes, _raw_stream(index))
    if rc != N.OK:
        N.check(rc, fn.__name__)


def _rows(*ts: Optional[torch.Tensor]):
    """Each tensor as a matrix of rows: a view where its strides allow one, else a copy, which the
    caller holds until the launch (a descriptor keeps only its address)."""
    return [t if t is None or t.dim() == 2 else t.reshape(-1, t.shape[-1]) for t in ts]


def _mat(t: Optional[torch.Tensor]) -> Optional[bytes]:
    return None if t is None else pack_matrix(t)


def _vec(t: Optional[torch.Tensor]) -> Optional[bytes]:
    return None if t is None else pack_vector(t)


# ---------------------------------------------------------------------------
# the linear map
# ---------------------------------------------------------------------------
def _linear(x, weight, bias, act, scale, residual, out, out_dtype):
    # (one token's call is bound by this function: no helper calls, descriptors packed in place)
    if out is None:
        out = x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype or x.dtype)
    if x.dim() == 2:
        dx, do = pack_matrix(x), pack_matrix(out)
        dr = None if residual is None else pack_matrix(residual)
    else:
        if x.numel() == 0:
            return out
        held = _rows(x, out, residual)
        dx, do, dr = map(_mat, held)
    dw = pack_matrix(weight)
    db = None if bias is None else pack_vector(bias)
    ds = None if scale is None else pack_vector(scale)
    lib = N.lib()
    index = x.get_device()
    rc = N.ERR_WORKSPACE
    # most calls need no scratch memory: tried without (refused before any launch)
    if index == _current_device():
        rc = lib.maba_linear(dx, dw, db, act, ds, dr, do, None, 0, _raw_stream(index))
    if rc:
        if rc != N.ERR_WORKSPACE:
            N.check(rc, "maba_linear")
        _call(lib.maba_linear, lib.maba_linear_workspace_size, x, (dx, dw, db, act, ds, dr, do), (dx, dw, dr, do))
    return out


def _linear_backward(grad_out, x, weight, bias, act, scale, needs):
    need_x, need_w, need_b, need_s = needs
    dx = x.new_empty(x.shape) if need_x else None
    dw = x.new_empty(weight.shape) if need_w else None
    db = bias.new_empty(bias.shape) if need_b else None
    ds = scale.new_empty(scale.shape) if need_s else None
    if need_x or need_w or need_b or need_s:
        lib = N.lib()
        held = _rows(grad_out, x, weight, dx, dw)
        mg, mx, mw, mdx, mdw = map(_mat, held)
        args = (mg, mx, mw, _vec(bias), act, _vec(scale), mdx, mdw, _vec(db), _vec(ds))
        _call(lib.maba_linear_backward, lib.maba_linear_backward_workspace_size, x, args, args)
    return dx, dw, db, ds


class _LinearFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, scale, residual, act, out_dtype):
        ctx.save_for_backward(x, weight, bias, scale)
        ctx.act, ctx.res_dtype = act, None if residual is None else residual.dtype
        return _linear(x, weight, bias, act, scale, residual, None, out_dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        x, weight, bias, scale = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _no_tangents("linear_backward", grad_out, x, weight, bias, scale)
        dx, dw, db, ds = _linear_backward(grad_out, x, weight, bias, ctx.act, scale, ctx.needs_input_grad[:4])
        dr = grad_out.to(ctx.res_dtype) if ctx.needs_input_grad[4] else None
        return dx, dw, db, ds, dr, None, None


def b200_linear(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    activation: str = "none",
    scale: Optional[torch.Tensor] = None,
    residual: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
    out_dtype: Optional[torch.dtype] = None,
) -> torch.Tensor:
    """``residual + scale * act(x weight^T + bias)``, the epilogue applied to the float32 sums.
    One launch, and one more each where 16-bit inputs have rows off 16-byte boundaries (they are
    copied first) and where few outputs with a long contraction split it.

    x [..., K], weight [N, K] (nn.Linear's layout), bias and scale [N] and residual [..., N] in x's
    dtype or float32; ``activation`` one of ``none``, ``relu``, ``silu``, ``gelu`` (the erf form).
    The result [..., N] has x's dtype, or ``out_dtype=torch.float32``; ``out`` receives it in
    place and may be ``residual`` (a residual stream updated where it is), not another input.
    With the residual gates of MabaBlock as ``scale``: maba_sparse/model.py:107-108, 126-127.
    """
    act = ACTIVATIONS.get(activation)
    if act is None:
        _activation(activation, True)
    n, _ = _check_x(x, weight, "weight")
    shape = (*x.shape[:-1], n)
    if bias is not None:
        _check_side(bias, "bias", x, (n,))
    if scale is not None:
        _check_side(scale, "scale", x, (n,))
    if residual is not None:
        _check_side(residual, "residual", x, shape)
    if out_dtype is not None and out_dtype is not torch.float32 and out_dtype is not x.dtype:
        raise TypeError(f"out_dtype must be {x.dtype} or torch.float32, got {out_dtype}")
    if forward_ad._current_level >= 0:
        _no_tangents("linear", x, weight, bias, scale, residual, out)
    if not x.is_cuda:
        N.require_cuda(x, op="linear")
    tracked = torch.is_grad_enabled() and (
        weight.requires_grad or x.requires_grad or (bias is not None and bias.requires_grad)
        or (scale is not None and scale.requires_grad) or (residual is not None and residual.requires_grad))
    if out is not None:
        if tracked or out.requires_grad:
            raise RuntimeError("linear: out= does not support automatic differentiation")
        if out_dtype is not None and out.dtype != out_dtype:
            raise TypeError(f"out must be {out_dtype}, got {out.dtype}")
        _check_out(out, x, shape, (("x", x), ("weight", weight), ("bias", bias), ("scale", scale)), residual)
    if tracked:
        return _LinearFunction.apply(x, weight, bias, scale, residual, act, out_dtype)
    y = _linear(x, weight, bias, act, scale, residual, out, out_dtype)
    if out is not None:
        increment_version(out)
    return y


def b200_linear_backward(
    grad_out: torch.Tensor,
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    activation: str = "none",
    scale: Optional[torch.Tensor] = None,
    needs: Tuple[bool, bool, bool, bool] = (True, True, True, True),
) -> Tuple[Optional[torch.Tensor], ...]:
    """Gradients ``(dx, dweight, dbias, dscale)`` of ``b200_linear`` for its output's gradient
    ``grad_out`` [..., N] (x's dtype or float32); the residual's is grad_out itself.  ``needs``
    says which are computed (dbias / dscale only where bias / scale are given); the rest are None.

    z = x weight^T + bias is computed again where an activation or a scale is given, so the forward
    pass keeps nothing but its inputs.  grad_out * scale * act'(z) is rounded to x's dtype between the
    products; the column sums of dbias and dscale are taken before that rounding.
    """
    act = _activation(activation, True)
    n, _ = _check_x(x, weight, "weight")
    if bias is not None:
        _check_side(bias, "bias", x, (n,))
    if scale is not None:
        _check_side(scale, "scale", x, (n,))
    _check_side(grad_out, "grad_out", x, (*x.shape[:-1], n))
    if forward_ad._current_level >= 0:
        _no_tangents("linear_backward", grad_out, x, weight, bias, scale)
    N.require_cuda(x, op="linear_backward")
    needs = (bool(needs[0]), bool(needs[1]), bool(needs[2]) and bias is not None, bool(needs[3]) and scale is not None)
    return _linear_backward(grad_out, x, weight, bias, act, scale, needs)


# ---------------------------------------------------------------------------
# the gated feed-forward block
# ---------------------------------------------------------------------------
def _gated_ffn(x, w_gate, w_up, act, out):
    if out is None:
        out = x.new_empty((*x.shape[:-1], w_gate.shape[0]))
    if x.dim() == 2:
        dx, do = pack_matrix(x), pack_matrix(out)
    else:
        if x.numel() == 0:
            return out
        held = _rows(x, out)
        dx, do = map(_mat, held)
    dg, du = pack_matrix(w_gate), pack_matrix(w_up)
    lib = N.lib()
    index = x.get_device()
    rc = N.ERR_WORKSPACE
    if index == _current_device():  # (as in _linear)
        rc = lib.maba_gated_ffn(dx, dg, du, act, do, None, 0, _raw_stream(index))
    if rc:
        if rc != N.ERR_WORKSPACE:
            N.check(rc, "maba_gated_ffn")
        _call(lib.maba_gated_ffn, lib.maba_gated_ffn_workspace_size, x, (dx, dg, du, act, do), (dx, dg, du, do))
    return out


def _gated_ffn_backward(grad_out, x, w_gate, w_up, act, needs):
    need_x, need_g, need_u = needs
    dx = x.new_empty(x.shape) if need_x else None
    dg = x.new_empty(w_gate.shape) if need_g else None
    du = x.new_empty(w_up.shape) if need_u else None
    if need_x or need_g or need_u:
        lib = N.lib()
        held = _rows(grad_out, x, w_gate, w_up, dx, dg, du)
        packed = [_mat(t) for t in held]
        ins, outs = packed[:4], packed[4:]
        _call(lib.maba_gated_ffn_backward, lib.maba_gated_ffn_backward_workspace_size, x, (*ins, act, *outs),
              (*ins, *outs))
    return dx, dg, du


class _GatedFFNFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, act):
        ctx.save_for_backward(x, w_gate, w_up)
        ctx.act = act
        return _gated_ffn(x, w_gate, w_up, act, None)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        x, w_gate, w_up = ctx.saved_tensors
        if forward_ad._current_level >= 0:
            _no_tangents("gated_ffn_backward", grad_out, x, w_gate, w_up)
        return (*_gated_ffn_backward(grad_out, x, w_gate, w_up, ctx.act, ctx.needs_input_grad[:3]), None)


def b200_gated_ffn(
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    activation: str = "silu",
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``act(x w_gate^T) * (x w_up^T)``: both projections, the activation and the product; the
    projections are never stored, but for float32 partial sums where few outputs with a long
    contraction split it.  Launches as for ``b200_linear``.

    x [..., K], w_gate and w_up [I, K]; ``activation`` one of ``silu``, ``gelu`` (the erf form),
    ``relu``.  The result is [..., I] in x's dtype.  Reference: maba_sparse/model.py:28-37
    (SwiGLUFFN without its down projection, which is ``b200_linear``).
    """
    act = _activation(activation, False)
    n, k = _check_x(x, w_gate, "w_gate")
    _check_weight(w_up, "w_up", x, n, k)
    if forward_ad._current_level >= 0:
        _no_tangents("gated_ffn", x, w_gate, w_up, out)
    if not x.is_cuda:
        N.require_cuda(x, op="gated_ffn")
    tracked = torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad)
    if out is not None:
        if tracked or out.requires_grad:
            raise RuntimeError("gated_ffn: out= does not support automatic differentiation")
        _check_side(out, "out", x, (*x.shape[:-1], n), f32=False)
        _check_out(out, x, out.shape, (("x", x), ("w_gate", w_gate), ("w_up", w_up)), None)
    if tracked:
        return _GatedFFNFunction.apply(x, w_gate, w_up, act)
    y = _gated_ffn(x, w_gate, w_up, act, out)
    if out is not None:
        increment_version(out)
    return y


def b200_gated_ffn_backward(
    grad_out: torch.Tensor,
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    activation: str = "silu",
    needs: Tuple[bool, bool, bool] = (True, True, True),
) -> Tuple[Optional[torch.Tensor], ...]:
    """Gradients ``(dx, dw_gate, dw_up)`` of ``b200_gated_ffn`` for ``grad_out`` [..., I] (x's dtype);
    ``needs`` says which are computed.  The projections are computed again from the inputs; their
    gradients are rounded to x's dtype between the products."""
    act = _activation(activation, False)
    n, k = _check_x(x, w_gate, "w_gate")
    _check_weight(w_up, "w_up", x, n, k)
    _check_side(grad_out, "grad_out", x, (*x.shape[:-1], n), f32=False)
    if forward_ad._current_level >= 0:
        _no_tangents("gated_ffn_backward", grad_out, x, w_gate, w_up)
    N.require_cuda(x, op="gated_ffn_backward")
    return _gated_ffn_backward(grad_out, x, w_gate, w_up, act, tuple(bool(n) for n in needs))


__all__ = ["b200_linear", "b200_linear_backward", "b200_gated_ffn", "b200_gated_ffn_backward"]
