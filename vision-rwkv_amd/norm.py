"""The root-mean-square norm with the residual's addition in front of it, with its gradients, or with an output in 8 bits for a product that takes such.

    r = x + residual          y = r / sqrt(mean(r^2) + eps) weight

The LayerNorm forms of row_fuse are the reference's; this one it lacks."""
import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .decay import _call, _check, _check_recorders, _eager, _resolved
from .ops import _DT, batched_cotangent

_KINDS = {None: 0, torch.float8_e4m3fn: 1, torch.int8: 2}


def _check_norm(x, weight, residual):
    _check(x, "x")
    if x.dim() < 1 or x.dtype not in _DT or x.shape[-1] == 0:
        raise RuntimeError("x must be (..., C) of one of float32 / bfloat16 / float16")
    _check(weight, "weight", x)
    if tuple(weight.shape) != (x.shape[-1],) or weight.dtype not in (torch.float32, x.dtype):
        raise RuntimeError(f"weight must be ({x.shape[-1]},) of x's dtype or float32")
    if residual is not None:
        _check(residual, "residual", x)
        if residual.shape != x.shape or residual.dtype not in (torch.float32, x.dtype):
            raise RuntimeError("residual must have the shape of x, and its dtype or float32")
    if x.shape[-1] > 0x7fffffff or x.numel() // x.shape[-1] > 0x7fffffff:
        raise RuntimeError("a size of 2^31 or more")


def _as_rows(t):
    """t (..., C) as rows at one distance, elements side by side."""
    t = _resolved(t)
    if t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] == 1):
        return t
    try:
        rows = t.view(-1, t.shape[-1])
    except RuntimeError:
        return t.contiguous().view(-1, t.shape[-1])
    return rows if rows.stride(1) == 1 or rows.shape[1] == 1 else rows.contiguous()


def _distance(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _args(weight, C, rows, dtype, residual_dtype, eps):
    a = _lib.RmsnormArgs()
    a.weight, a.C, a.rows, a.eps = weight.data_ptr(), C, rows, eps
    a.dtype, a.residual_dtype, a.weight_dtype = _DT[dtype], _DT[residual_dtype], _DT[weight.dtype]
    return a


def _forward(x, weight, residual, eps, kind):
    """y, its scales (or None) and r (or None)."""
    shape, xr = x.shape, _as_rows(x)
    weight = _resolved(weight).contiguous()
    y = torch.empty(shape, dtype=kind or x.dtype, device=x.device)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=x.device) if kind else None
    r = torch.empty(shape, dtype=residual.dtype, device=x.device) if residual is not None else None
    if xr.shape[0] == 0:
        return y, scale, r
    a = _args(weight, shape[-1], xr.shape[0], x.dtype, residual.dtype if residual is not None else x.dtype, eps)
    a.x, a.x_stride, a.y, a.out_kind = xr.data_ptr(), _distance(xr), y.data_ptr(), _KINDS[kind]
    if residual is not None:
        rr = _as_rows(residual)
        a.residual, a.residual_stride, a.sum = rr.data_ptr(), _distance(rr), r.data_ptr()
    if kind:
        a.scale = scale.data_ptr()
    _call("vrwkv_rmsnorm", a, x.device)
    return y, scale, r


class RMSNormFunction(torch.autograd.Function):
    """rms_norm with its backward kernel."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        _check_norm(x, weight, residual)
        y, _, r = _forward(x, weight, residual, eps, None)
        ctx.save_for_backward(x if residual is None else r, weight)
        ctx.meta = x.shape, x.dtype, eps, residual is not None
        ctx.set_materialize_grads(False)
        return y, r

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, gr):
        r, weight = ctx.saved_tensors
        shape, dtype, eps, has_residual = ctx.meta
        _check(r, "the saved sum")
        _check(weight, "weight", r)
        if r.shape != shape or (r.dtype != dtype and not (has_residual and r.dtype == torch.float32)) or tuple(weight.shape) != shape[-1:] or weight.dtype not in _DT:   # (hooks on saved tensors may have changed them)
            raise RuntimeError("the saved tensors have other sizes or types than those of the call")
        if batched_cotangent(*(t for t in (gy, gr) if t is not None)):
            raise RuntimeError("rms_norm's gradients take one cotangent at a time")
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        weight = _resolved(weight).contiguous()
        new = lambda t: torch.empty(shape, dtype=t, device=r.device)  # noqa: E731
        dx = new(dtype) if need_x or not need_r else None
        # (one tensor for both where they are of one type, as an addition's gradients are)
        dresidual = None if not need_r else dx if dx is not None and r.dtype == dtype else new(r.dtype)
        dw = torch.empty_like(weight) if need_w else None
        out = dx, dw, dresidual, None
        rows = _as_rows(r)
        if rows.shape[0] == 0 or gy is None:
            if dw is not None:
                dw.zero_()
            for t in (dx, dresidual):
                if t is not None:
                    t.zero_() if gr is None else t.copy_(gr)
            return out
        g = _as_rows(gy.to(dtype))
        a = _args(weight, shape[-1], rows.shape[0], dtype, r.dtype if has_residual else dtype, eps)
        a.sum, a.x_stride, a.gy, a.gy_stride = rows.data_ptr(), _distance(rows), g.data_ptr(), _distance(g)
        if gr is not None:
            gr = _as_rows(gr.to(r.dtype))
            a.gsum, a.gsum_stride = gr.data_ptr(), _distance(gr)
        a.dx = dx.data_ptr() if dx is not None else None
        a.dresidual = dresidual.data_ptr() if dresidual is not None and dresidual is not dx else None
        a.dweight = dw.data_ptr() if dw is not None else None
        _call("vrwkv_rmsnorm_bwd", a, r.device, "vrwkv_rmsnorm_bwd_workspace_bytes")
        return out


def rms_norm(x, weight, residual=None, eps=1e-6, quantize=None):
    """y, or (y, r) with a residual: r = x + residual, rounded to the residual's type, and y = r / sqrt(mean(r^2) + eps) weight of x's type, over the last dimension.

    x (..., C) float32, bfloat16 or float16, weight (C,) of x's dtype or float32, residual of x's shape and of its dtype or float32.  The mean and everything behind it is
    fp32, rounded once.  Gradients for all three; no second ones, no forward mode, no tracing (a compiled program makes the call as it is).
    quantize: torch.float8_e4m3fn or torch.int8: (q, scale) or (q, scale, r) instead, y = q scale with scale (...) in float32, the row's largest |y| over 448 or 127 (2^-126 at least) and
    q = y / scale, a quotient of fp32 numbers, rounded to the nearest (even) of 8 bits; y is not rounded to x's type before.  A row with a NaN has a scale of NaN.  Forward only."""
    if torch.compiler.is_compiling():
        return _eager(rms_norm)(x, weight, residual, eps, quantize)
    if isinstance(eps, torch.Tensor):                      # (it would go in without its gradient)
        raise RuntimeError("eps must be a number")
    if quantize not in _KINDS:
        raise RuntimeError("quantize must be None, torch.float8_e4m3fn or torch.int8")
    out = _lib.host().rms_norm(x, weight, residual, float(eps), _KINDS[quantize])
    if out is not None:
        y, scale, r = out
        return ((y, scale) if r is None else (y, scale, r)) if quantize is not None else y if r is None else (y, r)
    _check_recorders("rms_norm", x, weight, residual)
    _check_norm(x, weight, residual)
    record = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual))
    if quantize is not None:
        if record:
            raise RuntimeError("an output in 8 bits has no backward: call rms_norm under torch.no_grad(), or without quantize")
        q, scale, r = _forward(x, weight, residual, float(eps), quantize)
        return (q, scale) if residual is None else (q, scale, r)
    y, r = RMSNormFunction.apply(x, weight, residual, float(eps)) if record else _forward(x, weight, residual, float(eps), None)[::2]
    return y if residual is None else (y, r)
