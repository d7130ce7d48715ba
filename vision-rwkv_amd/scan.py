"""The selective state space scan with the short causal convolution in front of it, over whole sequences (with gradients) and one token at a time.

    h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t^T          y_t = (C_t h_t + D u_t) silu(z_t)          dt = softplus(delta + delta_bias)

Beside wkv6, whose decays belong to a key channel, and decay_attention, whose decays belong to a head, every channel and state of it has one of its own at every token.  The
convolution is to it what q_shift is to Bi-WKV: a channel's look at its neighbours, here those in front.  Their states can be kept in pages, which copy_states copies.  The
reference has no counterpart.
"""
import ctypes

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .decay import _call, _changed, _check, _check_in_place, _check_index, _check_recorders, _check_sizes, _eager, _pages_fit, _resolved
from .ops import _DT, batched_cotangent

_FLOATS = "one of float32 / bfloat16 / float16"


def _tokens(t):
    """t as the kernels read it: any strides, but channels side by side and tokens less than 2^22 elements apart."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) and (t.dim() == 2 or t.shape[1] == 1 or t.stride(1) < 1 << 22) else t.contiguous()


def _token_strides(t):
    """Strides of batch and token (and group); a row of one token has none to a next one, whatever the view says."""
    return (t.stride(0), 0 if t.shape[1] == 1 else t.stride(1)) + t.stride()[2:-1]


def _pointer(t):
    return t.data_ptr() if t is not None else None


def _set(args, **fields):
    for name, value in fields.items():
        setattr(args, name, value)


def _check_param(t, name, shape, like, also=()):
    """A parameter of the operator: of `like`'s type or float32 (or those in `also`)."""
    _check(t, name, like)
    if tuple(t.shape) != tuple(shape) or t.dtype not in (torch.float32, like.dtype, *also):
        raise RuntimeError(f"{name} must be float32 or have the others' dtype, of shape {tuple(shape)}")


def _check_sequences(x, offsets):
    """The number of sequences in rows x (B, T, ..)."""
    if offsets is None:
        return x.shape[0]
    _check_index(offsets, "offsets", x)
    if x.shape[0] != 1 or offsets.numel() < 1:
        raise RuntimeError("packed sequences (offsets) come as one row, B = 1, with N + 1 offsets")
    return offsets.numel() - 1


def _check_pool(pool, name, page, dtype, like):
    _check(pool, name, like)
    _check_in_place(pool, name)
    _check_sizes(pool.shape)
    if pool.dim() != 3 or tuple(pool.shape[1:]) != page or pool.dtype != dtype or not _pages_fit(pool):
        raise RuntimeError(f"{name} must be {str(dtype)[6:]} (P, {page[0]}, {page[1]}) with contiguous pages")


def _check_slots(slots, pool, rows, like):
    if slots is None:
        if rows > pool.shape[0]:
            raise RuntimeError(f"{rows} rows without slots, and {pool.shape[0]} pages")
        return None
    slots = _check_index(slots, "slots", like)
    if slots.numel() != rows:
        raise RuntimeError(f"{slots.numel()} slots for {rows} rows")
    return slots


def _no_gradients(name, instead, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} has no backward: call it under torch.no_grad(), or {instead}")


def _outside(y, slots):
    """The results of rows where the pool has no page: zeros for slot -1, NaN for any other."""
    return y.copy_(torch.where(slots == -1, 0.0, float("nan"))[:, None].expand_as(y))


def _like(t, need):
    return torch.empty(t.shape, dtype=t.dtype, device=t.device) if need and t is not None else None


def _zero_all(*tensors):
    for t in tensors:
        if t is not None:
            t.zero_()


def _state_only(last, state):
    """last where there is no token: the states stay what they are."""
    if last is not None:
        last.zero_() if state is None else last.copy_(state)


# ---- the convolution ---------------------------------------------------------------------------------------------------

def _check_taps(x, weight, bias, activation):
    if x.dtype not in _DT:
        raise RuntimeError(f"x must be {_FLOATS}")
    if x.shape[-1] == 0:
        raise RuntimeError("x has no channels")
    _check(weight, "weight", x)
    if weight.dim() != 2 or not 2 <= weight.shape[1] <= 8:
        raise RuntimeError("weight must be (E, K) with 2 to 8 taps")
    _check_param(weight, "weight", (x.shape[-1], weight.shape[1]), x)
    if bias is not None:
        _check_param(bias, "bias", (x.shape[-1],), x)
        if bias.dtype != weight.dtype:
            raise RuntimeError("weight and bias must have one dtype")
    if activation not in (None, "silu"):
        raise RuntimeError("activation must be None or 'silu'")
    _check_sizes(x.shape)
    return weight.shape[1]


def _check_conv(x, weight, bias, activation, state, offsets):
    """causal_conv's checks; the number of sequences."""
    _check(x, "x")
    if x.dim() != 3:
        raise RuntimeError("x must be (B, T, E)")
    K = _check_taps(x, weight, bias, activation)
    N = _check_sequences(x, offsets)
    if state is not None:
        _check(state, "state", x)
        if tuple(state.shape) != (N, K - 1, x.shape[2]) or state.dtype != x.dtype:
            raise RuntimeError(f"state must be of x's dtype and of shape {(N, K - 1, x.shape[2])}")
    return N


def _conv_args(x, weight, bias, activation, state, offsets, N):
    a = _lib.ConvArgs()
    _set(a, x=x.data_ptr(), weight=weight.data_ptr(), bias=_pointer(bias), state=_pointer(state), offsets=_pointer(offsets), x_stride=_token_strides(x), N=N, T=x.shape[1],
         E=x.shape[2], K=weight.shape[1], dtype=_DT[x.dtype], param_dtype=_DT[weight.dtype], silu=activation is not None, offsets64=offsets is not None and offsets.dtype == torch.int64)
    return a


def _conv_inputs(x, weight, bias, state, offsets):
    x, weight, bias, state, offsets = (_resolved(t) for t in (x, weight, bias, state, offsets))
    return (_tokens(x), *(t.contiguous() if t is not None else None for t in (weight, bias, state, offsets)))


class CausalConv(torch.autograd.Function):
    """causal_conv with its backward kernels."""

    @staticmethod
    def forward(ctx, x, weight, bias, state, offsets, activation, N, keep_state):
        if N != _check_conv(x, weight, bias, activation, state, offsets):
            raise RuntimeError(f"{N} sequences are not those of the tensors")
        x, weight, bias, state, offsets = _conv_inputs(x, weight, bias, state, offsets)
        ctx.save_for_backward(x, weight, bias, state, offsets)
        ctx.meta = activation, N
        ctx.set_materialize_grads(False)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        last = torch.empty((N, weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device) if keep_state else None
        if N == 0 or x.shape[1] == 0:
            _state_only(last, state)
            return y.zero_(), last
        a = _conv_args(x, weight, bias, activation, state, offsets, N)
        _set(a, y=y.data_ptr(), last=_pointer(last))
        _call("vrwkv_conv_fwd", a, x.device)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, glast):
        x, weight, bias, state, offsets = ctx.saved_tensors
        activation, N = ctx.meta
        if N != _check_conv(x, weight, bias, activation, state, offsets):   # (hooks on saved tensors may have moved or changed them)
            raise RuntimeError("the saved tensors have other sizes than those of the call")
        if batched_cotangent(*(t for t in (gy, glast) if t is not None)):
            raise RuntimeError("causal_conv's gradients take one cotangent at a time")
        x, weight, bias, state, offsets = _conv_inputs(x, weight, bias, state, offsets)
        need = ctx.needs_input_grad
        dx, dw = _like(x, True), _like(weight, True)
        db, dstate = _like(bias, need[2]), _like(state, need[3])
        out = dx, dw, db, dstate, None, None, None, None
        if N == 0 or x.shape[1] == 0 or (gy is None and glast is None):
            _zero_all(dx, dw, db)
            if dstate is not None:
                dstate.zero_() if glast is None else dstate.copy_(glast)
            return out
        gy = torch.zeros_like(x, memory_format=torch.contiguous_format) if gy is None else _tokens(_resolved(gy.to(x.dtype)))
        glast = _resolved(glast.to(x.dtype)).contiguous() if glast is not None else None
        a = _conv_args(x, weight, bias, activation, state, offsets, N)
        _set(a, gy=gy.data_ptr(), gy_stride=_token_strides(gy), glast=_pointer(glast), dx=dx.data_ptr(), dweight=dw.data_ptr(), dbias=_pointer(db), dstate=_pointer(dstate))
        _call("vrwkv_conv_bwd", a, x.device, "vrwkv_conv_bwd_workspace_bytes")
        return out


def causal_conv(x, weight, bias=None, activation=None, state=None, offsets=None, return_state=False):
    """y (B, T, E), y_t = sum_j weight[:, j] x_{t - (K - 1) + j} + bias, and silu of that with activation "silu": each channel over the K - 1 tokens in front of it and its own.  With
    return_state also the last K - 1 tokens of each sequence (N, K - 1, E), for the call or the step that goes on from there.

    x (B, T, E), float32, bfloat16 or float16, at any strides (half of a projection's result).  weight (E, K), K 2 to 8, and bias (E,): x's dtype or float32.
    state: the K - 1 tokens in front of the first, (N, K - 1, E) of x's dtype, zeros without; N = B.
    offsets (N + 1,), int32 or int64 on the device, ascending from 0 to T: N sequences packed behind each other in one row (B = 1), sequence n the tokens
    offsets[n] to offsets[n + 1] (an empty one leaves its state as it is); y of rows behind the last sequence is zero, and so are their gradients.
    Gradients for x, weight, bias and state, sums in fp32, rounded once to their inputs' types; no second ones, no forward mode, no tracing (a compiled
    program makes the call as it is)."""
    if torch.compiler.is_compiling():
        return _eager(causal_conv)(x, weight, bias, activation, state, offsets, return_state)
    if activation in (None, "silu"):
        out = _lib.host().causal_conv(x, weight, bias, activation is not None, state, offsets, return_state)
        if out is not None:
            return out
    _check_recorders("causal_conv", x, weight, bias, state, offsets)
    N = _check_conv(x, weight, bias, activation, state, offsets)
    y, last = CausalConv.apply(x, weight, bias, state, offsets, activation, N, bool(return_state))
    return (y, last) if return_state else y


def causal_conv_step(x, weight, pool, slots=None, bias=None, activation=None):
    """y (N, E) for one more token of each of N sequences, whose last K - 1 tokens are pages of `pool` (P, K - 1, E) of x's dtype and are updated in place.

    x (N, E), weight, bias and activation as in causal_conv; slots as in decay_attention_step: row n's page, 0, 1, .. without; rows that name the same page are tokens
    behind each other; -1 gives zeros and touches nothing, any other slot outside the pool NaN.  Forward only: inputs that want gradients or carry tangents are refused, and so is tracing."""
    if torch.compiler.is_compiling():
        return _eager(causal_conv_step)(x, weight, pool, slots, bias, activation)
    if activation in (None, "silu"):
        y = _lib.host().causal_conv_step(x, weight, pool, slots, bias, activation is not None)
        if y is not None:
            return y
    _check_recorders("causal_conv_step", x, weight, bias, pool, slots)
    x, weight, bias, slots = (_resolved(t) for t in (x, weight, bias, slots))
    _check(x, "x")
    if x.dim() != 2:
        raise RuntimeError("x must be (N, E)")
    K = _check_taps(x, weight, bias, activation)
    N, E = x.shape
    _check_pool(pool, "pool", (K - 1, E), x.dtype, x)
    slots = _check_slots(slots, pool, N, x)
    _no_gradients("causal_conv_step", "causal_conv", x, weight, bias, pool)
    y = torch.empty((N, E), dtype=x.dtype, device=x.device)
    if N == 0:
        return y
    if pool.shape[0] == 0:
        return _outside(y, slots)
    x, weight = _tokens(x), weight.contiguous()
    bias = bias.contiguous() if bias is not None else None
    a = _lib.ConvStepArgs()
    _set(a, x=x.data_ptr(), weight=weight.data_ptr(), bias=_pointer(bias), slots=_pointer(slots), pool=pool.data_ptr(), y=y.data_ptr(), x_stride=x.stride(0),
         page_stride=pool.stride(0) if pool.shape[0] > 1 else (K - 1) * E, N=N, P=pool.shape[0], E=E, K=K, dtype=_DT[x.dtype], param_dtype=_DT[weight.dtype],
         silu=activation is not None, slots64=slots is not None and slots.dtype == torch.int64)
    _call("vrwkv_conv_step", a, x.device)
    _changed(pool)
    return y


# ---- the scan ----------------------------------------------------------------------------------------------------------

def _check_scan_inputs(u, delta, A, B, C, D, z, delta_bias, lead):
    """What selective_scan (lead 2) and its step (lead 1) check of their inputs; E, S and the groups."""
    _check(u, "u")
    if u.dim() != lead + 1 or u.dtype not in _DT:
        raise RuntimeError(f"u must be {'(B, T, E)' if lead == 2 else '(N, E)'} of {_FLOATS}")
    E = u.shape[-1]
    for t, n in ((delta, "delta"), (z, "z")):
        if t is None and n == "z":
            continue
        _check(t, n, u)
        if t.shape != u.shape or t.dtype != u.dtype:
            raise RuntimeError(f"{n} must have the shape and dtype of u")
    _check(A, "A", u)
    if A.dim() != 2 or A.shape[0] != E or A.dtype != torch.float32 or not 1 <= A.shape[1] <= 64:
        raise RuntimeError(f"A must be float32 of shape ({E}, S) with 1 to 64 states")
    S = A.shape[1]
    groups = B.shape[lead] if isinstance(B, torch.Tensor) and B.dim() == lead + 2 else 1
    for t, n in ((B, "B"), (C, "C")):
        _check(t, n, u)
        if t.dtype != u.dtype or t.dim() not in (lead + 1, lead + 2) or t.shape[:lead] != u.shape[:lead] or t.shape[-1] != S or (t.dim() == lead + 2 and t.shape[lead] != groups) or (t.dim() == lead + 1 and groups != 1):
            raise RuntimeError(f"{n} must be {'(B, T, S) or (B, T, G, S)' if lead == 2 else '(N, S) or (N, G, S)'} with u's dtype, B and C with as many groups")
    if E == 0 or groups == 0 or E % groups:
        raise RuntimeError(f"{groups} groups must divide {E} channels")
    for t, n in ((D, "D"), (delta_bias, "delta_bias")):
        if t is not None:
            _check_param(t, n, (E,), u)
    _check_sizes(u.shape, B.shape, C.shape)
    return E, S, groups


def _check_scan(u, delta, A, B, C, D, z, delta_bias, state, offsets):
    """selective_scan's checks; the number of sequences and groups."""
    E, S, groups = _check_scan_inputs(u, delta, A, B, C, D, z, delta_bias, 2)
    N = _check_sequences(u, offsets)
    if state is not None:
        _check(state, "state", u)
        if tuple(state.shape) != (N, E, S) or state.dtype != torch.float32:
            raise RuntimeError(f"state must be float32 of shape {(N, E, S)}")
    return N, groups


def _grouped(t, lead):
    t = _resolved(t)
    return _tokens(t if t.dim() == lead + 2 else t.unsqueeze(lead))


def _scan_inputs(u, delta, A, B, C, D, z, delta_bias, state, offsets):
    u, delta, z = (_tokens(_resolved(t)) if t is not None else None for t in (u, delta, z))
    A, D, delta_bias, state, offsets = (_resolved(t).contiguous() if t is not None else None for t in (A, D, delta_bias, state, offsets))
    return u, delta, A, _grouped(B, 2), _grouped(C, 2), D, z, delta_bias, state, offsets


def _scan_args(u, delta, A, B, C, D, z, delta_bias, state, offsets, softplus, N):
    a = _lib.ScanArgs()
    _set(a, u=u.data_ptr(), delta=delta.data_ptr(), A=A.data_ptr(), B=B.data_ptr(), C=C.data_ptr(), D=_pointer(D), z=_pointer(z), delta_bias=_pointer(delta_bias), state=_pointer(state),
         offsets=_pointer(offsets), u_stride=_token_strides(u), delta_stride=_token_strides(delta), B_stride=_token_strides(B), C_stride=_token_strides(C), N=N, T=u.shape[1], E=u.shape[2],
         S=A.shape[1], G=B.shape[2], dtype=_DT[u.dtype], D_dtype=_DT[D.dtype] if D is not None else 0, bias_dtype=_DT[delta_bias.dtype] if delta_bias is not None else 0, softplus=softplus,
         offsets64=offsets is not None and offsets.dtype == torch.int64)
    if z is not None:
        a.z_stride = _token_strides(z)
    return a


class SelectiveScan(torch.autograd.Function):
    """selective_scan with its backward kernels."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, state, offsets, softplus, N, keep_state, record):
        if N != _check_scan(u, delta, A, B, C, D, z, delta_bias, state, offsets)[0]:
            raise RuntimeError(f"{N} sequences are not those of the tensors")
        ctx.shapes = B.shape, C.shape
        inputs = _scan_inputs(u, delta, A, B, C, D, z, delta_bias, state, offsets)
        u, state = inputs[0], inputs[8]
        E, S = inputs[2].shape
        ctx.meta = softplus, N
        ctx.set_materialize_grads(False)
        y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
        last = torch.empty((N, E, S), dtype=torch.float32, device=u.device) if keep_state else None
        if N == 0 or u.shape[1] == 0:
            _state_only(last, state)
            ctx.save_for_backward(*inputs, None)
            return y.zero_(), last
        a = _scan_args(*inputs, softplus, N)
        # the states in front of every sixteenth token, which the backward goes back from
        kept = torch.empty(_lib.lib().vrwkv_scan_kept_bytes(ctypes.byref(a)) // 4, dtype=torch.float32, device=u.device) if record else None
        ctx.save_for_backward(*inputs, kept)
        _set(a, y=y.data_ptr(), last=_pointer(last), kept=_pointer(kept))
        _call("vrwkv_scan_fwd", a, u.device, "vrwkv_scan_fwd_workspace_bytes")
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, glast):
        *inputs, kept = ctx.saved_tensors
        softplus, N = ctx.meta
        if N != _check_scan(*inputs)[0]:                   # (hooks on saved tensors may have moved or changed them)
            raise RuntimeError("the saved tensors have other sizes than those of the call")
        if batched_cotangent(*(t for t in (gy, glast) if t is not None)):
            raise RuntimeError("selective_scan's gradients take one cotangent at a time")
        inputs = _scan_inputs(*inputs)
        u, delta, A, B, C, D, z, delta_bias, state, offsets = inputs
        need = ctx.needs_input_grad
        du, dd, dA, dB, dC, dz = (_like(t, True) for t in (u, delta, A, B, C, z))
        dD, dbias, dstate = _like(D, need[5]), _like(delta_bias, need[7]), _like(state, need[8])
        out = du, dd, dA, dB.view(ctx.shapes[0]), dC.view(ctx.shapes[1]), dD, dz, dbias, dstate, None, None, None, None, None
        if N == 0 or u.shape[1] == 0 or (gy is None and glast is None):
            _zero_all(du, dd, dA, dB, dC, dD, dz, dbias)
            if dstate is not None:
                dstate.zero_() if glast is None else dstate.copy_(glast)
            return out
        gy = torch.zeros_like(u, memory_format=torch.contiguous_format) if gy is None else _tokens(_resolved(gy.to(u.dtype)))
        glast = _resolved(glast.float()).contiguous() if glast is not None else None
        a = _scan_args(*inputs, softplus, N)
        _check(kept, "the kept states", u)
        if kept.dtype != torch.float32 or not kept.is_contiguous() or kept.numel() * 4 != _lib.lib().vrwkv_scan_kept_bytes(ctypes.byref(a)):
            raise RuntimeError("the saved tensors have other sizes than those of the call")
        _set(a, kept=kept.data_ptr(), gy=gy.data_ptr(), gy_stride=_token_strides(gy), glast=_pointer(glast), du=du.data_ptr(), ddelta=dd.data_ptr(), dz=_pointer(dz), dB=dB.data_ptr(),
             dC=dC.data_ptr(), dA=dA.data_ptr(), dstate=_pointer(dstate), dD=_pointer(dD), dbias=_pointer(dbias))
        _call("vrwkv_scan_bwd", a, u.device, "vrwkv_scan_bwd_workspace_bytes")
        return out


def selective_scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, state=None, offsets=None, return_state=False):
    """y (B, T, E), and with return_state the states behind the last tokens (N, E, S) in fp32, of whole sequences.

    u, delta and z (B, T, E), B and C (B, T, S) or (B, T, G, S) of one type (float32, bfloat16, float16), at any strides; channel e reads group e // (E // G) of B and C.
    A (E, S) float32, S 1 to 64, negative where states are to decay.  The step sizes are delta + delta_bias, with softplus log(1 + exp of that); delta_bias and D (E,): u's dtype or float32.
    state: the states in front, (N, E, S) float32, zeros without; N = B.
    offsets (N + 1,), int32 or int64 on the device, ascending from 0 to T: N sequences packed behind each other in one row (B = 1), sequence n the tokens
    offsets[n] to offsets[n + 1] (an empty one leaves its state as it is); y of rows behind the last sequence is zero, and so are their gradients.
    Gradients for all of them, sums in fp32, rounded once to their inputs' types; a call that records keeps the states in front of every sixteenth token for them (S / 16
    fp32 numbers a channel and token, S rounded up to 8, 16, 32 or 64).  No second gradients, no forward mode, no tracing (a compiled program makes the call as it is)."""
    if torch.compiler.is_compiling():
        return _eager(selective_scan)(u, delta, A, B, C, D, z, delta_bias, softplus, state, offsets, return_state)
    out = _lib.host().selective_scan(u, delta, A, B, C, D, z, delta_bias, softplus, state, offsets, return_state)
    if out is not None:
        return out
    tensors = u, delta, A, B, C, D, z, delta_bias, state
    _check_recorders("selective_scan", *tensors, offsets)
    N, _ = _check_scan(*tensors, offsets)
    record = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)
    y, last = SelectiveScan.apply(*tensors, offsets, bool(softplus), N, bool(return_state), record)
    return (y, last) if return_state else y


def selective_scan_step(u, delta, A, B, C, pool, slots=None, D=None, z=None, delta_bias=None, softplus=False):
    """y (N, E) for one more token of each of N sequences, whose states are pages of `pool` (P, E, S) in float32 and are updated in place.

    u, delta, z (N, E), B and C (N, S) or (N, G, S), the others as in selective_scan; slots as in decay_attention_step: row n's page, 0, 1, .. without; rows that name the same
    page are tokens behind each other; -1 gives zeros and touches nothing, any other slot outside the pool NaN.  Forward only: inputs that want gradients or carry
    tangents are refused, and so is tracing."""
    if torch.compiler.is_compiling():
        return _eager(selective_scan_step)(u, delta, A, B, C, pool, slots, D, z, delta_bias, softplus)
    y = _lib.host().selective_scan_step(u, delta, A, B, C, pool, slots, D, z, delta_bias, softplus)
    if y is not None:
        return y
    tensors = u, delta, A, B, C, D, z, delta_bias
    _check_recorders("selective_scan_step", *tensors, pool, slots)
    E, S, G = _check_scan_inputs(*tensors, 1)
    N = u.shape[0]
    _check_pool(pool, "pool", (E, S), torch.float32, u)
    slots = _check_slots(_resolved(slots), pool, N, u)
    _no_gradients("selective_scan_step", "selective_scan", *tensors, pool)
    y = torch.empty((N, E), dtype=u.dtype, device=u.device)
    if N == 0:
        return y
    if pool.shape[0] == 0:
        return _outside(y, slots)
    u, delta, z = (_tokens(_resolved(t)) if t is not None else None for t in (u, delta, z))
    A, D, delta_bias = (_resolved(t).contiguous() if t is not None else None for t in (A, D, delta_bias))
    B, C = (_step_group(t) for t in (B, C))
    a = _lib.ScanStepArgs()
    _set(a, u=u.data_ptr(), delta=delta.data_ptr(), A=A.data_ptr(), B=B.data_ptr(), C=C.data_ptr(), D=_pointer(D), z=_pointer(z), delta_bias=_pointer(delta_bias), slots=_pointer(slots),
         pool=pool.data_ptr(), y=y.data_ptr(), u_stride=u.stride(0), delta_stride=delta.stride(0), z_stride=z.stride(0) if z is not None else 0, B_stride=B.stride()[:2], C_stride=C.stride()[:2],
         page_stride=pool.stride(0) if pool.shape[0] > 1 else E * S, N=N, P=pool.shape[0], E=E, S=S, G=G, dtype=_DT[u.dtype], D_dtype=_DT[D.dtype] if D is not None else 0,
         bias_dtype=_DT[delta_bias.dtype] if delta_bias is not None else 0, softplus=bool(softplus), slots64=slots is not None and slots.dtype == torch.int64)
    _call("vrwkv_scan_step", a, u.device)
    _changed(pool)
    return y


def _step_group(t):
    t = _resolved(t)
    t = t if t.dim() == 3 else t.unsqueeze(1)
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()
