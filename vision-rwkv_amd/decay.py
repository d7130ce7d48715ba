"""Causal attention whose state decays head by head, over whole sequences (with gradients) and one token at a time, and the pages its states are kept in.

    S_t = exp(g_t) S_{t-1} + k_t v_t^T          y_t = scale * S_t^T q_t

Beside wkv6, which looks both ways and returns no state, this is the form for sequences that go on: prompts and the tokens behind them, frames of
a video, rows of an image in order.  The reference has no counterpart.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ops import _DT, _forward_mode, _on, _stream_ptr, batched_cotangent


def _eager(f):
    """f as a call that a compiled program makes and does not look into: its kernels take memory, not traces."""
    return torch.compiler.disable(f)


def _check_recorders(name, *tensors):
    """Refuses what a kernel would drop without a word: recordings of tensor operations, in which it leaves no trace, tangents, and tensors whose memory is
    elsewhere."""
    if torch.jit.is_tracing() or torch._C._get_dispatch_mode(torch._C._TorchDispatchModeKey.PROXY) is not None:
        raise RuntimeError(f"{name} cannot be traced")
    for t in tensors:
        if not isinstance(t, torch.Tensor):
            continue
        if _forward_mode() and (t.is_floating_point() or t.is_complex()) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{name} has no forward mode")
        if t.is_cuda and t.numel() and not t.data_ptr():
            raise RuntimeError(f"{name} takes tensors with memory of their own")


def _resolved(t):
    """t with the values that its memory holds (a view of another's imaginary part may be marked as negated)."""
    return t.resolve_conj().resolve_neg() if isinstance(t, torch.Tensor) else t


def _check_in_place(t, name):
    if t.is_neg() or t.is_conj():
        raise RuntimeError(f"{name} is a negated or conjugated view: it cannot be written in place")


def _rows(t):
    """t as the kernels read it: any strides, but the channels of a head side by side and tokens less than 2^22 elements apart."""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) and (t.dim() == 3 or t.stride(1) < 1 << 22) else t.contiguous()


def _check(t, name, like=None):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if like is not None and t.device != like.device:
        raise RuntimeError(f"{name} must be on {like.device}, as the others")


def _check_sizes(*shapes):
    if any(n > 0x7fffffff for shape in shapes for n in shape):
        raise RuntimeError("a size of 2^31 or more")       # (the library's are 32 bits)


def _check_scale(scale):
    if isinstance(scale, torch.Tensor):                    # (it would go in without its gradient)
        raise RuntimeError("scale must be a number")
    return float(scale)


def _check_heads(q, k, v, g, lead):
    """The numbers of heads and the head sizes of q, k, v, g with `lead` dimensions in front of the heads."""
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (g, "g")):
        _check(t, n, q if t is not q else None)
    if q.dim() != lead + 2 or k.dim() != lead + 2 or v.dim() != lead + 2 or k.shape[:lead] != q.shape[:lead] or v.shape[:lead] != q.shape[:lead]:
        raise RuntimeError(f"q, k and v must be ({'B, T' if lead == 2 else 'N'}, heads, channels) of the same {'batch and tokens' if lead == 2 else 'rows'}")
    if k.shape[-1] != q.shape[-1]:
        raise RuntimeError(f"q has {q.shape[-1]} channels a head, k {k.shape[-1]}")
    if q.dtype not in _DT or k.dtype != q.dtype or v.dtype != q.dtype:
        raise RuntimeError("q, k and v must share one of float32 / bfloat16 / float16")
    if g.dtype != torch.float32 and g.dtype != q.dtype:
        raise RuntimeError("g must be float32 or have the dtype of q, k, v")
    if g.dim() != 1 and (g.dim() != lead + 1 or g.shape[:lead] != q.shape[:lead]):
        raise RuntimeError(f"g must be ({'B, T' if lead == 2 else 'N'}, H), or (H,) for one decay a head")
    _check_sizes(*(t.shape for t in (q, k, v, g)))
    H = g.shape[-1]
    if H == 0 or any(t.shape[-2] == 0 or H % t.shape[-2] for t in (q, k, v)):
        raise RuntimeError(f"the heads of q, k and v ({q.shape[-2]}, {k.shape[-2]}, {v.shape[-2]}) must each divide those of g ({H})")
    Dk, Dv = q.shape[-1], v.shape[-1]
    if not (1 <= Dk <= 128 and 1 <= Dv <= 128):
        raise RuntimeError(f"head sizes ({Dk}, {Dv}) must be 1 to 128")
    return H, Dk, Dv


def _check_index(t, name, like):
    _check(t, name, like)
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name} must be a vector of int32 or int64")
    return t.contiguous()


def _check_call(q, k, v, g, state, offsets):
    """decay_attention's checks; the numbers of sequences and heads."""
    H, Dk, Dv = _check_heads(q, k, v, g, 2)
    N = q.shape[0]
    if offsets is not None:
        _check_index(offsets, "offsets", q)
        if q.shape[0] != 1 or offsets.numel() < 1:
            raise RuntimeError("packed sequences (offsets) come as one row, B = 1, with N + 1 offsets")
        N = offsets.numel() - 1
    if state is not None:
        _check(state, "state", q)
        if tuple(state.shape) != (N, H, Dk, Dv) or state.dtype != torch.float32:
            raise RuntimeError(f"state must be float32 of shape {(N, H, Dk, Dv)}")
    return N, H


def _strides(t):
    """Strides of batch, token and head; a row of one token has none to a next one, whatever the view says."""
    return t.stride(0), 0 if t.shape[1] == 1 else t.stride(1), t.stride(2)


def _call(name, args, device, ws_name=None):
    L = _lib.lib()
    with _on(device):
        if ws_name is not None:
            size = getattr(L, ws_name)(args)
            ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
            args.workspace, args.workspace_bytes = ws.data_ptr() if size else None, size
        _lib.check(getattr(L, name)(args, _stream_ptr(device)))


def _decay_args(q, k, v, g, state, offsets, scale, N, H):
    """vrwkv_decay_args of the inputs."""
    a = _lib.DecayArgs()
    a.q, a.k, a.v, a.g = q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr()
    a.state = state.data_ptr() if state is not None else None
    a.offsets = offsets.data_ptr() if offsets is not None else None
    for name, t in (("q_stride", q), ("k_stride", k), ("v_stride", v)):
        setattr(a, name, _strides(t))
    a.g_stride = (0, 0, g.stride(0)) if g.dim() == 1 else _strides(g)
    a.N, a.T, a.H, a.Hq, a.Hk, a.Hv, a.Dk, a.Dv = N, q.shape[1], H, q.shape[2], k.shape[2], v.shape[2], q.shape[3], v.shape[3]
    a.dtype, a.g_dtype, a.g_per_head, a.offsets64, a.scale = _DT[q.dtype], _DT[g.dtype], g.dim() == 1, offsets is not None and offsets.dtype == torch.int64, scale
    return a


class DecayAttention(torch.autograd.Function):
    """decay_attention with its backward kernels."""

    @staticmethod
    def forward(ctx, q, k, v, g, state, offsets, scale, N, H, keep_state):
        q, k, v, g, state, offsets = (_resolved(t) for t in (q, k, v, g, state, offsets))
        if (N, H) != _check_call(q, k, v, g, state, offsets):
            raise RuntimeError(f"{N} sequences and {H} heads are not those of the tensors")
        offsets = offsets.contiguous() if offsets is not None else None
        q, k, v = _rows(q), _rows(k), _rows(v)
        g = g if g.dim() == 1 or g.stride(1) < 1 << 22 else g.contiguous()
        state = state.contiguous() if state is not None else None
        ctx.save_for_backward(q, k, v, g, state, offsets)
        ctx.meta = scale, N, H
        ctx.set_materialize_grads(False)
        y = torch.empty((*q.shape[:2], H, v.shape[3]), dtype=q.dtype, device=q.device)
        last = torch.empty((N, H, q.shape[3], v.shape[3]), dtype=torch.float32, device=q.device) if keep_state else None
        if N == 0 or q.shape[1] == 0:                      # no token anywhere: the states stay what they are
            if last is not None:
                last.zero_() if state is None else last.copy_(state)
            return y.zero_(), last
        a = _decay_args(q, k, v, g, state, offsets, scale, N, H)
        a.y, a.last = y.data_ptr(), last.data_ptr() if keep_state else None
        _call("vrwkv_decay_fwd", a, q.device, "vrwkv_decay_fwd_workspace_bytes")
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, gy, glast):
        q, k, v, g, state, offsets = ctx.saved_tensors
        scale, N, H = ctx.meta
        if (N, H) != _check_call(q, k, v, g, state, offsets):   # (hooks on saved tensors may have moved or changed them)
            raise RuntimeError("the saved tensors have other sizes than those of the call")
        q, k, v, g, state, offsets, gy, glast = (_resolved(t) for t in (q, k, v, g, state, offsets, gy, glast))
        if batched_cotangent(*(t for t in (gy, glast) if t is not None)):
            raise RuntimeError("decay_attention's gradients take one cotangent at a time")
        q, k, v = _rows(q), _rows(k), _rows(v)
        g = g if g.dim() == 1 or g.stride(1) < 1 << 22 else g.contiguous()
        state, offsets = (t.contiguous() if t is not None else None for t in (state, offsets))
        new = lambda t, need: torch.empty(t.shape, dtype=t.dtype, device=t.device) if need else None
        dq, dk, dv, dg, dstate = (new(t, n) for t, n in zip((q, k, v, g, state), ctx.needs_input_grad[:5]))
        out = dq, dk, dv, dg, dstate, None, None, None, None, None
        if N == 0 or q.shape[1] == 0 or (gy is None and glast is None):
            for t in (dq, dk, dv, dg):
                if t is not None:
                    t.zero_()
            if dstate is not None:
                dstate.zero_() if glast is None else dstate.copy_(glast)
            return out
        gy = torch.zeros((*q.shape[:2], H, v.shape[3]), dtype=q.dtype, device=q.device) if gy is None else _rows(gy.to(q.dtype))
        glast = glast.float().contiguous() if glast is not None else None
        a = _decay_args(q, k, v, g, state, offsets, scale, N, H)
        a.gy, a.gy_stride = gy.data_ptr(), _strides(gy)
        for name, t in (("glast", glast), ("dq", dq), ("dk", dk), ("dv", dv), ("dg", dg), ("dstate", dstate)):
            setattr(a, name, t.data_ptr() if t is not None else None)
        _call("vrwkv_decay_bwd", a, q.device, "vrwkv_decay_bwd_workspace_bytes")
        return out


def decay_attention(q, k, v, g, scale=1.0, state=None, offsets=None, return_state=False):
    """y (B, T, H, Dv), and with return_state the states behind the last tokens (N, H, Dk, Dv) in fp32, of whole sequences.

    q (B, T, Hq, Dk), k (B, T, Hk, Dk), v (B, T, Hv, Dv) of one type (float32, bfloat16, float16), at any strides; each number of heads divides H, and
    head h reads head h // (H // Hq) of q, and so on.  g: log decays, (B, T, H) or one for each head (H,), float32 or q's type; zero keeps, -inf
    forgets.  Head sizes 1 to 128.  state: the states in front, (N, H, Dk, Dv) float32, zeros without; N = B.
    offsets (N + 1,), int32 or int64 on the device, ascending from 0 to T: N sequences packed behind each other in one row (B = 1), sequence n the tokens
    offsets[n] to offsets[n + 1] (an empty one leaves its state as it is); y of rows behind the last sequence is zero, and so are their gradients.
    Gradients for q, k, v, g and state, sums in fp32 (those of (H,) decays in 64 bits), rounded once to their inputs' types; no second ones, no
    forward mode, no tracing (a compiled program makes the call as it is)."""
    if torch.compiler.is_compiling():
        return _eager(decay_attention)(q, k, v, g, scale, state, offsets, return_state)
    scale = _check_scale(scale)
    out = _lib.host().decay_attention(q, k, v, g, scale, state, offsets, return_state)
    if out is not None:
        return out
    _check_recorders("decay_attention", q, k, v, g, state, offsets)
    N, H = _check_call(q, k, v, g, state, offsets)
    y, last = DecayAttention.apply(q, k, v, g, state, offsets, scale, N, H, bool(return_state))
    return (y, last) if return_state else y


def decay_attention_step(q, k, v, g, pool, slots=None, scale=1.0):
    """y (N, H, Dv) for one more token of each of N sequences, whose states are pages of `pool` (P, H, Dk, Dv) in float32 and are updated in place.

    q (N, Hq, Dk), k (N, Hk, Dk), v (N, Hv, Dv) and g (N, H) or (H,) as in decay_attention.  slots (N,), int32 or int64 on the device: row n's
    page, 0, 1, .. without.  Rows that name the same page are tokens behind each other, in their order.  A row of slot -1 (a place of the batch that is not
    taken) gives zeros and touches nothing, one of any other slot outside the pool NaN.  Pages may lie at any distance (pool[:, layer] of a pool for all
    layers), each contiguous.  Forward only: inputs that want gradients or carry tangents are refused, and so is tracing."""
    if torch.compiler.is_compiling():
        return _eager(decay_attention_step)(q, k, v, g, pool, slots, scale)
    scale = _check_scale(scale)
    y = _lib.host().decay_step(q, k, v, g, pool, slots, scale)
    if y is not None:
        return y
    _check_recorders("decay_attention_step", q, k, v, g, pool, slots)
    q, k, v, g, slots = (_resolved(t) for t in (q, k, v, g, slots))
    H, Dk, Dv = _check_heads(q, k, v, g, 1)
    N = q.shape[0]
    _check(pool, "pool", q)
    _check_in_place(pool, "pool")
    _check_sizes(pool.shape)
    if pool.dim() != 4 or tuple(pool.shape[1:]) != (H, Dk, Dv) or pool.dtype != torch.float32 or not _pages_fit(pool):
        raise RuntimeError(f"pool must be float32 (P, {H}, {Dk}, {Dv}) with contiguous pages")
    if slots is not None:
        slots = _check_index(slots, "slots", q)
        if slots.numel() != N:
            raise RuntimeError(f"{slots.numel()} slots for {N} rows")
    elif N > pool.shape[0]:
        raise RuntimeError(f"{N} rows without slots, and {pool.shape[0]} pages")
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, g, pool)):
        raise RuntimeError("decay_attention_step has no backward: call it under torch.no_grad(), or decay_attention")
    y = torch.empty((N, H, Dv), dtype=q.dtype, device=q.device)
    if N == 0:
        return y
    if pool.shape[0] == 0:                                 # no page: every slot lies outside
        return y.copy_(torch.where(slots == -1, 0.0, float("nan"))[:, None, None].expand_as(y))
    q, k, v = _rows(q), _rows(k), _rows(v)
    a = _lib.DecayStepArgs()
    a.q, a.k, a.v, a.g, a.pool, a.y = q.data_ptr(), k.data_ptr(), v.data_ptr(), g.data_ptr(), pool.data_ptr(), y.data_ptr()
    a.slots = slots.data_ptr() if slots is not None else None
    for name, t in (("q_stride", q), ("k_stride", k), ("v_stride", v)):
        setattr(a, name, (t.stride(0), t.stride(1)))
    a.g_stride = (0, g.stride(0)) if g.dim() == 1 else g.stride()
    a.page_stride = pool.stride(0) if pool.shape[0] > 1 else H * Dk * Dv
    a.N, a.P, a.H, a.Hq, a.Hk, a.Hv, a.Dk, a.Dv = N, pool.shape[0], H, q.shape[1], k.shape[1], v.shape[1], Dk, Dv
    a.dtype, a.g_dtype, a.slots64, a.scale = _DT[q.dtype], _DT[g.dtype], slots is not None and slots.dtype == torch.int64, scale
    _call("vrwkv_decay_step", a, q.device)
    _changed(pool)
    return y


def _changed(pool):
    if not pool.is_inference():                            # (those have no version)
        torch.autograd.graph.increment_version(pool)


def _pages_fit(pool):
    """Whether every page of pool (P, ...) is contiguous and none overlaps another."""
    want = 1
    for size, stride in zip(reversed(pool.shape[1:]), reversed(pool.stride()[1:])):
        if size != 1 and stride != want:
            return False
        want *= size
    return pool.shape[0] <= 1 or pool.stride(0) >= want


def _page_index(t, name, pool, lowest, pages):
    """A page list on the pool's device; one that comes from the host is looked through first."""
    if isinstance(t, torch.Tensor) and t.is_cuda:
        return _check_index(t, name, pool)
    t = torch.as_tensor(t)
    if t.numel() == 0:
        t = t.to(torch.int64)
    if t.dim() != 1 or t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name} must be a vector of int32 or int64")
    if t.numel() and not (lowest <= int(t.min()) and int(t.max()) < pages):
        raise RuntimeError(f"{name} names pages outside -1 .. {pages - 1}")
    return t.to(pool.device)


def copy_states(pool, src, dst, source=None):
    """Page dst[i] of `pool` (P, ...) becomes page src[i] of `source` (by default the pool itself) as it was before the call; returns the pool.

    One list forks a state (one src, several dst), moves pages together (over pages that move as well, in any order), exchanges them, copies them in
    from another pool or out to one.  src -1 clears the page, dst -1 is a place of the list that is not taken; of several entries with the same dst the
    last counts.  src, dst: vectors of up to 4096 int32 or int64, on the device -- where entries outside the pools are left out -- or on the host, where
    they are refused.  Pools of any type whose pages are contiguous, at any distance; a source is the pool, or its pages overlap none of
    the pool's: memory of its own, or gaps between the pool's pages at the same distance (pool[:, 0] and pool[:, 1] of a pool for all layers, or one page of it).  No gradients, tangents or tracing, as in decay_attention_step."""
    if torch.compiler.is_compiling():
        return _eager(copy_states)(pool, src, dst, source)
    if _lib.host().copy_pages(pool, src, dst, source):
        return pool
    _check_recorders("copy_states", pool, src, dst, source)
    _check(pool, "pool")
    _check_in_place(pool, "pool")
    source = pool if source is None else source
    _check(source, "source", pool)
    src, dst, source = _resolved(src), _resolved(dst), _resolved(source)
    if pool.dim() < 1 or source.shape[1:] != pool.shape[1:] or source.dtype != pool.dtype:
        raise RuntimeError("pool and source must hold pages of one shape and type")
    _check_sizes(pool.shape[:1], source.shape[:1])
    if not _pages_fit(pool) or not _pages_fit(source):
        raise RuntimeError("the pages of pool and source must be contiguous and apart")
    if torch.is_grad_enabled() and (pool.requires_grad or source.requires_grad):
        raise RuntimeError("copy_states has no backward: call it under torch.no_grad()")
    src, dst = _page_index(src, "src", pool, -1, source.shape[0]), _page_index(dst, "dst", pool, -1, pool.shape[0])
    M = src.numel()
    if dst.numel() != M:
        raise RuntimeError(f"{M} pages in src, {dst.numel()} in dst")
    if M > 4096:
        raise RuntimeError(f"{M} entries, at most 4096")
    size = pool.element_size()
    page = pool.numel() // max(pool.shape[0], 1) * size
    if M == 0 or pool.shape[0] == 0 or page == 0:
        return pool
    empty = source.shape[0] == 0                           # nothing to read: only -1 is inside
    origin, pages = (pool, 0) if empty else (source, source.shape[0])
    distance = lambda t: t.stride(0) * size if t.shape[0] > 1 else page
    L = _lib.lib()
    ws = torch.empty(L.vrwkv_copy_pages_workspace_bytes(M), dtype=torch.uint8, device=pool.device)
    with _on(pool.device):
        _lib.check(L.vrwkv_copy_pages(pool.data_ptr(), distance(pool), pool.shape[0], origin.data_ptr(), distance(origin), pages, page,
                                      src.data_ptr(), src.dtype == torch.int64, dst.data_ptr(), dst.dtype == torch.int64, M,
                                      ws.data_ptr() if ws.numel() else None, ws.numel(), _stream_ptr(pool.device)))
    _changed(pool)
    return pool
