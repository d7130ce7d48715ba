"""decay_attention, decay_attention_step and copy_states at the edges of what they take: sums that cancel, infinities and NaN, what is refused, and the ways
through the kernels that ordinary sizes do not take.

The reference and the bounds of ordinary results are those of test_decay_attention_gpu.py."""
import math

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import vision_rwkv_amd as vr
from test_decay_attention_gpu import DEV, DT, HALF_STEP, check_all, make, reference


def short(x, bits):
    """x with `bits` bits of mantissa."""
    m, e = torch.frexp(x)
    return torch.ldexp(torch.round(m * 2.0 ** bits) / 2.0 ** bits, e)


def pairs(x, first, second):
    """Rows (B, n, ..) as (B, 2 n, ..): each row times `first`, and behind it times `second`."""
    return torch.stack([first * x, second * x], 2).flatten(1, 2)


def cancelled(got, spread, what):
    """Bound: terms that cancel leave the rounding of their running sum, whose size is their root of squares: 2^-24 of it a step, of random sign, for the up
    to 64 sums that a matrix instruction and the chunk's terms make: 2^-21.  A factor of 16 bits would leave 2^-19.3 (an error of up to half a step
    of 2^-17, evenly spread, times 2^-0.8)."""
    err = got.detach().double().cpu().norm() / spread.norm()
    assert err <= 2.0 ** -21, f"{what}: 2^{math.log2(err):.1f}"


@pytest.mark.gpu
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 64), (100, 72)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_sums_that_cancel_keep_32_bits(dtype, Dk, Dv):
    """Of 16-bit rows: tokens two by two with k and 3 v, then 3 k and -v.  Behind each second one the state is zero, and y and dq are what is left of sums that cancel; with q and
    gy made the same way, dk and dv of each first one."""
    B, n, H = 1, 20, 2
    bits = {"bf16": 6, "fp16": 9}[dtype]
    gen = torch.Generator(DEV).manual_seed(Dk)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    rows = lambda x, a, b: pairs(short(x, bits), a, b).to(DT[dtype])
    free = lambda d: r(B, 2 * n, H, d).to(DT[dtype])
    g = torch.zeros(H, device=DEV)
    wide = lambda *ts: [t.detach().double().cpu().transpose(1, 2) for t in ts]          # (B, H, T, D)
    ahead = torch.ones(2 * n, 2 * n, dtype=torch.float64).tril()

    def run(q, k, v, gy):
        ts = [t.requires_grad_() for t in (q, k, v)]
        y = vr.decay_attention(*ts, g, scale=0.25)
        return [y, *torch.autograd.grad(y, ts, gy)], wide(q, k, v, gy)

    def spread(weights, x):
        """Root of the summed squares of the terms weights (.., t, s) x (.., s, d), as (B, T, H, d)."""
        return ((weights * weights) @ (x * x)).sqrt().transpose(1, 2)
    (y, dq, _, _), (Q, K, V, GY) = run(free(Dk), rows(r(B, n, H, Dk), 1, 3), rows(r(B, n, H, Dv), 3, -1), free(Dv))
    cancelled(y[:, 1::2], spread(0.25 * (Q @ K.mT) * ahead, V)[:, 1::2], "y")
    cancelled(dq[:, 1::2], spread(0.25 * (GY @ V.mT) * ahead, K)[:, 1::2], "dq")
    (_, _, dk, dv), (Q, K, V, GY) = run(rows(r(B, n, H, Dk), 1, 3), free(Dk), free(Dv), rows(r(B, n, H, Dv), 3, -1))
    cancelled(dv[:, 0::2], spread((0.25 * (Q @ K.mT) * ahead).mT, GY)[:, 0::2], "dv")
    cancelled(dk[:, 0::2], spread((0.25 * (GY @ V.mT) * ahead).mT, Q)[:, 0::2], "dk")


@pytest.mark.gpu
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 64)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_states_that_cancel_keep_32_bits(dtype, Dk, Dv):
    """A state whose rows lie two by two as S, -3 S, read with 3 q, q; a state's gradient the same way for dv.  What is left is the rounding of -3 S."""
    H, T = 2, 3
    gen = torch.Generator(DEV).manual_seed(Dv)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    bits = {"bf16": 6, "fp16": 9}[dtype]
    two = lambda x, a, b: torch.stack([a * x, b * x], -1).flatten(-2)
    row = two(short(r(1, T, H, Dk // 2), bits), 3, 1).to(DT[dtype])
    S = two(r(1, H, Dv, Dk // 2), 1, -3).mT.contiguous()
    zk, zv = torch.zeros(1, T, H, Dk, device=DEV, dtype=DT[dtype]), torch.zeros(1, T, H, Dv, device=DEV, dtype=DT[dtype])
    g = torch.zeros(H, device=DEV)
    f = lambda t: t.detach().double().cpu()
    exact = torch.einsum("bthk,bhkv->bthv", f(row), f(S))
    spread = torch.einsum("bthk,bhkv->bthv", f(row) ** 2, f(S) ** 2).sqrt()
    y = vr.decay_attention(row, zk, zv, g, state=S)
    cancelled(f(y) - exact, spread, "y")
    k, v = row.clone(), zv.clone().requires_grad_()
    _, last = vr.decay_attention(zk, k, v, g, return_state=True)
    cancelled(f(torch.autograd.grad(last, v, S)[0]) - exact, spread, "dv")


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
def test_what_the_library_refuses_raises_its_own_error(host, monkeypatch):
    """Calls that every check in front of the library lets through."""
    if not host:
        monkeypatch.setattr(vr._lib, "_host", vr._lib._NoHost)
    z = lambda *s: torch.zeros((1,) * len(s), device=DEV).expand(*s)
    for grads in (False, True):
        g = torch.zeros(2, device=DEV, requires_grad=grads)
        with pytest.raises(vr.VrwkvError, match="too many tokens and heads"):
            vr.decay_attention(z(1 << 18, 1, 1, 1), z(1 << 18, 1, 1, 1), z(1 << 18, 1, 1, 1), g)
        with pytest.raises(vr.VrwkvError, match="elements apart"):
            vr.decay_attention(z(1, 1, 1, 64), z(1, 1, 1, 64), z(1, 1, 1, 64), z(1 << 16).contiguous().requires_grad_(grads))
    x, g = z(1 << 19, 1, 1), torch.zeros(16, device=DEV)
    with pytest.raises(vr.VrwkvError, match="too many rows and heads"):
        vr.decay_attention_step(x, x, x, g, torch.zeros(1, 16, 1, 1, device=DEV), torch.zeros(1 << 19, dtype=torch.int32, device=DEV))
    with pytest.raises(vr.VrwkvError, match="overlaps the pool"):
        pool = torch.zeros(5, 8, device=DEV)
        vr.copy_states(pool[:4], torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV), source=pool[1:])
    q = torch.ones(1, 3, 2, 8, device=DEV)                 # (and the call behind is as before)
    assert torch.isfinite(vr.decay_attention(q, q, q, torch.zeros(2, device=DEV))).all()


def small_calls():
    """{name: (call, its float inputs)} of the three operators."""
    gen = torch.Generator(DEV).manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    q, g, pool = r(1, 5, 2, 8), -r(1, 5, 2).abs(), r(4, 2, 8, 8)
    src, dst = (torch.tensor(x, device=DEV) for x in ([0, 2], [1, 3]))
    return {"attention": (lambda q, g, S: vr.decay_attention(q, q, q, g, state=S), (q, g, pool[:1].clone())),
            "step": (lambda q, g, pool: vr.decay_attention_step(q, q, q, g, pool, src), (q[0, :2], g[0, :2], pool)),
            "pages": (lambda pool, source: vr.copy_states(pool, src, dst, source=source), (pool, r(4, 2, 8, 8)))}


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
@pytest.mark.parametrize("name", ["attention", "step", "pages"])
def test_tangents_are_refused(name, host, monkeypatch):
    if not host:
        monkeypatch.setattr(vr._lib, "_host", vr._lib._NoHost)
    call, args = small_calls()[name]
    for i in range(len(args)):
        before = [a.clone() for a in args]
        for mode in (torch.no_grad, torch.enable_grad):
            with forward_ad.dual_level(), mode():
                dual = [forward_ad.make_dual(a, torch.ones_like(a)) if i == j else a for j, a in enumerate(args)]
                with pytest.raises(RuntimeError):
                    call(*dual)
                call(*(a.clone() for a in args))           # (a level by itself is no tangent)
        assert all(torch.equal(a, b) for a, b in zip(args, before))


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attention", "step", "pages"])
def test_recordings_are_refused(name):
    """A trace would hold the outputs' allocations and nothing that fills them."""
    call, args = small_calls()[name]
    copies = lambda: tuple(a.clone() for a in args)
    want = call(*copies())
    for record in (lambda: torch.jit.trace(call, copies(), check_trace=False), lambda: make_fx(call)(*copies())):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            record()
    assert torch.equal(call(*copies()), want)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["attention", "step", "pages"])
def test_transforms_are_refused(name):
    call, args = small_calls()[name]
    copies = lambda: tuple(a.clone() for a in args)
    for transform in (lambda: torch.func.vmap(call)(*(torch.stack([a, a]) for a in copies())), lambda: torch.func.grad(lambda *a: call(*a).sum())(*copies()),
                      lambda: torch.func.jvp(call, copies(), copies()), lambda: torch.func.functionalize(call)(*copies())):
        with pytest.raises(RuntimeError):
            transform()
    # lists or a state alone that a transform has wrapped: not taken for ones that are not there
    q, g, pool = small_calls()["step"][1]
    before = pool.clone()
    with pytest.raises(RuntimeError):
        torch.func.functionalize(lambda s: vr.decay_attention_step(q, q, q, g, pool, s))(torch.tensor([3, 1], device=DEV))
    with pytest.raises(RuntimeError):
        torch.func.functionalize(lambda s: vr.decay_attention(q[None], q[None], q[None], g[None], state=s))(pool[:1])
    with pytest.raises(RuntimeError):
        torch.func.functionalize(lambda s: vr.copy_states(pool, s, s))(torch.tensor([3, 1], device=DEV))
    assert torch.equal(pool, before)


@pytest.mark.gpu
def test_negated_and_conjugated_views():
    """Tensors whose memory holds the negative or the conjugate of what they are: read as what they are, not written."""
    gen = torch.Generator(DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    neg = torch._neg_view
    q, k, v, g, S, gy = r(2, 5, 2, 8), r(2, 5, 2, 8), r(2, 5, 2, 8), -r(2, 5, 2).abs(), r(2, 2, 8, 8), r(2, 5, 2, 8)
    want = None
    for view in (lambda t: t, lambda t: neg(-t)):
        ts = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
        y, last = vr.decay_attention(*(view(t) for t in ts[:4]), state=view(ts[4]), return_state=True)
        results = [y, last, *torch.autograd.grad(y, ts, view(gy))]
        want = want or results
        assert all(torch.equal(a, b) for a, b in zip(results, want))
    pool, step = S.clone(), [t[:, 0] for t in (q, k, v, g)]
    y = vr.decay_attention_step(*step, S.clone())
    assert torch.equal(vr.decay_attention_step(*(neg(-t) for t in step), pool), y)
    slots = torch.tensor([0, 1], device=DEV)
    with pytest.raises(RuntimeError, match="in place"):
        vr.decay_attention_step(*step, neg(pool), slots)
    assert torch.equal(vr.decay_attention_step(*step, S.clone(), neg(-slots)), y)
    c = torch.complex(r(4, 3), r(4, 3))
    pages = torch.zeros(4, 3, device=DEV, dtype=torch.complex64)
    vr.copy_states(pages, slots, slots + 2, source=c.conj())
    assert torch.equal(pages[2:], c[:2].conj().resolve_conj())
    with pytest.raises(RuntimeError, match="in place"):
        vr.copy_states(pages.conj(), slots, slots + 2)
    vr.copy_states(pages, neg(-slots), neg(-slots), source=c)
    assert torch.equal(pages[:2], c[:2])


@pytest.mark.gpu
def test_the_class_by_itself_checks_what_it_is_given():
    gen = torch.Generator(DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    q, g, S, off = r(2, 6, 2, 8), -r(2, 6, 2).abs(), r(2, 2, 8, 8), torch.tensor([0, 9, 2, 9, 6, 9], device=DEV)[::2]
    good = dict(q=q, k=q, v=q, g=g, state=S, offsets=None, scale=0.5, N=2, H=2, keep=True)
    call = lambda **change: vr.DecayAttention.apply(*{**good, **change}.values())
    for a, b in zip(call(), vr.decay_attention(q, q, q, g, scale=0.5, state=S, return_state=True)):
        assert torch.equal(a, b)
    row = dict(q=q[:1], k=q[:1], v=q[:1], g=g[:1], offsets=off)
    for a, b in zip(call(**row), vr.decay_attention(q[:1], q[:1], q[:1], g[:1], scale=0.5, state=S, offsets=off, return_state=True)):
        assert torch.equal(a, b)
    for change in (dict(N=3), dict(N=1), dict(H=4), dict(H=1), dict(state=S[:1]), dict(k=q[:1]), dict(v=q[:, :5]), dict(g=g[:, :3]), dict(q=q.half()), dict(offsets=off), dict(row, N=3),
                   dict(row, offsets=off.float())):
        with pytest.raises(RuntimeError):
            call(**change)


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
def test_saved_tensors_that_a_hook_has_changed(host, monkeypatch):
    if not host:
        monkeypatch.setattr(vr._lib, "_host", vr._lib._NoHost)
    gen = torch.Generator(DEV).manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    ins = [r(2, 6, 2, 8), r(2, 6, 1, 8), r(2, 6, 2, 4), -r(2, 6, 2).abs(), r(2, 2, 8, 4)]

    def grads(ins, unpack, offsets=None):
        ts = [t.clone().requires_grad_() for t in ins]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), unpack):
            y = vr.decay_attention(*ts[:4], state=ts[4], offsets=offsets)
        return torch.autograd.grad(y, ts, torch.ones_like(y))
    want = grads(ins, lambda t: t)
    far = lambda t: torch.stack([t, t], -1)[..., 0] if t.dtype == torch.float32 else t       # (the same values at other strides)
    for a, b in zip(grads(ins, far), want):
        assert torch.equal(a, b)
    for like in ins:
        shorter = lambda t: t[:1] if t.shape == like.shape else t
        narrower = lambda t: t[..., :-1] if t.shape == like.shape else t
        wider = lambda t: t.double() if t.shape == like.shape else t
        for change in (shorter, narrower, wider):
            with pytest.raises(RuntimeError):
                grads(ins, change)
    row = [t.flatten(0, 1)[None] for t in ins[:4]] + ins[4:]
    for change in (lambda t: t[:-1], lambda t: t.float()):
        with pytest.raises(RuntimeError):
            grads(row, lambda t: change(t) if t.dim() == 1 else t, offsets=torch.tensor([0, 4, 12], device=DEV))


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
def test_one_page_of_a_layer(host, monkeypatch):
    """A pool or a source of a single page between another layer's pages: nothing overlaps, whatever distance its view says."""
    if not host:
        monkeypatch.setattr(vr._lib, "_host", vr._lib._NoHost)
    at = lambda *x: torch.tensor(x, device=DEV)
    layers = torch.randn(6, 3, 2, 8, 8, device=DEV)
    want = layers.clone()
    want[[0, 5], 0] = want[2, 1]
    vr.copy_states(layers[:, 0], at(0, 0), at(0, 5), source=layers[2:3, 1])
    assert torch.equal(layers, want)
    want[3, 2] = want[4, 0]
    vr.copy_states(layers[3:4, 2], at(4), at(0), source=layers[:, 0])
    assert torch.equal(layers, want)
    want[1, 1] = want[5, 2]
    vr.copy_states(layers[1:2, 1], at(0), at(0), source=layers[5:6, 2])
    assert torch.equal(layers, want)
    want[[3, 4], 1] = torch.stack([want[0, 1], torch.zeros_like(want[0, 1])])
    vr.copy_states(layers[:, 1], at(0, -1), at(3, 4), source=layers[:1, 1])        # the pool's own first page
    assert torch.equal(layers, want)
    flat = layers.flatten(1)
    for pool, source in ((flat[:, :128], flat[2:3, 64:192]), (flat[2:3, 64:192], flat[:, :128]), (flat[:, :128], flat[5:, :128]), (flat[5:, 1:129], flat[5:, :128])):
        with pytest.raises(RuntimeError):
            vr.copy_states(pool, at(0), at(0), source=source)
    assert torch.equal(layers, want)


def as_defined(got, want, name, dtype, T, Dk, Dv):
    """NaN where the recurrence in 64 bits has NaN, infinities where it has them, and what is finite within the bounds of ordinary results (compare())."""
    x, (ref, scale) = got.detach().double().cpu(), want
    for what, a, b in (("NaN", torch.isnan(x), torch.isnan(ref)), ("+inf", x == math.inf, ref == math.inf), ("-inf", x == -math.inf, ref == -math.inf)):
        assert torch.equal(a, b), f"{name}: {int((a != b).sum())} of {a.numel()} {what} otherwise"
    good = torch.isfinite(ref)
    inner = (Dk + Dv + 128 + 3 * math.ceil(T / 32)) * 2.0 ** -24
    # (a sum of absolute terms that is not finite belongs to a result that an infinity has reached and left again, as by a decay of -inf: none here)
    limit = HALF_STEP[dtype] * ref.abs() + inner * scale + (2.0 ** -25 if dtype == "fp16" else 0.0) + 1e-30
    over = ((x - ref).abs() / limit)[good & torch.isfinite(scale)]
    assert not over.numel() or over.max() <= 1.0, f"{name}: {over.max():.3g} of the bound"


def poison(ts, marks):
    """Copies of q, k, v, g, S, gy, glast with numbers put where marks say: (tensor, index, value)."""
    ts = {n: t.clone() for n, t in ts.items() if t is not None}
    for n, at, x in marks:
        ts[n][at] = x
    return ts


INF, NAN, HUGE = math.inf, math.nan, 3.4e38                # (finite in fp32; to bf16 it rounds up to infinity)
#   what is where, in a row of 150 tokens; head 1 stays clean
MARKS = {"k inf": [("k", (0, 70, 0, 3), INF)], "v inf": [("v", (0, 70, 0, 3), -INF)], "q inf": [("q", (0, 70, 0, 3), INF)], "v nan": [("v", (0, 40, 0, 5), NAN)], "k nan": [("k", (0, 149, 0, 0), NAN)],
         "q nan": [("q", (0, 0, 0, 0), NAN)], "state inf": [("S", (0, 0, 2, 3), INF)], "state nan": [("S", (0, 0, 2, 3), NAN)], "last v": [("v", (0, 149, 0, 0), INF)],
         "two": [("k", (0, 10, 0, 3), INF), ("v", (0, 130, 0, 1), -INF)], "against": [("v", (0, 20, 0, 3), INF), ("v", (0, 21, 0, 3), -INF)], "g nan": [("g", (0, 80, 0), NAN)],
         "both rows": [("k", (0, 66, 0, 3), INF), ("k", (1, 5, 0, 3), NAN)]}


@pytest.mark.gpu
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 72), (20, 13)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_infinities_and_nan_go_where_the_definition_takes_them(dtype, Dk, Dv):
    """Forwards: from a token to those behind it, and nowhere else."""
    q, k, v, g, S = make(2, 150, 2, 2, 2, 2, Dk, Dv, dtype, state=2, seed=3)
    positive = dict(q=q.abs(), k=k.abs(), v=v, g=g, S=S)   # (an infinity of v comes out as one)
    for name, marks in [*MARKS.items(), ("v inf alone", MARKS["v inf"]), ("last v alone", MARKS["last v"])]:
        ts = poison(positive if "alone" in name else dict(q=q, k=k, v=v, g=g, S=S), marks)
        y, last = vr.decay_attention(*(ts[n] for n in "qkvg"), scale=0.3, state=ts["S"], return_state=True)
        want = reference(*(ts[n] for n in "qkvg"), 0.3, ts["S"], [(0, 0, 150), (1, 0, 150)])
        as_defined(y, want["y"], f"{name}: y", dtype, 150, Dk, Dv)
        as_defined(last, want["last"], f"{name}: last", "fp32", 150, Dk, Dv)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,Dk,Dv", [("fp32", 64, 64), ("bf16", 64, 64), ("bf16", 100, 64), ("fp16", 40, 100)])
def test_infinities_and_nan_in_cut_and_packed_sequences(dtype, Dk, Dv):
    """In front of a cut, in the middle of one, between sequences; the padding behind them holds what it likes."""
    for offsets in (None, [0, 700], [5, 400, 400, 1100, 1150]):
        T = 1160 if offsets else 700
        N = len(offsets) - 1 if offsets else 1
        q, k, v, g, S = make(1, T, 1, 1, 1, 1, Dk, Dv, dtype, state=N, seed=4, strong=0.1)
        bounds = [(0, a, e) for a, e in zip(offsets[:-1], offsets[1:])] if offsets else [(0, 0, T)]
        off = torch.tensor(offsets, device=DEV) if offsets else None
        for name, marks in (("early", [("k", (0, 30, 0, 3), INF)]), ("late", [("v", (0, 620, 0, 3), NAN)]), ("cut", [("v", (0, 447, 0, 0), INF), ("k", (0, 448, 0, 1), INF)]),
                            ("outside", [(n, (0, slice(1150, None)), NAN) for n in "qkvg"] if offsets and offsets[0] else [("q", (0, 5, 0, 0), INF)])):
            ts = poison(dict(q=q, k=k, v=v, g=g, S=S), marks)
            y, last = vr.decay_attention(*(ts[n] for n in "qkvg"), scale=0.3, state=ts["S"], offsets=off, return_state=True)
            want = reference(*(ts[n] for n in "qkvg"), 0.3, ts["S"], bounds)
            as_defined(y, want["y"], f"{offsets} {name}: y", dtype, T, Dk, Dv)
            as_defined(last, want["last"], f"{offsets} {name}: last", "fp32", T, Dk, Dv)


@pytest.mark.gpu
def test_finite_numbers_above_those_of_bf16():
    """fp32 rows and states near the type's largest number; products that stay in range."""
    q, k, v, g, S = make(1, 100, 2, 2, 2, 2, 64, 64, "fp32", state=1, seed=6)
    k, q = k * 1e-3, q * 1e-2
    for name, marks in (("v", [("v", (0, 50, 0, 3), HUGE)]), ("state", [("S", (0, 0, 2, 3), -HUGE)]), ("small k", [("k", (0, 50, 0), 1e-30), ("v", (0, 50, 0), HUGE)])):
        ts = poison(dict(q=q, k=k, v=v, g=g, S=S), marks)
        y, last = vr.decay_attention(*(ts[n] for n in "qkvg"), scale=0.3, state=ts["S"], return_state=True)
        want = reference(*(ts[n] for n in "qkvg"), 0.3, ts["S"], [(0, 0, 100)])
        assert torch.isfinite(want["y"][0]).all() and torch.isfinite(want["last"][0]).all()
        as_defined(y, want["y"], f"{name}: y", "fp32", 100, 64, 64)
        as_defined(last, want["last"], f"{name}: last", "fp32", 100, 64, 64)


def gradients_as_defined(ts, marks, dtype, what, offsets=None, scale=0.3):
    """Of all inputs (a decay a token or a head), against the recurrence."""
    ts = poison(ts, marks)
    T = ts["q"].shape[1]
    bounds = [(b, 0, T) for b in range(ts["q"].shape[0])] if offsets is None else [(0, a, e) for a, e in zip(offsets[:-1], offsets[1:])]
    names = [n for n in "qkvgS" if n in ts]
    leaves = [ts[n].clone().requires_grad_() for n in names]
    y, last = vr.decay_attention(*leaves[:4], scale=scale, state=leaves[4] if "S" in ts else None, offsets=torch.tensor(offsets, device=DEV) if offsets else None, return_state=True)
    got = torch.autograd.grad((y, last), leaves, (ts["gy"], ts["gl"]))
    want = reference(*(ts[n] for n in "qkvg"), scale, ts.get("S"), bounds, ts["gy"], ts["gl"])
    for n, x in zip(names, got):
        kind = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}[x.dtype]
        as_defined(x, want["dstate" if n == "S" else "d" + n], f"{what}: d{n}", kind, T, ts["q"].shape[-1], ts["v"].shape[-1])


def backward_inputs(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype, N, g="fp32", seed=3, strong=1.0):
    q, k, v, g, S = make(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype, g=g, state=N, seed=seed, strong=strong)
    gen = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    return dict(q=q, k=k, v=v, g=g, S=S, gy=r(B, T, H, Dv).to(q.dtype), gl=r(N, H, Dk, Dv))


BACK_MARKS = {**MARKS, "gy inf": [("gy", (0, 70, 0, 3), INF)], "gy nan": [("gy", (0, 149, 0, 3), NAN)], "gl inf": [("gl", (0, 0, 2, 3), INF)], "gl nan": [("gl", (1, 0, 2, 3), NAN)]}


@pytest.mark.gpu
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (72, 128), (20, 13)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_gradients_of_infinities_and_nan(dtype, Dk, Dv):
    """Backwards: into the gradients that the formulas give them to."""
    ts = backward_inputs(2, 150, 2, 2, 2, 2, Dk, Dv, dtype, 2)
    for name, marks in BACK_MARKS.items():
        gradients_as_defined(ts, marks, dtype, name)
    ts.update({n: ts[n].abs() for n in ("q", "k", "gl")})  # (an infinity of v or gy comes out as one)
    for name in ("v inf", "gy inf", "last v"):
        gradients_as_defined(ts, BACK_MARKS[name], dtype, name + ", positive")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,Dk,Dv,g", [("fp32", 64, 64, "fp32"), ("bf16", 64, 64, "head"), ("bf16", 100, 64, "same"), ("fp16", 40, 100, "fp32")])
def test_gradients_of_infinities_and_nan_in_cut_and_packed_sequences(dtype, Dk, Dv, g):
    for offsets in (None, [0, 700], [5, 400, 400, 1100, 1150]):
        T = 1160 if offsets else 700
        ts = backward_inputs(1, T, 2, 1, 2, 1, Dk, Dv, dtype, len(offsets) - 1 if offsets else 1, g=dtype if g == "same" else g, seed=4, strong=0.1)
        for name, marks in (("early", [("k", (0, 30, 0, 3), INF)]), ("late", [("v", (0, 620, 0, 3), NAN)]), ("cut", [("v", (0, 447, 0, 0), INF), ("gy", (0, 448, 0, 1), INF)]),
                            ("outside", [(n, (0, slice(1150, None)), NAN) for n in ("q", "k", "v", "gy") + (("g",) if g != "head" else ())] if offsets and offsets[0] else [("q", (0, 5, 0, 0), INF)]),
                            ("end", [("gl", (-1, 0, 0, 0), INF)])):
            gradients_as_defined(ts, marks, dtype, f"{offsets} {name}", offsets)


@pytest.mark.gpu
def test_gradients_of_numbers_above_those_of_bf16():
    ts = backward_inputs(1, 100, 2, 2, 2, 2, 64, 64, "fp32", 1, seed=6)
    for n in "kqv":
        ts[n] = ts[n] * 1e-3
    ts["S"], ts["gl"] = ts["S"] * 1e-3, ts["gl"] * 1e-3
    for name, marks in (("gy", [("gy", (0, 50, 0, 3), HUGE)]), ("gl", [("gl", (0, 0, 2, 3), HUGE)]), ("S", [("S", (0, 0, 2, 3), -HUGE)])):
        gradients_as_defined(ts, marks, "fp32", name)


@pytest.mark.gpu
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (48, 80), (7, 13), (100, 66)])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_steps_with_infinities_and_nan(dtype, Dk, Dv):
    """Row by row, and as tokens of one page behind each other."""
    N, H = 6, 2
    q, k, v, g, S = make(N, 1, H, H, H, H, Dk, Dv, dtype, state=N, seed=8)
    marks = [("v", (0, 0, 0, 3), INF), ("k", (1, 0, 0, 2), -INF), ("q", (2, 0, 0, 2), INF), ("S", (3, 0, 2, 3), INF), ("v", (4, 0, 0, 1), NAN), ("g", (5, 0, 0), NAN)]
    q[0], k[0] = q[0].abs(), k[0].abs()                    # (so that an infinity of v comes out as one)
    ts = poison(dict(q=q, k=k, v=v, g=g, S=S), marks)
    row = [ts[n][:, 0] for n in "qkvg"]
    pool = ts["S"].clone()
    y = vr.decay_attention_step(*row, pool, scale=0.3)
    want = reference(*(ts[n] for n in "qkvg"), 0.3, ts["S"], [(n, 0, 1) for n in range(N)])
    as_defined(y[:, None], want["y"], "y", dtype, 1, Dk, Dv)
    as_defined(pool, want["last"], "pool", "fp32", 1, Dk, Dv)
    pool = ts["S"].clone()
    y = vr.decay_attention_step(*row, pool, torch.zeros(N, dtype=torch.int32, device=DEV), scale=0.3)
    want = reference(*(t[None] for t in row), 0.3, ts["S"][:1], [(0, 0, N)])
    as_defined(y[None], want["y"], "tokens: y", dtype, N, Dk, Dv)
    as_defined(pool[:1], want["last"], "tokens: pool", "fp32", N, Dk, Dv)


# ---- instances and ways through the kernels that the sizes of test_decay_attention_gpu.py do not take -------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Dk,Dv", [(128, 64), (100, 128), (72, 24)])
def test_cut_sequences_of_large_heads(Dk, Dv, dtype):
    """Outputs of more than 64 channels that start from a segment's state; gradients of cut sequences in two tiles of k and v."""
    q, k, v, g, S = make(1, 700, 2, 2, 1, 2, Dk, Dv, dtype, state=1, strong=0.1)
    check_all(q, k, v, g, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_many_pieces_of_one_sequence(dtype):
    """More segments, forwards and back, than the scan over their states asks for at a time."""
    q, k, v, g, S = make(1, 2100, 1, 1, 1, 1, 16, 24, dtype, state=1, strong=0.02)
    check_all(q, k, v, g, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,D,dtype,state", [(900, 2, 8, "fp32", True), (900, 2, 8, "bf16", True), (800, 1, 128, "fp16", False)])
def test_long_sequences_among_many_short_ones(N, H, D, dtype, state):
    """More sequences than a workgroup has threads, most of a token or none and two that are cut: their segments' places are searched, and a scan in few
    workgroups carries a state along them."""
    lens = np.random.default_rng(N).integers(0, 4, N)
    lens[[N // 3, N - 2]] = 1500, 700
    offsets = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, g, S = make(1, offsets[-1], H, H, H, H, D, D, dtype, state=N if state else None, strong=0.1)
    check_all(q, k, v, g, S, dtype, offsets=offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (128, 80)])
def test_packed_and_cut_in_fp16(Dk, Dv):
    q, k, v, g, S = make(1, 1200, 2, 1, 2, 2, Dk, Dv, "fp16", state=4, strong=0.1)
    check_all(q, k, v, g, S, "fp16", offsets=[0, 700, 701, 701, 1150])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 7, 8, 9, 33, 64, 65])
def test_infinities_in_short_sequences(T):
    """Outputs and gradients; blocks of tokens that are not full, chunks that are."""
    for dtype, g in (("fp32", "fp32"), ("bf16", "head"), ("fp16", "same")):
        ts = backward_inputs(3, T, 2, 2, 1, 2, 24, 40, dtype, 3, g=dtype if g == "same" else g, seed=T)
        marks = [("k", (0, 0, 0, 3), INF), ("v", (1, T - 1, 0, 3), -INF), ("gy", (2, T // 2, 1, 0), NAN)]
        gradients_as_defined(ts, marks, dtype, f"{T}")
        bad = poison(ts, marks)
        y, last = vr.decay_attention(*(bad[n] for n in "qkvg"), scale=0.3, state=bad["S"], return_state=True)
        want = reference(*(bad[n] for n in "qkvg"), 0.3, bad["S"], [(b, 0, T) for b in range(3)])
        as_defined(y, want["y"], f"{T}: y", dtype, T, 24, 40)
        as_defined(last, want["last"], f"{T}: last", "fp32", T, 24, 40)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("offsets", [None, [0, 900, 1000, 1700]])
def test_an_infinite_state_under_decays_that_leave_fp32(offsets, dtype):
    """It stays infinite through segments whose whole decay is below fp32's least number; a token that forgets makes NaN of it.  The gradient of the last states the same way."""
    T, N = (offsets[-1], 3) if offsets else (900, 1)
    ts = backward_inputs(1, T, 2, 2, 2, 2, 64, 64, dtype, N, seed=9)
    ts["g"] = torch.full_like(ts["g"], -0.7)
    for name, marks in (("kept", []), ("forgotten", [("g", (0, 500, 0), -INF)]), ("late", [("g", (0, 890, 0), -INF)])):
        gradients_as_defined(ts, [("S", (0, 0, 2, 3), INF), ("gl", (0, 0, 5, 7), -INF), *marks], dtype, name, offsets)
        y, last = vr.decay_attention(*(poison(ts, marks)[n] for n in "qkvg"), scale=0.3, state=poison(ts, [("S", (0, 0, 2, 3), INF)])["S"],
                                     offsets=torch.tensor(offsets, device=DEV) if offsets else None, return_state=True)
        want = reference(*(poison(ts, marks)[n] for n in "qkvg"), 0.3, poison(ts, [("S", (0, 0, 2, 3), INF)])["S"], [(0, a, e) for a, e in zip(offsets[:-1], offsets[1:])] if offsets else [(0, 0, T)])
        as_defined(y, want["y"], f"{name}: y", dtype, T, 64, 64)
        as_defined(last, want["last"], f"{name}: last", "fp32", T, 64, 64)


@pytest.mark.gpu
def test_a_long_sequence_that_is_nan_from_its_front_on():
    """Its segments start from states that are NaN already, and none goes back to its front: 400 000 tokens take no second."""
    T = 400_000
    q, k, v, g, S = make(1, T, 1, 1, 1, 1, 64, 64, "bf16", seed=2)
    k[0, 0] = NAN
    off = torch.tensor([0, T], device=DEV)
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    vr.decay_attention(q[:, :300], k[:, :300], v[:, :300], g[:, :300])
    begin.record()
    y, last = vr.decay_attention(q, k, v, g, offsets=off, return_state=True)
    end.record()
    torch.cuda.synchronize()
    assert torch.isnan(y).all() and torch.isnan(last).all()
    assert begin.elapsed_time(end) < 200                   # (ms; each of 1 562 segments from the front on would have been 18 s of workgroups on 512 places)


def test_the_workspace_of_many_packed_sequences():
    """States are kept for the segments that there can be, not for every sequence: two to each length of a segment."""
    a, lib = vr._lib.DecayArgs(), vr.lib()
    a.offsets = 4096
    a.N, a.T, a.H, a.Hq, a.Hk, a.Hv, a.Dk, a.Dv = 4096, 4096 * 64, 16, 16, 16, 16, 128, 64
    page = 16 * 128 * 64 * 4
    many = lib.vrwkv_decay_fwd_workspace_bytes(a)
    assert 0 < many <= 2 * (a.T // 256 + 1) * page         # (a segment has 256 tokens or more)
    a.N = 1
    assert 0 < lib.vrwkv_decay_fwd_workspace_bytes(a) <= many
    a.N = 1 << 14
    assert lib.vrwkv_decay_fwd_workspace_bytes(a) == many
