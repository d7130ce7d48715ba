"""decay_attention, decay_attention_step and copy_states on the GPU against the recurrence token by token in 64 bits.

Bounds.  Beside every result the reference forms the same sums of absolute values, A.  With u the half step of the result's type:
  * a 16-bit result is u |x| off by its own rounding, and y and dv carry operands of two bf16 terms (2^-16 each, three of them on the way: 2^-14 A);
  * operands of fp32 rows, of dq, dk and of the states have three terms (2^-24); what is left is the rounding of fp32 sums, one half step of 2^-24 a term at
    most, over Dk + Dv channels, two chunks' tokens and the chunks: N_SUM 2^-24 A, and the exponentials, whose argument is off by 2^-24 of itself:
    at most 2^-24 x e^-x <= 2^-25 each, two of them, in front of the first chunk as many as there are chunks.
A result far inside 16 bits' own step is dominated by it; fp32 results are also held to 2e-6 of their norm: errors of random sign, 2^-24 sqrt(2 N_SUM)
for the 300 to 700 roundings here, 1.5e-6 to 2.2e-6 where every one were a full half step."""
import math

import numpy as np
import pytest
import torch

import vision_rwkv_amd as vr

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def reference(q, k, v, g, scale, state, bounds, gy=None, glast=None):
    """Everything in float64 on the CPU: {name: (value, sum of absolute terms)}.  bounds: [(batch row, first, end)] of the sequences."""
    f = lambda t: t.detach().double().cpu()
    q, k, v, g = f(q), f(k), f(v), f(g)
    B, T = q.shape[:2]
    H = g.shape[-1]
    per_head = g.dim() == 1
    g = g.expand(B, T, H)
    Hq, Hk, Hv, Dk, Dv = q.shape[2], k.shape[2], v.shape[2], q.shape[3], v.shape[3]
    rep = lambda t: t.repeat_interleave(H // t.shape[2], 2)
    q, k, v = rep(q), rep(k), rep(v)
    N = len(bounds)
    S0 = f(state) if state is not None else torch.zeros(N, H, Dk, Dv, dtype=torch.float64)
    out = {}
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)
    for kind, a in (("x", lambda t: t), ("abs", torch.abs)):
        Q, K, V = a(q), a(k), a(v)
        y, last = zeros(B, T, H, Dv), zeros(N, H, Dk, Dv)
        GY = a(f(gy)) if gy is not None else zeros(B, T, H, Dv)
        dq, dk, dv, dg, dS = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(g), zeros(N, H, Dk, Dv)
        sc = abs(scale) if kind == "abs" else scale
        for n, (b, first, end) in enumerate(bounds):
            S, kept = a(S0[n]), []
            for t in range(first, end):
                kept.append(S)
                S = g[b, t].exp()[:, None, None] * S + K[b, t][:, :, None] * V[b, t][:, None, :]
                y[b, t] = sc * (Q[b, t][:, :, None] * S).sum(1)
                dq[b, t] = sc * (S * GY[b, t][:, None, :]).sum(2)
            last[n] = S
            R = a(f(glast)[n]) if glast is not None else zeros(H, Dk, Dv)
            for t in reversed(range(first, end)):
                R = R + sc * Q[b, t][:, :, None] * GY[b, t][:, None, :]
                dk[b, t] = (R * V[b, t][:, None, :]).sum(2)
                dv[b, t] = (R * K[b, t][:, :, None]).sum(1)
                R = g[b, t].exp()[:, None, None] * R
                dg[b, t] = (R * kept[t - first]).sum((1, 2))
            dS[n] = R
        fold = lambda t, h: t.reshape(B, T, h, H // h, t.shape[-1]).sum(3)
        out[kind] = dict(y=y, last=last, dq=fold(dq, Hq), dk=fold(dk, Hk), dv=fold(dv, Hv), dg=dg.sum((0, 1)) if per_head else dg, dstate=dS)
    return {n: (out["x"][n], out["abs"][n]) for n in out["x"]}


def compare(got, want, name, dtype, Dk, Dv, T):
    x, (ref, scale) = got.detach().double().cpu(), want
    assert x.shape == ref.shape, name
    assert torch.isfinite(x).all(), name
    u = HALF_STEP[dtype]
    n_sum = Dk + Dv + 128 + 3 * math.ceil(T / 32)
    inner = n_sum * 2.0 ** -24 + (2.0 ** -14 if dtype != "fp32" and name in ("y", "dv") else 0.0)
    # (per-head decays add up all tokens' gradients, in 64 bits, and round once more)
    limit = u * ref.abs() + inner * scale + 1e-30
    if dtype == "fp16":
        limit = limit + 2.0 ** -25                         # half a step of fp16's subnormal numbers
    over = ((x - ref).abs() / limit).max().item() if x.numel() else 0.0
    assert over <= 1.0, f"{name}: {over:.3g} of the bound"
    if dtype == "fp32" and ref.norm() > 0:
        assert (x - ref).norm() <= 2e-6 * max(ref.norm(), 2.0 ** -4 * scale.norm()), f"{name}: {(x - ref).norm() / ref.norm():.3g}"


def make(B, T, H, Hq, Hk, Hv, Dk, Dv, dtype, g="fp32", seed=0, state=None, strong=1.0):
    gen = torch.Generator(DEV).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV)
    q, k, v = r(B, T, Hq, Dk).to(DT[dtype]), r(B, T, Hk, Dk).to(DT[dtype]), r(B, T, Hv, Dv).to(DT[dtype])
    gate = -strong * torch.exp(r(H) - 2.5) if g == "head" else (-strong * torch.exp(r(B, T, H) - 2.5)).to(DT[g])
    S = r(state, H, Dk, Dv) if state else None
    return q, k, v, gate, S


def check_all(q, k, v, g, S, dtype, scale=0.3, offsets=None, grads=True, seed=1):
    B, T = q.shape[:2]
    N = B if offsets is None else len(offsets) - 1
    bounds = [(b, 0, T) for b in range(B)] if offsets is None else [(0, a, e) for a, e in zip(offsets[:-1], offsets[1:])]
    off = None if offsets is None else torch.tensor(offsets, dtype=torch.int64 if N % 2 else torch.int32, device=DEV)
    H, Dk, Dv = g.shape[-1], q.shape[-1], v.shape[-1]
    leaves = {n: t.detach().clone().requires_grad_(grads) for n, t in zip("qkvgS", (q, k, v, g, S)) if t is not None}
    y, last = vr.decay_attention(*(leaves[n] for n in "qkvg"), scale=scale, state=leaves.get("S"), offsets=off, return_state=True)
    gen = torch.Generator(DEV).manual_seed(seed)
    gy = torch.randn(y.shape, generator=gen, device=DEV).to(y.dtype)
    glast = torch.randn(last.shape, generator=gen, device=DEV) if S is not None else None
    want = reference(q, k, v, g, scale, S, bounds, gy, glast)
    longest = max([e - a for _, a, e in bounds] + [1])
    size = (Dk, Dv, longest)
    compare(y, want["y"], "y", dtype, *size)
    compare(last, want["last"], "last", "fp32", *size)
    if not grads:
        return
    outs, cot = ([y, last], [gy, glast]) if glast is not None else ([y], [gy])
    got = torch.autograd.grad(outs, list(leaves.values()), cot)
    for n, t in zip(leaves, got):
        assert t.dtype == leaves[n].dtype
        kind = {torch.float32: "fp32", torch.bfloat16: "bf16", torch.float16: "fp16"}[t.dtype]
        compare(t, want["dstate" if n == "S" else "d" + n], "dstate" if n == "S" else "d" + n, kind, *size)


SIZES = [(1, 1, 1, 64, 64), (2, 3, 2, 64, 64), (1, 63, 2, 64, 64), (1, 64, 1, 64, 64), (2, 65, 3, 64, 64), (1, 31, 2, 16, 8), (1, 33, 2, 128, 64),
         (1, 130, 2, 64, 128), (2, 97, 1, 128, 128), (1, 70, 2, 48, 80), (1, 129, 1, 1, 1), (1, 40, 2, 7, 13), (1, 200, 1, 127, 65)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("B,T,H,Dk,Dv", SIZES)
def test_sizes(B, T, H, Dk, Dv, dtype):
    q, k, v, g, S = make(B, T, H, H, H, H, Dk, Dv, dtype, state=B if T % 2 else None, seed=T)
    check_all(q, k, v, g, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("H,Hq,Hk,Hv,Dk,Dv,g", [(6, 6, 2, 6, 64, 64, "fp32"), (6, 1, 3, 2, 32, 64, "head"), (4, 2, 2, 4, 128, 96, "same"), (4, 4, 4, 1, 64, 64, "head")])
def test_shared_heads_and_kinds_of_decay(H, Hq, Hk, Hv, Dk, Dv, g, dtype):
    q, k, v, g, S = make(2, 77, H, Hq, Hk, Hv, Dk, Dv, dtype, g=dtype if g == "same" else g, state=2)
    check_all(q, k, v, g, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("offsets", [[0, 5, 5, 70, 71, 200], [0, 0, 0, 130], [0, 64, 128, 150], [3, 60, 100]])
@pytest.mark.parametrize("state", [False, True])
def test_packed(offsets, state, dtype):
    T = offsets[-1] + (9 if offsets[0] else 0)             # rows in front of the first sequence and behind the last
    q, k, v, g, S = make(1, T, 2, 2, 1, 2, 64, 64, dtype, state=len(offsets) - 1 if state else None)
    for t in (q, k, v, g):
        t[:, :offsets[0]] = float("nan")
        t[:, offsets[-1]:] = float("nan")
    zero = lambda t: torch.where(torch.isnan(t), 0, t)
    off = torch.tensor(offsets, device=DEV)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, g)]
    y = vr.decay_attention(*leaves, state=S, offsets=off)
    for t in (y, *torch.autograd.grad(y, leaves, torch.ones_like(y))):
        assert not t[:, :offsets[0]].any() and not t[:, offsets[-1]:].any() and torch.isfinite(t).all()
    check_all(zero(q), zero(k), zero(v), zero(g), S, dtype, offsets=offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("Dk,Dv", [(64, 64), (32, 100)])
def test_cut_into_segments(Dk, Dv, dtype):
    """One sequence of few heads is cut, forward and backward; its parts join as if it were whole."""
    q, k, v, g, S = make(1, 700, 2, 2, 2, 2, Dk, Dv, dtype, state=1, strong=0.1)
    check_all(q, k, v, g, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_packed_and_cut(dtype):
    q, k, v, g, S = make(1, 1200, 2, 2, 2, 2, 64, 64, dtype, state=4, strong=0.1)
    check_all(q, k, v, g, S, dtype, offsets=[0, 700, 701, 701, 1150])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
def test_whole_sequences_of_many_heads(dtype):
    q, k, v, g, S = make(24, 140, 16, 16, 16, 16, 16, 16, dtype, strong=0.2)
    check_all(q, k, v, g, S, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strong_and_missing_decays(dtype):
    """Decays of thousands beside ones of a hundredth, none at all, resets: -inf and the type's lowest value forget what was before."""
    q, k, v, g, S = make(1, 150, 4, 4, 4, 4, 64, 64, dtype, state=1)
    g[0, ::7, 0] = -5000.0
    g[0, :, 1] = 0.0
    g[0, 20::50, 2] = -1000.0
    g[0, ::3, 3] = -40.0
    check_all(q, k, v, g, S, dtype)
    for low in (-math.inf, torch.finfo(torch.float32).min):
        h = g.clone()
        h[0, 20::50, 2] = low
        a, b = (vr.decay_attention(q, k, v, x, state=S, return_state=True) for x in (g, h))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        leaves = [t.clone().requires_grad_() for t in (q, k, v, h, S)]
        y = vr.decay_attention(*leaves[:4], state=leaves[4])
        for t in torch.autograd.grad(y, leaves, torch.ones_like(y)):
            assert torch.isfinite(t).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strides(dtype):
    """Slices of one projection, other orders of dimensions, rows off 16 bytes, expanded heads and decays: as the contiguous copies."""
    B, T, H, D = 2, 50, 3, 64
    gen = torch.Generator(DEV).manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=gen, device=DEV).to(DT[dtype])
    qkv = r(B, T, 3 * H * D + 5)
    slices = [qkv[..., 5 + i * H * D:5 + (i + 1) * H * D].unflatten(-1, (H, D)) for i in range(3)]
    swapped = [r(B, H, T, D).transpose(1, 2) for _ in range(3)]
    last_first = [r(D, B, T, H).permute(1, 2, 3, 0) for _ in range(3)]
    same = [r(B, 1, 1, D).expand(B, T, H, D) for _ in range(3)]
    gates = [-torch.rand(B, H, T, generator=gen, device=DEV).transpose(1, 2), -torch.rand(H, generator=gen, device=DEV).expand(B, T, H)]
    for i, (q, k, v) in enumerate((slices, swapped, last_first, same)):
        g = gates[i % 2]
        S = torch.randn(B, H, D, D, generator=gen, device=DEV).transpose(-1, -2)
        def run(dense):
            ts = [t.detach().clone(memory_format=torch.contiguous_format) if dense else t.detach() for t in (q, k, v, g, S)]
            ts = [t.requires_grad_() for t in ts]
            y, last = vr.decay_attention(*ts[:4], state=ts[4], return_state=True)
            gy = torch.linspace(-1, 1, y.numel(), device=DEV).to(y.dtype).view(B, H, T, D).transpose(1, 2)
            return [y, last, *torch.autograd.grad(y, ts, gy.contiguous() if dense else gy)]
        for a, b in zip(run(False), run(True)):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_gradients_against_differences():
    """fp32, central differences along random directions: the loss is smooth, its third derivative h^2 / 6 small beside 1e-3."""
    q, k, v, g, S = make(1, 40, 2, 1, 2, 2, 16, 24, "fp32", state=1)
    leaves = [t.double().cpu().float().to(DEV).requires_grad_() for t in (q, k, v, g, S)]
    gen = torch.Generator(DEV).manual_seed(9)
    wy, wl = torch.randn(1, 40, 2, 24, generator=gen, device=DEV), torch.randn(1, 2, 16, 24, generator=gen, device=DEV)

    def loss(ts):
        y, last = vr.decay_attention(*ts[:4], scale=0.3, state=ts[4], return_state=True)
        return (y.double() * wy).sum() + (last.double() * wl).sum()
    grads = torch.autograd.grad(loss(leaves), leaves)
    for i, t in enumerate(leaves):
        d = torch.randn(t.shape, generator=gen, device=DEV) * (1.0 if i != 3 else 0.1)
        h = 1e-2
        move = lambda s: [x.detach() + s * h * d if j == i else x.detach() for j, x in enumerate(leaves)]
        num = (loss(move(1)) - loss(move(-1))).item() / (2 * h)
        ana = (grads[i].double() * d).sum().item()
        assert abs(num - ana) <= 2e-3 * max(abs(ana), grads[i].double().norm().item() * d.double().norm().item() / math.sqrt(t.numel())), (i, num, ana)


@pytest.mark.gpu
def test_only_some_gradients():
    q, k, v, g, S = make(1, 90, 2, 2, 1, 2, 64, 64, "bf16", state=1)
    every = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
    y, last = vr.decay_attention(*every[:4], state=every[4], return_state=True)
    full = torch.autograd.grad(y, every, torch.ones_like(y), retain_graph=True)
    from_last = torch.autograd.grad(last, every, torch.ones_like(last))
    assert not from_last[0].any() and all(t.any() for t in from_last[1:])
    for i in range(5):
        some = [t.clone().requires_grad_(i == j) for j, t in enumerate((q, k, v, g, S))]
        y = vr.decay_attention(*some[:4], state=some[4])
        assert torch.equal(torch.autograd.grad(y, some[i], torch.ones_like(y))[0], full[i])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,H,Hq,Hk,Hv,Dk,Dv", [(1, 1, 1, 1, 1, 64, 64), (5, 6, 2, 3, 6, 64, 64), (3, 2, 2, 2, 1, 128, 128), (4, 2, 1, 1, 2, 7, 13), (300, 2, 2, 2, 2, 32, 16), (2, 3, 3, 3, 3, 100, 66)])
def test_step(N, H, Hq, Hk, Hv, Dk, Dv, dtype):
    q, k, v, g, _ = make(1, N, H, Hq, Hk, Hv, Dk, Dv, dtype, seed=N)
    q, k, v, g = q[0], k[0], v[0], g[0]
    P = N + 3
    gen = torch.Generator(DEV).manual_seed(3)
    pool = torch.randn(P, H, Dk, Dv, generator=gen, device=DEV)
    slots = torch.randperm(P, generator=gen, device=DEV)[:N].to(torch.int32 if N % 2 else torch.int64)
    before = pool.clone()
    y = vr.decay_attention_step(q, k, v, g, pool, slots, scale=0.3)
    state = before[slots.long()]
    want = reference(q[:, None], k[:, None], v[:, None], g[:, None], 0.3, state, [(n, 0, 1) for n in range(N)])
    compare(y[:, None], want["y"], "y", dtype, Dk, Dv, 1)
    compare(pool[slots.long()], want["last"], "last", "fp32", Dk, Dv, 1)
    rest = torch.ones(P, dtype=torch.bool, device=DEV)
    rest[slots.long()] = False
    assert torch.equal(pool[rest], before[rest])
    # without slots: pages in order; one decay a head
    pool2 = before.clone()
    y2 = vr.decay_attention_step(q, k, v, g[0].contiguous(), pool2, scale=0.3)
    want = reference(q[:, None], k[:, None], v[:, None], g[0], 0.3, before[:N], [(n, 0, 1) for n in range(N)])
    compare(y2[:, None], want["y"], "y", dtype, Dk, Dv, 1)
    compare(pool2[:N], want["last"], "last", "fp32", Dk, Dv, 1)


@pytest.mark.gpu
def test_step_repeated_missing_and_bad_slots():
    H, D = 2, 64
    q, k, v, g, _ = make(1, 9, H, H, H, H, D, D, "bf16")
    q, k, v, g = q[0], k[0], v[0], g[0]
    layers = torch.randn(6, 3, H, D, D, device=DEV)        # pages of one layer lie three states apart
    before = layers.clone()
    pool = layers[:, 1]
    slots = torch.tensor([2, -1, 5, 2, 6, 2, -7, 0, 1 << 40], device=DEV)
    y = vr.decay_attention_step(q, k, v, g, pool, slots, scale=0.5)
    assert not y[1].any() and all(torch.isnan(y[i]).all() for i in (4, 6, 8))
    order = torch.tensor([0, 3, 5], device=DEV)            # the rows of page 2 are three tokens of one sequence
    want = reference(q[order][None], k[order][None], v[order][None], g[order][None], 0.5, before[2:3, 1], [(0, 0, 3)])
    compare(y[order][None], want["y"], "y", "bf16", D, D, 3)
    compare(pool[2][None], want["last"], "last", "fp32", D, D, 3)
    for i, s in ((2, 5), (7, 0)):
        want = reference(q[i:i + 1, None], k[i:i + 1, None], v[i:i + 1, None], g[i:i + 1, None], 0.5, before[s:s + 1, 1], [(0, 0, 1)])
        compare(y[i:i + 1, None], want["y"], "y", "bf16", D, D, 1)
        compare(pool[s][None], want["last"], "last", "fp32", D, D, 1)
    untouched = [(p, l) for p in range(6) for l in range(3) if l != 1 or p not in (0, 2, 5)]
    for p, l in untouched:
        assert torch.equal(layers[p, l], before[p, l])


def pages_reference(pool, src, dst, source=None):
    source = pool if source is None else source
    out = pool.copy()
    for a, b in zip(src, dst):
        if 0 <= b < len(pool) and -1 <= a < len(source):
            out[b] = source[a] if a >= 0 else 0
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("shape,dtype", [((2, 8, 8), torch.float32), ((3, 5, 7), torch.float32), ((5, 7), torch.bfloat16), ((3,), torch.uint8), ((12, 64, 64), torch.float32)])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("how", ["fork", "shift", "back", "cycle", "swap", "tree", "clear", "mixed", "random"])
def test_pages(how, shape, dtype, long):
    P = 40
    gen = np.random.default_rng(7)
    host = torch.from_numpy(gen.integers(0, 200, (P, *shape))).to(dtype)
    pool = host.to(DEV)
    lists = {"fork": ([3] * 6, [1, 7, 9, 20, 39, 0]), "shift": (list(range(1, 40)), list(range(39))), "back": (list(range(39)), list(range(1, 40))),
             "cycle": ([4, 8, 15, 16, 23], [8, 15, 16, 23, 4]), "swap": ([0, 39], [39, 0]), "tree": ([1, 1, 2, 2, 3, 0, 5], [2, 3, 4, 5, 6, 1, 0]),
             "clear": ([-1, -1, -1], [5, 0, 39]), "mixed": ([5, -1, 7, 50, 9, 9, -3, 2, 30], [7, 5, -1, 9, 40, 9, 11, 2, 30]),
             "random": (gen.integers(-1, P, 60).tolist(), gen.integers(-1, P, 60).tolist())}
    src, dst = lists[how]
    if long:                                               # places that are not taken, up to a list of the length that is planned by itself
        src, dst = src[:1] + [5] * 130 + src[1:] + [-9] * 130, dst[:1] + [-1] * 130 + dst[1:] + [3] * 130
    want = torch.from_numpy(pages_reference(host.float().numpy(), src, dst)).to(dtype)
    out = vr.copy_states(pool, torch.tensor(src, device=DEV, dtype=torch.int32), torch.tensor(dst, device=DEV))
    assert out is pool and torch.equal(pool.cpu(), want)


@pytest.mark.gpu
def test_pages_between_pools_and_long_lists():
    a, b = torch.randn(3000, 2, 4, 4, device=DEV), torch.randn(50, 3, 2, 4, 4, device=DEV)
    host, before = a.cpu().numpy(), b.clone()
    src, dst = list(range(7, 57)), [(7 * i) % 50 for i in range(50)]
    vr.copy_states(b[:, 2], src, dst, source=a)            # lists from the host, a layer of a pool of three
    want = pages_reference(before[:, 2].cpu().numpy(), src, dst, host)
    assert torch.equal(b[:, 2].cpu(), torch.from_numpy(want)) and torch.equal(b[:, :2], before[:, :2])
    gen = np.random.default_rng(0)
    src, dst = gen.integers(-1, 3000, 4096), gen.integers(-1, 3000, 4096)
    vr.copy_states(a, torch.from_numpy(src).to(DEV), torch.from_numpy(dst).to(DEV))
    assert torch.equal(a.cpu(), torch.from_numpy(pages_reference(host, src.tolist(), dst.tolist())))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_prompt_and_the_tokens_behind_it(dtype):
    """Used together: packed prompts, their states into a pool, a fork, steps, pages moved together, steps; as one long sequence each."""
    H, D, lens, more = 3, 64, [70, 1, 133], 5
    full = [make(1, n + 2 * more, H, H, 1, H, D, D, dtype, seed=n)[:4] for n in lens]
    packed = [torch.cat([f[i][:, :n] for f, n in zip(full, lens)], 1) for i in range(4)]
    offsets = torch.tensor([0, 70, 71, 204], device=DEV, dtype=torch.int32)
    ys = [[] for _ in lens]
    with torch.no_grad():
        y, last = vr.decay_attention(*packed, scale=0.2, offsets=offsets, return_state=True)
        for i, (a, e) in enumerate(zip([0, 70, 71], [70, 71, 204])):
            ys[i].append(y[0, a:e])
        pool = torch.full((8, H, D, D), float("nan"), device=DEV)
        vr.copy_states(pool, [0, 1, 2, 2], [6, 3, 5, 1], source=last)       # sequence 2 twice: a fork
        slots = torch.tensor([6, 3, 5, 1], device=DEV, dtype=torch.int32)
        for t in range(2 * more):
            if t == more:
                vr.copy_states(pool, slots, torch.arange(4, device=DEV))    # moved together, over one another
                slots = torch.arange(4, device=DEV)
            rows = [[f[i][0, n + t] for f, n in zip(full, lens)] for i in range(4)]
            q, k, v, g = (torch.stack(r + [r[2]]) for r in rows)
            y = vr.decay_attention_step(q, k, v, g, pool, slots, scale=0.2)
            assert torch.equal(y[2], y[3])
            for i in range(3):
                ys[i].append(y[i:i + 1])
    for i, (f, n) in enumerate(zip(full, lens)):
        want = reference(*f, 0.2, None, [(0, 0, n + 2 * more)])
        compare(torch.cat(ys[i])[None], want["y"], "y", dtype, D, D, n + 2 * more)
        compare(pool[i][None], want["last"], "last", "fp32", D, D, n + 2 * more)


@pytest.mark.gpu
def test_captured_and_replayed():
    """Forward, backward, steps and pages in one graph, replayed on new inputs with eager work between: bit for bit the eager calls."""
    q, k, v, g, S = make(2, 300, 2, 2, 1, 2, 64, 64, "bf16", state=2)
    pool0 = torch.randn(6, 2, 64, 64, device=DEV)
    ins = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
    pool, slots, src, dst = pool0.clone(), torch.tensor([4, 1], device=DEV), torch.tensor([4, 1, 2], device=DEV), torch.tensor([1, 2, 4], device=DEV)
    gy = torch.randn(2, 300, 2, 64, device=DEV).bfloat16()

    def work(ins, pool):
        y, last = vr.decay_attention(*ins[:4], state=ins[4], return_state=True)
        grads = torch.autograd.grad((y, last), ins, (gy, torch.ones_like(last)))
        with torch.no_grad():
            s = vr.decay_attention_step(*(t[:, 0] for t in ins[:4]), pool, slots)
            vr.copy_states(pool, src, dst)
        return [y.detach(), last.detach(), *grads, s]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work([t.detach().clone().requires_grad_() for t in ins], pool0.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(ins, pool)
    for seed in range(3):
        new = make(2, 300, 2, 2, 1, 2, 64, 64, "bf16", state=2, seed=10 + seed)
        with torch.no_grad():
            for t, x in zip(ins, new):
                t.copy_(x)
            pool.copy_(pool0)
        graph.replay()
        torch.cuda.synchronize()
        pool_e = pool0.clone()
        eager = work([t.detach().clone().requires_grad_() for t in new], pool_e)
        for a, b in zip(outs + [pool], eager + [pool_e]):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_on_another_stream_and_twice_at_once():
    q, k, v, g, S = make(1, 2000, 2, 2, 2, 2, 64, 64, "bf16", state=1)
    want = vr.decay_attention(q, k, v, g, state=S, return_state=True)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(vr.decay_attention(q, k, v, g, state=S, return_state=True))
    torch.cuda.synchronize()
    for y, last in got:
        assert torch.equal(y, want[0]) and torch.equal(last, want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("N", [255, 256, 800])
def test_many_short_sequences(N):
    """More sequences than a workgroup reads offsets at once; most of a token or none."""
    lens = np.random.default_rng(N).integers(0, 4, N)
    lens[N // 2] = 70
    offsets = np.concatenate([[0], np.cumsum(lens)]).tolist()
    q, k, v, g, S = make(1, offsets[-1], 2, 2, 2, 2, 8, 8, "fp32", state=N)
    check_all(q, k, v, g, S, "fp32", offsets=offsets)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [3000, 300000])
def test_packed_rows_of_one_token(N):
    """Thousands of packed sequences of one token, empty ones among them, are the rows of a batch of one token each: the same bits."""
    gen = torch.Generator(DEV).manual_seed(N)
    taken = torch.rand(N, generator=gen, device=DEV) < 0.8
    offsets = torch.cat([torch.zeros(1, dtype=torch.long, device=DEV), taken.long().cumsum(0)])
    B = int(offsets[-1])
    q, k, v, g, S = make(B, 1, 1, 1, 1, 1, 8, 8, "fp32", state=N, seed=1)
    gy = torch.randn(B, 1, 1, 8, generator=gen, device=DEV)
    gl = torch.randn(N, 1, 8, 8, generator=gen, device=DEV)

    def run(packed):
        ts = [(t.transpose(0, 1) if packed else t).clone().requires_grad_() for t in (q, k, v, g)] + [(S if packed else S[taken]).clone().requires_grad_()]
        y, last = vr.decay_attention(*ts[:4], scale=0.5, state=ts[4], offsets=offsets if packed else None, return_state=True)
        grads = torch.autograd.grad((y, last), ts, (gy.transpose(0, 1), gl) if packed else (gy, gl[taken]))
        return [y, *grads[:4]], last, grads[4]
    rows, last, dstate = run(True)
    want_rows, want_last, want_dstate = run(False)
    for a, b in zip(rows, want_rows):
        assert torch.equal(a.transpose(0, 1), b)
    assert torch.equal(last[taken], want_last) and torch.equal(last[~taken], S[~taken])
    assert torch.equal(dstate[taken], want_dstate) and torch.equal(dstate[~taken], gl[~taken])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_the_same_without_the_host_module(dtype, monkeypatch):
    """Through the Python classes: the same kernels, bit for bit."""
    q, k, v, g, S = make(2, 150, 4, 2, 1, 4, 64, 80, dtype, state=2)
    gen = torch.Generator(DEV).manual_seed(2)
    gy, gl = torch.randn(2, 150, 4, 80, generator=gen, device=DEV).to(DT[dtype]), torch.randn(2, 4, 64, 80, generator=gen, device=DEV)
    pool0 = torch.randn(5, 4, 64, 80, generator=gen, device=DEV)

    def run():
        ts = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
        y, last = vr.decay_attention(*ts[:4], scale=0.5, state=ts[4], return_state=True)
        grads = torch.autograd.grad((y, last), ts, (gy, gl))
        off = torch.tensor([0, 40, 150], device=DEV)
        with torch.no_grad():
            packed = vr.decay_attention(q[:1], k[:1], v[:1], g[:1], offsets=off)
            pool = pool0.clone()
            s = vr.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], pool, torch.tensor([3, 1], device=DEV))
            vr.copy_states(pool, torch.tensor([3, 0], device=DEV), torch.tensor([0, 3], device=DEV))
        return [y, last, *grads, packed, s, pool]
    a = run()
    monkeypatch.setattr(vr._lib, "_host", vr._lib._NoHost)
    for x, y in zip(a, run()):
        assert torch.equal(x, y)


@pytest.mark.gpu
def test_hooks_on_saved_tensors_and_gradients_in_batches():
    q, k, v, g, S = make(1, 100, 2, 2, 2, 2, 64, 64, "bf16", state=1)
    ts = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
    y = vr.decay_attention(*ts[:4], state=ts[4])
    want = torch.autograd.grad(y, ts, torch.ones_like(y))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(DEV)):
        y = vr.decay_attention(*ts[:4], state=ts[4])
    for a, b in zip(torch.autograd.grad(y, ts, torch.ones_like(y)), want):
        assert torch.equal(a, b)
    y = vr.decay_attention(*ts[:4], state=ts[4])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, ts, torch.ones(2, *y.shape, device=DEV, dtype=y.dtype), is_grads_batched=True)


@pytest.mark.gpu
def test_inside_a_compiled_program():
    """The calls are left as they are."""
    q, k, v, g, S = make(1, 70, 2, 2, 2, 2, 64, 64, "fp32", state=1)

    def layer(q, k, v, g, S):
        y, last = vr.decay_attention(q * 2, k, v, g, state=S, return_state=True)
        return y + 1, last

    def token(q, pool):
        y = vr.decay_attention_step(q, q, q, g[:, 0], pool)
        return y, vr.copy_states(pool, torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV))
    for f, args in ((layer, (q, k, v, g, S)), (token, (q[:, 0], S))):
        with torch.no_grad():
            want = f(*(t.clone() for t in args))
            got = torch.compile(f, backend="eager")(*(t.clone() for t in args))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    ts = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
    want = torch.autograd.grad(layer(*ts)[0].sum(), ts)
    for a, b in zip(torch.autograd.grad(torch.compile(layer, backend="eager")(*ts)[0].sum(), ts), want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_the_same_bits_twice():
    for dtype, T, offsets in (("bf16", 900, None), ("fp32", 300, None), ("bf16", 900, [0, 500, 510, 900])):
        q, k, v, g, S = make(1, T, 3, 1, 3, 3, 64, 64, dtype, g="head", state=3 if offsets else 1)
        off = torch.tensor(offsets, device=DEV) if offsets else None
        def run():
            ts = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
            y, last = vr.decay_attention(*ts[:4], state=ts[4], offsets=off, return_state=True)
            return [y, last, *torch.autograd.grad((y, last), ts, (torch.ones_like(y), torch.ones_like(last)))]
        for a, b in zip(run(), run()):
            assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_hundred_thousand_tokens():
    """As two halves, the second going on from the first's state.  Bound: both sides are within that of compare(), whose absolute sums are at most
    64 max|q| max|k| max|v| (tokens that a decay of 0.03 keeps: 1 / 0.03)."""
    T, D = 100_000, 16
    q, k, v, _, _ = make(1, T, 2, 2, 2, 2, D, D, "fp32", seed=4)
    g = torch.full((2,), -0.03, device=DEV)
    y, last = vr.decay_attention(q, k, v, g, scale=0.25, return_state=True)
    h = T // 2 + 13
    a, mid = vr.decay_attention(q[:, :h], k[:, :h], v[:, :h], g, scale=0.25, return_state=True)
    b, end = vr.decay_attention(q[:, h:], k[:, h:], v[:, h:], g, scale=0.25, state=mid, return_state=True)
    bound = 2 * (D + D + 128) * 2.0 ** -24 * 0.25 * D * (1 / 0.03) * q.abs().max() * k.abs().max() * v.abs().max()
    assert (torch.cat([a, b], 1) - y).abs().max() <= bound and (end - last).abs().max() <= bound


@pytest.mark.gpu
def test_strides_and_pages_beyond_32_bits():
    """A batch whose rows, and pools whose pages, lie 2^31 and more elements apart."""
    far = (1 << 31) + 64
    big = torch.empty(far + 4096, dtype=torch.bfloat16, device=DEV)
    q, k, v, g, S = make(2, 40, 1, 1, 1, 1, 64, 64, "bf16", state=2)
    views = []
    for t, at in ((q, 0),):
        w = big.as_strided(t.shape, (far, 64, 64, 1), at)
        w.copy_(t)
        views.append(w)
    a = vr.decay_attention(q, k, v, g, state=S, return_state=True)
    b = vr.decay_attention(views[0], k, v, g, state=S, return_state=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    del big, views, w
    torch.cuda.empty_cache()
    big = torch.empty(far + 8192, device=DEV)
    pool = big.as_strided((2, 1, 64, 64), (far, 4096, 64, 1))
    pool.copy_(S)
    dense = S.clone()
    slots = torch.tensor([1, 0], device=DEV)
    ys = [vr.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g[:, 0], p, slots) for p in (pool, dense)]
    assert torch.equal(*ys) and torch.equal(pool, dense)
    vr.copy_states(pool, torch.tensor([1, 0], device=DEV), torch.tensor([0, 1], device=DEV))
    assert torch.equal(pool, dense.flip(0))


@pytest.mark.gpu
def test_nothing_in_it():
    r = lambda *s: torch.randn(*s, device=DEV, requires_grad=True)
    for B, T in ((0, 5), (2, 0)):
        q, g, S = r(B, T, 2, 8), r(B, T, 2), r(B, 2, 8, 8)
        y, last = vr.decay_attention(q, q, q, g, state=S, return_state=True)
        assert y.shape == (B, T, 2, 8) and torch.equal(last, S)
        dq, dg, dS = torch.autograd.grad((y, last), (q, g, S), (torch.ones_like(y), torch.ones_like(last)))
        assert dq.shape == q.shape and dg.shape == g.shape and torch.equal(dS, torch.ones_like(S))
    y, last = vr.decay_attention(r(1, 0, 2, 8), r(1, 0, 2, 8), r(1, 0, 2, 8), r(2), offsets=torch.zeros(4, dtype=torch.int32, device=DEV), return_state=True)
    assert y.shape == (1, 0, 2, 8) and last.shape == (3, 2, 8, 8) and not last.any()
    with torch.no_grad():
        pool = torch.randn(3, 2, 8, 8, device=DEV)
        assert vr.decay_attention_step(r(0, 2, 8), r(0, 2, 8), r(0, 2, 8), r(0, 2), pool).shape == (0, 2, 8)
        assert vr.copy_states(pool, [], []) is pool


@pytest.mark.gpu
@pytest.mark.parametrize("mode", [torch.no_grad, torch.inference_mode])
def test_serving_without_gradients(mode):
    """Inference tensors have no version; others count the changes that are made in place."""
    q, k, v, g, S = make(2, 6, 2, 2, 2, 2, 64, 64, "bf16", state=2)
    with mode():
        pool = S.clone()
        version = None if pool.is_inference() else pool._version
        y = torch.stack([vr.decay_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], pool) for t in range(6)], 1)
        vr.copy_states(pool, [1, 0], [0, 1])
        vr.copy_states(pool, torch.tensor([1, 0], device=DEV), torch.tensor([0, 1], device=DEV))
        assert version is None or pool._version == version + 8
    want = reference(q, k, v, g, 1.0, S, [(0, 0, 6), (1, 0, 6)])
    compare(y, want["y"], "y", "bf16", 64, 64, 6)
    compare(pool, want["last"], "last", "fp32", 64, 64, 6)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    r = lambda *s, dt=torch.float32: torch.randn(*s, device=DEV).to(dt)
    q, g = r(1, 4, 2, 8), r(1, 4, 2)
    bad = [dict(q=r(1, 4, 8)), dict(k=r(1, 5, 2, 8)), dict(k=r(1, 4, 2, 9)), dict(v=r(1, 4, 2, 8, dt=torch.bfloat16)), dict(g=r(1, 4, 3)), dict(g=r(1, 5, 2)),
           dict(g=r(1, 4, 2, dt=torch.float16)), dict(q=r(1, 4, 2, 129), k=r(1, 4, 2, 129)), dict(state=r(1, 2, 8, 9)), dict(state=r(1, 2, 8, 8, dt=torch.bfloat16)),
           dict(offsets=torch.tensor([0.0, 4.0], device=DEV)), dict(offsets=torch.tensor([0, 4])), dict(q=q.cpu()), dict(q=r(1, 4, 2, 0), k=r(1, 4, 2, 0))]
    for change in bad:
        with pytest.raises(RuntimeError):
            vr.decay_attention(**{**dict(q=q, k=q, v=q, g=g), **change})
    with pytest.raises(RuntimeError):
        vr.decay_attention(*(t.expand(2, *t.shape[1:]) for t in (q, q, q, g)), offsets=torch.tensor([0, 4], device=DEV))
    pool = r(3, 2, 8, 8)
    step = dict(q=q[0], k=q[0], v=q[0], g=g[0], pool=pool, slots=torch.arange(4, device=DEV))
    for change in (dict(pool=r(3, 2, 8, 9)), dict(pool=pool.transpose(2, 3)), dict(pool=pool.bfloat16()), dict(slots=None), dict(slots=torch.arange(3, device=DEV)),
                   dict(slots=torch.arange(4, device=DEV).float()), dict(q=q[0].clone().requires_grad_()), dict(pool=pool[:1].expand(3, 2, 8, 8))):
        with pytest.raises(RuntimeError):
            vr.decay_attention_step(**{**step, **change})
    for a in ((pool, [0, 1], [0]), (pool, [3], [0]), (pool, [0], [3]), (pool, [-2], [0]), (pool, [0.5], [1]), (pool, [0] * 4097, [1] * 4097), (pool, [0], [1], r(3, 2, 8, 9)),
              (pool, [0], [1], pool[1:]), (pool.transpose(2, 3), [0], [1])):
        with pytest.raises(RuntimeError):
            vr.copy_states(*a)
    x = q.clone().requires_grad_()
    first = torch.autograd.grad(vr.decay_attention(x, q, q, g).sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        first.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("host", [True, False])
def test_one_token_of_rows_that_lie_far_apart(host, monkeypatch):
    """(T, B, H, D) with T = 1 seen as (B, T, H, D): the stride of tokens that are not there may be anything."""
    if not host:
        monkeypatch.setattr(vr._lib, "_host", vr._lib._NoHost)
    q, k, v, g, S = make(3, 1, 2, 2, 2, 2, 64, 64, "bf16", state=3)
    gy = torch.randn(3, 1, 2, 64, generator=torch.Generator(DEV).manual_seed(5), device=DEV).bfloat16()
    results = []
    for far in (False, True):
        view = (lambda t: t.as_strided(t.shape, (t.stride(0), 1 << 23, *t.stride()[2:]))) if far else lambda t: t
        ts = [t.clone().requires_grad_() for t in (q, k, v, g, S)]
        y, last = vr.decay_attention(*(view(t) for t in ts[:4]), state=ts[4], return_state=True)
        results.append((y, last, *torch.autograd.grad(y, ts, view(gy))))
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_pages_of_one_layer_from_another():
    layers = torch.randn(6, 3, 2, 8, 8, device=DEV)
    before = layers.clone()
    vr.copy_states(layers[:, 0], [5, 0, -1], [1, 5, 2], source=layers[:, 2])
    before[1, 0], before[5, 0], before[2, 0] = before[5, 2], before[0, 2], 0
    assert torch.equal(layers, before)
    flat = layers.flatten(1)
    for pool, source in ((flat[:, :256], flat[:, 128:]), (flat[:, :192], flat[:, 191:383]), (flat[:, :128], flat[::2, 128:256])):
        with pytest.raises(RuntimeError):                  # overlapping by half, by one number; at another distance
            vr.copy_states(pool, [0], [1], source=source)


@pytest.mark.gpu
def test_refusals_of_sizes_and_of_moved_tensors():
    wide = torch.zeros(1, 1, 1, 1, device=DEV).expand(1, (1 << 31) + 5, 1, 1)
    for call in (lambda: vr.decay_attention(wide, wide, wide, torch.zeros(1, device=DEV)),
                 lambda: vr.decay_attention_step(wide[0], wide[0], wide[0], torch.zeros(1, device=DEV), torch.zeros(2, 1, 1, 1, device=DEV))):
        with pytest.raises(RuntimeError, match="2\\^31"):
            call()
    q, k, v, g, S = make(1, 20, 2, 2, 2, 2, 64, 64, "bf16", state=1)
    for name, t in (("g", g), ("state", S), ("q", q)):
        x = q.clone().requires_grad_()
        back = lambda u, like=t: u.cpu() if u.shape == like.shape and u.dtype == like.dtype else u
        with torch.autograd.graph.saved_tensors_hooks(lambda u: u, back):
            y = vr.decay_attention(x, k, v, g, state=S)
        with pytest.raises(RuntimeError):
            y.float().sum().backward()


def test_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="number"):
        vr.decay_attention(torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2), scale=torch.ones(()))
    q, g = torch.randn(1, 4, 2, 8), torch.randn(1, 4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        vr.decay_attention(q, q, q, g)
    with pytest.raises(RuntimeError, match="CUDA"):
        vr.decay_attention_step(q[0], q[0], q[0], g[0], torch.zeros(4, 2, 8, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        vr.copy_states(torch.zeros(4, 8), [0], [1])


def test_the_library_refuses_before_it_launches():
    """Every check of the C entries, without a device."""
    L, lib = vr._lib, vr.lib()

    def args(cls, **change):
        a = cls()
        for n in cls.POINTERS:
            setattr(a, n, 4096)
        if cls is L.DecayArgs:
            a.offsets = a.gy = a.glast = None
            a.workspace, a.workspace_bytes, a.T = 4096, 1 << 40, 9
        else:
            a.P, a.page_stride = 5, 2 * 64
        a.N = a.H = a.Hq = a.Hk = a.Hv = 2
        a.Dk = a.Dv = 8
        for n, x in change.items():
            setattr(a, n, x)
        return a
    A, S = L.DecayArgs, L.DecayStepArgs
    assert lib.vrwkv_decay_fwd(None, None) == 1 and lib.vrwkv_decay_step(None, None) == 1
    for change, status in ((dict(N=0), 1), (dict(T=0), 1), (dict(H=-1), 1), (dict(Hq=3), 3), (dict(Hv=0), 1), (dict(Dk=129), 3), (dict(Dv=0), 3), (dict(dtype=3), 2), (dict(g_dtype=-1), 2),
                           (dict(q=None), 1), (dict(g=None), 1), (dict(y=None), 1), (dict(k=4097), 1), (dict(g=4098), 1), (dict(state=4098), 1), (dict(offsets=4098), 1),
                           (dict(N=1 << 24), 3), (dict(N=1 << 20, H=16, Hq=16, Hk=16, Hv=16), 3)):
        assert lib.vrwkv_decay_fwd(args(A, **change), None) == status, change
        if "N" not in change and "y" not in change:
            assert lib.vrwkv_decay_bwd(args(A, gy=4096, **change), None) == status, change
    assert lib.vrwkv_decay_bwd(args(A), None) == 1         # no gy
    long = dict(N=1, T=5000)
    assert lib.vrwkv_decay_fwd_workspace_bytes(args(A, **long)) > 0 and lib.vrwkv_decay_fwd_workspace_bytes(args(A, T=0)) == 0
    for change, status in ((dict(workspace=None), 5), (dict(workspace_bytes=64), 5), (dict(workspace=4100), 1)):
        assert lib.vrwkv_decay_fwd(args(A, **long, **change), None) == status, change
        assert lib.vrwkv_decay_bwd(args(A, gy=4096, **long, **change), None) == status, change
    for change, status in ((dict(N=0), 1), (dict(P=0), 1), (dict(slots=None, N=6), 1), (dict(page_stride=127), 1), (dict(Hk=4), 3), (dict(Dv=200), 3), (dict(dtype=7), 2), (dict(q=4097), 1),
                           (dict(pool=4098), 1), (dict(slots=4100, slots64=1), 1), (dict(N=1 << 23), 3), (dict(y=None), 1)):
        assert lib.vrwkv_decay_step(args(S, **change), None) == status, change

    def pages(pool=1 << 20, stride=64, P=4, source=1 << 20, source_stride=64, source_P=4, size=64, src=4096, s64=0, dst=4096, d64=0, M=3, ws=4096, ws_bytes=1 << 20):
        return lib.vrwkv_copy_pages(pool, stride, P, source, source_stride, source_P, size, src, s64, dst, d64, M, ws, ws_bytes, None)
    for change, status in ((dict(pool=None), 1), (dict(src=None), 1), (dict(P=0), 1), (dict(M=0), 1), (dict(size=0), 1), (dict(M=4097), 3), (dict(stride=63), 1), (dict(source_stride=60), 1),
                           (dict(src=4100, s64=1), 1), (dict(ws=None, M=300), 5), (dict(ws_bytes=1199, M=300), 5), (dict(ws=4097, M=300), 1), (dict(source=(1 << 20) + 64), 1), (dict(source_stride=128), 1),
                           (dict(size=1 << 30, stride=1 << 30, source_stride=1 << 30, M=4096), 3), (dict(size=(1 << 23) + 1, stride=1 << 24, source_stride=1 << 24, M=4096), 3)):
        assert pages(**change) == status, change
    assert lib.vrwkv_copy_pages_workspace_bytes(300) == 1200 and lib.vrwkv_copy_pages_workspace_bytes(5) == lib.vrwkv_copy_pages_workspace_bytes(0) == 0
