"""causal_conv, its gradients and its step on the GPU against the sums written out in 64 bits.

Bounds.  A result is off by the half step u of its type, and inside by fp32 roundings, each 2^-24 of the sum of absolute values A at most: K + 1 of a sum of taps, eight of silu or its slope (argument,
exponential, sum, reciprocal, three products and a sum), K + 1 of the sum over the tokens behind: N = 2 K + 12.  silu' is at most 1.1 and its own slope at most 0.5, so that an error of the argument
weighs no more than itself.  Sums over all tokens (weight, bias) add their number.  fp32 results are also held to 2e-6 of their norm."""
import pytest
import torch

import vision_rwkv_amd as vr
from vision_rwkv_amd import _lib

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=[True, False], ids=["compiled", "python"])
def host(request, monkeypatch):
    """The operators through the compiled host module, and through the Python classes alone."""
    if not request.param:
        monkeypatch.setattr(_lib, "host", lambda: _lib._NoHost)


def reference(x, w, b, act, state, bounds, gy=None, glast=None):
    """Everything in float64 on the CPU: {name: (value, sum of absolute terms)}."""
    f = lambda t: None if t is None else t.detach().double().cpu()
    x, w, b, state, gy, glast = (f(t) for t in (x, w, b, state, gy, glast))
    rows, T, E = x.shape
    K, N = w.shape[1], len(bounds)
    out = {}
    for kind, a in (("x", lambda t: t), ("abs", torch.abs)):
        r = dict(y=torch.zeros(rows, T, E).double(), dx=torch.zeros(rows, T, E).double(), dw=torch.zeros(E, K).double(), db=torch.zeros(E).double(), last=torch.zeros(N, K - 1, E).double(),
                 dstate=torch.zeros(N, K - 1, E).double())
        for n, (row, i, j) in enumerate(bounds):
            whole = torch.cat([state[n] if state is not None else torch.zeros(K - 1, E).double(), x[row, i:j]])
            r["last"][n] = a(whole[j - i:])
            back = torch.zeros_like(whole)
            if glast is not None:
                back[j - i:] += a(glast[n])
            for t in range(j - i):
                pre = (whole[t:t + K].T * w).sum(1) + (b if b is not None else 0)
                pre_abs = (whole[t:t + K].T * w).abs().sum(1) + (b.abs() if b is not None else 0)
                s = torch.sigmoid(pre)
                if kind == "x":
                    r["y"][row, i + t] = pre * s if act else pre
                    slope = s * (1 + pre * (1 - s)) if act else torch.ones_like(pre)
                else:
                    r["y"][row, i + t] = pre_abs if act else pre_abs
                    slope = s * (1 + pre.abs() * (1 - s)) + 0.5 * pre_abs if act else torch.ones_like(pre)
                if gy is None:
                    continue
                g = a(gy[row, i + t]) * slope
                r["db"] += g
                r["dw"] += a(whole[t:t + K].T) * g[:, None]
                back[t:t + K] += a(w.T) * g
            r["dx"][row, i:j] = back[K - 1:]
            r["dstate"][n] = back[:K - 1]
        out[kind] = r
    return {n: (out["x"][n], out["abs"][n]) for n in out["x"]}


def compare(got, want, name, K, tokens=0):
    x, (ref, scale) = got.detach().double().cpu(), want
    assert x.shape == ref.shape and torch.isfinite(x).all(), name
    limit = HALF_STEP[got.dtype] * ref.abs() + (2 * K + 12 + (tokens if name in ("dw", "db") else 0)) * 2.0 ** -24 * scale + 1e-30
    if got.dtype == torch.float16:
        limit = limit + 2.0 ** -25
    over = ((x - ref).abs() / limit).max().item() if x.numel() else 0.0
    assert over <= 1.0, f"{name}: {over:.3g} of the bound"
    if got.dtype == torch.float32 and ref.norm() > 0:
        assert (x - ref).norm() <= 2e-6 * max(ref.norm(), 2.0 ** -4 * scale.norm()), name


def inputs(N, T, E, K, dtype, params="fp32", bias=True, state=0, seed=0):
    gen = torch.Generator().manual_seed(seed * 1000 + N + 7 * T + 13 * E + K)
    normal = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    dt, pt = DT[dtype], DT[dtype if params == "same" else params]
    return normal(N, T, E).to(dt), normal(E, K).to(pt), normal(E).to(pt) if bias else None, normal(state, K - 1, E).to(dt) if state else None, normal


def run_and_compare(x, w, b, state, normal, bounds, act="silu", offsets=None, glast=True):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, state) if t is not None]
    named = [n for n, t in (("dx", x), ("dw", w), ("db", b), ("dstate", state)) if t is not None]
    it = iter(leaves)
    a = [next(it) if t is not None else None for t in (x, w, b, state)]
    y, last = vr.causal_conv(a[0], a[1], a[2], act, state=a[3], offsets=offsets, return_state=True)
    gy, gl = normal(*y.shape).to(y.dtype), normal(*last.shape).to(y.dtype) if glast else None
    grads = torch.autograd.grad([y, last] if glast else [y], leaves, [gy, gl] if glast else [gy])
    want = reference(x, w, b, act, state, bounds, gy, gl)
    K, tokens = w.shape[1], sum(j - i for _, i, j in bounds)
    compare(y, want["y"], "y", K)
    assert torch.equal(last.double().cpu(), reference(x, w, b, act, state, bounds)["last"][0])
    for n, g, t in zip(named, grads, leaves):
        assert g.dtype == t.dtype
        compare(g, want[n], n, K, tokens)
    with torch.no_grad():
        y2, last2 = vr.causal_conv(x, w, b, act, state=state, offsets=offsets, return_state=True)
    assert torch.equal(y2, y) and torch.equal(last2, last)
    return y, last, grads


@pytest.mark.parametrize("dtype,params", [("fp32", "fp32"), ("bf16", "same"), ("bf16", "fp32"), ("fp16", "same")])
@pytest.mark.parametrize("N,T,E,K", [(2, 50, 96, 4), (3, 1, 40, 4), (1, 2, 65, 4), (2, 3, 64, 4), (1, 9, 130, 2), (2, 40, 33, 3), (1, 17, 600, 8), (2, 30, 18, 6), (1, 7, 1, 5), (2, 100, 520, 4), (1, 300, 16, 7)])
def test_sequences_and_gradients(N, T, E, K, dtype, params):
    x, w, b, state, normal = inputs(N, T, E, K, dtype, params, state=N)
    run_and_compare(x, w, b, state, normal, [(n, 0, T) for n in range(N)])


@pytest.mark.parametrize("bias,state,act,glast", [(False, 0, None, False), (True, 2, None, True), (False, 2, "silu", False), (True, 0, "silu", True)])
def test_what_may_be_left_out(bias, state, act, glast):
    x, w, b, state, normal = inputs(2, 60, 72, 4, "bf16", bias=bias, state=state)
    run_and_compare(x, w, b, state, normal, [(0, 0, 60), (1, 0, 60)], act=act, glast=glast)


@pytest.mark.parametrize("K", [2, 4, 5, 8])
@pytest.mark.parametrize("lengths,front,behind,dtype,E,index", [([5, 0, 100, 1, 17, 0, 0, 180], 0, 0, "fp32", 20, torch.int32), ([0, 33, 64, 0], 3, 21, "bf16", 64, torch.int64), ([1] * 40, 0, 5, "fp32", 7, torch.int32),
                                                              ([290], 20, 3, "fp16", 34, torch.int64), ([3, 2, 1, 2, 3, 8, 7], 0, 0, "bf16", 200, torch.int32)])
def test_packed_sequences(lengths, front, behind, dtype, E, index, K):
    first = [front]
    for n in lengths:
        first.append(first[-1] + n)
    T = first[-1] + behind
    x, w, b, state, normal = inputs(1, T, E, K, dtype, state=len(lengths))
    outside = torch.ones(T, dtype=torch.bool)
    outside[front:first[-1]] = False
    x[0, outside] = float("nan")                           # rows of no sequence hold anything
    y, last, grads = run_and_compare(x, w, b, state, normal, [(0, i, j) for i, j in zip(first[:-1], first[1:])], offsets=torch.tensor(first, dtype=index, device=DEV))
    assert not y[0, outside].any() and not grads[0][0, outside].any()


def test_long_rows_and_many_runs():
    """Runs of 64 tokens, workgroups that take several: more tokens than the chip has lanes for."""
    x, w, b, state, normal = inputs(2, 30000, 256, 4, "bf16")
    x32, w32 = x.float(), w.float()
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = vr.causal_conv(*leaves, "silu")
    gy = normal(*y.shape).bfloat16()
    grads = torch.autograd.grad(y, leaves, gy)
    want = [t.detach().double().requires_grad_() for t in leaves]
    padded = torch.nn.functional.pad(want[0], (0, 0, 3, 0))
    pre = sum(padded[:, j:j + 30000] * want[1][:, j] for j in range(4)) + want[2]
    exact = pre * torch.sigmoid(pre)
    # (sums of random sign over 60 000 tokens: their error goes by the root of that, 2^-24 x 250; a sum's own size by it as well)
    for got, ref, bound in zip([y, *grads], [exact, *torch.autograd.grad(exact, want, gy.double())], [2.0 ** -8, 2.0 ** -8, 1e-5, 1e-5]):
        assert (got.double() - ref).norm() <= bound * ref.norm()


def test_strides_and_views():
    N, T, E, K = 3, 37, 48, 4
    x, w, b, state, normal = inputs(N, T, E, K, "bf16", state=N)
    views = [torch.cat([x, x], -1)[..., E:], torch.stack([x] * 3, 2)[:, :, 1], x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x, x[..., :1]], -1)[..., :E], x.transpose(1, 2).contiguous().transpose(1, 2)]
    plain = run_and_compare(x, w, b, state, normal, [(n, 0, T) for n in range(N)])
    for v in views:
        leaves = [t.detach().requires_grad_() for t in (v, w.t().contiguous().t(), b, torch.cat([state] * 2, -1)[..., :E])]
        y, last = vr.causal_conv(*leaves[:3], "silu", state=leaves[3], return_state=True)
        assert torch.equal(y, plain[0]) and torch.equal(last, plain[1])
        ones = [torch.ones_like(x), torch.ones_like(state)]
        base = [t.detach().requires_grad_() for t in (x, w, b, state)]
        want = torch.autograd.grad(vr.causal_conv(*base[:3], "silu", state=base[3], return_state=True), base, ones)
        got = torch.autograd.grad([y, last], leaves, [ones[0].transpose(0, 1).contiguous().transpose(0, 1), ones[1]])
        for n, (p, q) in enumerate(zip(got, want)):
            # (sums over tokens are taken in other orders where other numbers of channels go together)
            assert torch.equal(p, q) if n in (0, 3) else (p.float() - q.float()).norm() <= 1e-5 * q.float().norm()


def test_no_tokens():
    x, w, b, state, _ = inputs(2, 0, 20, 4, "fp32", state=2)
    state.requires_grad_()
    y, last = vr.causal_conv(x, w, b, "silu", state=state, return_state=True)
    assert y.shape == (2, 0, 20) and torch.equal(last, state)
    assert torch.equal(torch.autograd.grad(last, state, torch.ones_like(last))[0], torch.ones_like(last))
    x, w, b, _, _ = inputs(1, 7, 20, 4, "fp32")
    y, last = vr.causal_conv(x, w, b, offsets=torch.tensor([0], device=DEV), return_state=True)
    assert not y.any() and last.shape == (0, 3, 20)


def test_infinities_and_nan_stay_within_reach():
    for K in (3, 4, 6):
        x, w, b, _, _ = inputs(2, 60, 24, K, "bf16")
        clean = vr.causal_conv(x, w, b, "silu")
        for bad in (float("inf"), float("nan")):
            v = x.clone()
            v[0, 20, 5] = bad
            y = vr.causal_conv(v, w, b, "silu")
            same = torch.ones_like(y, dtype=torch.bool)
            same[0, 20:20 + K, 5] = False
            assert torch.equal(y[same], clean[same])


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E,K", [(96, 4), (33, 2), (64, 3), (50, 8), (2056, 4), (18, 6)])
def test_steps_are_what_sequences_are(E, K, dtype):
    N, T = 5, 9
    x, w, b, state, _ = inputs(N, T, E, K, dtype, state=N)
    want = reference(x, w, b, "silu", state, [(n, 0, T) for n in range(N)])
    pool = torch.full((9, K - 1, E), 7.0, device=DEV, dtype=DT[dtype])
    slots = torch.tensor([8, 0, 3, 5, 1], device=DEV)
    pool[slots] = state
    ys = [vr.causal_conv_step(x[:, t], w, pool, slots if t % 2 else slots.int(), bias=b, activation="silu") for t in range(T)]
    compare(torch.stack(ys, 1), want["y"], "y", K)
    assert torch.equal(pool[slots].double().cpu(), want["last"][0])
    rest = torch.ones(9, dtype=torch.bool)
    rest[slots.cpu()] = False
    assert (pool[rest] == 7).all()


def test_step_slots_and_pools():
    N, E, K = 600, 40, 4
    x, w, b, _, normal = inputs(1, N, E, K, "fp32")
    pool = normal(4, K - 1, E)
    before = pool.clone()
    page = torch.tensor([n % 3 if n % 7 else (-1 if n % 2 else 4 + n) for n in range(N)], device=DEV)
    y = vr.causal_conv_step(x[0], w, pool, page, bias=b)
    for p in range(3):
        mine = (page == p).nonzero()[:, 0]
        want = reference(x[:, mine], w, b, None, before[p:p + 1], [(0, 0, len(mine))])
        compare(y[mine][None], want["y"], "y", K)
        assert torch.equal(pool[p].double().cpu(), want["last"][0][0])
    assert torch.equal(pool[3], before[3]) and not y[page == -1].any() and torch.isnan(y[page >= 4]).all()
    layers = normal(5, 2, K - 1, E)
    alone, kept = layers[:, 1].clone(), layers[:, 0].clone()
    assert torch.equal(vr.causal_conv_step(x[0, :3], w, layers[:, 1]), vr.causal_conv_step(x[0, :3], w, alone)) and torch.equal(layers[:, 1], alone) and torch.equal(layers[:, 0], kept)
    y = vr.causal_conv_step(x[0, :2], w, torch.empty(0, K - 1, E, device=DEV), torch.tensor([-1, 2], device=DEV))
    assert not y[0].any() and torch.isnan(y[1]).all()


def test_refusals():
    x, w, b, state, normal = inputs(2, 9, 20, 4, "bf16", state=2)
    ok = dict(x=x, weight=w, bias=b, activation="silu", state=state)
    for change in (dict(x=x.double()), dict(x=x.cpu()), dict(x=x[0]), dict(weight=w[:, :1]), dict(weight=normal(20, 9)), dict(weight=w[:10]), dict(weight=w.half()), dict(bias=b.bfloat16()), dict(bias=b[:3]),
                   dict(activation="relu"), dict(state=state.float()), dict(state=state[:, :2]), dict(state=state[:1]), dict(offsets=torch.tensor([0, 9], device=DEV))):
        with pytest.raises(RuntimeError):
            vr.causal_conv(**{**ok, **change})
    pool = normal(4, 3, 20).bfloat16()
    for p, s in ((pool.float(), None), (pool[:, :2], None), (pool.transpose(1, 2).contiguous().transpose(1, 2), None), (pool[:1], None), (pool[:1].expand(4, 3, 20), None), (pool, torch.tensor([0], device=DEV)),
                 (pool, torch.tensor([0.0, 1.0], device=DEV)), (pool, torch.tensor([0, 1])), (pool.clone().requires_grad_(), None)):
        with pytest.raises(RuntimeError):
            vr.causal_conv_step(x[:, 0], w, p, s)
    with pytest.raises(RuntimeError, match="forward mode"), torch.autograd.forward_ad.dual_level():
        vr.causal_conv(torch.autograd.forward_ad.make_dual(x, x), w)
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda t: vr.causal_conv(t, w), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: vr.causal_conv(t, w))(torch.stack([x, x]))


def test_other_streams_and_graphs():
    x, w, b, state, normal = inputs(2, 150, 64, 4, "bf16", state=2)
    leaves = [t.detach().requires_grad_() for t in (x, w, b, state)]
    gy, gl = normal(2, 150, 64).bfloat16(), normal(2, 3, 64).bfloat16()

    def call():
        y, last = vr.causal_conv(*leaves[:3], "silu", state=leaves[3], return_state=True)
        return [y.detach(), last.detach(), *torch.autograd.grad([y, last], leaves, [gy, gl])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for p, q in zip(got, call()):
        assert torch.equal(p, q)
    del p, q, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = call()
    for k in range(3):
        with torch.no_grad():
            for t in (*leaves, gy, gl):
                t.copy_(normal(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(recorded, call()):
            assert torch.equal(p, q), k
