"""selective_scan, its gradients and its step on the GPU against the recurrence token by token in 64 bits.

Bounds.  Beside every result the reference forms the same sums of absolute values, A.  With u the half step of the result's type a result is u |x| off by its own rounding, and
inside by at most N 2^-24 A: a term passes at most T products with an exponential (each off by two half steps: its own and the product's rounding, 2 T) and T + 64 additions; the step
size is off by at most eight half steps of itself (bias, exponential, quotient, series), and with it the decay over a stretch by 8 X e^-X <= 3 for its exponent X, and the terms by 8, in the
gradients by 16; the gate and its slope by another eight.  N = 3 T + 64 + 40 + 16.  Sums over all tokens of a batch (A, D, the bias) add their number of terms.
fp32 results are also held to 3e-6 of their norm: errors of random sign, 2^-24 sqrt(N) for the N up to 2 000 here."""
import math

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


def reference(x, bounds, softplus, gy=None, glast=None):
    """Everything in float64 on the CPU: {name: (value, sum of absolute terms)}.  x: the inputs by name; bounds: [(batch row, first, end)] of the sequences."""
    f = lambda t: None if t is None else t.detach().double().cpu()
    u, raw, A, D, z, bias, state = (f(x.get(n)) for n in ("u", "delta", "A", "D", "z", "delta_bias", "state"))
    wide = lambda t: (t if t.dim() == 4 else t.unsqueeze(2)).repeat_interleave(u.shape[2] // (t.shape[2] if t.dim() == 4 else 1), 2)
    B, C = wide(f(x["B"])), wide(f(x["C"]))
    G = x["B"].shape[2] if x["B"].dim() == 4 else 1
    rows, T, E = u.shape
    S = A.shape[1]
    raw = raw if bias is None else raw + bias
    dt = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)
    out = {}
    for kind, a in (("x", lambda t: t), ("abs", torch.abs)):
        U, Bk, Ck, Dt, Ak = a(u), a(B), a(C), a(dt), a(A)
        Dk = a(D) if D is not None else zeros(E)
        gate = a(z * torch.sigmoid(z)) if z is not None else torch.ones_like(u)
        # (the slope of silu is a sum of two terms, 1 and z (1 - sigmoid), that cancel at z = -1.28: its error goes by their absolute values)
        bend = torch.sigmoid(z) * (1 + a(z) * (1 - torch.sigmoid(z))) if z is not None else None
        GY = a(f(gy)) if gy is not None else zeros(rows, T, E)
        r = {n: zeros(*s) for n, s in dict(y=(rows, T, E), du=(rows, T, E), ddelta=(rows, T, E), dz=(rows, T, E), dB=(rows, T, E, S), dC=(rows, T, E, S), dA=(E, S), dD=(E,), dbias=(E,),
                                           last=(len(bounds), E, S), dstate=(len(bounds), E, S)).items()}
        for n, (b, i, j) in enumerate(bounds):
            h, kept = a(state[n]) if state is not None else zeros(E, S), []
            for t in range(i, j):
                kept.append(h)
                h = torch.exp(dt[b, t, :, None] * A) * h + (Dt[b, t] * U[b, t])[:, None] * Bk[b, t]
                inner = (h * Ck[b, t]).sum(1) + Dk * U[b, t]
                r["y"][b, t] = inner * gate[b, t]
                g = GY[b, t] * gate[b, t]
                r["dC"][b, t] = g[:, None] * h
                r["dD"] += g * U[b, t]
                if z is not None:
                    r["dz"][b, t] = GY[b, t] * inner * bend[b, t]
            r["last"][n] = h
            R = a(f(glast)[n]) if glast is not None else zeros(E, S)
            for t in reversed(range(i, j)):
                g = GY[b, t] * gate[b, t]
                R = R + g[:, None] * Ck[b, t]
                r["dB"][b, t] = R * (Dt[b, t] * U[b, t])[:, None]
                along = (R * Bk[b, t]).sum(1)
                r["du"][b, t] = Dt[b, t] * along + Dk * g
                R = torch.exp(dt[b, t, :, None] * A) * R
                q = R * kept[t - i]
                d = ((q * Ak).sum(1) + U[b, t] * along) * slope[b, t]
                r["ddelta"][b, t] = d
                r["dbias"] += d
                r["dA"] += q * Dt[b, t][:, None]
            r["dstate"][n] = R
        for n in ("dB", "dC"):
            r[n] = r[n].reshape(rows, T, G, E // G, S).sum(3).reshape(x["B"].shape)
        out[kind] = r
    return {n: (out["x"][n], out["abs"][n]) for n in out["x"]}


def compare(got, want, name, T, tokens=0):
    x, (ref, scale) = got.detach().double().cpu(), want
    assert x.shape == ref.shape, (name, x.shape, ref.shape)
    assert torch.isfinite(x).all(), name
    n = 3 * T + 120 + (tokens if name in ("dA", "dD", "dbias") else 0)
    limit = HALF_STEP[got.dtype] * ref.abs() + n * 2.0 ** -24 * scale + 1e-30
    if got.dtype == torch.float16:
        limit = limit + 2.0 ** -25                         # half a step of fp16's subnormal numbers
    over = ((x - ref).abs() / limit).max().item() if x.numel() else 0.0
    assert over <= 1.0, f"{name}: {over:.3g} of the bound"
    if got.dtype == torch.float32 and ref.norm() > 0:
        assert (x - ref).norm() <= 3e-6 * max(ref.norm(), 2.0 ** -4 * scale.norm()), f"{name}: {(x - ref).norm() / ref.norm():.3g}"


def inputs(N, T, E, S, G, dtype, seed=0, z=True, D=True, bias=True, state=False, params="fp32", softplus=True, flat=False):
    gen = torch.Generator().manual_seed(seed * 1000 + N + 7 * T + 13 * E + S)
    normal = lambda *s: torch.randn(*s, generator=gen)
    dt, pt = DT[dtype], DT[params] if params != "same" else DT[dtype]
    x = dict(u=normal(N, T, E).to(dt), A=-torch.arange(1, S + 1) * torch.exp(0.2 * normal(E, S)))
    size = torch.exp(math.log(1e-3) + torch.rand(E, generator=gen) * math.log(2e2))
    x["delta"] = (0.5 * normal(N, T, E) if softplus else size * torch.exp(0.5 * normal(N, T, E))).to(dt)
    x["delta_bias"] = (size + torch.log(-torch.expm1(-size))).to(pt) if bias and softplus else (0.01 * size).to(pt) if bias else None
    shape = (N, T, S) if flat else (N, T, G, S)
    x["B"], x["C"] = normal(*shape).to(dt), normal(*shape).to(dt)
    x["D"] = (1 + 0.2 * normal(E)).to(pt) if D else None
    x["z"] = normal(N, T, E).to(dt) if z else None
    x["state"] = normal(state, E, S) if state else None
    return {n: t.to(DEV) if t is not None else None for n, t in x.items()}, lambda *s: normal(*s).to(DEV)


NAMES = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "dbias", "state": "dstate"}


def run_and_compare(x, normal, bounds, softplus=True, offsets=None, glast=True, T=None):
    """A call with all its results and gradients; T: the longest sequence."""
    T = T or max([j - i for _, i, j in bounds] + [1])
    leaves = {n: t.clone().requires_grad_() for n, t in x.items() if t is not None}
    y, last = vr.selective_scan(**{n: leaves.get(n) for n in x}, softplus=softplus, offsets=offsets, return_state=True)
    gy, gl = normal(*y.shape).to(y.dtype), normal(*last.shape) if glast else None
    grads = torch.autograd.grad([y, last] if glast else [y], list(leaves.values()), [gy, gl] if glast else [gy])
    want = reference(x, bounds, softplus, gy, gl)
    compare(y, want["y"], "y", T)
    compare(last, want["last"], "last", T)
    for n, g in zip(leaves, grads):
        assert g.dtype == x[n].dtype and g.shape == x[n].shape
        compare(g, want[NAMES[n]], NAMES[n], T, tokens=sum(j - i for _, i, j in bounds))
    with torch.no_grad():                                  # without a record of it: the same
        y2, last2 = vr.selective_scan(**x, softplus=softplus, offsets=offsets, return_state=True)
    assert torch.equal(y2, y) and torch.equal(last2, last)
    return y, last, grads


@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("N,T,E,S,G", [(2, 196, 96, 16, 1), (3, 1, 40, 16, 2), (1, 16, 65, 16, 1), (2, 17, 130, 16, 2), (1, 33, 24, 4, 1), (2, 50, 70, 3, 5), (1, 40, 300, 1, 1), (2, 64, 33, 8, 3),
                                       (1, 47, 129, 6, 1), (2, 31, 48, 32, 2), (1, 90, 20, 27, 1), (1, 35, 18, 64, 2), (2, 20, 17, 50, 1), (1, 577, 12, 16, 1)])
def test_sequences_and_gradients(N, T, E, S, G, dtype):
    x, normal = inputs(N, T, E, S, G, dtype, state=N)
    run_and_compare(x, normal, [(n, 0, T) for n in range(N)])


@pytest.mark.parametrize("segments", [2, 5, 13])
@pytest.mark.parametrize("dtype,S", [("fp32", 16), ("bf16", 16), ("fp32", 5), ("fp16", 40)])
def test_cut_sequences(segments, dtype, S, force):
    force("scan_segments", segments)
    x, normal = inputs(2, 403, 40, S, 2, dtype, state=2)
    run_and_compare(x, normal, [(0, 0, 403), (1, 0, 403)])


@pytest.mark.parametrize("segments", [0, 1])
@pytest.mark.parametrize("N,T,E,S,G,dtype", [(1, 1024, 8, 16, 1, "bf16"), (2, 513, 10, 3, 2, "fp32"), (1, 512, 9, 64, 1, "fp32"), (1, 300, 21, 29, 3, "fp16"), (3, 129, 14, 50, 1, "bf16"), (2, 257, 34, 8, 2, "fp16")])
def test_few_channels_with_and_without_rounds(N, T, E, S, G, dtype, segments, force):
    force("scan_segments", segments)
    x, normal = inputs(N, T, E, S, G, dtype, state=N)
    run_and_compare(x, normal, [(n, 0, T) for n in range(N)])


def test_long_packed_rows_of_few_channels():
    lengths = [3, 0, 250, 16, 1, 1, 240, 0, 300, 45]
    first = [5]
    for n in lengths:
        first.append(first[-1] + n)
    x, normal = inputs(1, first[-1] + 9, 6, 16, 1, "fp32", state=len(lengths))
    offsets = torch.tensor(first, dtype=torch.int32, device="cuda")
    run_and_compare(x, normal, [(0, a, b) for a, b in zip(first, first[1:])], offsets=offsets)


@pytest.mark.parametrize("z,D,bias,softplus,state,glast,params", [(False, False, False, False, 0, False, "fp32"), (True, False, True, False, 2, False, "same"), (False, True, False, True, 0, True, "same"),
                                                                  (True, True, True, True, 0, False, "same"), (False, False, True, True, 2, True, "fp32")])
def test_what_may_be_left_out(z, D, bias, softplus, state, glast, params):
    x, normal = inputs(2, 60, 50, 16, 1, "bf16", z=z, D=D, bias=bias, state=state, params=params, softplus=softplus, flat=True)
    run_and_compare(x, normal, [(0, 0, 60), (1, 0, 60)], softplus=softplus, glast=glast)


@pytest.mark.parametrize("segments", [0, 1, 4, 9])
@pytest.mark.parametrize("lengths,front,behind,dtype,S,index", [([5, 0, 100, 1, 17, 0, 0, 180], 0, 0, "fp32", 16, torch.int32), ([0, 33, 64, 0], 3, 21, "bf16", 16, torch.int64), ([1] * 40, 0, 5, "fp32", 7, torch.int32),
                                                              ([290], 20, 3, "fp16", 16, torch.int64), ([16, 16, 32, 15, 17], 0, 0, "fp32", 33, torch.int32)])
def test_packed_sequences(lengths, front, behind, dtype, S, index, segments, force):
    force("scan_segments", segments)
    first = [front]
    for n in lengths:
        first.append(first[-1] + n)
    T = first[-1] + behind
    x, normal = inputs(1, T, 36, S, 2, dtype, state=len(lengths))
    outside = torch.ones(T, dtype=torch.bool)
    outside[front:first[-1]] = False
    for n in ("u", "delta", "B", "C", "z"):                # rows of no sequence hold anything
        x[n][0, outside] = float("nan")
    bounds = [(0, i, j) for i, j in zip(first[:-1], first[1:])]
    clean = {n: t.clone().nan_to_num_(0.0) if t is not None else None for n, t in x.items()}
    offsets = torch.tensor(first, dtype=index, device=DEV)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items() if t is not None}
    y, last = vr.selective_scan(**leaves, softplus=True, offsets=offsets, return_state=True)
    gy, gl = normal(*y.shape).to(y.dtype), normal(*last.shape)
    grads = torch.autograd.grad([y, last], list(leaves.values()), [gy, gl])
    want = reference(clean, bounds, True, gy, gl)
    compare(y, want["y"], "y", max(lengths))
    compare(last, want["last"], "last", max(lengths))
    for n, g in zip(leaves, grads):
        compare(g, want[NAMES[n]], NAMES[n], max(lengths), tokens=sum(lengths))
    assert not y[0, outside].any() and not any(g[0, outside].any() for g, n in zip(grads, leaves) if n in ("u", "delta", "B", "C", "z"))


def test_packed_is_what_the_sequences_are_alone():
    """A sequence's results do not depend on where it lies, to the bit where it is not cut."""
    x, _ = inputs(1, 90, 64, 16, 1, "bf16", state=3)
    first = [0, 32, 48, 90]
    with torch.no_grad(), vr.option("scan_segments", 1):
        y, last = vr.selective_scan(**x, softplus=True, offsets=torch.tensor(first, device=DEV), return_state=True)
        for n, (i, j) in enumerate(zip(first[:-1], first[1:])):
            part = {k: t[:, i:j] if k in ("u", "delta", "B", "C", "z") else t[n:n + 1] if k == "state" else t for k, t in x.items()}
            y1, last1 = vr.selective_scan(**part, softplus=True, return_state=True)
            assert torch.equal(y1, y[:, i:j]) and torch.equal(last1[0], last[n])


def test_strides_and_views():
    """Halves and slices of projections, transposed batches, shared rows: the same as their copies, gradients too."""
    N, T, E, S, G = 3, 37, 48, 16, 2
    x, normal = inputs(N, T, E, S, G, "bf16", state=N)
    views = dict(x)
    views["u"] = torch.cat([x["u"], x["u"]], -1)[..., E:]
    views["z"] = x["z"].transpose(0, 1).contiguous().transpose(0, 1)
    views["delta"] = torch.stack([x["delta"]] * 3, 2)[:, :, 1]
    low = torch.cat([x["B"].flatten(2), x["C"].flatten(2), normal(N, T, 5).to(x["B"].dtype)], -1)
    views["B"], views["C"] = low[..., :G * S].unflatten(-1, (G, S)), low[..., G * S:2 * G * S].unflatten(-1, (G, S))
    views["A"] = x["A"].t().contiguous().t()
    views["state"] = torch.cat([x["state"]] * 2, -1)[..., :S]
    results = []
    for v in (x, views):
        leaves = [t.detach().requires_grad_() for t in v.values()]
        y, last = vr.selective_scan(**dict(zip(v, leaves)), softplus=True, return_state=True)
        results.append([y, last, *torch.autograd.grad([y, last], leaves, [torch.ones_like(y).transpose(0, 1).contiguous().transpose(0, 1), torch.ones_like(last)])])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    u = x["u"][:, :1].expand(N, T, E)                      # one row for all tokens
    with torch.no_grad():
        assert torch.equal(vr.selective_scan(**{**x, "u": u}, softplus=True), vr.selective_scan(**{**x, "u": u.contiguous()}, softplus=True))


def test_no_tokens():
    x, normal = inputs(2, 0, 20, 16, 1, "fp32", state=2)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    y, last = vr.selective_scan(**leaves, softplus=True, return_state=True)
    assert y.shape == (2, 0, 20) and torch.equal(last, x["state"])
    g = torch.autograd.grad(last, leaves["state"], torch.ones_like(last))[0]
    assert torch.equal(g, torch.ones_like(last))
    x, _ = inputs(1, 7, 20, 16, 1, "fp32")
    y, last = vr.selective_scan(**x, offsets=torch.tensor([0], device=DEV), return_state=True)
    assert not y.any() and last.shape == (0, 20, 16)


def test_gradients_against_differences():
    """The sum of the results' products with given numbers, moved along a direction in every input, in steps of 2^-7: the difference's error is of third order, (2^-7)^2 / 6 of derivatives
    of a few units, 1e-4 of a gradient of order one, and the results' rounding 2^-24 over 2^-7."""
    x, normal = inputs(1, 21, 8, 5, 1, "fp32", state=1)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    weight = normal(1, 21, 8)
    f = lambda v: (vr.selective_scan(**v, softplus=True).double() * weight.double()).sum()
    grads = dict(zip(leaves, torch.autograd.grad(f(leaves), list(leaves.values()))))
    with torch.no_grad():
        for n in x:
            d = normal(*x[n].shape)
            d = d / d.norm()
            step = 2.0 ** -7
            up, down = f({**x, n: x[n] + step * d}), f({**x, n: x[n] - step * d})
            slope, want = (up - down).item() / (2 * step), (grads[n].double() * d.double()).sum().item()
            assert abs(slope - want) <= 2e-3 * max(1.0, grads[n].norm().item()), (n, slope, want)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("segments", [1, 6])
def test_infinities_and_nan_stay_with_their_tokens(dtype, segments, force):
    """An infinite or NaN token changes nothing in front of it, in other channels or in other sequences; behind it its channel holds what the recurrence makes of it."""
    force("scan_segments", segments)
    for bad in (float("inf"), float("nan")):
        x, _ = inputs(2, 100, 20, 10, 1, dtype)
        clean = vr.selective_scan(**x, softplus=True)
        x["u"][0, 40, 3] = bad
        y, last = vr.selective_scan(**x, softplus=True, return_state=True)
        same = torch.ones_like(y, dtype=torch.bool)
        same[0, 40:, 3] = False
        assert torch.equal(y[same], clean[same])
        want = reference({n: t for n, t in x.items()}, [(0, 0, 100), (1, 0, 100)], True)
        assert torch.equal(torch.isnan(last.cpu()), torch.isnan(want["last"][0])) and torch.equal(torch.isinf(last.cpu()), torch.isinf(want["last"][0]))
        assert torch.equal(torch.isfinite(y.cpu()), torch.isfinite(want["y"][0]))


@pytest.mark.parametrize("S", [10, 16, 35])
@pytest.mark.parametrize("segments", [0, 1, 6])
def test_infinite_step_sizes(segments, S, force):
    """A step of any length forgets what is in front of it: no gradient comes to that, and nothing else knows of it."""
    force("scan_segments", segments)
    x, normal = inputs(2, 300, 12, S, 1, "fp32", state=2)
    x["delta"][0, 40, 3] = x["u"][1, 290, 5] = float("inf")
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    y, last = vr.selective_scan(**leaves, softplus=True, return_state=True)
    gy = normal(*y.shape)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), gy)))
    want = reference(x, [(0, 0, 300), (1, 0, 300)], True, gy)
    assert torch.equal(torch.isfinite(y.cpu()), torch.isfinite(want["y"][0])) and torch.equal(torch.isfinite(last.cpu()), torch.isfinite(want["last"][0]))
    others = torch.ones(2, 300, 12, dtype=torch.bool)
    others[0, 40:, 3] = others[1, 290:, 5] = False
    for n in ("u", "delta", "z"):
        ref, scale = want[NAMES[n]]
        compare(grads[n].cpu()[others], (ref[others], scale[others]), NAMES[n], 300)
    rows = others.all(2)
    for n in ("B", "C"):
        ref, scale = want[NAMES[n]]
        compare(grads[n].cpu()[rows], (ref[rows], scale[rows]), NAMES[n], 300)
    compare(grads["state"], want["dstate"], "dstate", 300)
    clean = torch.tensor([e not in (3, 5) for e in range(12)])
    compare(grads["A"].cpu()[clean], tuple(t[clean] for t in want["dA"]), "dA", 300, tokens=600)


def test_states_far_from_one():
    """Decays that leave fp32 over a segment meet states of any size: nothing becomes NaN that the recurrence leaves finite."""
    x, _ = inputs(1, 640, 8, 16, 1, "fp32", state=1, softplus=False, bias=False)
    x["delta"].fill_(0.5)
    x["A"].copy_(torch.linspace(-300, -0.001, 128).reshape(8, 16))
    x["state"].fill_(3e38)
    x["state"][0, 7, 15] = float("inf")
    with vr.option("scan_segments", 10):
        y, last = vr.selective_scan(**x, return_state=True)
    want = reference(x, [(0, 0, 640)], False)
    assert torch.equal(torch.isinf(last.cpu()), torch.isinf(want["last"][0])) and not torch.isnan(last).any()
    keep = torch.isfinite(want["last"][0])
    assert ((last.cpu().double() - want["last"][0]).abs()[keep] <= 2100 * 2.0 ** -24 * want["last"][1][keep] + 1e-37).all()
    x["A"].copy_(torch.linspace(0.001, 0.3, 128).reshape(8, 16))   # growth: up to e^96 over the whole, from zeros and from small numbers
    x["state"].fill_(1e-30)
    x["B"].zero_()
    x["state"][0, 0].zero_()
    with vr.option("scan_segments", 10):
        last = vr.selective_scan(**x, return_state=True)[1]
    want = reference(x, [(0, 0, 640)], False)
    # (growth multiplies the argument's own error: 96 half steps more)
    assert ((last.cpu().double() - want["last"][0]).abs() <= 2300 * 2.0 ** -24 * want["last"][1]).all() and not last[0, 0].any()


# ---- one token at a time -----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("E,S,G", [(96, 16, 1), (33, 16, 3), (20, 4, 2), (50, 7, 1), (130, 8, 1), (24, 32, 1), (17, 64, 1), (9, 61, 1), (2000, 16, 2)])
def test_steps_are_what_sequences_are(E, S, G, dtype):
    N, T = 5, 6
    x, _ = inputs(N, T, E, S, G, dtype, state=N)
    bounds = [(n, 0, T) for n in range(N)]
    want = reference(x, bounds, True)
    pool = torch.full((9, E, S), 7.0, device=DEV)
    slots = torch.tensor([8, 0, 3, 5, 1], device=DEV)
    pool[slots] = x["state"]
    ys = []
    for t in range(T):
        tok = {n: x[n][:, t] for n in ("u", "delta", "B", "C", "z")}
        ys.append(vr.selective_scan_step(tok["u"], tok["delta"], x["A"], tok["B"], tok["C"], pool, slots if t % 2 else slots.int(), D=x["D"], z=tok["z"], delta_bias=x["delta_bias"], softplus=True))
    compare(torch.stack(ys, 1), want["y"], "y", T)
    compare(pool[slots], want["last"], "last", T)
    rest = torch.ones(9, dtype=torch.bool)
    rest[slots.cpu()] = False
    assert (pool[rest] == 7).all()


def test_step_slots():
    """Rows of one page are tokens behind each other; -1 is no place, other slots outside give NaN; neither touches a page."""
    N, E, S = 600, 40, 16
    x, normal = inputs(1, N, E, S, 1, "fp32")
    pool = normal(4, E, S)
    page = torch.tensor([n % 3 if n % 7 else (-1 if n % 2 else 4 + n) for n in range(N)], device=DEV)
    before = pool.clone()
    args = lambda r: (x["u"][0, r], x["delta"][0, r], x["A"], x["B"][0, r], x["C"][0, r])
    more = lambda r: dict(D=x["D"], z=x["z"][0, r], delta_bias=x["delta_bias"], softplus=True)
    everything = slice(0, N)
    y = vr.selective_scan_step(*args(everything), pool, page, **more(everything))
    for p in range(3):
        mine = (page == p).nonzero()[:, 0]
        one = {k: x[k][:, mine] for k in ("u", "delta", "B", "C", "z")}
        want = reference({**x, **one, "state": before[p:p + 1]}, [(0, 0, len(mine))], True)
        compare(y[mine][None], want["y"], "y", len(mine))
        compare(pool[p:p + 1], want["last"], "last", len(mine))
    assert torch.equal(pool[3], before[3])
    assert not y[page == -1].any() and torch.isnan(y[page >= 4]).all()


@pytest.mark.parametrize("E,S,G,dtype,shift", [(1100, 16, 2, "bf16", 0), (1090, 16, 1, "fp32", 1), (2200, 5, 2, "fp16", 0)])
def test_steps_of_many_rows(E, S, G, dtype, shift):
    """Pages named once, several times next to each other and far apart, and none, in a batch that fills the chip; a pool that does not lie at a multiple of 16 bytes."""
    N, P = 530, 300
    x, normal = inputs(1, N, E, S, G, dtype)
    gen = torch.Generator().manual_seed(E)
    page = torch.cat([torch.arange(200), torch.randint(180, P, (N - 220,), generator=gen), torch.tensor([5, 5, 5, 7, 7, 299, 299, 299, 299, 299, 5, 9, -1, -1, P, 9, 9, -7, 0, 0])])
    page = page.view(-1, 2).flip(1).reshape(-1)
    pool = torch.empty(P * E * S + shift, device=DEV)[shift:].view(P, E, S).copy_(normal(P, E, S))
    before = pool.clone()
    y = vr.selective_scan_step(x["u"][0], x["delta"][0], x["A"], x["B"][0], x["C"][0], pool, page.to(DEV), D=x["D"], z=x["z"][0], delta_bias=x["delta_bias"], softplus=True)
    known = (page >= 0) & (page < P)
    order = torch.arange(N)[known]
    order = order[page[order].argsort(stable=True)]        # the rows of each page one after the other
    pages, counts = page[order].unique_consecutive(return_counts=True)
    ends = counts.cumsum(0).tolist()
    rows = {n: x[n][:, order.to(DEV)] for n in ("u", "delta", "B", "C", "z")}
    want = reference({**x, **rows, "state": before[pages.to(DEV)]}, [(0, j - n, j) for j, n in zip(ends, counts.tolist())], True)
    compare(y[order.to(DEV)][None], want["y"], "y", int(counts.max()))
    compare(pool[pages.to(DEV)], want["last"], "last", int(counts.max()))
    rest = torch.ones(P, dtype=torch.bool)
    rest[pages] = False
    assert torch.equal(pool[rest.to(DEV)], before[rest.to(DEV)])
    assert not y[(page == -1).to(DEV)].any() and torch.isnan(y[((page < -1) | (page >= P)).to(DEV)]).all()


def test_step_pools():
    """Pages at a distance (one layer of a pool for all), without slots, pools without pages."""
    E, S = 24, 16
    x, normal = inputs(1, 3, E, S, 1, "bf16")
    tok = lambda n: x[n][0]
    call = lambda pool, slots=None: vr.selective_scan_step(tok("u"), tok("delta"), x["A"], tok("B"), tok("C"), pool, slots, D=x["D"], z=tok("z"), delta_bias=x["delta_bias"], softplus=True)
    layers = normal(5, 2, E, S)
    alone = layers[:, 1].clone()
    kept = layers[:, 0].clone()
    assert torch.equal(call(layers[:, 1]), call(alone)) and torch.equal(layers[:, 1], alone) and torch.equal(layers[:, 0], kept)
    odd = torch.zeros(5 * E * S + 1, device=DEV)[1:].view(5, E, S)   # (not at a multiple of 16 bytes)
    odd.copy_(kept)
    even = kept.clone()
    assert torch.equal(call(odd), call(even)) and torch.equal(odd, even)
    y = call(torch.empty(0, E, S, device=DEV), torch.tensor([-1, 0, 3], device=DEV))
    assert not y[0].any() and torch.isnan(y[1:]).all()
    version = alone._version
    call(alone)
    assert alone._version > version


# ---- how it is called --------------------------------------------------------------------------------------------------

def test_refusals():
    x, normal = inputs(2, 9, 20, 16, 2, "bf16", state=2)
    ok = dict(x, softplus=True)
    bad = [dict(u=x["u"].float()), dict(u=x["u"].cpu()), dict(u=x["u"][0]), dict(delta=x["delta"][:, :8]), dict(A=x["A"].bfloat16()), dict(A=normal(20, 65)), dict(A=x["A"][:10]), dict(B=x["B"][:, :, :1]),
           dict(B=x["B"].float()), dict(C=x["C"][:, :, :, :8]), dict(D=x["D"].half()), dict(D=x["D"][:5]), dict(delta_bias=x["delta_bias"][:3]), dict(z=x["z"][:1]), dict(state=x["state"].bfloat16()),
           dict(state=x["state"][:1]), dict(offsets=torch.tensor([0, 9], device=DEV)), dict(B=x["B"][:, :, :1].expand(2, 9, 3, 16), C=x["C"][:, :, :1].expand(2, 9, 3, 16))]
    for change in bad:
        with pytest.raises(RuntimeError):
            vr.selective_scan(**{**ok, **change})
    one = {n: (t[:1] if n in ("u", "delta", "B", "C", "z", "state") else t) for n, t in x.items()}
    for offsets in (torch.tensor([0.0, 9.0], device=DEV), torch.tensor([0, 9]), torch.tensor([[0, 9]], device=DEV), torch.tensor([], dtype=torch.int32, device=DEV), torch.tensor([0, 3, 9], device=DEV)):
        with pytest.raises(RuntimeError):
            vr.selective_scan(**one, offsets=offsets)
    tok = {n: x[n][:, 0] for n in ("u", "delta", "B", "C", "z")}
    step = lambda pool, slots=None, **k: vr.selective_scan_step(**{**dict(u=tok["u"], delta=tok["delta"], A=x["A"], B=tok["B"], C=tok["C"]), **k}, pool=pool, slots=slots)
    pool = normal(4, 20, 16)
    for p, s in ((pool.bfloat16(), None), (pool[:, :10], None), (pool.transpose(1, 2).contiguous().transpose(1, 2), None), (pool[:1], None), (pool[:1].expand(4, 20, 16), None), (pool, torch.tensor([0], device=DEV)),
                 (pool, torch.tensor([0.0, 1.0], device=DEV)), (pool, torch.tensor([0, 1])), (pool.clone().requires_grad_(), None)):
        with pytest.raises(RuntimeError):
            step(p, s)
    with pytest.raises(RuntimeError):
        step(pool, u=tok["u"].clone().requires_grad_())


def test_other_streams_and_graphs(force):
    """On a stream of its own, and recorded into a graph that is replayed with new numbers in the same memory, gradients too."""
    force("scan_segments", 3)
    x, normal = inputs(2, 150, 64, 16, 1, "bf16", state=2)
    leaves = {n: t.clone().requires_grad_() for n, t in x.items()}
    gy, gl = normal(2, 150, 64).bfloat16(), normal(2, 64, 16)

    def call():
        y, last = vr.selective_scan(**leaves, softplus=True, return_state=True)
        return [y.detach(), last.detach(), *torch.autograd.grad([y, last], list(leaves.values()), [gy, gl])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            got = call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b in zip(got, call()):
        assert torch.equal(a, b)
    del a, b, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = call()
    for k in range(3):
        with torch.no_grad():
            for n in ("u", "delta", "B", "C", "z", "state"):
                leaves[n].copy_(normal(*leaves[n].shape) * (0.5 if n == "delta" else 1.0))
            gy.copy_(normal(2, 150, 64))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(recorded, call()):
            assert torch.equal(a, b), k


def test_recordings_and_transforms_are_refused():
    x, normal = inputs(2, 9, 20, 16, 1, "fp32")
    call = lambda u: vr.selective_scan(**{**x, "u": u}, softplus=True)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward mode"):
            call(torch.autograd.forward_ad.make_dual(x["u"], x["u"]))
    with pytest.raises(RuntimeError):
        torch.jit.trace(call, (x["u"],))
    with pytest.raises(RuntimeError):
        torch.func.vmap(call)(torch.stack([x["u"]] * 2))
    u = x["u"].clone().requires_grad_()
    y = call(u)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, u, torch.stack([y.detach()] * 2), is_grads_batched=True)
    g = torch.autograd.grad(call(u).sum(), u, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), u)


def test_inputs_that_change_before_the_backward_are_noticed():
    x, _ = inputs(1, 20, 20, 16, 1, "fp32")
    u = x["u"].clone().requires_grad_()
    y = vr.selective_scan(**{**x, "u": u * 1.0, "B": x["B"]}, softplus=True)
    x["B"].add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_workspaces_that_hold_anything():
    """Memory that the allocator hands out again is not read before it is written."""
    x, normal = inputs(2, 150, 40, 10, 2, "bf16", state=2)
    bounds = [(0, 0, 150), (1, 0, 150)]
    for _ in range(2):
        junk = [torch.full((1 << k,), float("nan"), device=DEV) for k in range(10, 24)]
        del junk
        with vr.option("scan_segments", 4):
            run_and_compare(x, normal, bounds)
