"""Cases of the selective state space scan, the short causal convolution in front of it and the root-mean-square norm around both.

With u (E channels), a step size dt for each token and channel, A (E, S), B and C (G groups of S states) and h (E, S) one sequence's state:

    h_t = exp(dt_t A) h_{t-1} + dt_t u_t B_t^T          y_t = (h_t C_t + D u_t) silu(z_t)          dt = softplus(delta + delta_bias)

Kinds
  conv, conv_train   y_t = silu(sum_j w_j x_{t-K+1+j} + b) of whole sequences and the last K - 1 tokens of each; with the gradients of x, w, b and the first state
  conv_step          one more token for each of N sequences, whose last K - 1 tokens are pages of a pool that is updated in place
  scan, scan_train   y and the last states of whole sequences (rows of a batch, or packed behind each other); with all gradients
  scan_step          one more token for each of N sequences, whose states are pages of such a pool
  norm, norm_train   r = x + residual, y = r / sqrt(mean(r^2) + eps) w, y in 16 or 32 bits or in 8 with a scale for each row; with all gradients

`run` computes them in elementary torch operations, or with `own` through the package's entry points.
"""
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_DEV = "cuda"
_EPS = 1e-6


def listed():
    return [
        # a server's batch of prompts of all lengths, packed, that go on from earlier tokens
        dict(name="conv_packed_states", kind="conv", N=48, T=2048, E=1536, K=4, dtype="bf16", params="bf16", act=True, bias=True, packed=True, state=True),
        # one layer's convolution in bf16 training of a base-size model with twice as many inner channels
        dict(name="conv_train_base", kind="conv_train", N=64, T=196, E=1536, K=4, dtype="bf16", params="bf16", act=True, bias=True, packed=False, state=False),
        # the next token of one sequence of a tiny model: latency
        dict(name="conv_step_one", kind="conv_step", N=1, P=4, E=384, K=4, dtype="bf16", params="bf16", act=True, bias=True),
        # the next token of a server's whole batch
        dict(name="conv_step_batch", kind="conv_step", N=512, P=640, E=1536, K=4, dtype="bf16", params="bf16", act=True, bias=True),
        # one image's tokens through a layer of a tiny model: the smallest prompt, all latency
        dict(name="scan_one_image", kind="scan", N=1, T=196, E=384, S=16, G=1, dtype="bf16", params="fp32", gate=True, skip=True, soft=True, packed=False, state=False),
        # packed prompts of all lengths that go on from earlier states, groups of channels with their own B and C, an odd number of channels
        dict(name="scan_packed_fp16", kind="scan", N=48, T=2048, E=1110, S=16, G=2, dtype="fp16", params="fp32", gate=True, skip=True, soft=True, packed=True, state=True),
        # one layer's scan in bf16 training of a base-size model
        dict(name="scan_train_base", kind="scan_train", N=64, T=196, E=1536, S=16, G=1, dtype="bf16", params="fp32", gate=True, skip=True, soft=True, packed=False, state=False),
        # detection fine-tuning: two images of about 1333 x 800 in fp32
        dict(name="scan_train_dense_fp32", kind="scan_train", N=2, T=4150, E=768, S=16, G=1, dtype="fp32", params="fp32", gate=True, skip=True, soft=True, packed=False, state=False),
        # the next token of one sequence of a tiny model: latency
        dict(name="scan_step_one", kind="scan_step", N=1, P=4, E=384, S=16, G=1, dtype="bf16", params="fp32", gate=True, skip=True, soft=True),
        # the next token of a server's whole batch
        dict(name="scan_step_batch", kind="scan_step", N=512, P=640, E=1536, S=16, G=1, dtype="bf16", params="fp32", gate=True, skip=True, soft=True),
        # the norm in front of an 8-bit product: a batch of images of a base-size model, with the residual's addition
        dict(name="norm_8bit_residual", kind="norm", rows=12544, E=768, dtype="bf16", params="bf16", residual="bf16", eight=True),
        # the same norm in bf16 training, its residual in fp32
        dict(name="norm_train_base", kind="norm_train", rows=12544, E=768, dtype="bf16", params="bf16", residual="fp32", eight=False),
    ]


def _log_int(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["conv", "conv_train", "conv_step", "scan", "scan", "scan_train", "scan_train", "scan_step", "norm", "norm_train"])
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    params = rng.choice(["fp32", dtype])
    E = rng.choice([192, 384, 768, 1536]) if rng.random() < 0.5 else _log_int(rng, 16, 2048)
    if kind.startswith("norm"):
        E = E if rng.random() < 0.6 else _log_int(rng, 16, 8192)
        rows = _log_int(rng, 1, min(16384, 12544 * 768 // E))
        return dict(kind=kind, rows=rows, E=E, dtype=dtype, params=params, residual=rng.choice(["none", "fp32", dtype]), eight=kind == "norm" and rng.random() < 0.5)
    S = 16 if rng.random() < 0.6 else rng.choice([8, 32, 64]) if rng.random() < 0.5 else rng.randint(1, 64)
    G = 1 if rng.random() < 0.7 else rng.choice([d for d in (1, 2, 3, 4) if E % d == 0])
    K = 4 if rng.random() < 0.6 else rng.randint(2, 8)
    sizes = dict(E=E, K=K, dtype=dtype, params=params, act=rng.random() < 0.8, bias=rng.random() < 0.8) if kind.startswith("conv") else \
        dict(E=E, S=S, G=G, dtype=dtype, params=params, gate=rng.random() < 0.7, skip=rng.random() < 0.8, soft=rng.random() < 0.8)
    if kind.endswith("_step"):
        N = _log_int(rng, 1, max(1, min(512, 512 * 1536 * 16 // (E * (S if kind == "scan_step" else 16)))))
        return dict(kind=kind, N=N, P=N + rng.randint(0, N // 2 + 3), **sizes)
    # one token up to long sequences; the cost goes by tokens, channels and, for a scan, by its states in fours
    each = E if kind.startswith("conv") else E * -(-S // 4) * 4 // 16
    most = 64 * 196 * 1536 // max(each, 1) // (2 if dtype == "fp32" or S > 16 else 1)
    T = _log_int(rng, 1, min(8192 if not kind.endswith("train") else 4150, most))
    N = _log_int(rng, 1, max(1, min(64, most // T)))
    return dict(kind=kind, N=N, T=T, **sizes, packed=rng.random() < 0.4, state=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lengths(case):
    """The lengths of a packed case's sequences, the same for every seed: spread over the logarithm of 1 .. T, one of them T, and one empty where
    there are several."""
    r = np.random.default_rng(case["N"] * 100_000 + case["T"])
    n = np.maximum(1, np.round(case["T"] ** r.random(case["N"]))).astype(np.int64)
    n[r.integers(case["N"])] = case["T"]
    if case["N"] > 2:
        n[(int(np.argmax(n)) + 1) % case["N"]] = 0
    return n


def _generator(seed):
    gen = torch.Generator(_DEV).manual_seed(seed)
    return lambda *s: torch.randn(*s, generator=gen, device=_DEV), lambda *s: torch.rand(*s, generator=gen, device=_DEV)


def _batch(case, s):
    """The rows of a case's token tensors; a packed one has the offsets of its sequences too."""
    if case["kind"].endswith("_step"):
        return (case["N"],)
    if not case["packed"]:
        return case["N"], case["T"]
    n = _lengths(case)
    s["offsets"] = torch.from_numpy(np.concatenate([[0], np.cumsum(n)])).to(device=_DEV, dtype=torch.int32)
    return 1, int(n.sum())


def _pages(case, seed, s):
    s["slots"] = torch.from_numpy(np.random.default_rng(seed).permutation(case["P"])[:case["N"]].astype(np.int32)).to(_DEV)


def prepare(case, seed):
    kind, dt, pt = case["kind"].split("_")[0], _DTYPES[case["dtype"]], _DTYPES[case["params"]]
    normal, uniform = _generator(seed)
    E, s = case["E"], {"case": case, "state": None}
    train = case["kind"].endswith("_train")
    if kind == "norm":
        s["x"] = normal(case["rows"], E).to(dt)
        s["w"] = (1 + 0.2 * normal(E)).to(pt)
        s["residual"] = None if case["residual"] == "none" else (2 * normal(case["rows"], E)).to(_DTYPES[case["residual"]])
        names = ("x", "w", "residual")
        outs = [((case["rows"], E), dt)] + ([((case["rows"], E), s["residual"].dtype)] if s["residual"] is not None else [])
    elif kind == "conv":
        rows = _batch(case, s)
        s["x"] = normal(*rows, 2 * E).to(dt)[..., :E]                          # one half of a projection's result
        s["w"] = (normal(E, case["K"]) * case["K"] ** -0.5).to(pt)
        s["b"] = (0.2 * normal(E)).to(pt) if case["bias"] else None
        if case["kind"] == "conv_step":
            s["pool"] = normal(case["P"], case["K"] - 1, E).to(dt)
            _pages(case, seed, s)
            return s
        if case["state"]:
            s["state"] = normal(case["N"], case["K"] - 1, E).to(dt)
        names = ("x", "w", "b", "state")
        outs = [((*rows, E), dt), ((case["N"], case["K"] - 1, E), dt)]
    else:
        rows, S, G = _batch(case, s), case["S"], case["G"]
        s["u"] = normal(*rows, E).to(dt)
        dt0 = torch.exp(math.log(1e-3) + uniform(E) * math.log(1e2))           # step sizes of 1e-3 to 1e-1, token by token around them
        if case["soft"]:
            s["delta"] = (0.5 * normal(*rows, E)).to(dt)
            s["delta_bias"] = (dt0 + torch.log(-torch.expm1(-dt0))).to(pt)
        else:
            s["delta"] = (dt0 * torch.exp(0.5 * normal(*rows, E))).to(dt)
            s["delta_bias"] = None
        s["A"] = -torch.arange(1, S + 1, device=_DEV) * torch.exp(0.1 * normal(E, S))
        low = (normal(*rows, 48 + 2 * G * S)).to(dt)                           # the projection that step sizes, B and C come from
        s["B"], s["C"] = (low[..., 48 + i * G * S:48 + (i + 1) * G * S].unflatten(-1, (G, S)) for i in (0, 1))
        s["D"] = (1 + 0.1 * normal(E)).to(pt) if case["skip"] else None
        s["z"] = normal(*rows, 2 * E).to(dt)[..., E:] if case["gate"] else None
        if case["kind"] == "scan_step":
            s["pool"] = normal(case["P"], E, S)
            _pages(case, seed, s)
            return s
        if case["state"]:
            s["state"] = normal(case["N"], E, S)
        names = ("u", "delta", "A", "B", "C", "D", "z", "delta_bias", "state")
        outs = [((*rows, E), dt), ((case["N"], E, S), torch.float32)]
    if train:
        s["leaves"] = []
        for n in names:
            if s[n] is not None:
                s[n] = s[n].detach().requires_grad_()
                s["leaves"].append(s[n])
        s["grads"] = [normal(*shape).to(t) for shape, t in outs]
        if kind != "norm" and not case["state"]:
            s["grads"][1] = None                                               # no gradient comes to the last states
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(s):
    kind = s["case"]["kind"]
    if own:
        out = _own(s)
        if not kind.endswith("_train"):
            return out
        some = [(y, g) for y, g in zip(out, s["grads"]) if g is not None]
        grads = torch.autograd.grad([y for y, _ in some], s["leaves"], [g for _, g in some])
        return [y.detach() for y in out] + list(grads)
    with torch.no_grad():
        return {"conv": _plain_conv, "scan": _plain_scan, "norm": _plain_norm}[kind.split("_")[0]](s) if not kind.endswith("_step") else \
            (_plain_conv_step if kind == "conv_step" else _plain_scan_step)(s)


def _own(s):
    import vision_rwkv_amd as vr
    case, kind = s["case"], s["case"]["kind"]
    if kind.startswith("norm"):
        out = vr.rms_norm(s["x"], s["w"], s["residual"], eps=_EPS, quantize=torch.float8_e4m3fn if case["eight"] else None)
        return out if isinstance(out, tuple) else (out,)
    if kind == "conv_step":
        return vr.causal_conv_step(s["x"], s["w"], s["pool"], s["slots"], bias=s["b"], activation="silu" if case["act"] else None), s["pool"]
    if kind.startswith("conv"):
        return vr.causal_conv(s["x"], s["w"], s["b"], activation="silu" if case["act"] else None, state=s["state"], offsets=s.get("offsets"), return_state=True)
    args = s["u"], s["delta"], s["A"], s["B"], s["C"]
    more = dict(D=s["D"], z=s["z"], delta_bias=s["delta_bias"], softplus=case["soft"])
    if kind == "scan_step":
        return vr.selective_scan_step(*args, s["pool"], s["slots"], **more), s["pool"]
    return vr.selective_scan(*args, **more, state=s["state"], offsets=s.get("offsets"), return_state=True)


def _silu(x):
    return x / (1 + torch.exp(-x))


def _silu_slope(x):
    p = 1 / (1 + torch.exp(-x))
    return p * (1 + x * (1 - p))


def _places(s, rows):
    """For each row of tokens (batch, T): its sequence, its place in it and the places behind it, and whether there is a sequence at all."""
    if "offsets" not in s:
        t = torch.arange(rows[1], device=_DEV).expand(rows)
        n = torch.arange(rows[0], device=_DEV)[:, None].expand(rows)
        return n, t, rows[1] - 1 - t, torch.ones(rows, dtype=torch.bool, device=_DEV)
    off = s["offsets"].long()
    t = torch.arange(rows[1], device=_DEV)
    n = torch.searchsorted(off[1:], t, right=True)
    inside = n < off.numel() - 1
    n = n.clamp(max=off.numel() - 2)
    return n[None], (t - off[n])[None], (off[n + 1] - 1 - t)[None], inside[None]


# -- the convolution

def _plain_conv(s):
    case, K = s["case"], s["case"]["K"]
    x, w = s["x"].float(), s["w"].float()
    rows, E, N = x.shape[:2], case["E"], case["N"]
    n, t, behind, inside = _places(s, rows)
    first = torch.zeros(N, K - 1, E, device=_DEV) if s["state"] is None else s["state"].float()
    taps = []                                              # tap j of every row: the token K - 1 - j places in front, or one of the first state
    for j in range(K):
        back = K - 1 - j
        shifted = torch.nn.functional.pad(x, (0, 0, back, 0))[:, :rows[1]]
        taps.append(shifted if back == 0 else torch.where((t >= back)[..., None], shifted, first[n, (K - 1 + t - back).clamp(max=K - 2)]))
    pre = sum(w[:, j] * taps[j] for j in range(K)) + (0 if s["b"] is None else s["b"].float())
    y = torch.where(inside[..., None], _silu(pre) if case["act"] else pre, 0)
    last = first.clone()
    for i in range(K - 1):                                 # places length - (K - 1) + i, in the sequence or in the state in front of it
        at = (behind == K - 2 - i) & inside
        last[n[at], i] = x[at]
    length = torch.zeros(N, dtype=torch.long, device=_DEV).index_add_(0, n.expand(rows)[inside], torch.ones_like(n.expand(rows)[inside]))
    moved = torch.arange(K - 1, device=_DEV) + length[:, None]
    last = torch.where((moved < K - 1)[..., None], first.gather(1, moved.clamp(max=K - 2)[..., None].expand(-1, -1, E)), last)
    out = [y.to(s["x"].dtype), last.to(s["x"].dtype)]
    if not case["kind"].endswith("_train"):
        return tuple(out)
    gy, glast = s["grads"]
    g = torch.where(inside[..., None], gy.float() * (_silu_slope(pre) if case["act"] else 1), 0)
    dx, dfirst, dw = torch.zeros_like(x), torch.zeros_like(first), []
    for j in range(K):
        back = K - 1 - j
        dw.append((g * taps[j]).sum((0, 1)))
        part = torch.nn.functional.pad(g * w[:, j], (0, 0, 0, back))[:, back:]
        dx += torch.where(((behind >= back) & inside)[..., None], part, 0)
        if back:
            early = (t < back) & inside
            dfirst.index_put_((n[early], K - 1 + t[early] - back), (g * w[:, j])[early], accumulate=True)
    if glast is not None:
        for i in range(K - 1):
            at = (behind == K - 2 - i) & inside
            dx[at] += glast[n[at], i].float()
        keep = torch.where((moved < K - 1)[..., None], glast.float(), 0)
        dfirst.scatter_add_(1, moved.clamp(max=K - 2)[..., None].expand(-1, -1, E), keep)
    grads = [dx.to(s["x"].dtype), torch.stack(dw, 1).to(s["w"].dtype)]
    grads += [g.sum((0, 1)).to(s["b"].dtype)] if s["b"] is not None else []
    return out + grads + ([dfirst.to(s["x"].dtype)] if s["state"] is not None else [])


def _plain_conv_step(s):
    case, slots = s["case"], s["slots"].long()
    window = torch.cat([s["pool"][slots], s["x"][:, None]], 1)
    pre = (window.float() * s["w"].float().T).sum(1) + (0 if s["b"] is None else s["b"].float())
    s["pool"][slots] = window[:, 1:]
    return (_silu(pre) if case["act"] else pre).to(s["x"].dtype), s["pool"]


# -- the scan

def _step_size(s):
    raw = s["delta"].float()
    raw = raw if s["delta_bias"] is None else raw + s["delta_bias"].float()
    return raw, torch.logaddexp(raw, torch.zeros_like(raw)) if s["case"]["soft"] else raw


def _of_channels(x, E):
    """x (..., G, S) for each of E channels: (..., E, S)."""
    x = x.float()
    return x.repeat_interleave(E // x.shape[-2], -2) if x.shape[-2] > 1 else x.expand(*x.shape[:-2], E, x.shape[-1])


def _carried(h, e):
    """h_t + e_t h_{t-1} + e_t e_{t-1} h_{t-2} + .. along dimension 1, by doubling; h and e are overwritten."""
    d = 1
    while d < h.shape[1]:
        h[:, d:] += e[:, d:] * h[:, :-d]
        e[:, d:] = e[:, d:] * e[:, :-d]
        d *= 2
    return h


def _plain_scan(s):
    case, E, G, N = s["case"], s["case"]["E"], s["case"]["G"], s["case"]["N"]
    u, rows = s["u"].float(), s["u"].shape[:2]
    n, t, behind, inside = _places(s, rows)
    raw, dt = _step_size(s)
    B, C = _of_channels(s["B"], E), _of_channels(s["C"], E)
    starts, ends, there = (t == 0) & inside, (behind == 0) & inside, inside[..., None, None]
    state = torch.zeros(N, E, case["S"], device=_DEV) if s["state"] is None else s["state"]
    e = torch.exp(dt[..., None] * s["A"])
    h = torch.where(there, (dt * u)[..., None] * B, 0)
    h[starts] += e[starts] * state[n[starts]]
    onward = torch.where(starts[..., None, None] | ~there, 0, e)
    train = case["kind"].endswith("_train")
    h = _carried(h, onward.clone() if train else onward)
    inner = (h * C).sum(-1) + (0 if s["D"] is None else s["D"].float() * u)
    z = None if s["z"] is None else s["z"].float()
    y = torch.where(inside[..., None], inner if z is None else inner * _silu(z), 0)
    last = state.clone()
    last[n[ends]] = h[ends]
    out = [y.to(s["u"].dtype), last]
    if not train:
        return tuple(out)
    gy, glast = s["grads"]
    gy = torch.where(inside[..., None], gy.float(), 0)
    g = gy if z is None else gy * _silu(z)
    R = g[..., None] * C
    if glast is not None:
        R[ends] += glast[n[ends]]
    back = torch.cat([onward[:, 1:], torch.zeros_like(onward[:, :1])], 1)
    R = _carried(R.flip(1), back.flip(1)).flip(1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    before[starts] = state[n[starts]]
    through = R * e
    dstate = torch.zeros_like(state) if glast is None else glast.clone()
    dstate[n[starts]] = through[starts]
    through *= before                                      # the gradient of dt A
    along_B = (R * B).sum(-1)
    ddt = (through * s["A"]).sum(-1) + u * along_B
    ddt = torch.where(inside[..., None], ddt / (1 + torch.exp(-raw)) if case["soft"] else ddt, 0)
    du = dt * along_B + (0 if s["D"] is None else s["D"].float() * g)
    share = lambda x: x.unflatten(2, (G, E // G)).sum(3)  # noqa: E731
    through = torch.where(there, through * dt[..., None], 0)
    grads = [torch.where(inside[..., None], du, 0), ddt, through.sum((0, 1)), torch.where(there, share(R * (dt * u)[..., None]), 0), share(g[..., None] * h)]
    grads += [(g * u).sum((0, 1))] if s["D"] is not None else []
    grads += [gy * inner * _silu_slope(z)] if z is not None else []
    grads += [ddt.sum((0, 1))] if s["delta_bias"] is not None else []
    grads += [dstate] if s["state"] is not None else []
    return out + [g.to(x.dtype) for g, x in zip(grads, s["leaves"])]


def _plain_scan_step(s):
    case, slots = s["case"], s["slots"].long()
    u = s["u"].float()
    _, dt = _step_size(s)
    h = torch.exp(dt[..., None] * s["A"]) * s["pool"][slots] + (dt * u)[..., None] * _of_channels(s["B"], case["E"])
    s["pool"][slots] = h
    y = (h * _of_channels(s["C"], case["E"])).sum(-1) + (0 if s["D"] is None else s["D"].float() * u)
    return (y if s["z"] is None else y * _silu(s["z"].float())).to(s["u"].dtype), s["pool"]


# -- the norm

def _plain_norm(s):
    case, x, w = s["case"], s["x"], s["w"].float()
    r = x if s["residual"] is None else (x.float() + s["residual"].float()).to(s["residual"].dtype)
    v = r.float()
    scale = torch.rsqrt((v * v).mean(-1, keepdim=True) + _EPS)
    normed = v * scale
    y = normed * w
    if case["eight"]:
        step = (y.abs().amax(-1) / 448).clamp(min=2.0 ** -126)
        out = [(y / step[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn), step]
    else:
        out = [y.to(x.dtype)]
    out += [] if s["residual"] is None else [r]
    if case["kind"] == "norm":
        return tuple(out)
    gy = s["grads"][0].float()
    gn = gy * w
    dr = scale * (gn - normed * (gn * normed).mean(-1, keepdim=True))
    dw = (gy * normed).sum(0).to(s["w"].dtype)
    if s["residual"] is None:
        return out + [dr.to(x.dtype), dw]
    dr = dr + s["grads"][1].float()
    return out + [dr.to(x.dtype), dw, dr.to(s["residual"].dtype)]


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    kind, e, p, E = case["kind"], _BYTES[case["dtype"]], _BYTES[case["params"]], case["E"]
    train = kind.endswith("_train")
    if kind.startswith("norm"):
        n, r = case["rows"] * E, _BYTES.get(case["residual"], 0)
        moved = n * (e + (1 if case["eight"] else e) + 2 * r) + E * p + (4 * case["rows"] if case["eight"] else 0)
        return {"bytes": moved + (n * (2 * e + 2 * r) + E * p if train else 0), "flops": n * (5 + (8 if train else 0))}
    if kind.endswith("_step"):
        rows = case["N"]
    else:
        rows = case["N"] * case["T"] if not case["packed"] else int(_lengths(case).sum())
    if kind.startswith("conv"):
        K = case["K"]
        page, params = (K - 1) * E * e, E * p * (K + case["bias"])
        if kind == "conv_step":
            return {"bytes": rows * E * e * 2 + rows * page * 2 + params, "flops": rows * E * 2 * K}
        states = case["N"] * page * (2 if case["state"] else 1)
        moved = rows * E * e * 2 + states + params
        if train:
            moved += rows * E * e * 2 + params + (2 * case["N"] * page if case["state"] else 0)
        return {"bytes": moved, "flops": rows * E * 2 * K * (3 if train else 1)}
    S, G = case["S"], case["G"]
    page = E * S * 4
    tokens = rows * (E * (3 + case["gate"]) + 2 * G * S) * e
    params = page + E * p * (case["skip"] + case["soft"])
    # for each token, channel and state: the decay's argument and exponential, the token's part and its addition, the product with C
    if kind == "scan_step":
        return {"bytes": tokens + params + 2 * rows * page, "flops": rows * E * S * 7}
    moved = tokens + params + case["N"] * page * (2 if case["state"] else 1)
    if train:                                              # gy read, the inputs' gradients written; the state again, its gradient, and six sums of both
        moved += tokens + params + (2 * case["N"] * page if case["state"] else 0)
    return {"bytes": moved, "flops": rows * E * S * (7 + (16 if train else 0))}


# ---- the definition, token by token, in 64 bits ----------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    wide = {n: v.detach().double().requires_grad_(v.requires_grad) if isinstance(v, torch.Tensor) and v.is_floating_point() else v for n, v in s.items()}
    with torch.set_grad_enabled(kind.endswith("_train")):
        if kind.endswith("_step"):
            return (_exact_conv_step if kind == "conv_step" else _exact_scan_step)(wide)
        out = {"conv": _exact_conv, "scan": _exact_scan, "norm": _exact_norm}[kind.split("_")[0]](wide, s)
    if not kind.endswith("_train"):
        return out
    names = {id(v): n for n, v in s.items() if isinstance(v, torch.Tensor)}
    leaves = [wide[names[id(v)]] for v in s["leaves"]]
    some = [(y, g.double()) for y, g in zip(out, s["grads"]) if g is not None]
    grads = torch.autograd.grad([y for y, _ in some], leaves, [g for _, g in some])
    return [y.detach() for y in out] + list(grads)


def _sequences(w):
    """The (batch row, first, end) of each sequence."""
    if "offsets" in w:
        off = w["offsets"].tolist()
        return [(0, a, b) for a, b in zip(off[:-1], off[1:])]
    x = w["x"] if "x" in w else w["u"]
    return [(n, 0, x.shape[1]) for n in range(x.shape[0])]


def _exact_conv(w, s):
    K, ys, last = w["case"]["K"], [], []
    for n, (b, i, j) in enumerate(_sequences(w)):
        front = w["x"].new_zeros(K - 1, w["x"].shape[2]) if w["state"] is None else w["state"][n]
        whole = torch.cat([front, w["x"][b, i:j]])
        pre = torch.einsum("tck,ck->tc", whole.unfold(0, K, 1), w["w"]) if j > i else whole[:0]
        pre = pre if w["b"] is None else pre + w["b"]
        ys.append(pre * torch.sigmoid(pre) if w["case"]["act"] else pre)
        last.append(whole[whole.shape[0] - (K - 1):])
    return [torch.cat(ys).reshape(w["x"].shape), torch.stack(last)]


def _exact_conv_step(w):
    pool, ys = w["pool"], []
    for n, slot in enumerate(w["slots"].tolist()):
        whole = torch.cat([pool[slot], w["x"][n][None]])
        pre = torch.einsum("kc,ck->c", whole, w["w"])
        pre = pre if w["b"] is None else pre + w["b"]
        ys.append(pre * torch.sigmoid(pre) if w["case"]["act"] else pre)
        pool[slot] = whole[1:]
    return torch.stack(ys), pool


def _exact_size(w):
    raw = w["delta"] if w["delta_bias"] is None else w["delta"] + w["delta_bias"]
    return torch.where(raw > 0, raw, 0) + torch.log1p(torch.exp(-raw.abs())) if w["case"]["soft"] else raw


def _exact_scan(w, s):
    """Along the tokens, all sequences that still have one at a time; the gradients by automatic differentiation of that."""
    case, seqs = w["case"], _sequences(w)
    E, S, group = case["E"], case["S"], case["E"] // case["G"]
    order = sorted(range(len(seqs)), key=lambda n: seqs[n][1] - seqs[n][2])    # the longest first
    row = torch.tensor([seqs[n][0] for n in order], device=_DEV)
    first = torch.tensor([seqs[n][1] for n in order], device=_DEV)
    length = [seqs[n][2] - seqs[n][1] for n in order]
    perm = torch.tensor(order, device=_DEV)
    h = w["u"].new_zeros(len(seqs), E, S) if w["state"] is None else w["state"][perm]
    dt, g = _exact_size(w), torch.arange(E, device=_DEV) // group
    done, ys, at = [], [], []
    for t in range(max(length)):
        n = sum(x > t for x in length)
        if n < h.shape[0]:
            done.append(h[n:])
            h = h[:n]
        i = (row[:n], first[:n] + t)
        d = dt[i]
        h = torch.exp(d[:, :, None] * w["A"]) * h + (d * w["u"][i])[:, :, None] * w["B"][i][:, g]
        y = torch.einsum("nes,nes->ne", h, w["C"][i][:, g])
        y = y if w["D"] is None else y + w["D"] * w["u"][i]
        ys.append(y if w["z"] is None else y * w["z"][i] * torch.sigmoid(w["z"][i]))
        at.append(i)
    ended = torch.cat([h] + done[::-1])
    y = torch.zeros_like(w["u"]).index_put((torch.cat([a for a, _ in at]), torch.cat([b for _, b in at])), torch.cat(ys))
    return [y, torch.zeros_like(ended).index_copy(0, perm, ended)]


def _exact_scan_step(w):
    case, pool, ys = w["case"], w["pool"], []
    g, dt = torch.arange(case["E"], device=_DEV) // (case["E"] // case["G"]), _exact_size(w)
    for n, slot in enumerate(w["slots"].tolist()):
        pool[slot] = torch.exp(dt[n][:, None] * w["A"]) * pool[slot] + (dt[n] * w["u"][n])[:, None] * w["B"][n][g]
        y = torch.einsum("es,es->e", pool[slot], w["C"][n][g])
        y = y if w["D"] is None else y + w["D"] * w["u"][n]
        ys.append(y if w["z"] is None else y * w["z"][n] * torch.sigmoid(w["z"][n]))
    return torch.stack(ys), pool


def _exact_norm(w, s):
    r = w["x"] if w["residual"] is None else w["x"] + w["residual"]
    if w["residual"] is not None:                          # the sum is rounded to the residual's type: the definition's norm is of what is returned
        r = r + ((s["x"].detach().float() + s["residual"].detach().float()).to(s["residual"].dtype).double() - r).detach()
    y = r / torch.sqrt((r ** 2).mean(-1, keepdim=True) + _EPS) * w["w"]
    more = [] if w["residual"] is None else [r]
    if w["case"]["eight"]:
        step = torch.linalg.vector_norm(y, math.inf, dim=-1) / 448
        return [y / step[:, None], step, *more]
    return [y, *more]
