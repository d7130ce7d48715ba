"""rms_norm, causal_conv, selective_scan, their steps and copy_states together, as a layer of a model uses them: training, a prompt, tokens behind it, a fork."""
import math

import pytest
import torch
from torch.nn.functional import linear

import vision_rwkv_amd as vr

DEV = "cuda"
pytestmark = pytest.mark.gpu
W, E, S, K, R = 48, 96, 16, 4, 6                           # width of the model, channels inside, states, taps, rank of the step sizes


def weights(seed=0):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    size = torch.exp(math.log(1e-3) + torch.rand(E, generator=gen).to(DEV) * math.log(100))
    return dict(norm=1 + 0.1 * normal(W), inside=normal(2 * E, W) * W ** -0.5, conv=normal(E, K) * 0.5, conv_b=0.1 * normal(E), low=normal(R + 2 * S, E) * E ** -0.5, up=normal(E, R) * R ** -0.5,
                bias=size + torch.log(-torch.expm1(-size)), A=torch.log(torch.arange(1, S + 1, device=DEV).float()).expand(E, S).contiguous(), D=1 + 0.1 * normal(E), out=normal(W, E) * E ** -0.5), normal


def layer(p, x, residual, offsets=None, states=(None, None)):
    """The layer's results, its residual and its states; x, residual (B, T, W)."""
    h, r = vr.rms_norm(x, p["norm"], residual)
    u, z = linear(h, p["inside"]).chunk(2, -1)
    u, tail = vr.causal_conv(u, p["conv"], p["conv_b"], "silu", state=states[0], offsets=offsets, return_state=True)
    size, B, C = linear(u, p["low"]).split([R, S, S], -1)
    y, state = vr.selective_scan(u, linear(size, p["up"]), -torch.exp(p["A"]), B, C, p["D"], z, p["bias"], True, state=states[1], offsets=offsets, return_state=True)
    return linear(y, p["out"]), r, (tail, state)


def layer_step(p, x, residual, pools, slots):
    h, r = vr.rms_norm(x, p["norm"], residual)
    u, z = linear(h, p["inside"]).chunk(2, -1)
    u = vr.causal_conv_step(u, p["conv"], pools[0], slots, p["conv_b"], "silu")
    size, B, C = linear(u, p["low"]).split([R, S, S], -1)
    y = vr.selective_scan_step(u, linear(size, p["up"]), -torch.exp(p["A"]), B, C, pools[1], slots, p["D"], z, p["bias"], True)
    return linear(y, p["out"]), r


def plain(p, x, residual):
    r = x + residual
    h = r / torch.sqrt((r * r).mean(-1, keepdim=True) + 1e-6) * p["norm"]
    u, z = linear(h, p["inside"]).chunk(2, -1)
    padded = torch.nn.functional.pad(u, (0, 0, K - 1, 0))
    u = sum(padded[:, j:j + u.shape[1]] * p["conv"][:, j] for j in range(K)) + p["conv_b"]
    u = u * torch.sigmoid(u)
    size, B, C = linear(u, p["low"]).split([R, S, S], -1)
    dt = torch.nn.functional.softplus(linear(size, p["up"]) + p["bias"])
    state, ys = u.new_zeros(u.shape[0], E, S), []
    for t in range(u.shape[1]):
        state = torch.exp(dt[:, t, :, None] * -torch.exp(p["A"])) * state + (dt[:, t] * u[:, t])[..., None] * B[:, t, None]
        ys.append((state * C[:, t, None]).sum(-1) + p["D"] * u[:, t])
    return linear(torch.stack(ys, 1) * z * torch.sigmoid(z), p["out"]), r


def test_two_layers_train():
    """Results and all gradients of two layers against the same in 64 bits.  Some 300 roundings of 2^-24 on the way to a number, of random sign, and the products' own: 2e-6 of a tensor's norm;
    ten times that through two layers and back."""
    (p, normal), (q, _) = weights(1), weights(2)
    x, res = normal(2, 83, W), normal(2, 83, W)
    gy, gr = normal(2, 83, W), normal(2, 83, W)
    results = []
    for dtype, f in ((torch.float32, lambda *a: layer(*a)[:2]), (torch.float64, plain)):
        leaves = [t.to(dtype).detach().requires_grad_() for t in (x, res, *p.values(), *q.values())]
        P, Q = dict(zip(p, leaves[2:2 + len(p)])), dict(zip(q, leaves[2 + len(p):]))
        out = f(Q, *f(P, leaves[0], leaves[1]))
        results.append([*out, *torch.autograd.grad(out, leaves, [gy.to(dtype), gr.to(dtype)])])
    for n, (a, b) in enumerate(zip(*results)):
        assert (a.double() - b).norm() <= 2e-5 * b.norm(), n


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_prompts_steps_and_forks(dtype):
    """Packed prompts, their states put in pages, pages forked, tokens behind them one at a time: what whole sequences give.  16-bit results differ by a few roundings of 2^-8 each
    (products of other shapes round otherwise): 3e-2 of the norm."""
    p, normal = weights(3)
    p = {n: t if n in ("A", "bias", "D") else t.to(dtype) for n, t in p.items()}
    lengths, more = [5, 40, 1, 19], 7
    x, res = normal(4, 60, W).to(dtype), normal(4, 60, W).to(dtype)
    bound = 2e-5 if dtype == torch.float32 else 3e-2
    first = [0]
    for n in lengths:
        first.append(first[-1] + n)
    with torch.no_grad():
        packed = [torch.cat([t[n, :k] for n, k in enumerate(lengths)])[None] for t in (x, res)]
        y, r, (tail, state) = layer(p, *packed, offsets=torch.tensor(first, device=DEV))
        pools = torch.zeros(9, K - 1, E, dtype=dtype, device=DEV), torch.zeros(9, E, S, device=DEV)
        pages = torch.tensor([3, 0, 7, 1], device=DEV)
        for pool, rows in zip(pools, (tail, state)):
            vr.copy_states(pool, torch.arange(4, device=DEV), pages, source=rows)
            vr.copy_states(pool, pages[1:2], torch.tensor([8], device=DEV))    # the second sequence once more
        slots = torch.cat([pages, torch.tensor([8, -1], device=DEV)])
        who = [0, 1, 2, 3, 1, 0]
        for t in range(more):
            rows = [t_[who, [lengths[n] + t for n in who]] for t_ in (x, res)]
            out, _ = layer_step(p, *rows, pools, slots)
            for i, n in enumerate(who[:5]):
                want = layer(p, x[n:n + 1, :lengths[n] + t + 1], res[n:n + 1, :lengths[n] + t + 1])[0][0, -1]
                assert (out[i].double() - want.double()).norm() <= bound * want.double().norm(), (t, i)
            assert (out[4].double() - out[1].double()).norm() <= bound * out[1].double().norm()
        for n, k in enumerate(lengths):
            want = layer(p, x[n:n + 1, :k], res[n:n + 1, :k])[0][0]
            assert (y[0, first[n]:first[n + 1]].double() - want.double()).norm() <= bound * want.double().norm()


def test_a_step_in_a_graph():
    p, normal = weights(4)
    pools = torch.zeros(6, K - 1, E, device=DEV), torch.zeros(6, E, S, device=DEV)
    mine = [t.clone() for t in pools]
    x, res, slots = normal(3, W), normal(3, W), torch.tensor([4, 0, -1], device=DEV)
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer_step(p, x, res, mine, slots)
        torch.cuda.current_stream().wait_stream(side)
        for t in mine:
            t.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, _ = layer_step(p, x, res, mine, slots)
        for k in range(4):
            x.copy_(normal(3, W))
            slots.copy_(torch.tensor([[4, 0, -1], [1, 4, 0], [-1, 2, 5], [0, 1, 4]][k]))
            graph.replay()
            torch.cuda.synchronize()
            want, _ = layer_step(p, x, res, pools, slots)
            assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(pools, mine)), k


def test_two_calls_at_once():
    """The same operators on two streams, with workspaces of their own."""
    p, normal = weights(5)
    x = [normal(2, 700, W) for _ in range(2)]
    with torch.no_grad(), vr.option("scan_segments", 9):
        want = [layer(p, t, t)[0] for t in x]
        streams = [torch.cuda.Stream() for _ in x]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(5):
            for k, s in enumerate(streams):
                with torch.cuda.stream(s):
                    got[k].append(layer(p, x[k], x[k])[0])
        torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(t, want[k]) for t in got[k])
