"""Where the scan's, the convolution's and the norm's operators can go wrong beyond ordinary calls: quotients on the border of two 8-bit numbers, rows and launches at their limits, offsets that
do not ascend, values that are not finite beside lanes and channels that are not there."""
import pytest
import torch

import vision_rwkv_amd as vr
from vision_rwkv_amd import _lib
import test_selective_scan_gpu as scans

DEV = "cuda"
pytestmark = pytest.mark.gpu


@pytest.fixture(params=[True, False], ids=["compiled", "python"])
def host(request, monkeypatch):
    """The operators through the compiled host module, and through the Python classes alone."""
    if not request.param:
        monkeypatch.setattr(_lib, "host", lambda: _lib._NoHost)


# ---- the norm ------------------------------------------------------------------------------------------------------------

def _borders(kind, C, unit):
    """Rows of results that are whole, half and quarter steps of the 8-bit type times `unit`, rounded to fp32: next to the border of two numbers, or on it."""
    if kind == torch.int8:
        t = (torch.arange(C) % 509 - 254).float() / 2
        t[0] = 127
    else:
        t = (16 + (torch.arange(C) % 64).float() / 4) * 2.0 ** ((torch.arange(C) // 64 % 12) - 8)
        t[0] = 448
    return t * unit


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("C", [64, 768, 1024, 2048, 4096, 8192, 70, 1021])
def test_eight_bits_are_the_quotient_by_the_scale(C, kind):
    """Rows of one and minus one have a root of exactly one and results that are the weights, so that scale and quotient can be said to the bit: both rounded once to fp32, the quotient then to 8 bits."""
    top = 127 if kind == torch.int8 else 448
    x = torch.where(torch.arange(3 * C).view(3, C) % 3 == 1, -1.0, 1.0)
    for unit in (1.1, 0.013, 777.7, 1.0 + 2.0 ** -23, 1.9999998, 3e33, 2e-33):
        w = _borders(kind, C, unit)
        q, scale = vr.rms_norm(x.to(DEV), w.to(DEV), eps=0.0, quantize=kind)
        want_scale = w.abs().max() / torch.tensor(float(top))
        ratio = (x * w / want_scale).clamp(-top, top)
        want = ratio.round().to(kind) if kind == torch.int8 else ratio.to(kind)
        assert (scale.cpu() == want_scale).all()
        assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8)), unit


@pytest.mark.parametrize("C", [768, 70])
def test_eight_bits_beside_an_infinity(C):
    """A row with an infinite result has an infinite scale: the others are zeros, the infinite one is NaN (0 in int8)."""
    x, w = torch.ones(2, C, device=DEV), torch.ones(C, device=DEV)
    w[3] = float("inf")
    for kind in (torch.float8_e4m3fn, torch.int8):
        q, scale = vr.rms_norm(x, w, eps=0.0, quantize=kind)
        others = torch.arange(C) != 3
        assert torch.isinf(scale).all() and not q.float().cpu()[:, others].any()
        assert torch.isnan(q[:, 3].float()).all() if kind != torch.int8 else not q[:, 3].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("contiguous", [True, False])
def test_saved_rows_of_another_type_are_refused(host, contiguous, dtype):
    """A hook on saved tensors that hands fp32 rows back where the forward kept 16 bits: refused without a residual; with one (whose sum may be either) the same gradients."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 96, generator=g).to(DEV, dtype)
    x = (x if contiguous else torch.cat([x, x], -1)[:, :96]).detach().requires_grad_()
    w = (1 + 0.3 * torch.randn(96, generator=g)).to(DEV, dtype).requires_grad_()
    res = torch.randn(6, 96, generator=g).to(DEV, dtype).requires_grad_()
    gy = torch.randn(6, 96, generator=g).to(DEV, dtype)
    hooks = torch.autograd.graph.saved_tensors_hooks(lambda t: t.float(), lambda t: t)
    with hooks:
        y = vr.rms_norm(x, w)
    with pytest.raises(RuntimeError, match="saved tensors"):
        torch.autograd.grad(y, [x, w], gy)
    with hooks:
        y, r = vr.rms_norm(x, w, res)
    got = torch.autograd.grad([y, r], [x, w, res], [gy, gy])
    want = torch.autograd.grad(vr.rms_norm(x, w, res), [x, w, res], [gy, gy])
    assert all(a.dtype == dtype and torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("C", [64, 2048, 70])
def test_rows_whose_mean_square_is_subnormal(host, C):
    """eps may be zero: a mean of squares below 2^-126 still has its root.  2e-20 squared is 4e-40, 285 000 steps of 2^-149: each square is off by 2^-19 of itself at most, the root by half of
    that (2^-20), C / 64 + 24 half steps of fp32 beside it."""
    x = torch.where(torch.arange(4 * C).view(4, C) % 3 == 1, -2e-20, 2e-20).to(DEV)
    w = torch.linspace(0.5, 2, C, device=DEV)
    leaves = [x.requires_grad_(), w.requires_grad_()]
    y = vr.rms_norm(*leaves, eps=0.0)
    bound = 2.0 ** -20 + (C / 64 + 24) * 2.0 ** -24
    want = torch.sign(x.detach()).double() * w.detach().double()
    assert ((y.detach().double() - want).abs() <= bound * want.abs()).all()
    dw = torch.autograd.grad(y, w, torch.sign(x.detach()))[0]
    assert ((dw.double() - 4).abs() <= 4 * bound).all()


# ---- the convolution -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("N", [(1 << 24) + 3, (1 << 26) + 5])
def test_more_runs_than_a_launch_has_in_one_dimension(N):
    """Sequences of one token, as many as there are waves: 2^22 workgroups and 2^24, which a launch's first dimension has no room for, and some more."""
    x, state = (torch.arange(N, device=DEV, dtype=torch.int32).remainder_(k).sub_(k // 2).to(torch.bfloat16) for k in (251, 127))
    w = torch.tensor([[0.5, 2.0]], device=DEV)
    leaves = [t.requires_grad_() for t in (x.view(N, 1, 1), w, state.view(N, 1, 1))]
    y, last = vr.causal_conv(leaves[0], leaves[1], state=leaves[2], return_state=True)
    # (products and sums are exact in fp32: what is left is the one rounding)
    assert torch.equal(y.view(N), (2 * x.float() + 0.5 * state.float()).bfloat16()) and torch.equal(last, leaves[0])
    dx, dstate = torch.autograd.grad([y, last], [leaves[0], leaves[2]], [torch.ones_like(y), 3 * torch.ones_like(last)])
    assert (dx == 5).all() and (dstate == 0.5).all()


# ---- the scan ------------------------------------------------------------------------------------------------------------

def _same_kinds(x, gy, glast, segments):
    """All results and gradients of a call have infinities and NaN where the recurrence in 64 bits has them, of the same sign, and the other numbers are its own."""
    N, T, _ = x["u"].shape
    leaves = {n: t.clone().requires_grad_() for n, t in x.items() if t is not None}
    with vr.option("scan_segments", segments):
        y, last = vr.selective_scan(**leaves, softplus=True, return_state=True)
        grads = torch.autograd.grad([y, last], list(leaves.values()), [gy, glast])
    want = scans.reference(x, [(n, 0, T) for n in range(N)], True, gy, glast)
    for name, got in (("y", y), ("last", last), *((scans.NAMES[n], g) for n, g in zip(leaves, grads))):
        v, (ref, scale) = got.detach().cpu().double(), want[name]
        assert torch.equal(torch.isnan(v), torch.isnan(ref)), (name, torch.isnan(v).sum(), torch.isnan(ref).sum())
        assert torch.equal(torch.isinf(v), torch.isinf(ref)) and torch.equal(torch.sign(v)[torch.isinf(v)], torch.sign(ref)[torch.isinf(v)]), name
        fine = torch.isfinite(ref)
        if fine.any():
            scans.compare(got.detach().cpu()[fine], (ref[fine], scale[fine]), name, T, tokens=N * T)


@pytest.mark.parametrize("segments", [1, 6])
@pytest.mark.parametrize("S", [1, 3, 10, 20, 40])
def test_an_infinite_gradient_beside_states_that_are_not_there(S, segments):
    """A lane's states are filled up to four and a channel's to a power of two: what fills them up hands no NaN on.  All terms of a sum over states have one sign here, so that only
    the definition's own infinities meet."""
    x, normal = scans.inputs(2, 100, 20, S, 1, "fp32", state=2)
    for n in ("u", "B", "C", "state", "z"):
        x[n].abs_()
    gy, glast = normal(2, 100, 20), normal(2, 20, S)
    gy[0, 40, 3] = float("inf")
    _same_kinds(x, gy, glast, segments)
    gy[0, 40, 3] = 1
    glast[1, 7] = float("inf")
    _same_kinds(x, gy, glast, segments)


@pytest.mark.parametrize("segments", [1, 6])
@pytest.mark.parametrize("E,S,G", [(20, 16, 1), (70, 16, 1), (40, 8, 2), (20, 32, 1), (20, 5, 1)])
def test_an_infinity_in_the_channel_beside_those_that_are_not_there(E, S, G, segments):
    """A workgroup's lanes behind its last channel read that channel once more: whatever it holds, they add nothing to the sums over channels."""
    x, normal = scans.inputs(2, 100, E, S, G, "fp32", state=2)
    for n in ("u", "B", "C", "state", "z"):
        x[n].abs_()
    x["D"].abs_()
    gy, glast = normal(2, 100, E).abs(), normal(2, E, S).abs()
    inf = float("inf")
    for name, place in (("u", (0, 40, E - 1)), ("state", (1, E - 1)), ("glast", (1, E - 1)), ("delta", (0, 40, E // G - 1)), ("B", (0, 40)), ("C", (1, 50))):
        changed = {n: t.clone() if t is not None else None for n, t in x.items()}
        ends = glast.clone()
        (ends if name == "glast" else changed[name])[place] = inf
        _same_kinds(changed, gy, ends, segments)


# ---- offsets that do not ascend ------------------------------------------------------------------------------------------

class _Guarded:
    """Outputs inside one buffer, with room around each that nothing may write."""

    def __init__(self):
        self.parts = []

    def __call__(self, dtype, *shape):
        n, room = 1, 4096
        for k in shape:
            n *= k
        whole = torch.full((n + 2 * room,), 77.0, dtype=dtype, device=DEV)
        self.parts.append((whole, room, n))
        return whole[room:room + n]

    def untouched(self):
        return all((w[:r] == 77).all() and (w[r + n:] == 77).all() for w, r, n in self.parts)


def _disordered(count, seed):
    """Offsets out of order, outside the rows, and the ones that made the convolution's gradients write in front of the states': (T, offsets)."""
    g = torch.Generator().manual_seed(seed)
    yield 40, [0, 30, 10, 40]
    for k in range(count):
        T, N = int(torch.randint(1, 300, (1,), generator=g)), (1, 2, 5, 20, 150)[k % 5]
        yield T, torch.randint(-9, T + 9, (N + 1,), generator=g).tolist()


@pytest.mark.parametrize("K", [2, 4, 7])
@pytest.mark.parametrize("E", [24, 7])
def test_convolution_of_disordered_offsets_stays_in_its_tensors(K, E):
    L = _lib.lib()
    for T, first in _disordered(40, K):
        N, x = len(first) - 1, torch.randn(T, E, device=DEV)
        gy, w, state, glast = torch.randn(T, E, device=DEV), torch.randn(E, K, device=DEV), torch.randn(N, K - 1, E, device=DEV), torch.randn(N, K - 1, E, device=DEV)
        offsets, new = torch.tensor(first, device=DEV), _Guarded()
        a = _lib.ConvArgs()
        a.N, a.T, a.E, a.K, a.silu, a.offsets64 = N, T, E, K, 1, 1
        a.x_stride = a.gy_stride = (0, E)
        out = dict(y=new(torch.float32, T, E), last=new(torch.float32, N, K - 1, E), dx=new(torch.float32, T, E), dweight=new(torch.float32, E, K), dstate=new(torch.float32, N, K - 1, E))
        for n, t in dict(x=x, weight=w, state=state, offsets=offsets, gy=gy, glast=glast, **out).items():
            setattr(a, n, t.data_ptr())
        assert L.vrwkv_conv_fwd(a, None) == 0
        a.workspace_bytes = L.vrwkv_conv_bwd_workspace_bytes(a)
        workspace = torch.empty(a.workspace_bytes, dtype=torch.uint8, device=DEV)
        a.workspace = workspace.data_ptr()
        assert L.vrwkv_conv_bwd(a, None) == 0
        torch.cuda.synchronize()
        assert new.untouched(), first


@pytest.mark.parametrize("segments", [0, 1, 5])
@pytest.mark.parametrize("E,S", [(24, 16), (7, 5)])
def test_scan_of_disordered_offsets_stays_in_its_tensors(E, S, segments, force):
    force("scan_segments", segments)
    L = _lib.lib()
    for T, first in _disordered(25, S):
        N, normal, new, f = len(first) - 1, lambda *s: torch.randn(*s, device=DEV), _Guarded(), torch.float32
        offsets = torch.tensor(first, device=DEV)
        a = _lib.ScanArgs()
        a.N, a.T, a.E, a.S, a.G, a.softplus, a.offsets64 = N, T, E, S, 1, 1, 1
        a.u_stride = a.delta_stride = a.z_stride = a.gy_stride = (0, E)
        a.B_stride = a.C_stride = (0, S, S)
        inputs = dict(u=normal(T, E), delta=normal(T, E), z=normal(T, E), gy=normal(T, E), B=normal(T, S), C=normal(T, S), A=-normal(E, S).abs(), state=normal(N, E, S), glast=normal(N, E, S), offsets=offsets)
        kept = L.vrwkv_scan_kept_bytes(a) // 4
        out = dict(y=new(f, T, E), last=new(f, N, E, S), kept=new(f, kept), du=new(f, T, E), ddelta=new(f, T, E), dz=new(f, T, E), dB=new(f, T, S), dC=new(f, T, S), dA=new(f, E, S), dstate=new(f, N, E, S))
        for n, t in {**inputs, **out}.items():
            setattr(a, n, t.data_ptr())
        for call, size in ((L.vrwkv_scan_fwd, L.vrwkv_scan_fwd_workspace_bytes), (L.vrwkv_scan_bwd, L.vrwkv_scan_bwd_workspace_bytes)):
            room = new(torch.uint8, max(16, size(a)))
            a.workspace, a.workspace_bytes = room.data_ptr(), size(a)
            assert call(a, None) == 0
        torch.cuda.synchronize()
        assert new.untouched(), first


@pytest.mark.parametrize("segments", [0, 1, 6])
def test_other_lengths_on_each_replay(segments, force):
    """Packed sequences in a graph, forward and back, whose offsets change from replay to replay: what eager calls give, to the bit."""
    force("scan_segments", segments)
    T, E, S, K, N = 420, 72, 16, 4, 5
    x, normal = scans.inputs(1, T, E, S, 1, "bf16", state=N)
    taps, w = normal(N, K - 1, E).bfloat16(), normal(E, K)
    leaves = [t.requires_grad_() for t in (*x.values(), taps, w)]
    offsets = torch.tensor([0, 100, 130, 130, 300, 420], device=DEV)
    grads = normal(1, T, E).bfloat16(), normal(N, E, S), normal(N, K - 1, E).bfloat16()

    def call():
        c, tail = vr.causal_conv(x["u"], w, None, "silu", state=taps, offsets=offsets, return_state=True)
        y, last = vr.selective_scan(**{**x, "u": c}, softplus=True, offsets=offsets, return_state=True)
        return [c.detach(), tail.detach(), y.detach(), last.detach(), *torch.autograd.grad([y, last, tail], leaves, list(grads))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = call()
    for first in ([0, 100, 130, 130, 300, 420], [0, 0, 0, 0, 0, 420], [5, 21, 37, 53, 54, 60], [0, 400, 401, 402, 403, 404], [420] * 6, [1, 2, 3, 4, 5, 6]):
        offsets.copy_(torch.tensor(first))
        graph.replay()
        torch.cuda.synchronize()
        for n, (p, q) in enumerate(zip(recorded, call())):
            assert torch.equal(p, q), (first, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_and_rows_further_apart_than_32_bits(dtype):
    """Pages and batch rows more than 2^31 elements from each other: the same as of tensors next to each other, in place and out, gradients too."""
    g, far, E, S, K, T = torch.Generator().manual_seed(3), (1 << 31) + 40, 24, 16, 4, 9
    normal = lambda *s: torch.randn(*s, generator=g).to(DEV)
    space = torch.empty(2 * far + 4096, dtype=torch.float32, device=DEV)

    def apart(t, offset=0):
        """t (n, ..) with its rows `far` elements apart."""
        v = space.view(torch.uint8)[:(space.numel() // 4 * 4) * t.element_size()].view(t.dtype)
        v = v.as_strided(t.shape, (far, *t[0].contiguous().stride()), offset)
        return v.copy_(t)

    u, delta, z, B, C = normal(2, T, E).to(dtype), normal(2, T, E).to(dtype), normal(2, T, E).to(dtype), normal(2, T, S).to(dtype), normal(2, T, S).to(dtype)
    A, w = -normal(E, S).abs(), normal(E, K).to(dtype)
    near = [u, delta, z, B, C]
    split = [apart(t, 512 * i) for i, t in enumerate(near)]
    results = []
    for u_, delta_, z_, B_, C_ in (near, split):
        leaves = [t.detach().requires_grad_() for t in (u_, delta_, z_, B_, C_)]
        y, last = vr.selective_scan(leaves[0], leaves[1], A, leaves[3], leaves[4], z=leaves[2], softplus=True, return_state=True)
        c, tail = vr.causal_conv(leaves[0], w, None, "silu", return_state=True)
        results.append([y, last, c, tail, *torch.autograd.grad([y, last, c, tail], leaves, [torch.ones_like(v) for v in (y, last, c, tail)])])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    states, taps = normal(3, E, S), normal(3, K - 1, E).to(dtype)
    slots = torch.tensor([2, 0], device=DEV)
    for pool, other, f in ((states, apart(states), lambda p: vr.selective_scan_step(u[:, 0], delta[:, 0], A, B[:, 0], C[:, 0], p, slots, z=z[:, 0], softplus=True)),
                           (taps, apart(taps), lambda p: vr.causal_conv_step(u[:, 0], w, p, slots, activation="silu"))):
        other.copy_(pool)
        assert torch.equal(f(pool), f(other)) and torch.equal(pool, other)
    x = normal(3, 768).to(dtype)
    assert torch.equal(vr.rms_norm(x, torch.ones(768, device=DEV)), vr.rms_norm(apart(x), torch.ones(768, device=DEV)))
