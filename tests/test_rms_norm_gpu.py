"""rms_norm and its gradients on the GPU against the formulas in 64 bits.

Bounds.  With the sum r rounded as the operator says, a result is off by the half step u of its type, and inside by fp32 roundings: the mean of squares adds C terms in a tree of at most
C / 64 + 8 steps, half of which reaches the inverse root, with eight more for the root, the products and the division.  In the gradient the same once more for the mean over g n, relative to the
sum of the terms' absolute values.  dweight adds a term for each row.  In 8 bits a result is half a step (2^-4 of itself for e4m3, at least 2^-10; 1/2 for int8) from y / scale, and
y / scale off by four half steps of fp32 more."""
import pytest
import torch

import vision_rwkv_amd as vr
from vision_rwkv_amd import _lib

DEV = "cuda"
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
EPS = 1e-6
pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=[True, False], ids=["compiled", "python"])
def host(request, monkeypatch):
    """The operators through the compiled host module, and through the Python classes alone."""
    if not request.param:
        monkeypatch.setattr(_lib, "host", lambda: _lib._NoHost)


def inputs(shape, dtype, params="fp32", residual=None, seed=0):
    gen = torch.Generator().manual_seed(seed * 1000 + sum(shape))
    normal = lambda *s: torch.randn(*s, generator=gen).to(DEV)
    x, w = normal(*shape).to(DT[dtype]), (1 + 0.3 * normal(shape[-1])).to(DT[dtype if params == "same" else params])
    return x, w, None if residual is None else (2 * normal(*shape)).to(DT[dtype if residual == "same" else residual]), normal


def rounded_sum(x, residual):
    return x if residual is None else (x.float() + residual.float()).to(residual.dtype)


def steps(C):
    return C / 64 + 24


def near(got, ref, scale, n, name):
    limit = HALF_STEP[got.dtype] * ref.abs() + n * 2.0 ** -24 * scale + (2.0 ** -25 if got.dtype == torch.float16 else 1e-30)
    over = ((got.double() - ref).abs() / limit).max().item()
    assert over <= 1.0, f"{name}: {over:.3g} of the bound"


def run_and_compare(x, w, residual, normal):
    C = x.shape[-1]
    leaves = [t.detach().requires_grad_() for t in (x, w, residual) if t is not None]
    out = vr.rms_norm(*leaves, eps=EPS)
    y, r = out if residual is not None else (out, None)
    assert y.dtype == x.dtype
    if r is not None:
        assert r.dtype == residual.dtype and torch.equal(r, rounded_sum(x, residual))
    gy, gr = normal(*y.shape).to(y.dtype), normal(*y.shape).to(residual.dtype) if r is not None else None
    grads = torch.autograd.grad([y] if r is None else [y, r], leaves, [gy] if r is None else [gy, gr])
    v, W, g = rounded_sum(x, residual).double(), w.double(), gy.double()
    s = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    n = v * s
    near(y, n * W, (n * W).abs(), steps(C), "y")
    gw = g * W
    d = s * (gw - n * (gw * n).mean(-1, keepdim=True))
    size = s * (gw.abs() + 2 * n.abs() * (gw * n).abs().mean(-1, keepdim=True))
    if r is not None:
        d, size = d + gr.double(), size + gr.double().abs()
    near(grads[0], d, size, 2 * steps(C), "dx")
    near(grads[1], (g * n).flatten(0, -2).sum(0), (g * n).abs().flatten(0, -2).sum(0), steps(C) + x.numel() / C, "dweight")
    if r is not None:
        assert grads[2].dtype == residual.dtype
        near(grads[2], d, size, 2 * steps(C), "dresidual")
    with torch.no_grad():
        again = vr.rms_norm(x, w, residual, eps=EPS)
    assert torch.equal(again if r is None else again[0], y)


@pytest.mark.parametrize("dtype,params,residual", [("fp32", "fp32", None), ("fp32", "fp32", "same"), ("bf16", "same", None), ("bf16", "fp32", "same"), ("bf16", "same", "fp32"), ("fp16", "same", "same"), ("fp16", "fp32", "fp32")])
@pytest.mark.parametrize("shape", [(5, 768), (1, 1), (3, 7), (2, 9, 64), (300, 40), (4, 513), (2, 2048), (3, 4096), (5, 8192), (2, 10000), (2, 8190), (4100, 16), (1, 520)])
def test_rows_and_gradients(shape, dtype, params, residual):
    if len(shape) == 1:
        shape = (1, *shape)
    run_and_compare(*inputs(shape, dtype, params, residual))


@pytest.mark.parametrize("kind", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype,residual", [("fp32", None), ("bf16", "same"), ("bf16", "fp32"), ("fp16", None)])
@pytest.mark.parametrize("shape", [(5, 768), (1, 1), (3, 7), (2, 9, 64), (70, 4), (2, 8192), (3, 8190), (33, 100)])
def test_eight_bits(shape, dtype, residual, kind):
    x, w, res, _ = inputs(shape, dtype, residual=residual)
    x[0] = 0
    if res is not None:
        res[0] = 0
    q, scale, *r = vr.rms_norm(x, w, res, eps=EPS, quantize=kind)
    assert q.dtype == kind and q.shape == x.shape and scale.shape == x.shape[:-1] and scale.dtype == torch.float32
    assert not r or torch.equal(r[0], rounded_sum(x, res))
    v = rounded_sum(x, res).double()
    y = v / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS) * w.double()
    top = 448 if kind == torch.float8_e4m3fn else 127
    want = (y.abs().amax(-1) / top).clamp(min=2.0 ** -126)
    near(scale, want, want, steps(x.shape[-1]), "scale")
    ratio, got = y / scale.double()[..., None], q.float().double()
    slack = (steps(x.shape[-1]) + 4) * 2.0 ** -24 * ratio.abs()
    half = (2.0 ** -4 * ratio.abs()).clamp(min=2.0 ** -10) if kind == torch.float8_e4m3fn else torch.full_like(ratio, 0.5)
    assert ((got - ratio).abs() <= half + slack).all()
    # the largest of a row is the top of the type
    assert torch.equal(got.abs().amax(-1) == top, want > 2.0 ** -126)
    assert not got[0].any() and (scale[0] == 2.0 ** -126).all()


@pytest.mark.parametrize("C", [64, 70])
def test_infinities_and_nan(C):
    x, w, _, _ = inputs((6, C), "fp32")
    clean = vr.rms_norm(x, w, eps=EPS)
    x[1, 3], x[2, 5], x[4] = float("nan"), float("inf"), 1e30    # squares beyond fp32: the row's mean is infinite, its results zero
    y = vr.rms_norm(x, w, eps=EPS)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 5]) and not y[2, :5].any() and not y[2, 6:].any() and not y[4].any()
    assert torch.equal(y[[0, 3, 5]], clean[[0, 3, 5]])
    q, scale = vr.rms_norm(x, w, eps=EPS, quantize=torch.float8_e4m3fn)
    assert torch.isnan(scale[1]) and torch.isnan(q[1].float()).all() and torch.isnan(scale[2])
    q, scale = vr.rms_norm(x, w, eps=EPS, quantize=torch.int8)
    assert torch.isnan(scale[1]) and not q[1].any() and torch.isnan(scale[2])
    assert torch.isfinite(scale[[0, 3, 4, 5]]).all()


def test_strides_and_views():
    x, w, res, normal = inputs((4, 9, 64), "bf16", residual="same")
    want = vr.rms_norm(x, w, res, eps=EPS)
    for v in (torch.cat([x, x], -1)[..., 64:], x.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([x, x[..., :3]], -1)[..., :64], x.transpose(1, 2).contiguous().transpose(1, 2)):
        got = vr.rms_norm(v, torch.stack([w, w], 1)[:, 0], torch.stack([res] * 2, -1)[..., 0], eps=EPS)
        assert torch.equal(got[1], want[1]) and (got[0].float() - want[0].float()).abs().max() <= 2.0 ** -7 * want[0].float().abs().max()
    row = x[:1, :1].expand(4, 9, 64)
    assert torch.equal(vr.rms_norm(row, w, eps=EPS), vr.rms_norm(row.contiguous(), w, eps=EPS))
    assert vr.rms_norm(x[0, 0], w, eps=EPS).shape == (64,)
    assert vr.rms_norm(x[:0], w, eps=EPS).shape == (0, 9, 64)
    e = x[:0].clone().requires_grad_()
    wl = w.clone().requires_grad_()
    ge, gw = torch.autograd.grad(vr.rms_norm(e, wl, eps=EPS).sum(), [e, wl])
    assert ge.shape == e.shape and not gw.any()


def test_gradients_of_some():
    """Only the weight's, only the residual's, and only of the sum."""
    x, w, res, normal = inputs((7, 96), "bf16", residual="fp32")
    full = [t.detach().requires_grad_() for t in (x, w, res)]
    gy, gr = normal(7, 96).bfloat16(), normal(7, 96)
    want = torch.autograd.grad(vr.rms_norm(*full, eps=EPS), full, [gy, gr])
    for k in range(3):
        some = [t.detach().requires_grad_(i == k) for i, t in enumerate((x, w, res))]
        assert torch.equal(torch.autograd.grad(vr.rms_norm(*some, eps=EPS), some[k], [gy, gr])[0], want[k])
    y, r = vr.rms_norm(*full, eps=EPS)
    got = torch.autograd.grad(r, full, gr, allow_unused=True)
    assert torch.equal(got[2], gr) and torch.equal(got[0], gr.bfloat16()) and (got[1] is None or not got[1].any())


def test_refusals():
    x, w, res, normal = inputs((4, 64), "bf16", residual="fp32")
    for args, more in (((x.cpu(), w), {}), ((x.double(), w), {}), ((x, w[:9]), {}), ((x, w.half()), {}), ((x, w, res[:2]), {}), ((x, w, res.half()), {}), ((x, w), dict(quantize=torch.uint8)),
                       ((x, w), dict(eps=torch.tensor(1e-6))), ((x.clone().requires_grad_(), w), dict(quantize=torch.int8)), ((x[:, :0], w[:0]), {})):
        with pytest.raises(RuntimeError):
            vr.rms_norm(*args, **more)
    with pytest.raises(RuntimeError, match="forward mode"), torch.autograd.forward_ad.dual_level():
        vr.rms_norm(torch.autograd.forward_ad.make_dual(x, x), w)
    with pytest.raises(RuntimeError):
        torch.jit.trace(lambda t: vr.rms_norm(t, w), (x,))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: vr.rms_norm(t, w))(torch.stack([x, x]))


def test_other_streams_and_graphs():
    x, w, res, normal = inputs((300, 768), "bf16", residual="fp32")
    leaves = [t.detach().requires_grad_() for t in (x, w, res)]
    gy, gr = normal(300, 768).bfloat16(), normal(300, 768)

    def call():
        y, r = vr.rms_norm(*leaves, eps=EPS)
        with torch.no_grad():
            q, scale, _ = vr.rms_norm(*leaves, eps=EPS, quantize=torch.int8)
        return [y.detach(), r.detach(), q, scale, *torch.autograd.grad([y, r], leaves, [gy, gr])]

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
            for t in (*leaves, gy, gr):
                t.copy_(normal(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(recorded, call()):
            assert torch.equal(p, q), k


@pytest.mark.parametrize("rows,C", [((1 << 24) + 5, 4), ((1 << 22) + 3, 3)])
def test_more_rows_than_a_launch_has_in_one_dimension(rows, C):
    x = torch.arange(rows * C, device=DEV, dtype=torch.float32).view(rows, C).remainder_(1021).sub_(500.25)
    w = torch.linspace(0.5, 2, C, device=DEV).requires_grad_()
    leaf = x.requires_grad_()
    y = vr.rms_norm(leaf, w, eps=EPS)
    gy = torch.ones_like(x)
    gx, gw = torch.autograd.grad(y, [leaf, w], gy)
    v, W = x.detach().double(), w.detach().double()
    s = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    n = v * s
    near(y.detach(), n * W, (n * W).abs(), steps(C), "y")
    mean = (W * n).mean(-1, keepdim=True)
    near(gx, s * (W - n * mean), s * (W + n.abs() * (W * n.abs()).mean(-1, keepdim=True)), 2 * steps(C), "dx")
    near(gw, n.sum(0), n.abs().sum(0), 2 * steps(C) + rows / 256 + 512, "dweight")
