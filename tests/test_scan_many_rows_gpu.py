"""Gradients of the scan, the convolution and the norm where a workgroup takes several rows of a batch one after the other, and the convolution's runs of more tokens than are asked for at once: sizes
go by the device's compute units, as the kernels' plans do.  References in 64 bits, over the whole batch at once; bounds as in the operators' own tests."""
import pytest
import torch

import test_causal_conv_gpu as convs
import test_rms_norm_gpu as norms
import test_selective_scan_gpu as scans
import vision_rwkv_amd as vr

DEV = "cuda"
pytestmark = pytest.mark.gpu


def units():
    return torch.cuda.get_device_properties(0).multi_processor_count


@pytest.mark.parametrize("dtype,E,S,G,T,segments", [("fp32", 1600, 16, 1, 6, 0), ("bf16", 1600, 16, 1, 17, 0), ("fp32", 90, 16, 90, 20, 0), ("fp16", 700, 64, 1, 5, 0), ("fp32", 60, 40, 60, 18, 0),
                                                    ("bf16", 120, 5, 120, 7, 0), ("fp32", 100, 16, 100, 40, 2), ("fp32", 64, 29, 32, 35, 3)])
def test_scan_gradients_of_more_rows_than_workgroups(dtype, E, S, G, T, segments, force):
    """Half as many rows again as there are places for (eight workgroups a compute unit): some workgroups take one row, some two, and one case three."""
    force("scan_segments", segments)
    channels = 256 // (2 if S <= 8 else 4 if S <= 16 else 8 if S <= 32 else 16)
    blocks, cuts = G * -(-E // G // channels), max(1, segments)
    places = 8 * units() // (blocks * cuts)
    N = places * 3 // 2 + (places if G == 90 else 0) + 1
    assert 1 <= places < N < 400
    x, normal = scans.inputs(N, T, E, S, G, dtype, state=N)
    scans.run_and_compare(x, normal, [(n, 0, T) for n in range(N)])


def conv_reference(x, w, b, state, index, last_index, gy, glast):
    """convs.reference over all tokens at once, on the device.  index (M, K): the rows of [tokens, states, a row of zeros] under a token's taps, the last number for tokens of no sequence."""
    x, w, b, state, gy, glast = (t.detach().double() for t in (x, w, b, state, gy, glast))
    E, K, M = x.shape[-1], w.shape[1], index.shape[0]
    whole = torch.cat([x.reshape(M, E), state.reshape(-1, E), torch.zeros(1, E, device=DEV).double()])
    there = (index[:, -1] < whole.shape[0] - 1)[:, None].double()
    taps = whole[index]
    pre, size = (taps * w.T).sum(1) + b, (taps * w.T).abs().sum(1) + b.abs()
    s = torch.sigmoid(pre)
    out = {"last": (whole[last_index], whole[last_index].abs())}
    g, ga = gy.reshape(M, E) * s * (1 + pre * (1 - s)) * there, gy.reshape(M, E).abs() * (s * (1 + pre.abs() * (1 - s)) + 0.5 * size) * there
    out["y"] = (pre * s * there, size * there)
    out["db"] = (g.sum(0), ga.sum(0))
    out["dw"] = ((taps * g[:, None]).sum(0).T, (taps.abs() * ga[:, None]).sum(0).T)
    back = []
    for a, gg, gl in ((w, g, glast), (w.abs(), ga, glast.abs())):
        r = torch.zeros_like(whole)
        r.index_add_(0, index.flatten(), (a.T * gg[:, None]).reshape(-1, E))
        r.index_add_(0, last_index.flatten(), gl.reshape(-1, E))
        back.append(r)
    out["dx"], out["dstate"] = (tuple(r[:M] for r in back)), (tuple(r[M:-1] for r in back))
    return out


def run_conv(N, T, E, K, dtype, first=None):
    """A call of N rows of T tokens, or of one row of T with sequences from first[n] to first[n + 1], with all gradients."""
    rows = N if first is None else 1
    x, w, b, state, normal = convs.inputs(rows, T, E, K, dtype, state=N)
    M = rows * T
    if first is None:
        begin, end = torch.arange(N) * T, torch.arange(1, N + 1) * T
        offsets = None
    else:
        begin, end, offsets = torch.tensor(first[:-1]), torch.tensor(first[1:]), torch.tensor(first, device=DEV)
    t = torch.arange(M)
    n = torch.searchsorted(end, t, right=True)
    inside = (n < N) & (t >= begin[0])
    n = n.clamp(max=N - 1)
    place = lambda t, n: torch.where(t >= begin[n], t, M + n * (K - 1) + t - begin[n] + K - 1)   # where token t of sequence n lies in [tokens, states]
    index = torch.stack([torch.where(inside, place(t - (K - 1) + j, n), M + N * (K - 1)) for j in range(K)], 1).to(DEV)
    last_index = torch.stack([place(end - (K - 1) + j, torch.arange(N)) for j in range(K - 1)], 1).to(DEV)
    leaves = [v.detach().requires_grad_() for v in (x, w, b, state)]
    y, last = vr.causal_conv(leaves[0], leaves[1], leaves[2], "silu", state=leaves[3], offsets=offsets, return_state=True)
    gy, gl = normal(*y.shape).to(y.dtype), normal(*last.shape).to(y.dtype)
    grads = torch.autograd.grad([y, last], leaves, [gy, gl])
    want = conv_reference(x, w, b, state, index, last_index, gy, gl)
    assert torch.equal(last.double(), want["last"][0])
    for name, got in (("y", y), *zip(("dx", "dw", "db", "dstate"), grads)):
        shape = got.shape if name in ("dw", "db") else (-1, E)
        convs.compare(got.reshape(shape), tuple(v.cpu() for v in want[name]), name, K, tokens=M)


@pytest.mark.parametrize("E,K,dtype", [(8, 4, "fp32"), (16, 4, "bf16"), (12, 7, "fp16"), (3, 2, "fp32")])
@pytest.mark.parametrize("tokens", [17, 70])
def test_convolution_in_runs_of_several_batches(tokens, E, K, dtype):
    """Runs of 16 and of 64 tokens, whose rows come eight at a time: from 16 tokens for each of four waves a vector unit on.  Rows end inside a batch of eight."""
    T = (tokens * 16 * units() // 2) // 8 * 8 + 8 + 3
    run_conv(2, T, E, K, dtype)


@pytest.mark.parametrize("E,K,dtype", [(8, 4, "fp32"), (16, 5, "bf16"), (24, 3, "fp16")])
def test_packed_convolution_in_runs_of_several_batches(E, K, dtype):
    """Sequences of none to a hundred tokens, which begin and end anywhere in a run, tokens in front and behind."""
    want, g, first = 70 * 16 * units(), torch.Generator().manual_seed(K), [11]
    while first[-1] < want:
        first.append(first[-1] + int(torch.randint(0, 100, (1,), generator=g)) * int(torch.randint(0, 5, (1,), generator=g) > 0))
    run_conv(len(first) - 1, first[-1] + 37, E, K, dtype, first)


@pytest.mark.parametrize("E,K,dtype,waves", [(8, 4, "fp32", 1), (4, 4, "bf16", 1), (4096, 4, "bf16", 16), (2050, 6, "fp16", 17), (5, 8, "fp32", 1)])
def test_convolution_gradients_of_more_rows_than_waves(E, K, dtype, waves):
    """Three waves a vector unit at once, for a row's channels: a wave takes several rows, its sums of the weights' gradients over all of them."""
    run_conv(12 * units() // waves * 5 // 2 + 3, 5, E, K, dtype)


@pytest.mark.parametrize("C,dtype,params,residual", [(1536, "bf16", "same", "fp32"), (1536, "bf16", "fp32", None), (2048, "fp32", "fp32", "same"), (4096, "fp16", "same", "same"), (1100, "fp32", "fp32", None), (1544, "fp16", "fp32", "fp32")])
def test_norm_gradients_of_more_rows_than_workgroups(C, dtype, params, residual):
    """Rows of four waves, three for each of four workgroups a compute unit."""
    norms.run_and_compare(*norms.inputs((12 * units() + 5, C), dtype, params, residual))
