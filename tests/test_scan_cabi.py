"""Host-side checks of the scan's, the convolution's and the norm's entry points, without a GPU: bad arguments are refused with a status and a message before anything is launched, and the
ctypes structures are the header's."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import vision_rwkv_amd as vr
from vision_rwkv_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, INVALID, DTYPE, SHAPE, WORKSPACE = 0, 1, 2, 3, 5


def scan_args(**change):
    a = _lib.ScanArgs()
    for n in ("u", "delta", "B", "C", "A", "y", "gy", "kept", "du", "ddelta", "dA", "dB", "dC"):
        setattr(a, n, 64)
    a.N, a.T, a.E, a.S, a.G = 2, 300, 96, 16, 2
    a.u_stride = a.delta_stride = a.gy_stride = (300 * 96, 96)
    a.B_stride = a.C_stride = (300 * 32, 32, 16)
    a.workspace, a.workspace_bytes = 64, 1 << 40
    for n, v in change.items():
        setattr(a, n, v)
    return a


BAD_SCANS = [(dict(u=None), INVALID), (dict(A=None), INVALID), (dict(N=0), INVALID), (dict(T=-1), INVALID), (dict(E=0), INVALID), (dict(G=0), INVALID), (dict(dtype=3), DTYPE), (dict(D_dtype=-1), DTYPE),
             (dict(bias_dtype=5), DTYPE), (dict(S=0), SHAPE), (dict(S=65), SHAPE), (dict(G=5), SHAPE), (dict(u_stride=(0, 1 << 22)), SHAPE), (dict(C_stride=(0, -1, 0)), SHAPE), (dict(N=70000), SHAPE),
             (dict(T=1 << 30, N=1), SHAPE), (dict(u=66), INVALID), (dict(state=65), INVALID), (dict(kept=72), INVALID), (dict(offsets=68, offsets64=1), INVALID), (dict(delta_bias=65, bias_dtype=1), INVALID)]


@pytest.mark.parametrize("change,status", BAD_SCANS)
def test_bad_scans(change, status):
    L = _lib.lib()
    for f in (L.vrwkv_scan_fwd, L.vrwkv_scan_bwd):
        assert f(scan_args(**change), None) == status, L.vrwkv_last_error()
        assert L.vrwkv_last_error().startswith(b"vrwkv_scan_")


def test_scan_sizes():
    L = _lib.lib()
    for f in (L.vrwkv_scan_fwd, L.vrwkv_scan_bwd, L.vrwkv_scan_step):
        assert f(None, None) == INVALID
    a = scan_args()
    # the states in front of every sixteenth token, whatever the cuts
    assert L.vrwkv_scan_kept_bytes(a) == 2 * 19 * 96 * 16 * 4
    assert L.vrwkv_scan_kept_bytes(scan_args(S=5)) == 2 * 19 * 96 * 8 * 4
    assert L.vrwkv_scan_fwd_workspace_bytes(a) == 0        # few tokens of few channels: one launch
    with vr.option("scan_segments", 3):
        need = L.vrwkv_scan_fwd_workspace_bytes(a)
        assert need > 0                                    # two sequences are cut
        assert L.vrwkv_scan_fwd(scan_args(workspace_bytes=need - 1), None) == WORKSPACE and L.vrwkv_scan_fwd(scan_args(workspace=None), None) == WORKSPACE
    assert L.vrwkv_scan_fwd_workspace_bytes(scan_args(E=9600)) > 0
    need = L.vrwkv_scan_bwd_workspace_bytes(a)
    assert L.vrwkv_scan_bwd(scan_args(workspace_bytes=need - 1), None) == WORKSPACE
    for gone in ("gy", "kept", "du", "ddelta", "dA", "dB", "dC"):
        assert L.vrwkv_scan_bwd(scan_args(**{gone: None}), None) == INVALID
    assert L.vrwkv_scan_bwd(scan_args(z=64, z_stride=(300 * 96, 96)), None) == INVALID   # z without dz
    assert L.vrwkv_scan_fwd_workspace_bytes(scan_args(N=4096)) == 0
    for nothing in (dict(N=0), dict(T=0), dict(S=99), dict(G=0)):
        b = scan_args(**nothing)
        assert L.vrwkv_scan_kept_bytes(b) == L.vrwkv_scan_fwd_workspace_bytes(b) == L.vrwkv_scan_bwd_workspace_bytes(b) == 0


def test_bad_scan_steps():
    L = _lib.lib()

    def args(**change):
        a = _lib.ScanStepArgs()
        for n in ("u", "delta", "B", "C", "A", "pool", "y"):
            setattr(a, n, 64)
        a.N, a.P, a.E, a.S, a.G, a.page_stride = 3, 4, 96, 16, 1, 96 * 16
        for n, v in change.items():
            setattr(a, n, v)
        return a

    for change, status in ((dict(pool=None), INVALID), (dict(N=0), INVALID), (dict(P=0), INVALID), (dict(dtype=9), DTYPE), (dict(S=65), SHAPE), (dict(G=7), SHAPE), (dict(N=5), INVALID),
                           (dict(page_stride=96 * 16 - 1), INVALID), (dict(u=66), INVALID), (dict(slots=68, slots64=1), INVALID), (dict(D=65, D_dtype=1), INVALID)):
        assert L.vrwkv_scan_step(args(**change), None) == status, change


def conv_args(**change):
    a = _lib.ConvArgs()
    for n in ("x", "weight", "y", "gy", "dx", "dweight"):
        setattr(a, n, 64)
    a.N, a.T, a.E, a.K = 2, 300, 96, 4
    a.x_stride = a.gy_stride = (300 * 96, 96)
    a.workspace, a.workspace_bytes = 64, 1 << 40
    for n, v in change.items():
        setattr(a, n, v)
    return a


def test_bad_convolutions():
    L = _lib.lib()
    for change, status in ((dict(x=None), INVALID), (dict(weight=None), INVALID), (dict(N=0), INVALID), (dict(T=0), INVALID), (dict(E=-1), INVALID), (dict(K=1), SHAPE), (dict(K=9), SHAPE), (dict(dtype=4), DTYPE),
                           (dict(param_dtype=-1), DTYPE), (dict(x_stride=(0, 1 << 22)), SHAPE), (dict(T=1 << 30), SHAPE), (dict(x=66), INVALID), (dict(state=67), INVALID), (dict(bias=66), INVALID), (dict(offsets=66), INVALID)):
        for f in (L.vrwkv_conv_fwd, L.vrwkv_conv_bwd):
            assert f(conv_args(**change), None) == status, (change, L.vrwkv_last_error())
    for gone in ("gy", "dx", "dweight"):
        assert L.vrwkv_conv_bwd(conv_args(**{gone: None}), None) == INVALID
    need = L.vrwkv_conv_bwd_workspace_bytes(conv_args())
    assert need > 0 and need % (5 * 96 * 4) == 0           # one row of sums a part
    assert L.vrwkv_conv_bwd(conv_args(workspace_bytes=need - 1), None) == WORKSPACE
    assert L.vrwkv_conv_bwd_workspace_bytes(conv_args(K=12)) == 0

    def step(**change):
        a = _lib.ConvStepArgs()
        for n in ("x", "weight", "pool", "y"):
            setattr(a, n, 64)
        a.N, a.P, a.E, a.K, a.page_stride = 3, 4, 96, 4, 3 * 96
        for n, v in change.items():
            setattr(a, n, v)
        return L.vrwkv_conv_step(a, None)

    assert [step(pool=None), step(N=0), step(K=1), step(dtype=3), step(N=5), step(page_stride=287), step(x=65), step(slots=66)] == [INVALID, INVALID, SHAPE, DTYPE, INVALID, INVALID, INVALID, INVALID]


def test_more_channels_than_a_launch_takes():
    L = _lib.lib()
    assert L.vrwkv_scan_fwd(scan_args(E=(1 << 22) + 2), None) == SHAPE and L.vrwkv_scan_bwd(scan_args(G=(1 << 16) + 1, E=(1 << 16) + 1), None) == SHAPE
    for f in (L.vrwkv_conv_fwd, L.vrwkv_conv_bwd):
        assert f(conv_args(E=(1 << 22) - 63), None) == SHAPE
    a = _lib.ScanStepArgs()
    for n in ("u", "delta", "A", "B", "C", "pool", "y"):
        setattr(a, n, 64)
    a.N, a.P, a.E, a.S, a.G, a.page_stride = 1, 1, (1 << 22) + 1, 1, 1, 1 << 23
    assert L.vrwkv_scan_step(a, None) == SHAPE
    a.N, a.E = 1 << 30, 1
    assert L.vrwkv_scan_step(a, None) == SHAPE
    b = _lib.ConvStepArgs()
    for n in ("x", "weight", "pool", "y"):
        setattr(b, n, 64)
    b.N, b.P, b.E, b.K, b.page_stride = 1, 1, (1 << 22) + 1, 2, 1 << 23
    assert L.vrwkv_conv_step(b, None) == SHAPE
    b.N, b.E = 1 << 30, 1
    assert L.vrwkv_conv_step(b, None) == SHAPE


def test_bad_norms():
    L = _lib.lib()

    def call(backward=False, **change):
        a = _lib.RmsnormArgs()
        for n in ("x", "weight", "y", "sum", "scale", "gy", "dx", "workspace"):
            setattr(a, n, 64)
        a.rows, a.C, a.x_stride, a.gy_stride, a.workspace_bytes = 10, 64, 64, 64, 1 << 30
        for n, v in change.items():
            setattr(a, n, v)
        return (L.vrwkv_rmsnorm_bwd if backward else L.vrwkv_rmsnorm)(a, None)

    assert [call(x=None), call(y=None), call(weight=None), call(out_kind=1, scale=None), call(rows=0), call(C=0), call(rows=1 << 31), call(out_kind=3), call(dtype=3), call(dtype=1, residual_dtype=2),
            call(weight_dtype=7), call(x=66), call(residual=66), call(scale=66)] == [INVALID] * 6 + [SHAPE, INVALID] + [DTYPE] * 3 + [INVALID] * 3
    assert [call(True, sum=None), call(True, gy=None), call(True, dx=None), call(True, workspace_bytes=16), call(True, workspace=8)] == [INVALID, INVALID, INVALID, WORKSPACE, INVALID]


def test_structures_are_the_headers():
    cc = shutil.which("gcc")
    if not cc:
        pytest.skip("no C compiler")
    names = {"vrwkv_scan_args": _lib.ScanArgs, "vrwkv_scan_step_args": _lib.ScanStepArgs, "vrwkv_conv_args": _lib.ConvArgs, "vrwkv_conv_step_args": _lib.ConvStepArgs, "vrwkv_rmsnorm_args": _lib.RmsnormArgs}
    lines = []
    for n, s in names.items():
        lines.append(f'printf("%zu\\n", sizeof({n}));')
        lines += [f'printf("%zu\\n", offsetof({n}, {f[0]}));' for f in s._fields_]
    source = f'#include <stdio.h>\n#include <stddef.h>\n#include "{ROOT}/include/vrwkv_hip.h"\nint main(void) {{ {" ".join(lines)} return 0; }}\n'
    import tempfile
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "a.c"), "w") as f:
            f.write(source)
        subprocess.run([cc, os.path.join(d, "a.c"), "-o", os.path.join(d, "a")], check=True)
        got = [int(v) for v in subprocess.run([os.path.join(d, "a")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for s in names.values():
        want.append(ctypes.sizeof(s))
        want += [getattr(s, f[0]).offset for f in s._fields_]
    assert got == want


def test_options():
    with vr.option("scan_segments", 64):
        assert vr.get_option("scan_segments") == 64
    for bad in (-1, 65):
        with pytest.raises(vr.VrwkvError):
            vr.set_option("scan_segments", bad)


def test_tensors_on_the_host_are_refused():
    x, A, B, w = torch.zeros(1, 4, 8), torch.zeros(8, 2), torch.zeros(1, 4, 2), torch.zeros(8, 4)
    for f in (lambda: vr.selective_scan(x, x, A, B, B), lambda: vr.selective_scan_step(x[0], x[0], A, B[0], B[0], torch.zeros(4, 8, 2)), lambda: vr.causal_conv(x, w), lambda: vr.causal_conv_step(x[0], w, torch.zeros(4, 3, 8)),
              lambda: vr.rms_norm(x, torch.zeros(8)), lambda: vr.rms_norm([1.0], torch.zeros(1))):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            f()
