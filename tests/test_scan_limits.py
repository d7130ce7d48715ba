"""Sizes at whose end 32-bit counters of the scan's, the convolution's and the norm's kernels run over, refused by the entry points before anything is launched (no GPU needed)."""
import pytest

from test_scan_cabi import INVALID, SHAPE, conv_args, scan_args
from vision_rwkv_amd import _lib


@pytest.mark.parametrize("N", [1 << 30, 0x7fffffff])
def test_more_packed_sequences_than_a_counter_takes(N):
    L = _lib.lib()
    for f in (L.vrwkv_scan_fwd, L.vrwkv_scan_bwd):
        assert f(scan_args(N=N, offsets=64), None) == SHAPE
    for f in (L.vrwkv_conv_fwd, L.vrwkv_conv_bwd):
        assert f(conv_args(N=N, offsets=64), None) == SHAPE
        assert f(conv_args(N=(1 << 30) - 1, offsets=64, x=66), None) == INVALID   # (looked at behind the sizes: these are taken)


def test_wider_rows_than_a_counter_takes():
    L = _lib.lib()

    def call(f, C, **change):
        a = _lib.RmsnormArgs()
        for n in ("x", "weight", "y", "sum", "gy", "dx", "workspace"):
            setattr(a, n, 64)
        a.rows, a.C, a.workspace_bytes = 1, C, 1 << 50
        for n, v in change.items():
            setattr(a, n, v)
        return f(a, None)

    top = (1 << 31) - 256
    for f in (L.vrwkv_rmsnorm, L.vrwkv_rmsnorm_bwd):
        assert call(f, top + 1) == call(f, 0x7fffffff) == SHAPE
        assert call(f, top, weight=66) == INVALID
    top = (1 << 27) - 32                                   # the weight's gradient
    assert call(L.vrwkv_rmsnorm_bwd, top + 1, dweight=64) == SHAPE
    assert call(L.vrwkv_rmsnorm_bwd, top, dweight=64, workspace_bytes=0) == call(L.vrwkv_rmsnorm_bwd, top + 1, workspace_bytes=0) == 5   # (no workspace: looked at last)
