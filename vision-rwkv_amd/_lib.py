"""ctypes binding of libvrwkv_hip.so (the C ABI declared in include/vrwkv_hip.h).

The library is loaded from this directory; it is never compiled at import time and there
is no fallback: a missing library is a hard error.
"""
import ctypes
import importlib.util
import os
import subprocess
import warnings

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libvrwkv_hip.so")

VRWKV_F32, VRWKV_BF16, VRWKV_F16 = 0, 1, 2
STATUS_NAMES = {0: "OK", 1: "INVALID_ARG", 2: "UNSUPPORTED_DTYPE", 3: "UNSUPPORTED_SHAPE",
                4: "LAUNCH_FAILED", 5: "WORKSPACE_TOO_SMALL"}

_lib = None
_host = None


class BlockArgs(ctypes.Structure):
    """vrwkv_block_args of include/vrwkv_hip.h."""
    POINTERS_A = ("x", "out", "workspace")
    POINTERS_B = ("ln1_w", "ln1_b", "ln2_w", "ln2_b", "gamma1", "gamma2", "att_mix", "ffn_mix", "w", "u", "key", "value",
                  "receptance", "output", "att_kn_w", "att_kn_b", "ffn_key", "ffn_receptance", "ffn_value", "ffn_kn_w", "ffn_kn_b",
                  "gate", "maa", "maa_w1", "maa_w2", "decay", "decay_w1", "decay_w2", "gn_w", "gn_b")
    INTS = ("B", "T", "C", "hidden", "heads", "Hp", "Wp", "shift_pixel", "quarter", "post_norm", "dtype")
    FLOATS = ("ln1_eps", "ln2_eps", "att_kn_eps", "ffn_kn_eps", "gn_eps")
    _fields_ = ([(n, ctypes.c_void_p) for n in POINTERS_A] + [("workspace_bytes", ctypes.c_size_t)]
                + [(n, ctypes.c_void_p) for n in POINTERS_B] + [(n, ctypes.c_int) for n in INTS] + [(n, ctypes.c_float) for n in FLOATS])


class Linear(ctypes.Structure):
    """vrwkv_linear of include/vrwkv_hip.h."""
    POINTERS = ("a", "w", "out", "gate", "vec", "res", "raw")
    _fields_ = [(n, ctypes.c_void_p) for n in POINTERS] + [(n, ctypes.c_int) for n in ("N", "K", "lda", "epi")]


class Block6Params(ctypes.Structure):
    """vrwkv_block6_params of include/vrwkv_hip.h."""
    POINTERS = ("maa_w1", "maa_w2", "decay_w1", "decay_w2", "maa_x", "maa_w", "maa_k", "maa_v", "maa_r", "maa_g", "ffn_mix_k", "ffn_mix_r",
                "u", "att_kn_w", "att_kn_b")
    _fields_ = [(n, ctypes.c_void_p) for n in POINTERS] + [("fp32_vectors", ctypes.c_int)]


class DecayArgs(ctypes.Structure):
    """vrwkv_decay_args of include/vrwkv_hip.h."""
    STRIDES = ("q_stride", "k_stride", "v_stride", "g_stride", "gy_stride")
    POINTERS = ("q", "k", "v", "g", "offsets", "state", "y", "last", "gy", "glast", "dq", "dk", "dv", "dg", "dstate")
    INTS = ("N", "T", "H", "Hq", "Hk", "Hv", "Dk", "Dv", "dtype", "g_dtype", "g_per_head", "offsets64")
    _fields_ = ([(n, ctypes.c_void_p) for n in POINTERS] + [(n, ctypes.c_longlong * 3) for n in STRIDES] + [(n, ctypes.c_int) for n in INTS]
                + [("scale", ctypes.c_float), ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)])


class DecayStepArgs(ctypes.Structure):
    """vrwkv_decay_step_args of include/vrwkv_hip.h."""
    POINTERS = ("q", "k", "v", "g", "slots", "pool", "y")
    INTS = ("N", "P", "H", "Hq", "Hk", "Hv", "Dk", "Dv", "dtype", "g_dtype", "slots64")
    _fields_ = ([(n, ctypes.c_void_p) for n in POINTERS] + [(n, ctypes.c_longlong * 2) for n in ("q_stride", "k_stride", "v_stride", "g_stride")]
                + [("page_stride", ctypes.c_longlong)] + [(n, ctypes.c_int) for n in INTS] + [("scale", ctypes.c_float)])


def _fields(pointers=(), longs=(), ints=(), tail=()):
    """Fields of an argument structure: pointers, [(long longs, how many)], ints, and what stands behind them."""
    c = ctypes
    return ([(n, c.c_void_p) for n in pointers] + [(n, c.c_longlong * k if k > 1 else c.c_longlong) for n, k in longs] + [(n, c.c_int) for n in ints] + list(tail))


_WORKSPACE = [("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


class ScanArgs(ctypes.Structure):
    """vrwkv_scan_args of include/vrwkv_hip.h."""
    _fields_ = _fields(("u", "delta", "B", "C", "D", "z", "delta_bias", "offsets", "A", "state", "y", "last", "kept", "gy", "glast", "du", "ddelta", "dz", "dB", "dC", "dA", "dstate", "dD", "dbias"),
                       (("u_stride", 2), ("delta_stride", 2), ("z_stride", 2), ("gy_stride", 2), ("B_stride", 3), ("C_stride", 3)),
                       ("N", "T", "E", "S", "G", "dtype", "D_dtype", "bias_dtype", "softplus", "offsets64"), tail=_WORKSPACE)


class ScanStepArgs(ctypes.Structure):
    """vrwkv_scan_step_args of include/vrwkv_hip.h."""
    _fields_ = _fields(("u", "delta", "B", "C", "D", "z", "delta_bias", "slots", "A", "pool", "y"),
                       (("u_stride", 1), ("delta_stride", 1), ("z_stride", 1), ("B_stride", 2), ("C_stride", 2), ("page_stride", 1)),
                       ("N", "P", "E", "S", "G", "dtype", "D_dtype", "bias_dtype", "softplus", "slots64"))


class ConvArgs(ctypes.Structure):
    """vrwkv_conv_args of include/vrwkv_hip.h."""
    _fields_ = _fields(("x", "weight", "bias", "state", "offsets", "y", "last", "gy", "glast", "dx", "dweight", "dbias", "dstate"), (("x_stride", 2), ("gy_stride", 2)),
                       ("N", "T", "E", "K", "dtype", "param_dtype", "silu", "offsets64"), tail=_WORKSPACE)


class ConvStepArgs(ctypes.Structure):
    """vrwkv_conv_step_args of include/vrwkv_hip.h."""
    _fields_ = _fields(("x", "weight", "bias", "slots", "pool", "y"), (("x_stride", 1), ("page_stride", 1)), ("N", "P", "E", "K", "dtype", "param_dtype", "silu", "slots64"))


class RmsnormArgs(ctypes.Structure):
    """vrwkv_rmsnorm_args of include/vrwkv_hip.h."""
    _fields_ = _fields(("x", "residual", "weight", "y", "sum", "scale", "gy", "gsum", "dx", "dresidual", "dweight"),
                       (("rows", 1), ("x_stride", 1), ("residual_stride", 1), ("gy_stride", 1), ("gsum_stride", 1)), ("C", "dtype", "residual_dtype", "weight_dtype", "out_kind"),
                       tail=[("eps", ctypes.c_float)] + _WORKSPACE)


class VrwkvError(RuntimeError):
    """Non-zero status from the C ABI (mirrors the RuntimeError TORCH_CHECK raises at
    classification/mmcls_custom/models/backbones/cuda_new/bi_wkv.cpp:6-8)."""

    def __init__(self, status, message):
        super().__init__(f"vrwkv status {status} ({STATUS_NAMES.get(status, '?')}): {message}")
        self.status = status


class _NoHost:
    """What host() answers without the compiled module: None and False, with which the classes of ops.py go on by themselves."""
    @staticmethod
    def wkv(*args):
        return None

    wkv6 = block_forward = decay_attention = decay_step = copy_pages = causal_conv = causal_conv_step = selective_scan = selective_scan_step = rms_norm = wkv

    @staticmethod
    def weights_fit(*args):
        return False


def _load_host(path):
    """The module at path, or an ImportError that says why it cannot be this process's."""
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing")
    spec = importlib.util.spec_from_file_location("_host", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    built, here = module.torch_version, torch.__version__.split("+")[0]
    if built != here:                                        # it passes torch's own objects: another build's layout may differ
        raise ImportError(f"{path} was built with torch {built}, this is {here}")
    return module


def host():
    """The compiled module of csrc/host: the operators' host side in C++.  It belongs to the torch that it was built with; where it is missing or
    another's, the operators run through the classes of ops.py, the same kernels at more host time a call, after one warning."""
    global _host
    if _host is None:
        lib()
        try:
            _host = _load_host(os.path.join(_HERE, "_host.so"))
        except ImportError as e:
            warnings.warn(f"{e}: operators are called through Python, which takes longer (make -C vision-rwkv_amd/csrc builds it)", RuntimeWarning)
            _host = _NoHost
    return _host


def build(force=True):
    """Compile libvrwkv_hip.so for gfx950 and _host.so with the Makefile in csrc/ (hipcc cross-compiles
    without a GPU)."""
    cmd = ["make", "-C", os.path.join(_HERE, "csrc"), "-j8"]
    if force:
        cmd.append("-B")
    subprocess.run(cmd, check=True)
    return LIB_PATH


def _declare(lib):
    c = ctypes
    vp, fp, i, sz = c.c_void_p, c.c_void_p, c.c_int, c.c_size_t
    lib.vrwkv_version.argtypes = []
    lib.vrwkv_version.restype = i
    lib.vrwkv_last_error.argtypes = []
    lib.vrwkv_last_error.restype = c.c_char_p
    lib.vrwkv_set_option.argtypes = [c.c_char_p, i]
    lib.vrwkv_set_option.restype = i
    lib.vrwkv_get_option.argtypes = [c.c_char_p, c.POINTER(c.c_int)]
    lib.vrwkv_get_option.restype = i
    lib.vrwkv_biwkv_fwd_workspace_bytes.argtypes = [i, i, i, i]
    lib.vrwkv_biwkv_fwd_workspace_bytes.restype = sz
    lib.vrwkv_biwkv_fwd.argtypes = [fp, fp, vp, vp, vp, i, i, i, i, vp, sz, vp]
    lib.vrwkv_biwkv_fwd.restype = i
    lib.vrwkv_biwkv_fwd_gate.argtypes = [fp, fp, vp, vp, vp, vp, i, i, i, i, vp, sz, vp]
    lib.vrwkv_biwkv_fwd_gate.restype = i
    lib.vrwkv_biwkv_fwd_static_max_workspace_bytes.argtypes = []
    lib.vrwkv_biwkv_fwd_static_max_workspace_bytes.restype = sz
    lib.vrwkv_biwkv_fwd_static.argtypes = [fp, fp, vp, vp, vp, i, i, i, i, vp]
    lib.vrwkv_biwkv_fwd_static.restype = i
    lib.vrwkv_biwkv_bwd_workspace_bytes.argtypes = [i, i, i, i]
    lib.vrwkv_biwkv_bwd_workspace_bytes.restype = sz
    lib.vrwkv_biwkv_bwd.argtypes = [fp, fp, vp, vp, vp, fp, fp, vp, vp, i, i, i, i, vp, sz, vp]
    lib.vrwkv_biwkv_bwd.restype = i
    lib.vrwkv_wkv6_fwd_workspace_bytes.argtypes = [i, i, i, i]
    lib.vrwkv_wkv6_fwd_workspace_bytes.restype = sz
    lib.vrwkv_wkv6_fwd.argtypes = [vp, vp, vp, vp, fp, vp, i, i, i, i, i, i, i, vp, sz, vp]
    lib.vrwkv_wkv6_fwd.restype = i
    lib.vrwkv_wkv6_fwd_whole.argtypes = [vp, vp, vp, vp, fp, vp, i, i, i, i, i, i, i, vp]
    lib.vrwkv_wkv6_fwd_whole.restype = i
    lib.vrwkv_wkv6_fwd_phases_bytes.argtypes = [i, i, i]
    lib.vrwkv_wkv6_fwd_phases_bytes.restype = sz
    lib.vrwkv_wkv6_fwd_phases.argtypes = [vp, vp, vp, vp, vp, vp, i, i, i, i, vp, sz, vp]
    lib.vrwkv_wkv6_fwd_phases.restype = i
    lib.vrwkv_wkv6_bwd_workspace_bytes.argtypes = [i, i, i, i]
    lib.vrwkv_wkv6_bwd_workspace_bytes.restype = sz
    lib.vrwkv_wkv6_bwd.argtypes = [vp, vp, vp, vp, fp, fp, fp, fp, fp, fp, fp, i, i, i, i, i, i, i, vp, sz, vp]
    lib.vrwkv_wkv6_bwd.restype = i
    lib.vrwkv_wkv6_bwd_like_workspace_bytes.argtypes = [i, i, i, i, i, i]
    lib.vrwkv_wkv6_bwd_like_workspace_bytes.restype = sz
    lib.vrwkv_wkv6_bwd_like.argtypes = lib.vrwkv_wkv6_bwd.argtypes
    lib.vrwkv_wkv6_bwd_like.restype = i
    lib.vrwkv_qshift_mix.argtypes = [vp, fp, c.POINTER(c.c_void_p), i, i, i, i, i, i, i, i, i, i, vp]
    lib.vrwkv_qshift_mix.restype = i
    lib.vrwkv_qshift_mix_bwd_workspace_bytes.argtypes = [i, i, i, i]
    lib.vrwkv_qshift_mix_bwd_workspace_bytes.restype = sz
    lib.vrwkv_qshift_mix_bwd.argtypes = [vp, fp, c.POINTER(c.c_void_p), i, vp, fp, i, i, i, i, i, i, i, i, i, vp, sz, vp]
    lib.vrwkv_qshift_mix_bwd.restype = i
    lib.vrwkv_maa_lora_mix.argtypes = [vp, vp, vp, vp, fp, c.POINTER(c.c_void_p), c.c_longlong, i, i, vp]
    lib.vrwkv_maa_lora_mix.restype = i
    lib.vrwkv_maa_lora_mix_bwd_workspace_bytes.argtypes = [c.c_longlong, i]
    lib.vrwkv_maa_lora_mix_bwd_workspace_bytes.restype = sz
    lib.vrwkv_maa_lora_mix_bwd.argtypes = [vp, vp, vp, vp, fp, c.POINTER(c.c_void_p), vp, vp, vp, fp, c.c_longlong, i, i, vp, sz, vp]
    lib.vrwkv_maa_lora_mix_bwd.restype = i
    lib.vrwkv_column_sums_workspace_bytes.argtypes = [c.c_longlong, i]
    lib.vrwkv_column_sums_workspace_bytes.restype = sz
    lib.vrwkv_column_sums.argtypes = [vp, vp, c.c_longlong, i, i, vp, sz, vp]
    lib.vrwkv_column_sums.restype = i
    lib.vrwkv_qshift_mix_bwd_add.argtypes = [vp, fp, c.POINTER(c.c_void_p), i, c.POINTER(c.c_void_p), i, vp, vp, i, i, i, i, i, i, i, i, i, i, vp, sz, vp]
    lib.vrwkv_qshift_mix_bwd_add.restype = i
    lib.vrwkv_rowfuse.argtypes = [vp, vp, vp, vp, vp, vp, c.c_longlong, i, i, i, c.c_float, i, vp]
    lib.vrwkv_rowfuse.restype = i
    lib.vrwkv_rowfuse_bwd_workspace_bytes.argtypes = [c.c_longlong, i]
    lib.vrwkv_rowfuse_bwd_workspace_bytes.restype = sz
    lib.vrwkv_rowfuse_bwd.argtypes = [vp, vp, vp, vp, vp, vp, vp, vp, fp, c.c_longlong, i, i, i, c.c_float, i, vp, sz, vp]
    lib.vrwkv_rowfuse_bwd.restype = i
    lib.vrwkv_maa_mix.argtypes = [vp, vp, vp, fp, c.POINTER(c.c_void_p), c.c_longlong, i, i, vp]
    lib.vrwkv_maa_mix.restype = i
    lib.vrwkv_groupnorm_gate.argtypes = [vp, vp, vp, vp, vp, c.c_longlong, i, i, c.c_float, i, i, vp]
    lib.vrwkv_groupnorm_gate.restype = i
    lib.vrwkv_maa_mix_bwd_workspace_bytes.argtypes = [c.c_longlong, i]
    lib.vrwkv_maa_mix_bwd_workspace_bytes.restype = sz
    lib.vrwkv_maa_mix_bwd.argtypes = [vp, vp, vp, fp, c.POINTER(c.c_void_p), vp, vp, vp, fp, c.c_longlong, i, i, vp, sz, vp]
    lib.vrwkv_maa_mix_bwd.restype = i
    lib.vrwkv_groupnorm_gate_bwd_workspace_bytes.argtypes = [c.c_longlong, i]
    lib.vrwkv_groupnorm_gate_bwd_workspace_bytes.restype = sz
    lib.vrwkv_groupnorm_gate_bwd.argtypes = [vp, vp, vp, vp, vp, vp, vp, fp, c.c_longlong, i, i, c.c_float, i, i, vp, sz, vp]
    lib.vrwkv_groupnorm_gate_bwd.restype = i
    lib.vrwkv_pos_resize.argtypes = [vp, vp, i, i, i, i, i, i, i, vp]
    lib.vrwkv_pos_resize.restype = i
    lib.vrwkv_block_fwd_workspace_bytes.argtypes = [i, i, i, i, i, i]
    lib.vrwkv_block_fwd_workspace_bytes.restype = sz
    lib.vrwkv_block_fwd.argtypes = [c.POINTER(BlockArgs), vp]
    lib.vrwkv_block_fwd.restype = i
    lib.vrwkv_block6_fwd.argtypes = [c.POINTER(BlockArgs), c.POINTER(Block6Params), vp]
    lib.vrwkv_block6_fwd.restype = i
    lib.vrwkv_linear_group.argtypes = [c.POINTER(Linear), i, i, i, vp]
    lib.vrwkv_linear_group.restype = i
    lib.vrwkv_transpose_group.argtypes = [c.POINTER(vp), c.POINTER(vp), c.POINTER(i), c.POINTER(i), i, vp]
    lib.vrwkv_transpose_group.restype = i
    ll = c.c_longlong
    lib.vrwkv_wgrad_workspace_bytes.argtypes = [i, i, i, i]
    lib.vrwkv_wgrad_workspace_bytes.restype = sz
    lib.vrwkv_wgrad.argtypes = [vp, vp, vp, i, i, i, i, i, i, ll, ll, i, vp, sz, vp]
    lib.vrwkv_wgrad.restype = i
    lib.vrwkv_biwkv_fwd_as.argtypes = [vp, vp, i, c.c_float, vp, vp, vp, i, i, i, i, vp, sz, vp]
    lib.vrwkv_biwkv_fwd_as.restype = i
    lib.vrwkv_biwkv_bwd_as.argtypes = [vp, vp, i, c.c_float, vp, vp, vp, vp, vp, vp, vp, i, i, i, i, vp, sz, vp]
    lib.vrwkv_biwkv_bwd_as.restype = i
    pi, pv = c.POINTER(i), c.POINTER(vp)
    lib.vrwkv_wgrad_group_workspace_bytes.argtypes = [pi, pi, i, i]
    lib.vrwkv_wgrad_group_workspace_bytes.restype = sz
    lib.vrwkv_wgrad_group.argtypes = [pv, pv, pv, pi, pi, pi, pi, i, i, i, vp, sz, vp]
    lib.vrwkv_wgrad_group.restype = i
    for name in ("vrwkv_decay_fwd", "vrwkv_decay_bwd"):
        getattr(lib, name).argtypes, getattr(lib, name).restype = [c.POINTER(DecayArgs), vp], i
        size = getattr(lib, name + "_workspace_bytes")
        size.argtypes, size.restype = [c.POINTER(DecayArgs)], sz
    lib.vrwkv_decay_step.argtypes = [c.POINTER(DecayStepArgs), vp]
    lib.vrwkv_decay_step.restype = i
    lib.vrwkv_copy_pages_workspace_bytes.argtypes = [i]
    lib.vrwkv_copy_pages_workspace_bytes.restype = sz
    lib.vrwkv_copy_pages.argtypes = [vp, ll, i, vp, ll, i, ll, vp, i, vp, i, i, vp, sz, vp]
    lib.vrwkv_copy_pages.restype = i
    for name, args, size in (("scan_fwd", ScanArgs, True), ("scan_bwd", ScanArgs, True), ("scan_step", ScanStepArgs, False), ("conv_fwd", ConvArgs, False), ("conv_bwd", ConvArgs, True),
                             ("conv_step", ConvStepArgs, False), ("rmsnorm", RmsnormArgs, False), ("rmsnorm_bwd", RmsnormArgs, True)):
        call = getattr(lib, f"vrwkv_{name}")
        call.argtypes, call.restype = [c.POINTER(args), vp], i
        if size:
            call = getattr(lib, f"vrwkv_{name}_workspace_bytes")
            call.argtypes, call.restype = [c.POINTER(args)], sz
    lib.vrwkv_scan_kept_bytes.argtypes, lib.vrwkv_scan_kept_bytes.restype = [c.POINTER(ScanArgs)], sz
    for name in ("rowfuse_bwd", "qshift_mix_bwd", "groupnorm_gate_bwd", "biwkv_bwd"):
        like = getattr(lib, f"vrwkv_{name}_like")
        like.argtypes, like.restype = getattr(lib, f"vrwkv_{name}").argtypes, i
    return lib


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(
                f"{LIB_PATH} is missing: build it first (python -c 'import __graft_entry__ as g; g.build()' "
                "or make -C vision-rwkv_amd/csrc); there is no non-HIP fallback")
        _lib = _declare(ctypes.CDLL(LIB_PATH))
    return _lib


def get_option(name):
    """Value of a tuning / testing switch of the library (include/vrwkv_hip.h lists the names)."""
    out = ctypes.c_int(0)
    check(lib().vrwkv_get_option(name.encode(), ctypes.byref(out)))
    return out.value


def set_option(name, value):
    check(lib().vrwkv_set_option(name.encode(), int(value)))


class option:
    """with option("wkv6_fwd_scalar", 1): ...  -- sets a switch for the block and restores it afterwards."""

    def __init__(self, name, value):
        self.name, self.value = name, value

    def __enter__(self):
        self.old = get_option(self.name)
        set_option(self.name, self.value)
        return self

    def __exit__(self, *exc):
        set_option(self.name, self.old)
        return False


def check(status):
    if status != 0:
        raise VrwkvError(status, lib().vrwkv_last_error().decode("utf-8", "replace"))
