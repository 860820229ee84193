"""ctypes binding of ``libkdn_b200.so`` (C ABI in ``include/kdn_b200.h``).

The shared library is required: importing the operators works without a GPU,
but every call raises ``RuntimeError`` when the library or a CUDA device is
missing.  There is no CPU fallback.
"""
from __future__ import annotations

import ctypes
import glob
import importlib.util
import os
import sysconfig
import threading
import warnings

import torch
from torch.autograd import forward_ad

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("KDN_B200_LIB", os.path.join(_HERE, "lib", "libkdn_b200.so"))

KDN_OK = 0
KDN_ISO = 0
KDN_DIAG = 1
KDN_PREC_BF16 = 0
KDN_PREC_FP32 = 1
# passes of a scan call (KdnScanArgs.mode)
KDN_SCAN_FULL = 0
KDN_SCAN_FWD_RECORDS = 1
KDN_SCAN_FWD_SEQUENTIAL = 2
KDN_SCAN_FWD_STATE_MAP = 3
KDN_SCAN_BWD_STATE = 4

_lock = threading.Lock()
_lib = None


class KdnScanArgs(ctypes.Structure):
    _fields_ = [
        ("variant", ctypes.c_int32),
        ("precision", ctypes.c_int32),
        ("B", ctypes.c_int64),
        ("T", ctypes.c_int64),
        ("H", ctypes.c_int64),
        ("K", ctypes.c_int64),
        ("V", ctypes.c_int64),
        ("scale", ctypes.c_float),
        ("q", ctypes.c_void_p),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("g", ctypes.c_void_p),
        ("beta", ctypes.c_void_p),
        ("kappa", ctypes.c_void_p),
        ("initial_state", ctypes.c_void_p),
        ("o", ctypes.c_void_p),
        ("final_state", ctypes.c_void_p),
        ("saved", ctypes.c_void_p),
        ("dO", ctypes.c_void_p),
        ("d_final_state", ctypes.c_void_p),
        ("dq", ctypes.c_void_p),
        ("dk", ctypes.c_void_p),
        ("dv", ctypes.c_void_p),
        ("dg", ctypes.c_void_p),
        ("dbeta", ctypes.c_void_p),
        ("dkappa", ctypes.c_void_p),
        ("d_initial_state", ctypes.c_void_p),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
        ("mode", ctypes.c_int32),
        ("final_state_map", ctypes.c_void_p),
        ("varlen_table", ctypes.c_void_p),
        ("num_seqs", ctypes.c_int64),
        ("num_chunks", ctypes.c_int64),
    ]


def _struct(name, *groups):
    """A ctypes structure with the header's fields: (type, "names") groups in order."""
    fields = [(field, ctype) for ctype, names in groups for field in names.split()]
    return type(name, (ctypes.Structure,), {"_fields_": fields})


KdnStepArgs = _struct(
    "KdnStepArgs",
    (ctypes.c_int32, "variant act_bf16 swish slots_i64"),
    (ctypes.c_int64, "B H D num_slots"),
    (ctypes.c_void_p, "qkv decay_raw omega_raw r_raw gate"),
    (ctypes.c_int64, "qkv_stride decay_stride omega_stride r_stride gate_stride"),
    (ctypes.c_void_p, "conv_weight A_log dt_bias omega_bias r_bias norm_weight"),
    (ctypes.c_float, "omega_min r_min posterior_scale eps scale"),
    (ctypes.c_void_p, "slots memory covariance window y"),
)
KdnBlockNormArgs = _struct(
    "KdnBlockNormArgs",
    (ctypes.c_int32, "stream_bf16 act_bf16 weights_bf16 swish"),
    (ctypes.c_int64, "rows D"),
    (ctypes.c_float, "alpha eps"),
    (ctypes.c_void_p, "x y gate"),
    (ctypes.c_int64, "x_stride y_stride gate_stride"),
    (ctypes.c_void_p, "weight post_weight scale z h rstd dz dh dx dy dgate dweight dpost dscale workspace"),
    (ctypes.c_size_t, "workspace_bytes"),
)
KdnSampleArgs = _struct(
    "KdnSampleArgs",
    (ctypes.c_int32, "logits_bf16 top_k_i64"),
    (ctypes.c_int64, "rows V"),
    (ctypes.c_void_p, "logits noise"),
    (ctypes.c_int64, "logits_stride noise_stride"),
    (ctypes.c_void_p, "temperature top_k top_p min_p"),
    (ctypes.c_float, "temperature_all"),
    (ctypes.c_int64, "top_k_all"),
    (ctypes.c_float, "top_p_all min_p_all"),
    (ctypes.c_void_p, "token prob"),
)

_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_F = ctypes.c_float
_SZ = ctypes.c_size_t

_SIGNATURES = {
    "kdn_version": ([], ctypes.c_int),
    "kdn_last_error": ([], ctypes.c_char_p),
    "kdn_iso_gain_workspace_bytes": ([_I64, _I64, _I64], _SZ),
    "kdn_iso_gain_fwd": ([_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _F, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gain_bwd": (
        [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _F, _P, _SZ, _P],
        ctypes.c_int,
    ),
    "kdn_iso_gain_fwd_maps": ([_P, _P, _P, _P, _I64, _I64, _I64, _F, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gain_fwd_finish": ([_P] * 8 + [_I64, _I64, _I64, _F, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gain_bwd_maps": ([_P] * 6 + [_I64, _I64, _I64, _F, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gain_bwd_finish": ([_P] * 13 + [_I64, _I64, _I64, _F, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gain_varlen_workspace_bytes": ([_I64, _I64, _I64], _SZ),
    "kdn_iso_gain_fwd_varlen": ([_P] * 8 + [_I64, _I64, _F, _P, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gain_bwd_varlen": ([_P] * 13 + [_I64, _I64, _F, _P, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_iso_gate_workspace_bytes": ([_I64, _I64, _I64, _I64], _SZ),
    "kdn_iso_gate_fwd": (
        [_P, ctypes.c_int, _P, ctypes.c_int, _I64, _I64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
         _I64, _I64, _I64, _I64, _F, _F, _P],
        ctypes.c_int,
    ),
    "kdn_iso_gate_bwd": (
        [_P, ctypes.c_int, _P, ctypes.c_int, _I64, _I64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
         _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _SZ, _P],
        ctypes.c_int,
    ),
    "kdn_diag_gate_workspace_bytes": ([_I64, _I64, _I64, _I64], _SZ),
    "kdn_diag_gate_fwd": ([_P] * 11 + [_I64, _I64, _I64, _I64, _P], ctypes.c_int),
    "kdn_diag_gate_bwd": ([_P] * 17 + [_I64, _I64, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_carry_elems": ([_I64, _I64, _I64, _I64], _I64),
    "kdn_diag_gain_workspace_bytes": ([_I64, _I64, _I64, _I64], _SZ),
    "kdn_diag_gain_fwd": ([_P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_fwd_noalloc": ([_P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P], ctypes.c_int),
    "kdn_diag_gain_fwd_maps": ([_P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_fwd_finish": ([_P] * 9 + [_I64, _I64, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_bwd_maps": ([_P] * 7 + [_I64, _I64, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_bwd_finish": ([_P] * 17 + [_I64, _I64, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_bwd": (
        [_P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _I64, _I64, _P, _SZ, _P],
        ctypes.c_int,
    ),
    "kdn_diag_gain_varlen_carry_elems": ([_I64, _I64, _I64, _I64], _I64),
    "kdn_diag_gain_varlen_workspace_bytes": ([_I64, _I64, _I64, _I64], _SZ),
    "kdn_diag_gain_fwd_varlen": ([_P] * 9 + [_I64, _I64, _I64, _P, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_diag_gain_bwd_varlen": ([_P] * 17 + [_I64, _I64, _I64, _P, _I64, _I64, _P, _SZ, _P], ctypes.c_int),
    "kdn_varlen_table_len": ([_I64, _I64], _I64),
    "kdn_varlen_plan": ([_P, _I64, _P, _I64, ctypes.POINTER(ctypes.c_int64)], ctypes.c_int),
    "kdn_diag_norm_fwd": ([_P, _P, ctypes.c_int, _P, _P, _P, _P, _P, _I64, _I64, _P], ctypes.c_int),
    "kdn_diag_norm_bwd": ([_P, _P, ctypes.c_int, _P, _P, _P, _P, _P, _P, _P, _I64, _I64, _P], ctypes.c_int),
    "kdn_rmsnorm_gated_workspace_bytes": ([_I64, _I64], _SZ),
    "kdn_rmsnorm_gated_fwd": ([_P, ctypes.c_int, _P, ctypes.c_int, _P, _P, _P, _I64, _I64, _F, ctypes.c_int, _P],
                              ctypes.c_int),
    "kdn_rmsnorm_gated_bwd": ([_P, ctypes.c_int, _P, ctypes.c_int, _P, _P, _P, _P, _P, _P, _I64, _I64, ctypes.c_int,
                               _P, _SZ, _P], ctypes.c_int),
    "kdn_short_conv_workspace_bytes": ([_I64, _I64, _I64, _I64], _SZ),
    "kdn_short_conv_fwd": ([_P, ctypes.c_int, _P, ctypes.c_int, _P, _I64, _I64, _I64, _I64, _I64, ctypes.c_int, _P],
                           ctypes.c_int),
    "kdn_short_conv_bwd": ([_P, ctypes.c_int, _P, ctypes.c_int, _P, _I64, _P, _P, _I64, _I64, _I64, _I64,
                            ctypes.c_int, _P, _SZ, _P], ctypes.c_int),
    "kdn_scan_saved_bytes": ([ctypes.POINTER(KdnScanArgs)], _SZ),
    "kdn_scan_workspace_bytes": ([ctypes.POINTER(KdnScanArgs)], _SZ),
    "kdn_scan_fwd": ([ctypes.POINTER(KdnScanArgs), _P], ctypes.c_int),
    "kdn_scan_bwd": ([ctypes.POINTER(KdnScanArgs), _P], ctypes.c_int),
    "kdn_step": ([ctypes.POINTER(KdnStepArgs), _P], ctypes.c_int),
    "kdn_block_norm_workspace_bytes": ([_I64, _I64], _SZ),
    "kdn_block_norm_fwd": ([ctypes.POINTER(KdnBlockNormArgs), _P], ctypes.c_int),
    "kdn_block_norm_bwd": ([ctypes.POINTER(KdnBlockNormArgs), _P], ctypes.c_int),
    "kdn_sample": ([ctypes.POINTER(KdnSampleArgs), _P], ctypes.c_int),
}


def load_library():
    """Load the C-ABI library once; raise a clear error when it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"kdn_b200: native library not found at {LIB_PATH}; build it with "
                    "`python -m kdn_b200.build` (nvcc, sm_100a)"
                )
            lib = ctypes.CDLL(LIB_PATH)
            for name, (argtypes, restype) in _SIGNATURES.items():
                fn = getattr(lib, name)
                fn.argtypes = argtypes
                fn.restype = restype
            _lib = lib
    return _lib


def exported_symbols():
    return tuple(_SIGNATURES)


def check(rc: int, what: str) -> None:
    if rc != KDN_OK:
        msg = load_library().kdn_last_error().decode(errors="replace")
        raise RuntimeError(f"kdn_b200 {what} failed ({rc}): {msg}")


def require_cuda(*tensors: torch.Tensor) -> None:
    if not torch.cuda.is_available():
        raise RuntimeError("kdn_b200 kernels need a CUDA device (B200, sm_100a); there is no CPU fallback")
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise ValueError("kdn_b200 kernels need CUDA tensors")
    load_library()


def ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def stream_of(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


_HOST_ENTRIES = ("kdn_step", "kdn_block_norm_fwd", "kdn_block_norm_bwd", "kdn_block_norm_workspace_bytes", "kdn_sample",
                 "kdn_last_error")
# Named after the torch and the interpreter it is built against: a library of others is never loaded.
HOST_LIB = os.path.join(_HERE, "lib", f"_kdn_torch.{torch.__version__}.{sysconfig.get_config_var('SOABI')}.so")
_host = None


def _load_host():
    if not os.path.exists(HOST_LIB):
        others = glob.glob(os.path.join(glob.escape(os.path.dirname(HOST_LIB)), "_kdn_torch.*.so"))
        if others:
            warnings.warn(f"kdn_b200: the C++ host path is built for another torch or Python ({os.path.basename(others[0])}); "
                          "taking the Python path until `python -m kdn_b200.build` has run")
        return None
    try:
        spec = importlib.util.spec_from_file_location("_kdn_torch", HOST_LIB)
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
    except (ImportError, OSError) as e:
        warnings.warn(f"kdn_b200: the C++ host path does not load ({e}); taking the Python path")
        return None
    lib = load_library()
    module.bind(*(ctypes.cast(getattr(lib, name), ctypes.c_void_p).value for name in _HOST_ENTRIES))
    return module


def host():
    """The C++ host path of the token step, the block norms and the sampling (``csrc/host/kdn_torch.cpp``): their
    functions answer None for what they leave to the Python path.  None where it is not built or does not load (with one
    warning), or with ``KDN_B200_HOST=python``; both paths make the same calls into the C library."""
    global _host
    if _host is None:
        _host = (None if os.environ.get("KDN_B200_HOST", "") == "python" else _load_host()) or False
    return _host or None


def has_tangent(*tensors) -> bool:
    """Whether a tensor carries a forward-mode derivative (asked tensor by tensor only inside a dual level)."""
    return forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def launch(entry, args, t: torch.Tensor, what: str) -> None:
    """Call a C entry ``entry(args, stream)`` on t's current stream, with t's device current."""
    device = t.device
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return check(entry(args, stream_of(t)), what)
    check(entry(args, _raw_stream(device.index)), what)


def _raw_stream(index: int) -> int:
    """The handle of the device's current stream (what ``stream_of`` gives, without making a Stream object per call)."""
    return torch._C._cuda_getCurrentRawStream(index)


_PRECISION = {"bf16": KDN_PREC_BF16, "fp32": KDN_PREC_FP32}


def precision() -> int:
    """Arithmetic precision of the scan, chosen by ``KDN_B200_PRECISION``:
    "bf16" (the product: the tcgen05 tensor-core kernels with bf16 operands
    and fp32 accumulation) or "fp32" (a separate debug implementation of the
    same chunked algorithm: SIMT / fp32 kernels with fp32 operands and the
    diagonal scan on 32-token chunks, used as a tight cross-check of the
    algorithm, not of the tcgen05 kernels)."""
    name = os.environ.get("KDN_B200_PRECISION", "bf16").lower()
    if name not in _PRECISION:
        raise ValueError(f"KDN_B200_PRECISION must be one of {sorted(_PRECISION)}, got {name!r}")
    return _PRECISION[name]


def byte_buffer(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 1), dtype=torch.uint8, device=device)
