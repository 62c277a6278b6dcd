"""ctypes binding of libbfa.so (declared in include/bfa.h).

This module only moves pointers, strides and sizes across the C ABI; all
compute happens in the library's CUDA kernels. It never falls back to a CPU
implementation: if the library is missing, every call raises.
"""
from __future__ import annotations

import ctypes
import functools
import os
import struct
import threading

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libbfa.so")
ABI_VERSION = 6

DTYPE_F32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2
DEBUG_INJECT_STALL = 1
ERR_DEVICE_TIMEOUT = -6

EXPORTED = ("bfa_abi_version", "bfa_launch_count", "bfa_strerror", "bfa_last_error", "bfa_fwd",
            "bfa_fwd_workspace_bytes", "bfa_bwd_workspace_bytes", "bfa_bwd_delta", "bfa_bwd", "bfa_bwd_noalloc",
            "bfa_merge_partial", "bfa_rope", "bfa_tree_workspace_bytes", "bfa_tree_fwd", "bfa_verify_tree",
            "bfa_cache_append")
ERR_SCRATCH_LIMIT = -7
ERR_INDEX = -8
NOALLOC_MAX_ROWS = 1 << 21
PHASE_DELTA, PHASE_DKDV, PHASE_DQ = 1, 2, 4

_TORCH_TO_BFA = {torch.float32: DTYPE_F32, torch.float16: DTYPE_F16,
                 torch.bfloat16: DTYPE_BF16}


class Problem(ctypes.Structure):
    _fields_ = [("batch", ctypes.c_int32), ("heads_q", ctypes.c_int32),
                ("heads_kv", ctypes.c_int32), ("seqlen_q", ctypes.c_int32),
                ("seqlen_k", ctypes.c_int32), ("head_dim", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("causal", ctypes.c_int32),
                ("sliding_window", ctypes.c_int32), ("scale", ctypes.c_float),
                ("soft_cap", ctypes.c_float), ("alibi_slopes", ctypes.c_void_p),
                ("q_pos_offset", ctypes.c_int64), ("k_pos_offset", ctypes.c_int64),
                ("doc_start", ctypes.c_void_p), ("doc_end", ctypes.c_void_p),
                ("block_mask", ctypes.c_void_p), ("block_mask_stride", ctypes.c_int64 * 3)]


class Tensor(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("stride", ctypes.c_int64 * 4)]


class FwdArgs(ctypes.Structure):
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor),
                ("lse", ctypes.c_void_p), ("status", ctypes.c_void_p),
                ("wait_timeout_ns", ctypes.c_int64), ("debug_flags", ctypes.c_uint32),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t),
                ("accumulate", ctypes.c_uint32)]


class BwdArgs(ctypes.Structure):
    _fields_ = [("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor),
                ("dout", Tensor), ("lse", ctypes.c_void_p), ("dq", Tensor),
                ("dk", Tensor), ("dv", Tensor), ("status", ctypes.c_void_p),
                ("wait_timeout_ns", ctypes.c_int64), ("debug_flags", ctypes.c_uint32),
                ("phases", ctypes.c_uint32), ("accumulate", ctypes.c_uint32)]


def _wide(name, fields):
    """A ctypes mirror of a structure whose fields are all 8 bytes wide, and
    the struct.Struct that packs its fields in order, a tensor as its pointer
    and four strides: one pack() call fills an argument block several times
    faster than attribute by attribute, which is what a decoding step's calls
    spend most of their host time on."""
    cls = type(name, (ctypes.Structure,), {"_fields_": fields})
    code = ""
    for _, t in fields:
        code += {Tensor: "5q", ctypes.c_int64: "q", ctypes.c_int64 * 2: "2q", ctypes.c_void_p: "q", ctypes.c_double: "d"}[t]
    pack = struct.Struct("@" + code)
    assert pack.size == ctypes.sizeof(cls)
    return cls, pack.pack


_i64, _ptr = ctypes.c_int64, ctypes.c_void_p

RopeArgs, pack_rope = _wide("RopeArgs", [
    ("batch", _i64), ("heads_q", _i64), ("heads_k", _i64), ("seqlen", _i64), ("head_dim", _i64),
    ("rotary_dim", _i64), ("dtype", _i64), ("interleaved", _i64), ("inverse", _i64),
    ("q", Tensor), ("k", Tensor), ("q_out", Tensor), ("k_out", Tensor), ("cos", _ptr), ("sin", _ptr),
    ("table_rows", _i64), ("table_stride", _i64), ("positions", _ptr), ("positions_bytes", _i64),
    ("positions_stride", _i64 * 2), ("offsets", _ptr), ("offsets_bytes", _i64), ("status", _ptr)])

TreeArgs, pack_tree = _wide("TreeArgs", [
    ("batch", _i64), ("heads_q", _i64), ("heads_kv", _i64), ("nodes", _i64), ("head_dim", _i64), ("dtype", _i64),
    ("num_pages", _i64), ("page_size", _i64), ("max_pages", _i64), ("sliding_window", _i64),
    ("scale", ctypes.c_double), ("soft_cap", ctypes.c_double), ("alibi_slopes", _ptr),
    ("q", Tensor), ("k", Tensor), ("v", Tensor), ("o", Tensor), ("lse", _ptr), ("k_pages", Tensor), ("v_pages", Tensor),
    ("page_table", _ptr), ("page_table_stride", _i64), ("lens", _ptr), ("parents", _ptr), ("parents_stride", _i64),
    ("status", _ptr), ("workspace", _ptr), ("workspace_bytes", _i64)])

_TREE_VALUES = sum(5 if t is Tensor else 1 for _, t in TreeArgs._fields_)

VerifyArgs, pack_verify = _wide("VerifyArgs", [
    ("batch", _i64), ("nodes", _i64), ("vocab", _i64), ("dtype", _i64), ("target", _ptr), ("target_stride", _i64 * 2),
    ("draft", _ptr), ("draft_stride", _i64 * 2), ("tokens", _ptr), ("tokens_bytes", _i64), ("tokens_stride", _i64),
    ("parents", _ptr), ("parents_stride", _i64), ("uniforms", _ptr), ("uniforms_stride", _i64), ("noise", _ptr),
    ("noise_stride", _i64), ("path", _ptr), ("count", _ptr), ("next_token", _ptr), ("status", _ptr)])

AppendArgs, pack_append = _wide("AppendArgs", [
    ("batch", _i64), ("heads_kv", _i64), ("tokens", _i64), ("head_dim", _i64), ("dtype", _i64), ("num_pages", _i64),
    ("page_size", _i64), ("max_pages", _i64), ("k", Tensor), ("v", Tensor), ("k_pages", Tensor), ("v_pages", Tensor),
    ("page_table", _ptr), ("page_table_stride", _i64), ("lens", _ptr), ("take", _ptr), ("take_stride", _i64),
    ("count", _ptr), ("lens_out", _ptr), ("status", _ptr)])


_lib = None
_lock = threading.Lock()


def load() -> ctypes.CDLL:
    """Load libbfa.so once and declare its signatures."""
    global _lib
    with _lock:
        if _lib is not None:
            return _lib
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing; build it with `python {HERE}/build.py` "
                "(there is no CPU fallback)")
        lib = ctypes.CDLL(LIB_PATH)
        lib.bfa_abi_version.restype = ctypes.c_int
        lib.bfa_abi_version.argtypes = []
        lib.bfa_launch_count.restype = ctypes.c_uint64
        lib.bfa_launch_count.argtypes = []
        lib.bfa_strerror.restype = ctypes.c_char_p
        lib.bfa_strerror.argtypes = [ctypes.c_int]
        lib.bfa_last_error.restype = ctypes.c_char_p
        lib.bfa_last_error.argtypes = []
        lib.bfa_fwd.restype = ctypes.c_int
        lib.bfa_fwd.argtypes = [ctypes.POINTER(Problem), ctypes.POINTER(FwdArgs), ctypes.c_void_p]
        lib.bfa_fwd_workspace_bytes.restype = ctypes.c_size_t
        lib.bfa_fwd_workspace_bytes.argtypes = [ctypes.POINTER(Problem)]
        lib.bfa_bwd_workspace_bytes.restype = ctypes.c_size_t
        lib.bfa_bwd_workspace_bytes.argtypes = [ctypes.POINTER(Problem)]
        lib.bfa_bwd_delta.restype = ctypes.c_int
        lib.bfa_bwd_delta.argtypes = [ctypes.POINTER(Problem), ctypes.POINTER(BwdArgs),
                                      ctypes.c_void_p, ctypes.c_void_p]
        lib.bfa_bwd.restype = ctypes.c_int
        lib.bfa_bwd.argtypes = [ctypes.POINTER(Problem), ctypes.POINTER(BwdArgs),
                                ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
        lib.bfa_bwd_noalloc.restype = ctypes.c_int
        lib.bfa_bwd_noalloc.argtypes = [ctypes.POINTER(Problem), ctypes.POINTER(BwdArgs),
                                        ctypes.c_void_p]
        lib.bfa_merge_partial.restype = ctypes.c_int
        lib.bfa_merge_partial.argtypes = [ctypes.c_int32] * 4 + [
            Tensor, ctypes.c_int32, ctypes.c_void_p, Tensor, ctypes.c_int32, ctypes.c_void_p,
            ctypes.c_void_p]
        # Packed argument blocks travel as bytes objects (a read-only pointer to them).
        for name in ("bfa_rope", "bfa_tree_fwd", "bfa_verify_tree", "bfa_cache_append"):
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_char_p, ctypes.c_void_p]
        lib.bfa_tree_workspace_bytes.restype = ctypes.c_size_t
        lib.bfa_tree_workspace_bytes.argtypes = [ctypes.c_char_p]
        ver = lib.bfa_abi_version()
        if ver != ABI_VERSION:
            raise RuntimeError(f"libbfa ABI version {ver}, expected {ABI_VERSION}")
        _lib = lib
    return _lib


ERR_CUDA = -5


def check(rc: int) -> None:
    if rc != 0:
        lib = load()
        msg = lib.bfa_strerror(rc).decode()
        if rc == ERR_CUDA:
            detail = lib.bfa_last_error().decode()
            if detail:
                msg = f"{msg} ({detail})"
        raise RuntimeError(msg)


def bfa_dtype(dt: torch.dtype) -> int:
    if dt not in _TORCH_TO_BFA:
        raise RuntimeError(f"unsupported dtype {dt} (need float32, float16 or bfloat16)")
    return _TORCH_TO_BFA[dt]


def tensor(t: torch.Tensor | None) -> Tensor:
    out = Tensor()
    if t is None:
        return out
    out.data = t.data_ptr()
    for i, s in enumerate(t.stride()):
        out.stride[i] = s
    return out


def flat(t: torch.Tensor | None) -> tuple:
    """A [B, H, S, D] tensor's pointer and strides, as the packers take them."""
    return (0, 0, 0, 0, 0) if t is None else (t.data_ptr(), *t.stride())


def require_cuda(what: str, tensors, device=None) -> None:
    """Every tensor is on one CUDA device (`device`, or the first one's)."""
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError(f"{what} (B200 build) needs CUDA tensors; there is no CPU path")
        if device is None:
            device = t.device
        elif t.device != device:
            raise RuntimeError(f"{what}: tensors on {device} and {t.device}; they must share a device")


CHECK_STATUS = os.environ.get("BFA_CHECK_STATUS", "0") == "1"
_functions = {}


def launch(name: str, packed: bytes, device: torch.device) -> None:
    """One entry point that takes a packed argument block, on the device's
    current stream. The tensors exist, so CUDA is initialised and the raw
    calls (current device, current stream's handle) need no guard of torch's;
    a decoding step makes a few such calls per layer, and their host time is
    what it waits for."""
    fn = _functions.get(name)
    if fn is None:
        fn = _functions[name] = getattr(load(), name)
    index = device.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(packed, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(device):
            rc = fn(packed, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        check(rc)
    if CHECK_STATUS:
        check(read_and_clear_status(device))


_status_at = {}


def status_ptr(device: torch.device) -> int:
    """Address of the device's status word."""
    at = _status_at.get(device.index)
    if at is None:
        at = _status_at[device.index] = status_word(device).data_ptr()
    return at


@functools.lru_cache(maxsize=4096)
def tree_workspace_bytes(index: int, *sizes) -> int:
    """bfa_tree_workspace_bytes of a device and the sizes that open a
    bfa_tree_args block (batch ... soft_cap); it depends on nothing else."""
    with torch.cuda.device(index):
        return load().bfa_tree_workspace_bytes(pack_tree(*sizes, *[0] * (_TREE_VALUES - len(sizes))))


def stream_ptr(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


_status = {}


def status_word(device: torch.device) -> torch.Tensor:
    """Per-device int32 status word that bounded device waits report into."""
    key = device.index if device.index is not None else torch.cuda.current_device()
    if key not in _status:
        _status[key] = torch.zeros(1, dtype=torch.int32, device=device)
    return _status[key]


def read_and_clear_status(device: torch.device) -> int:
    """Synchronise the device, return its status word and reset it to 0."""
    w = status_word(device)
    val = int(w.item())
    w.zero_()
    return val
