"""ctypes loader for libfastbb_b200.so, the C-ABI shared library holding the sm_100a kernels.

Plays the role of the reference's driver-API loader (fastbb/kernels.py:71-133 `Kernels`): the host code stays
Python/PyTorch and crosses one thin FFI boundary per operator. Differences: the boundary is a C ABI with one
entry point per operator instead of a kernel-name + signature-string table; a non-zero status becomes a Python
exception; nothing is cached per device in Python, so several GPUs can be used from one process.
There is no CPU or PyTorch fallback: if the library is missing, importing an operator raises.

Attention on its own: `attention.py` + this file + `libfastbb_flash64.so` (`python -m fastbb_b200.build --flash-only`) are
all a project needs that vendors only the attention API, as several forks do with the reference's
attention.py + kernels.py. When the full library is absent, load() falls back to that one and sets up only the
entry points it exports.
"""
import contextlib
import ctypes
import os
import struct

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libfastbb_b200.so")
FLASH_LIB_PATH = os.path.join(_HERE, "libfastbb_flash64.so")   # attention kernel and its entry points only

FBB_OK = 0
DTYPE_CODE = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
EPI_NONE, EPI_GELU, EPI_SWIGLU = 0, 1, 2
ACC_F32, ACC_F16 = 0, 1
FLASH_VARIANT = {"ff": 0, "fh": 1, "hh": 2}

_vp, _i32, _i64, _f32 = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


def on(device):
    """Context manager that makes `device` current for the enclosed C calls (a no-op when it already is)."""
    return _HERE_ALREADY if device.index == torch._C._cuda_getDevice() else torch.cuda.device(device)


_HERE_ALREADY = contextlib.nullcontext()


class BlockDesc(ctypes.Structure):
    """fbb_block_desc of include/fastbb_b200.h: weight pointers and shapes of one transformer block."""
    _fields_ = ([(n, _vp) for n in ("ln1_w", "ln1_b", "qkv_w", "qkv_b", "proj_w", "proj_b", "gamma1", "ln2_w", "ln2_b",
                                    "fc1_w", "fc1_b", "fc2_w", "fc2_b", "gamma2")]
                + [(n, _i32) for n in ("C", "heads", "hidden", "mlp", "acc_main", "acc_fc2", "flash_variant")]
                + [(n, _f32) for n in ("eps1", "eps2", "scale")])


class RotaryTensor(ctypes.Structure):
    """fbb_rotary_tensor of include/fastbb_b200.h: one tensor to turn, [B, N, heads, D], and where to."""
    _fields_ = [("x", _vp), ("y", _vp), ("heads", _i32)] + [(n, _i64) for n in ("x_sb", "x_sn", "x_sh", "y_sb", "y_sn", "y_sh")]


# Arguments of a call as one record: converted one by one, 25 to 36 of them take 2 to 3.3 us of a call's 15 (packed, 0.7).
RotaryArgs = struct.Struct("=QQi4x6q QQi4x6q 4Q3q11i4x")     # fbb_rotary_args
Diff64Args = struct.Struct("=9Q16q6i3f4x")                   # fbb_diff64_args
AdapterLinearArgs = struct.Struct("=13Q6q6i")                # fbb_adapter_linear_args

MLP_GELU, MLP_SWIGLU = 0, 1
_bdp = ctypes.POINTER(BlockDesc)

# name -> (restype, argtypes); mirrors include/fastbb_b200.h one to one.
PROTOTYPES = {
    "fbb_version": (_i32, []),
    "fbb_status_string": (ctypes.c_char_p, [_i32]),
    "fbb_last_error": (ctypes.c_char_p, []),
    "fbb_device_status": (_i32, [ctypes.POINTER(ctypes.c_uint * 4)]),
    "fbb_diag_wait_timeout": (_i32, [ctypes.c_uint64, ctypes.c_uint, _vp]),
    "fbb_diag_sm_clock_mhz": (_i32, [_vp, _i64, _vp]),
    "fbb_linear_max_cta_pairs": (_i32, [_i32]),
    "fbb_linear_form": (_i32, [_i64, _i32, _i32, _i32, _i32, ctypes.c_char_p, _i32]),
    "fbb_layernorm_f16": (_i32, [_vp, _vp, _vp, _vp, _i64, _i32, _i64, _i64, _f32, _i32, _i32, _vp]),
    "fbb_layernorm_split_f16": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _i32, _i32, _i32, _i32, _f32, _i32, _i32, _vp]),
    "fbb_linear_f16": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i64, _i64, _i64, _i64, _i32, _i32, _vp]),
    "fbb_linear_layernorm_f16": (_i32, [_vp, _vp, _vp, _vp, _vp, _vp, _i64, _i32, _i32, _i64, _i64, _i64, _i64, _i32, _i32, _vp, _vp, _f32, _vp, _i64,
                                        _vp, _vp]),
    "fbb_linear_layernorm_launches": (_i32, [_i64, _i32, _i32, _i32]),
    "fbb_flash64_f16": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32] + [_i64] * 12 + [_f32, _i32, _vp]),
    "fbb_flash64_workspace_bytes": (_i64, [_i32, _i32, _i32]),
    "fbb_flash64_launches": (_i32, [_i32, _i32, _i32, _i32]),
    "fbb_flash64_f16_ws": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32] + [_i64] * 12 + [_f32, _i32, _vp, _i64, _vp]),
    "fbb_flash64_f16_static": (_i32, [_vp, _vp, _vp, _vp, _i32, _i32, _i32] + [_i64] * 12 + [_f32, _i32, _vp]),
    "fbb_adapter_linear_workspace_bytes": (_i64, [_i64] + [_i32] * 5),
    "fbb_adapter_linear_f16": (_i32, [_vp] * 6 + [_i64, _i32, _i32] + [_i64] * 4 + [_i32, _vp, _vp, _vp, _i32, _i32, _vp, _vp, _i32, _vp, _i64, _vp]),
    "fbb_adapter_linear_f16_from": (_i32, [ctypes.c_char_p]),
    "fbb_diff64_workspace_bytes": (_i64, [_i32] * 4),
    "fbb_diff64_launches": (_i32, [_i32] * 4),
    "fbb_diff64_f16": (_i32, [_vp] * 4 + [_i32] * 5 + [_i64] * 12 + [_vp] + [_i64] * 3 + [_vp, _i32, _f32, _f32, _f32, _vp, _vp, _i64, _vp]),
    "fbb_diff64_f16_from": (_i32, [ctypes.c_char_p]),
    "fbb_rotary": (_i32, [ctypes.POINTER(RotaryTensor)] + [_i32] * 7 + [_vp, _i32, _i32, _i64, _i64, _i64, _vp, _vp, _i32, _i32, _vp]),
    "fbb_rotary_from": (_i32, [ctypes.c_char_p]),
    "fbb_stack_scratch_bytes": (_i64, [_bdp, _i32, _i64]),
    "fbb_stack_launches": (_i32, [_bdp, _i32, _i64]),
    "fbb_stack_forward_f16": (_i32, [_bdp, _i32, _vp, _i32, _i32, _vp, _i64, _vp, _i64, _vp]),
    "fbb_block_forward_f16": (_i32, [_bdp, _vp, _i32, _i32, _vp, _i64, _vp, _i64, _vp]),
}


class FastbbError(RuntimeError):
    """A non-zero status from libfastbb_b200.so (negative: rejected arguments; positive: a CUDA error code)."""

    def __init__(self, status, message):
        super().__init__(f"fastbb_b200 status {status}: {message}")
        self.status = status


_LIB = None
LAUNCHES = 0  # kernels enqueued through this module since import (each operator call is exactly one launch)


def launched(n=1):
    global LAUNCHES
    LAUNCHES += n


# what libfastbb_flash64.so exports (the other prototypes are skipped when that library is the one loaded)
FLASH_ONLY_SYMBOLS = ("fbb_version", "fbb_status_string", "fbb_last_error", "fbb_device_status", "fbb_diag_wait_timeout",
                      "fbb_diag_sm_clock_mhz", "fbb_flash64_f16",
                      "fbb_flash64_workspace_bytes", "fbb_flash64_launches", "fbb_flash64_f16_ws", "fbb_flash64_f16_static")


def load(path=None):
    """Load (once) and return the ctypes handle with every prototype set. Without `path`: the full library, or, if only
    the attention-only library has been built, that one. Raises OSError if neither exists."""
    global _LIB
    if _LIB is None or path is not None:
        p = path or (LIB_PATH if os.path.exists(LIB_PATH) or not os.path.exists(FLASH_LIB_PATH) else FLASH_LIB_PATH)
        if not os.path.exists(p):
            raise OSError(f"{p} not found: build it with `python -m fastbb_b200.build` (needs nvcc with sm_100a support); "
                          "there is no fallback path")
        lib = ctypes.CDLL(p)
        lib.flash_only = not hasattr(lib, "fbb_linear_f16")
        for name, (res, args) in PROTOTYPES.items():
            if lib.flash_only and name not in FLASH_ONLY_SYMBOLS:
                continue
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        if path is not None:
            return lib
        _LIB = lib
    return _LIB


def check(status):
    if status != FBB_OK:
        lib = load()
        msg = lib.fbb_last_error().decode() or lib.fbb_status_string(status).decode()
        raise FastbbError(status, msg)


def stream_ptr(device=None):
    """cudaStream_t of torch's current stream on `device` as an integer (0 = legacy default stream)."""
    index = device.index if device is not None else None
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device() if index is None else index)


def ptr(t):
    return t.data_ptr() if t is not None else None


def address(t):
    """ptr() for a record's field."""
    return t.data_ptr() if t is not None else 0


def _nest(dims, span):
    """Whether every one of dims, (stride, size) innermost first, steps over what the dimensions inside it span, from `span` elements on."""
    for s, n in dims:
        if s < span:
            return False
        span += (n - 1) * s
    return True


def _nested(t):
    """(stride, size) of t's dimensions of more than one element, innermost first, and whether no two elements share an address
    (every stride steps over what the dimensions inside it span)."""
    dims = sorted([(s, n) for n, s in zip(t.shape, t.stride()) if n > 1])
    return dims, _nest(dims, 1)


def writable(t):
    """Whether every element of t has an address of its own (an expanded or self-overlapping view cannot be written by many threads)."""
    return t.is_contiguous() or t.numel() == 0 or _nested(t)[1]


def same_view(a, b):
    return a is b or (a.data_ptr() == b.data_ptr() and a.shape == b.shape and a.dtype == b.dtype and all(
        n == 1 or s == r for n, s, r in zip(a.shape, a.stride(), b.stride())))


def disjoint(a, b):
    """Whether a and b (of one dtype) surely share no element: byte ranges apart, or views of one buffer that lie beside each other
    within equal outer strides, like the queries and keys of a packed projection."""
    pa, pb = a.data_ptr(), b.data_ptr()
    if pa > pb:
        a, b, pa, pb = b, a, pb, pa
    size = a.element_size()
    if pb - pa >= size * a.numel() and a.is_contiguous():
        return True
    if a.numel() == 0 or b.numel() == 0:
        return True
    gap = (pb - pa) // size
    da, db = _nested(a)[0], _nested(b)[0]
    if gap > sum([(n - 1) * s for s, n in da]):
        return True
    for k in range(len(da)):  # the k innermost dimensions of a against what the next one leaves for b (if the outer ones step over all of that)
        outer = da[k:]
        m = len(db) - len(outer)
        if m < 0 or db[m:] != outer or not _nest(outer, outer[0][0]):
            continue
        span_a, span_b = 1 + sum([(n - 1) * s for s, n in da[:k]]), 1 + sum([(n - 1) * s for s, n in db[:m]])
        if gap >= span_a and gap + span_b <= outer[0][0]:
            return True
    return False


def apart(out, *others):
    """Whether an output surely shares no memory with any of the others (of any dtype; None: not there)."""
    lo = out.data_ptr()
    hi = lo + _bytes(out)
    for t in others:
        if t is not None:
            p = t.data_ptr()
            if p < hi and lo < p + _bytes(t) and not (t.dtype == out.dtype and disjoint(out, t)):
                return False
    return True


def _bytes(t):
    """From a tensor's first byte to behind its last one, holes included."""
    n = t.numel()
    if n and not t.is_contiguous():
        n = 1 + sum([(n - 1) * s for n, s in zip(t.shape, t.stride())])
    return n * t.element_size()


def device_status():
    """Synchronise the current device and raise FastbbError if any kernel gave up a bounded wait."""
    out = (ctypes.c_uint * 4)()
    check(load().fbb_device_status(ctypes.byref(out)))
    return tuple(out)
