"""What rotary.py and paged.py share: the library's handle with their
prototypes, argument checks, and the device and stream of a launch."""
from __future__ import annotations

import contextlib
import ctypes

import fp4attn_b200 as _fa

F32, F16 = 0, 1


class CacheStruct(ctypes.Structure):
    """fp4attn_cache of include/fp4attn.h."""
    _fields_ = [("k_codes", ctypes.c_void_p), ("k_scales", ctypes.c_void_p), ("v", ctypes.c_void_p),
                ("k_codes_stride", ctypes.c_int64), ("k_scales_stride", ctypes.c_int64), ("v_stride", ctypes.c_int64),
                ("pages", ctypes.c_int), ("page_size", ctypes.c_int), ("kv_heads", ctypes.c_int),
                ("head_dim", ctypes.c_int)]


def declare(L) -> None:
    """Prototypes of the serving entry points (called once by lib())."""
    vp, i32, i64, sz, f32, f64 = (ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t, ctypes.c_float,
                                  ctypes.c_double)
    cache = ctypes.POINTER(CacheStruct)
    L.fp4attn_rotary_table.argtypes = [vp, i32, i64, f64, vp, vp]
    L.fp4attn_rotary.argtypes = [vp, vp] + [i32] * 5 + [vp, vp, vp, i32, i64, vp, i64, i32, i32, vp]
    L.fp4attn_cache_append.argtypes = ([cache] + [vp] * 4 + [i32] * 3 + [vp] * 4 + [i64, i32, i32] + [vp] * 3 +
                                       [i32, i64, i32, i32, vp])
    L.fp4attn_cache_gather.argtypes = [cache, vp, i64, i32, i32, vp, vp, i32, i32, vp, vp, i32, vp]
    L.fp4attn_paged_attention_workspace_size.argtypes = [i32] * 4
    L.fp4attn_paged_attention.argtypes = ([cache, vp, vp, vp] + [i32] * 4 + [vp, vp, i64, i32, vp, f32, i32, vp, sz, vp])
    L.fp4attn_copy_pages.argtypes = [cache, i32, vp, vp, i32, vp]
    for name in ("rotary_table", "rotary", "cache_append", "cache_gather", "paged_attention", "copy_pages"):
        getattr(L, "fp4attn_" + name).restype = i32
    L.fp4attn_paged_attention_workspace_size.restype = sz


lib, check, scale_mode = _fa.lib, _fa._check, _fa._scale_mode
I2, I3 = ctypes.c_int64 * 2, ctypes.c_int64 * 3
_T = None
_CODES = {}


def torch():
    """torch, imported on the first call (these functions run once a layer and
    token, so what they look up is kept)."""
    global _T
    if _T is None:
        _T = _fa._torch()
        _CODES.update({_T.float16: F16, _T.float32: F32})
    return _T


def dtype_code(dtype) -> int:
    torch()
    code = _CODES.get(dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype}; use float16 or float32")
    return code


def check_index(t, name, device):
    if t.dtype is not torch().int32 or t.device != device:
        raise ValueError(f"{name} must be an int32 tensor on {device}")


def check_table(table, device, head_dim):
    """(pointer, rotary_dim, positions) of a rotary table."""
    shape = table.shape
    if (len(shape) != 3 or shape[2] != 2 or table.dtype is not torch().float32 or table.device != device or
            not table.is_contiguous()):
        raise ValueError(f"table must be a contiguous float32 [positions, rotary_dim / 2, 2] tensor on {device}")
    if 2 * shape[1] > head_dim:
        raise ValueError(f"the table's rotary_dim {2 * shape[1]} exceeds head_dim {head_dim}")
    return table.data_ptr(), 2 * shape[1], shape[0]


_HERE = contextlib.nullcontext()


def on(device, stream):
    """Context in which a call allocates and launches: the tensors' device
    current, and `stream` (default: that device's current stream) the stream
    its outputs and workspaces belong to."""
    T = torch()
    if stream is not None:
        if stream.device != device:
            raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
        return T.cuda.stream(stream)
    return _HERE if device.index == T.cuda.current_device() else T.cuda.device(device)


def stream_ptr(device) -> int:
    """The current stream of a device, as the library takes it."""
    return _T._C._cuda_getCurrentRawStream(device.index)
