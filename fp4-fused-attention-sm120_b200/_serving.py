"""What rotary.py and paged.py share: the library's handle with their
prototypes, the binding of their tensor calls, and the stream of a launch."""
from __future__ import annotations

import ctypes

import fp4attn_b200 as _fa


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
    L.fp4attn_selftest_paged_abort.argtypes = [cache, vp, vp, i32, i32, vp, i64, i32, vp, vp, sz, ctypes.c_uint, vp]
    L.fp4attn_copy_pages.argtypes = [cache, i32, vp, vp, i32, vp]
    for name in ("rotary_table", "rotary", "cache_append", "cache_gather", "paged_attention", "copy_pages",
                 "selftest_paged_abort"):
        getattr(L, "fp4attn_" + name).restype = i32
    L.fp4attn_paged_attention_workspace_size.restype = sz


lib, check, scale_mode = _fa.lib, _fa._check, _fa._scale_mode
_T = _NATIVE = None


def torch():
    """torch, imported on the first call (these functions run once a layer and
    token, so what they look up is kept)."""
    global _T
    if _T is None:
        _T = _fa._torch()
    return _T


def native():
    """The binding of the tensor calls (csrc/binding.cpp), bound to the library."""
    global _NATIVE
    if _NATIVE is None:
        torch()
        L = lib()
        try:
            from . import _native
        except ImportError as e:
            raise ImportError(f"{e}: build it with `make -C csrc` in the package directory "
                              "(there is no fallback implementation)") from e
        names = ("rotary", "cache_append", "cache_gather", "paged_attention_workspace_size", "paged_attention", "copy_pages")
        _native.bind(check, *[ctypes.cast(getattr(L, "fp4attn_" + n), ctypes.c_void_p).value for n in names])
        _NATIVE = _native
    return _NATIVE


def on(device, stream):
    """Context of a call on `stream`, which its outputs and workspaces belong to."""
    if stream.device != device:
        raise ValueError(f"the stream is on {stream.device}, the tensors on {device}")
    return torch().cuda.stream(stream)
