"""ctypes view of the attention launchers of include/futhark_amd_kernels.h.

The kernel library takes device pointers, sizes and a HIP stream; whose memory
it is (a context's arrays, another library's tensors) does not matter to it.
Pointers are integers or None, element types "f16" and "bf16".  A call that
the library rejects raises FutharkError with its code and text.
"""
from __future__ import annotations

import ctypes as C

from .capi import FutharkError, lib_path

DTYPES = {"i32": 0, "i64": 1, "f32": 2, "f64": 3, "u32": 4, "u64": 5, "f16": 6, "bf16": 7}


class Heads(C.Structure):
    """fa_heads: an array of rows of heads (strides in elements)."""
    _fields_ = [("data", C.c_void_p), ("row_stride", C.c_int64), ("head_stride", C.c_int64)]


def heads(data, row_stride: int, head_stride: int) -> Heads:
    return Heads(data, row_stride, head_stride)


_P, _I, _H = C.c_void_p, C.c_int64, C.POINTER(Heads)
_SEGS = [_P, _P]
_CACHE = [_P, _P, _I, _I, _P, _I]  # k_pages, v_pages, n_pages, page_size, page_table, table_cols
_FAILURE = [_P, C.c_int32]
_QKV = [_P, C.c_int, _H, _I, _H, _H, _I, _I, _I, _I] + _SEGS + _SEGS + [_I, C.c_float, C.c_int]
_LAUNCHERS = {
    "attention": _QKV + [_H, _P] + _FAILURE,
    "attention_grad": _QKV + [_H, _P, _H, _H, _H, _H, _P, C.c_size_t] + _FAILURE,
    "kv_append": [_P, C.c_int, _H, _H, _H, _H, _I, _I, _I, _I] + _SEGS + [_I, _P, _P, _I, C.c_int]
                 + _CACHE + _FAILURE,
    "attention_paged": [_P, C.c_int, _H, _I, _I, _I, _I] + _SEGS + [_I, _P, C.c_float]
                       + _CACHE + [_H, _P, _P, C.c_size_t] + _FAILURE,
}
_SIZES = {"attention_grad_workspace_bytes": 6, "attention_paged_workspace_bytes": 7}


class Kernels:
    """The launchers as methods, without their fa_ prefix and with the arguments
    of the header; `t` is the element type's name, arrays of heads are `Heads`."""

    def __init__(self, path=None):
        path = path or lib_path("libfuthark_amd_kernels.so")
        self.lib = C.CDLL(str(path))
        self.lib.fa_strerror.restype = C.c_char_p
        self.lib.fa_strerror.argtypes = [C.c_int]
        for name, args in _LAUNCHERS.items():
            f = getattr(self.lib, "fa_" + name)
            f.argtypes, f.restype = args, C.c_int
            setattr(self, name, self._launcher(f))
        for name, count in _SIZES.items():
            f = getattr(self.lib, "fa_" + name)
            f.argtypes, f.restype = [_I] * count, C.c_size_t
            setattr(self, name, f)

    def _launcher(self, f):
        def call(stream, t, *args):
            rc = f(stream, DTYPES[t], *args)
            if rc != 0:
                raise FutharkError(rc, self.lib.fa_strerror(rc).decode())
        call.__name__ = f.__name__
        return call
