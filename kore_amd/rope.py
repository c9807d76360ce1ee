"""ctypes binding of include/kore_rope.h (in kore_amd/libkore_paged.so): rotary
positions of rows of heads, in both pair layouts, over a part of the head, and
scaled for contexts past the trained one.

    r = Rope(Config(rot_dim=128, scaling="yarn", factor=4.0, orig_ctx=32768))
    r.apply_dev("f32", n_tok, n_head, head_dim, x_ptr, pos_ptr, out_ptr, stream=s)
    r.norm_dev("bf16", n_tok, head_dim, [Heads(q_ptr, q_ptr, n_head, head_dim, norm=q_norm_ptr),
                                         Heads(k_ptr, k_ptr, n_head_kv, head_dim, norm=k_norm_ptr)], pos_ptr, stream=s)

Device pointers are plain integers.  There is no CPU fallback: without the built
library or a GPU every call raises.
"""
from __future__ import annotations

import ctypes as C
import os

import numpy as np

from . import _lib as _attn_lib

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libkore_paged.so")

(KORE_PAGED_OK, KORE_PAGED_E_INVALID, KORE_PAGED_E_UNSUPPORTED, KORE_PAGED_E_HIP,
 KORE_PAGED_E_NOMEM) = 0, -1, -3, -4, -5
TYPES = {"f32": 0, "f16": 1, "bf16": 2}
LAYOUTS = {"half": 0, "interleaved": 1}
SCALINGS = {"none": 0, "linear": 1, "yarn": 2}

_vp, _i, _i64, _f = C.c_void_p, C.c_int, C.c_int64, C.c_float


class RopeConfig(C.Structure):
    """kore_rope_config"""
    _fields_ = [("rot_dim", _i), ("layout", _i), ("base", _f), ("scaling", _i), ("factor", _f), ("orig_ctx", _i),
                ("beta_fast", _f), ("beta_slow", _f), ("magnitude", _f), ("freq_factors", _vp)]


class HeadsStruct(C.Structure):
    """kore_rope_heads"""
    _fields_ = [("x", _vp), ("out", _vp), ("x_stride", _i64), ("out_stride", _i64), ("n_head", _i), ("norm", _vp)]


SYMBOLS = [
    ("kore_rope_create", _i, [C.POINTER(_vp), C.POINTER(RopeConfig)]),
    ("kore_rope_destroy", None, [_vp]),
    ("kore_rope_apply_dev", _i, [_vp, _i, _i, _i, _i, _vp, _i64, _vp, _vp, _i64, _i, _vp]),
    ("kore_rope_norm_dev", _i, [_vp, _i, _i, _i, C.POINTER(HeadsStruct), C.POINTER(HeadsStruct), _vp, _f, _vp]),
    ("kore_rope_get_freqs", _i, [_vp, _vp, C.POINTER(_f)]),
    ("kore_rope_sync", _i, [_vp]),
    ("kore_rope_last_error", C.c_char_p, [_vp]),
]

_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise _attn_lib.LibraryMissing(
                f"{LIB_PATH} is not built; run `make -C kore_amd/csrc` (or __graft_entry__.build())")
        L = C.CDLL(LIB_PATH)
        for name, res, args in SYMBOLS:
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _lib = L
    return _lib


class PagedError(RuntimeError):
    """A failed kore_rope_* or kore_paged_* call."""

    def __init__(self, code: int, message: str):
        super().__init__(f"[{code}] {message}")
        self.code = code
        self.message = message


def type_code(name: str) -> int:
    code = TYPES.get(name)
    if code is None:
        raise ValueError(f"type {name!r} is not one of {sorted(TYPES)}")
    return code


class Config:
    """The frequencies of a rotary plan (kore_rope_config)."""

    def __init__(self, rot_dim: int, layout: str = "half", base: float = 1e6, scaling: str = "none",
                 factor: float = 1.0, orig_ctx: int = 0, beta_fast: float = 0.0, beta_slow: float = 0.0,
                 magnitude: float = 0.0, freq_factors=None):
        if layout not in LAYOUTS:
            raise ValueError(f"layout {layout!r} is not one of {sorted(LAYOUTS)}")
        if scaling not in SCALINGS:
            raise ValueError(f"scaling {scaling!r} is not one of {sorted(SCALINGS)}")
        self.factors = None
        if freq_factors is not None:
            self.factors = np.ascontiguousarray(freq_factors, np.float32).reshape(-1)
            if self.factors.size != rot_dim // 2:
                raise ValueError(f"expected {rot_dim // 2} freq_factors, got {self.factors.size}")
        self.rot_dim = rot_dim
        self.struct = RopeConfig(rot_dim, LAYOUTS[layout], base, SCALINGS[scaling], factor, orig_ctx, beta_fast,
                                 beta_slow, magnitude, None if self.factors is None else self.factors.ctypes.data)


class Heads:
    """A set of rows of n_head heads of head_dim values (kore_rope_heads): device pointers of the rows, of those that they
    become and of the norm's weights (None: the heads are turned only).  Strides in elements, None: rows one behind the
    other."""

    def __init__(self, x: int, out: int, n_head: int, head_dim: int, norm: int | None = None, x_stride: int | None = None,
                 out_stride: int | None = None):
        n = n_head * head_dim
        self.struct = HeadsStruct(x, out, n if x_stride is None else x_stride, n if out_stride is None else out_stride, n_head,
                                  norm)
        self._ref = C.byref(self.struct)


class Rope:
    """kore_rope_t: a rotary plan on the current HIP device."""

    def __init__(self, config: Config):
        self._h = None
        h = _vp()
        rc = lib().kore_rope_create(C.byref(h), C.byref(config.struct))
        if rc != KORE_PAGED_OK:
            raise PagedError(rc, lib().kore_rope_last_error(None).decode())
        self._h = h
        self._norm = lib().kore_rope_norm_dev
        self.rot_dim = config.rot_dim

    def _check(self, rc: int) -> None:
        if rc != KORE_PAGED_OK:
            raise PagedError(rc, lib().kore_rope_last_error(self._h).decode())

    def apply_dev(self, dtype: str, n_tok: int, n_head: int, head_dim: int, x: int, pos: int, out: int,
                  x_stride: int | None = None, out_stride: int | None = None, transpose: bool = False,
                  stream=None) -> None:
        """Rows x [n_tok][n_head][head_dim] turned to the positions pos (int32) into out (device pointers; strides
        in elements, None: rows one behind the other).  transpose: the gradient of the same call."""
        n = n_head * head_dim
        self._check(lib().kore_rope_apply_dev(self._h, type_code(dtype), n_tok, n_head, head_dim, x,
                                              n if x_stride is None else x_stride, pos, out,
                                              n if out_stride is None else out_stride, int(transpose), stream))

    def norm_dev(self, dtype: str, n_tok: int, head_dim: int, sets, pos: int, eps: float = 1e-6, stream=None) -> None:
        """One or two sets (Heads) of n_tok rows: each head over its root mean square, times its set's weights, then turned
        to the row's position (pos: device, int32; rows with a negative one are left as they are)."""
        if len(sets) > 2:
            raise ValueError(f"{len(sets)} sets of heads (1 or 2)")
        q, k = sets[0]._ref if sets else None, sets[1]._ref if len(sets) == 2 else None
        rc = self._norm(self._h, type_code(dtype), n_tok, head_dim, q, k, pos, eps, stream)
        if rc:
            self._check(rc)

    def freqs(self):
        """(frequencies [rot_dim / 2], magnitude)"""
        f, m = np.empty(self.rot_dim // 2, np.float32), _f()
        self._check(lib().kore_rope_get_freqs(self._h, f.ctypes.data, C.byref(m)))
        return f, m.value

    def sync(self) -> None:
        self._check(lib().kore_rope_sync(self._h))

    def close(self) -> None:
        if self._h:
            lib().kore_rope_destroy(self._h)
            self._h = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
