"""ctypes binding of include/kore_paged.h (kore_amd/libkore_paged.so): a KV cache
of pages shared by several sequences, the append of their new rows and the
attention that reads it.

    kv = PagedKV(n_layer=28, n_pages=4096, page_size=64, n_head=28, n_head_kv=4, head_dim=128,
                 cache_type="bf16", rope=rope.Config(rot_dim=128))
    b = Batch(n_seq, n_tok, q_start_ptr, kv_len_ptr, pages_ptr, pages_stride, max_q=1)
    kv.append_dev(layer, b, "f32", k_ptr, v_ptr, q=q_ptr, q_out=q_ptr, stream=s)
    kv.attend_dev(layer, b, "f32", q_ptr, out_ptr, stream=s)

and, for steps of drafted tokens, the step's tables made on the GPU, the store by them, the attention of the trees and
what is kept of them:

    kv.plan_dev(Plan(...), stream=s)
    kv.append_rows_dev(layer, Rows(n_tok, pos_ptr, slot_ptr, q_norm=..., k_norm=...), "f32", k_ptr, v_ptr, q=q_ptr, q_out=q_ptr)
    kv.attend_tree_dev(layer, b, Tree(mask_ptr, mask_words), "f32", q_ptr, out_ptr, stream=s)
    kv.keep_dev(Keep(...), stream=s)

Device pointers are plain integers.  There is no CPU fallback: without the built
library or a GPU every call raises.
"""
from __future__ import annotations

import ctypes as C

from . import rope as _rope
from .rope import KORE_PAGED_OK, Config, PagedError, RopeConfig, type_code

_vp, _i, _i64, _f = C.c_void_p, C.c_int, C.c_int64, C.c_float


class PagedConfig(C.Structure):
    """kore_paged_config"""
    _fields_ = [("n_layer", _i), ("n_pages", _i), ("page_size", _i), ("n_head", _i), ("n_head_kv", _i),
                ("head_dim", _i), ("cache_type", _i), ("rope", RopeConfig), ("k_pool", _vp), ("v_pool", _vp)]


class BatchStruct(C.Structure):
    """kore_paged_batch"""
    _fields_ = [("n_seq", _i), ("n_tok", _i), ("q_start", _vp), ("kv_len", _vp), ("pages", _vp),
                ("pages_stride", _i), ("max_q", _i)]


class PagedInfo(C.Structure):
    """kore_paged_info"""
    _fields_ = [("config", PagedConfig), ("device", _i), ("num_cu", _i), ("pool_bytes", C.c_size_t), ("stream", _vp)]


class PlanStruct(C.Structure):
    """kore_paged_plan"""
    _fields_ = [("n_seq", _i), ("n_tok", _i), ("n_new", _vp), ("kv_held", _vp), ("kv_len", _vp), ("pages", _vp),
                ("pages_stride", _i), ("free_pages", _vp), ("n_free", _vp), ("n_free_out", _vp), ("parent", _vp),
                ("q_start", _vp), ("pos", _vp), ("slot", _vp), ("mask", _vp), ("mask_words", _i), ("status", _vp), ("window", _i)]


class RowsStruct(C.Structure):
    """kore_paged_rows"""
    _fields_ = [("n_tok", _i), ("pos", _vp), ("slot", _vp), ("q_norm", _vp), ("k_norm", _vp), ("norm_eps", _f)]


class TreeStruct(C.Structure):
    """kore_paged_tree"""
    _fields_ = [("mask", _vp), ("mask_words", _i), ("pos", _vp)]


class KeepStruct(C.Structure):
    """kore_paged_keep"""
    _fields_ = [("n_seq", _i), ("n_tok", _i), ("q_start", _vp), ("n_keep", _vp), ("rows", _vp), ("kv_len", _vp), ("kv_out", _vp),
                ("pages", _vp), ("pages_stride", _i), ("free_pages", _vp), ("n_free", _vp), ("n_free_out", _vp)]


SYMBOLS = [
    ("kore_paged_create", _i, [C.POINTER(_vp), C.POINTER(PagedConfig)]),
    ("kore_paged_destroy", None, [_vp]),
    ("kore_paged_append_dev", _i, [_vp, _i, C.POINTER(BatchStruct), _i, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    ("kore_paged_attend_dev", _i, [_vp, _i, C.POINTER(BatchStruct), _i, _vp, _i64, _vp, _i64, _f, _i, _vp, _vp]),
    ("kore_paged_plan_dev", _i, [_vp, C.POINTER(PlanStruct), _vp]),
    ("kore_paged_append_rows_dev", _i, [_vp, _i, C.POINTER(RowsStruct), _i, _vp, _i64, _vp, _i64, _vp, _i64, _vp, _i64, _vp]),
    ("kore_paged_attend_tree_dev", _i, [_vp, _i, C.POINTER(BatchStruct), C.POINTER(TreeStruct), _i, _vp, _i64, _vp, _i64, _f, _i,
                                        _vp, _vp]),
    ("kore_paged_keep_dev", _i, [_vp, C.POINTER(KeepStruct), _vp]),
    ("kore_paged_workspace_bytes", C.c_size_t, [_vp]),
    ("kore_paged_get_info", _i, [_vp, C.POINTER(PagedInfo)]),
    ("kore_paged_sync", _i, [_vp]),
    ("kore_paged_last_error", C.c_char_p, [_vp]),
]

_done = False


def lib() -> C.CDLL:
    global _done
    L = _rope.lib()
    if not _done:
        for name, res, args in SYMBOLS:
            fn = getattr(L, name)
            fn.restype, fn.argtypes = res, args
        _done = True
    return L


class Batch:
    """The new rows of a step (kore_paged_batch): device pointers to int32 arrays q_start [n_seq + 1], kv_len [n_seq]
    and pages [n_seq][pages_stride].  max_q: the most new rows of a sequence, where it is known."""

    def __init__(self, n_seq: int, n_tok: int, q_start: int, kv_len: int, pages: int, pages_stride: int,
                 max_q: int = 0):
        self.struct = BatchStruct(n_seq, n_tok, q_start, kv_len, pages, pages_stride, max_q)
        self._ref = C.byref(self.struct)


class Plan:
    """The requests of a step and the tables that are made of them (kore_paged_plan): device pointers, int32 but for slot
    [n_tok] and mask [n_tok][mask_words], which are 64-bit.  kv_len and n_free_out may be kv_held and n_free; parent and mask
    go together (None: every sequence's rows one behind the other); window: of the masks, as the attention's."""

    def __init__(self, n_seq: int, n_tok: int, n_new: int, kv_held: int, kv_len: int, pages: int, pages_stride: int,
                 free_pages: int, n_free: int, n_free_out: int, q_start: int, pos: int, slot: int, status: int,
                 parent: int | None = None, mask: int | None = None, mask_words: int = 0, window: int = 0):
        self.struct = PlanStruct(n_seq, n_tok, n_new, kv_held, kv_len, pages, pages_stride, free_pages, n_free, n_free_out, parent,
                                 q_start, pos, slot, mask, mask_words, status, window)
        self._ref = C.byref(self.struct)


class Rows:
    """New rows by their own positions (int32) and slots (int64: page * page_size + slot), as a plan leaves them, and the
    weights of their heads' norms (kore_paged_rows)."""

    def __init__(self, n_tok: int, pos: int, slot: int, q_norm: int | None = None, k_norm: int | None = None,
                 norm_eps: float = 1e-6):
        self.struct = RowsStruct(n_tok, pos, slot, q_norm, k_norm, norm_eps)
        self._ref = C.byref(self.struct)


class Tree:
    """Which of its sequence's new rows a row attends (kore_paged_tree): mask [n_tok][mask_words] of 64 bits each; pos (int32
    [n_tok]) where there is a window."""

    def __init__(self, mask: int, mask_words: int = 1, pos: int | None = None):
        self.struct = TreeStruct(mask, mask_words, pos)
        self._ref = C.byref(self.struct)


class Keep:
    """What is kept of a step's rows (kore_paged_keep).  rows None: the first n_keep[s] of each sequence; the three of the free
    pages None: no page is given back."""

    def __init__(self, n_seq: int, n_tok: int, q_start: int, n_keep: int, kv_len: int, kv_out: int, pages: int, pages_stride: int,
                 rows: int | None = None, free_pages: int | None = None, n_free: int | None = None, n_free_out: int | None = None):
        self.struct = KeepStruct(n_seq, n_tok, q_start, n_keep, rows, kv_len, kv_out, pages, pages_stride, free_pages, n_free,
                                 n_free_out)
        self._ref = C.byref(self.struct)


class PagedKV:
    """kore_paged_t: a pool of pages on the current HIP device.  k_pool, v_pool: the caller's device memory of
    [n_layer][n_pages][n_head_kv][page_size][head_dim] elements each, or None (the handle allocates them).  rope:
    the rotation of append (None: rows are stored as given)."""

    def __init__(self, n_layer: int, n_pages: int, page_size: int, n_head: int, n_head_kv: int, head_dim: int,
                 cache_type: str = "f32", rope: Config | None = None, k_pool: int | None = None,
                 v_pool: int | None = None):
        self._h = None
        cfg = PagedConfig(n_layer, n_pages, page_size, n_head, n_head_kv, head_dim, type_code(cache_type),
                          rope.struct if rope is not None else RopeConfig(), k_pool, v_pool)
        h = _vp()
        rc = lib().kore_paged_create(C.byref(h), C.byref(cfg))
        if rc != KORE_PAGED_OK:
            raise PagedError(rc, lib().kore_paged_last_error(None).decode())
        self._h = h
        L = lib()
        self._plan, self._rows, self._tree, self._keep = (L.kore_paged_plan_dev, L.kore_paged_append_rows_dev,
                                                          L.kore_paged_attend_tree_dev, L.kore_paged_keep_dev)
        self.kv_dim, self.E = n_head_kv * head_dim, n_head * head_dim

    def _check(self, rc: int) -> None:
        if rc != KORE_PAGED_OK:
            raise PagedError(rc, lib().kore_paged_last_error(self._h).decode())

    @property
    def handle(self):
        return self._h

    def append_dev(self, layer: int, batch: Batch, dtype: str, k: int, v: int, q: int | None = None,
                   q_out: int | None = None, k_stride: int | None = None, v_stride: int | None = None,
                   q_stride: int | None = None, q_out_stride: int | None = None, stream=None) -> None:
        """Rotates and stores the batch's k and v rows, and rotates q into q_out where given."""
        self._check(lib().kore_paged_append_dev(
            self._h, layer, batch._ref, type_code(dtype), k, self.kv_dim if k_stride is None else k_stride, v,
            self.kv_dim if v_stride is None else v_stride, q, self.E if q_stride is None else q_stride, q_out,
            self.E if q_out_stride is None else q_out_stride, stream))

    def attend_dev(self, layer: int, batch: Batch, dtype: str, q: int, out: int, q_stride: int | None = None,
                   out_stride: int | None = None, scale: float = 0.0, window: int = 0, workspace: int | None = None,
                   stream=None) -> None:
        """Attention of the batch's (rotated) q rows over their sequences' pages into out."""
        self._check(lib().kore_paged_attend_dev(
            self._h, layer, batch._ref, type_code(dtype), q, self.E if q_stride is None else q_stride, out,
            self.E if out_stride is None else out_stride, scale, window, workspace, stream))

    def plan_dev(self, plan: Plan, stream=None) -> None:
        """Makes a step's tables of the requests' lengths, and takes the pages that it needs."""
        rc = self._plan(self._h, plan._ref, stream)
        if rc:
            self._check(rc)

    def append_rows_dev(self, layer: int, rows: Rows, dtype: str, k: int, v: int, q: int | None = None, q_out: int | None = None,
                        k_stride: int | None = None, v_stride: int | None = None, q_stride: int | None = None,
                        q_out_stride: int | None = None, stream=None) -> None:
        """append_dev by the rows' own positions and slots, with the norms of q's and k's heads."""
        rc = self._rows(self._h, layer, rows._ref, type_code(dtype), k, self.kv_dim if k_stride is None else k_stride, v,
                        self.kv_dim if v_stride is None else v_stride, q, self.E if q_stride is None else q_stride, q_out,
                        self.E if q_out_stride is None else q_out_stride, stream)
        if rc:
            self._check(rc)

    def attend_tree_dev(self, layer: int, batch: Batch, tree: Tree, dtype: str, q: int, out: int, q_stride: int | None = None,
                        out_stride: int | None = None, scale: float = 0.0, window: int = 0, workspace: int | None = None,
                        stream=None) -> None:
        """attend_dev for new rows that are a tree: each attends what its sequence held before, and the new ones of its mask."""
        rc = self._tree(self._h, layer, batch._ref, tree._ref, type_code(dtype), q, self.E if q_stride is None else q_stride, out,
                        self.E if out_stride is None else out_stride, scale, window, workspace, stream)
        if rc:
            self._check(rc)

    def keep_dev(self, keep: Keep, stream=None) -> None:
        """Moves the kept rows together in every layer, and gives back lengths and pages."""
        rc = self._keep(self._h, keep._ref, stream)
        if rc:
            self._check(rc)

    def workspace_bytes(self) -> int:
        return int(lib().kore_paged_workspace_bytes(self._h))

    def info(self) -> PagedInfo:
        inf = PagedInfo()
        self._check(lib().kore_paged_get_info(self._h, C.byref(inf)))
        return inf

    def sync(self) -> None:
        self._check(lib().kore_paged_sync(self._h))

    def close(self) -> None:
        if self._h:
            lib().kore_paged_destroy(self._h)
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
