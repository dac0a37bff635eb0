"""Several requests over one paged cache of keys and values: the operators of
a pass (include/iris_hip.h), on device pointers.

``PagedKv``, ``PagedPlan``, ``PackedAttention`` and ``TreeAttention`` are the
header's structs: a program fills one in once (device addresses as integers,
``None`` for null) and passes it to each call. ``stream`` is a hipStream_t as
an integer (0 or None: the null stream). Nothing here synchronises; a refused
call raises ``native.IrisError``.
"""
from __future__ import annotations

import ctypes as C

from . import native

_P, _U, _I = C.c_void_p, C.c_uint32, C.c_int32


class PagedKv(C.Structure):
    """Key and value pages of one layer (IrisPagedKv)."""
    _fields_ = [("k", _P), ("v", _P), ("pages", _U), ("page_size", _U), ("kv_heads", _U), ("head_dim", _U)]


class PagedPlan(C.Structure):
    """The block tables and slot map of a pass (IrisPagedPlan)."""
    _fields_ = [(n, _P) for n in ("lengths", "added", "parents", "held", "held_out", "table", "ring", "ring_state",
                                  "ring_state_out", "row_start", "slots", "positions", "status")] + \
               [(n, _U) for n in ("requests", "table_stride", "pages", "page_size", "max_rows")]


class PackedAttention(C.Structure):
    """Causal attention over packed prompts (IrisPackedAttention)."""
    _fields_ = [(n, _P) for n in ("q", "k", "v", "out", "row_start", "status")] + \
               [(n, _U) for n in ("q_stride", "k_stride", "v_stride", "out_stride", "sequences", "rows", "max_length",
                                  "heads", "kv_heads", "head_dim", "window")] + [("scaled", _I), ("scale_q32", _U)]


class TreeAttention(C.Structure):
    """Attention of drafted trees over the cache (IrisTreeAttention)."""
    _fields_ = [(n, _P) for n in ("q", "out", "row_start", "lengths", "parents", "table", "status")] + \
               [(n, _U) for n in ("q_stride", "out_stride", "requests", "rows", "table_stride", "max_nodes",
                                  "max_positions", "heads", "window")] + [("scaled", _I), ("scale_q32", _U)]


_calls = None


def _lib():
    global _calls
    if _calls is None:
        L, u64 = native.lib(), C.c_uint64
        kv, plan, packed, tree = (C.POINTER(t) for t in (PagedKv, PagedPlan, PackedAttention, TreeAttention))
        sig = {
            "iris_paged_plan": (C.c_int, [plan, _P]),
            "iris_paged_store": (C.c_int, [kv, _P, _U, _P, _U, _P, _U, _P]),
            "iris_attention_packed_workspace_bytes": (u64, [packed]),
            "iris_attention_packed": (C.c_int, [packed, _P, u64, _P]),
            "iris_attention_tree_workspace_bytes": (u64, [kv, tree]),
            "iris_attention_tree": (C.c_int, [kv, tree, _P, u64, _P]),
        }
        for name, (res, args) in sig.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _calls = L
    return _calls


def plan(p: PagedPlan, stream=None):
    """Builds a pass's block tables, slot map, row starts and positions."""
    native.check(_lib().iris_paged_plan(p, stream), "paged plan")


def store(cache: PagedKv, k, k_stride: int, v, v_stride: int, slots, rows: int, stream=None):
    """Writes ``rows`` rows of keys and values to their slots."""
    native.check(_lib().iris_paged_store(cache, k, k_stride, v, v_stride, slots, rows, stream), "paged store")


def packed_workspace_bytes(a: PackedAttention) -> int:
    return _lib().iris_attention_packed_workspace_bytes(a)


def attend_packed(a: PackedAttention, workspace, workspace_bytes: int, stream=None):
    """Causal attention over whole prompts packed row after row."""
    native.check(_lib().iris_attention_packed(a, workspace, workspace_bytes, stream), "packed attention")


def tree_workspace_bytes(cache: PagedKv, a: TreeAttention) -> int:
    return _lib().iris_attention_tree_workspace_bytes(cache, a)


def attend_tree(cache: PagedKv, a: TreeAttention, workspace, workspace_bytes: int, stream=None):
    """Attention of each request's newest rows over the paged cache."""
    native.check(_lib().iris_attention_tree(cache, a, workspace, workspace_bytes, stream), "tree attention")
