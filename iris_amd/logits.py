"""Rows of logits to tokens, each request in its own way: penalties, biases and
masks, and the draw (include/iris_hip.h), on device pointers.

``TokenRule`` and ``Drawing`` are the requests' records, ``LogitsRules`` and
``LogitsDraw`` the header's structs of a call: a program fills one in once
(device addresses as integers, ``None`` for null) and passes it to each call.
``stream`` is a hipStream_t as an integer (0 or None: the null stream). Nothing
here synchronises; a refused call raises ``native.IrisError``.
"""
from __future__ import annotations

import ctypes as C
import math

from . import native

_P, _U, _I = C.c_void_p, C.c_uint32, C.c_int32

ONE = 1 << 16  # of Q16.16
CLOSED = -(1 << 31)  # the logit of a place that a mask closed


class TokenRule(C.Structure):
    """A request's penalties and biases (IrisTokenRule)."""
    _fields_ = [(n, _I) for n in ("repetition", "frequency", "presence")] + \
               [(n, _U) for n in ("window", "bias_start", "bias_count")]


class Drawing(C.Structure):
    """How a request draws (IrisDrawing)."""
    _fields_ = [("inverse_temperature", _I)] + [(n, _U) for n in ("top_k", "top_p", "max_gap")]


class LogitsRules(C.Structure):
    """Rules on rows of logits (IrisLogitsRules)."""
    _fields_ = [(n, _P) for n in ("logits", "out", "request", "rules", "history", "lengths", "row_start", "ids", "parents",
                                  "bias_ids", "bias_values", "masks", "mask_of", "status")] + \
               [(n, _U) for n in ("rows", "first_row", "vocab", "logits_stride", "out_stride", "requests",
                                  "history_stride", "biases", "mask_rows", "mask_stride")]


class LogitsDraw(C.Structure):
    """A token for each row of logits (IrisLogitsDraw)."""
    _fields_ = [(n, _P) for n in ("logits", "request", "drawings", "numbers", "tokens", "mass", "status")] + \
               [(n, _U) for n in ("rows", "vocab", "logits_stride", "requests")]


_calls = None


def _lib():
    global _calls
    if _calls is None:
        L, u64 = native.lib(), C.c_uint64
        rules, draw = C.POINTER(LogitsRules), C.POINTER(LogitsDraw)
        sig = {
            "iris_logits_rules": (C.c_int, [rules, _P]),
            "iris_logits_draw_workspace_bytes": (u64, [draw]),
            "iris_logits_draw": (C.c_int, [draw, _P, u64, _P]),
        }
        for name, (res, args) in sig.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _calls = L
    return _calls


def fixed(x: float) -> int:
    """A real number in Q16.16, ties to even (an import-time conversion)."""
    v = round(float(x) * ONE)
    if not -(1 << 31) <= v < 1 << 31:
        raise ValueError(f"{x} does not fit Q16.16")
    return v


def drawing(temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0, min_p: float = 0.0) -> Drawing:
    """The record of a temperature (0: the first maximum), top-k (0: all), top-p
    (1: all) and min-p (the least share of the first token's weight; 0: any)."""
    if not (temperature >= 0 and 0 < top_p <= 1 and 0 <= min_p <= 1 and 0 <= top_k < 1 << 32):
        raise ValueError("a temperature of at least 0, top_k of at least 0, top_p in (0, 1], min_p in [0, 1]")
    share = 0 if top_p == 1 else max(1, min(round(top_p * 2 ** 32), (1 << 32) - 1))
    # (0 would mean any gap: min_p of 1 keeps what rounds to the first's weight.)
    gap = max(1, round(-math.log(min_p) * ONE)) if min_p else 0
    # (Nor may a high temperature's inverse be 0, the first maximum.)
    inverse = max(1, round(min(1 / temperature * ONE, (1 << 31) - 1))) if temperature else 0
    return Drawing(inverse, top_k, share, gap)


def apply_rules(r: LogitsRules, stream=None):
    """Penalties, biases and masks on rows of logits."""
    native.check(_lib().iris_logits_rules(r, stream), "logits rules")


def draw_workspace_bytes(d: LogitsDraw) -> int:
    return _lib().iris_logits_draw_workspace_bytes(d)


def draw(d: LogitsDraw, workspace, workspace_bytes: int, stream=None):
    """A token for each row of logits."""
    native.check(_lib().iris_logits_draw(d, workspace, workspace_bytes, stream), "logits draw")
