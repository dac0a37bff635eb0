"""Low-rank adapters of many requests beside one product
(include/iris_hip.h, IrisAdapterBank).

An ``AdapterBank`` holds the adapters of one product; ``AdapterRows`` is the
header's struct of a call, filled in once with device addresses. ``stream`` is a
hipStream_t as an integer (0 or None: the null stream). ``apply`` does not
synchronise; a refused call raises ``native.IrisError``.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

from . import native

_P, _U = C.c_void_p, C.c_uint32

MAX_PARTS, MAX_RANK, MAX_WEIGHT, MAX_BITS = 3, 256, 32639, 40


class AdapterPart(C.Structure):
    """A product's part: output i is column first + i * step (IrisAdapterPart)."""
    _fields_ = [("rows", _U), ("first", _U), ("step", _U)]


class AdapterRows(C.Structure):
    """The rows of one call (IrisAdapterRows)."""
    _fields_ = [(n, _P) for n in ("x", "y", "out", "slots", "status")] + \
               [(n, _U) for n in ("x_stride", "y_stride", "out_stride", "rows")]


_calls = None


def _lib():
    global _calls
    if _calls is None:
        L, u64 = native.lib(), C.c_uint64
        sig = {
            "iris_adapters_create": (C.c_int, [_U, C.POINTER(AdapterPart), _U, _U, _U, C.POINTER(_P)]),
            "iris_adapters_free": (None, [_P]),
            "iris_adapters_device_bytes": (u64, [_P]),
            "iris_adapters_load": (C.c_int, [_P, _U, _U, _P, _U, _P, _U, _U]),
            "iris_adapters_workspace_bytes": (u64, [_P, _U]),
            "iris_adapters_apply": (C.c_int, [_P, C.POINTER(AdapterRows), _P, u64, _P]),
        }
        for name, (res, args) in sig.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        _calls = L
    return _calls


def to_fixed(weights: np.ndarray) -> tuple:
    """A matrix of real weights as 16-bit integers and the number of fraction
    bits, the most with which all of them fit: (integers, bits). Ties go to
    even. (An import-time conversion, on the host.)"""
    w = np.asarray(weights, dtype=np.float64)
    most = float(np.abs(w).max()) if w.size else 0.0
    if not math.isfinite(most) or most > MAX_WEIGHT:
        raise ValueError("an adapter's weights must be finite and at most 32639")
    # (Below 2^-MAX_BITS all have the most bits; the quotient of the smallest would be infinite.)
    bits = MAX_BITS if most < 2.0 ** -MAX_BITS else min(MAX_BITS, int(math.floor(math.log2(MAX_WEIGHT / most))))
    while np.rint(most * 2.0 ** bits) > MAX_WEIGHT:
        bits -= 1
    return np.rint(w * 2.0 ** bits).astype(np.int16), bits


class AdapterBank:
    """Up to ``slots`` adapters of rank up to ``max_rank`` beside one product of
    ``cols`` columns; ``parts`` are (rows, first output, step) each."""

    def __init__(self, cols: int, parts, slots: int, max_rank: int):
        self.cols, self.parts, self.slots, self.max_rank = cols, [tuple(p) for p in parts], slots, max_rank
        table = (AdapterPart * max(len(self.parts), 1))(*[AdapterPart(*p) for p in self.parts])
        h = _P()
        native.check(_lib().iris_adapters_create(cols, table, len(self.parts), slots, max_rank, C.byref(h)),
                     "adapter bank create")
        self._h = h

    @property
    def handle(self):
        return self._h

    def load(self, slot: int, part: int, a, a_bits: int = 0, b=None, b_bits: int = 0):
        """One part of an adapter: a [rank][cols] and b [rows][rank] (int16),
        weights a / 2^a_bits and b / 2^b_bits. ``a`` None empties the part.
        Waits for the device."""
        if a is None:
            native.check(_lib().iris_adapters_load(self._h, slot, part, None, 0, None, 0, 0), "adapter load")
            return
        if not 0 <= part < len(self.parts):
            raise native.IrisError(-1, "adapter load")
        a, b = np.asarray(a), np.asarray(b)
        if a.dtype != np.int16 or b.dtype != np.int16 or a.ndim != 2 or a.shape[1] != self.cols or \
                b.shape != (self.parts[part][0], a.shape[0]):
            raise ValueError(f"an adapter's part takes int16 [rank][{self.cols}] and [{self.parts[part][0]}][rank]")
        a, b = np.ascontiguousarray(a), np.ascontiguousarray(b)
        native.check(_lib().iris_adapters_load(self._h, slot, part, a.ctypes.data, a_bits, b.ctypes.data, b_bits, a.shape[0]),
                     "adapter load")

    def device_bytes(self) -> int:
        return _lib().iris_adapters_device_bytes(self._h)

    def workspace_bytes(self, rows: int) -> int:
        return _lib().iris_adapters_workspace_bytes(self._h, rows)

    def apply(self, a: AdapterRows, workspace, workspace_bytes: int, stream=None):
        """out = y + B (A x) for each row, by its slot's adapter."""
        native.check(_lib().iris_adapters_apply(self._h, a, workspace, workspace_bytes, stream), "adapters")

    def free(self):
        if getattr(self, "_h", None):
            _lib().iris_adapters_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
