"""Adapters, rules and draws: argument checks (no GPU: a refused call runs
nothing), structs against the header's, and the conversions of real numbers."""
import ctypes as C
import math
import os
import re

import numpy as np
import pytest

from iris_amd import adapters, logits, native
from tests import requests_reference as ref

A = 1 << 20  # an aligned address that nothing reads: every call here is refused


def refused(call, code):
    with pytest.raises(native.IrisError) as e:
        call()
    assert e.value.code == code


def rules(**kw):
    return logits.LogitsRules(**{**dict(logits=A, out=2 * A, request=A, rules=A, history=A, lengths=A, row_start=None, ids=None,
                                        parents=None, bias_ids=None, bias_values=None, masks=None, mask_of=None, status=None,
                                        rows=3, first_row=0, vocab=100, logits_stride=100, out_stride=100, requests=2,
                                        history_stride=64, biases=0, mask_rows=0, mask_stride=0), **kw})


def drawing(**kw):
    return logits.LogitsDraw(**{**dict(logits=A, request=A, drawings=A, numbers=A, tokens=A, mass=None, status=None, rows=3,
                                       vocab=100, logits_stride=100, requests=2), **kw})


@pytest.mark.parametrize("kw, code", [
    (dict(logits=None), -1), (dict(out=None), -1), (dict(vocab=0), -1), (dict(logits_stride=99), -1), (dict(out_stride=99), -1),
    (dict(out=A, out_stride=128), -1), (dict(request=None), -1), (dict(requests=0), -1), (dict(lengths=None), -1),
    (dict(ids=A), -1), (dict(biases=3), -1), (dict(biases=3, bias_ids=A), -1), (dict(mask_rows=1, mask_stride=4), -1),
    (dict(mask_rows=1, masks=A, mask_stride=4), -1), (dict(mask_rows=1, masks=A, mask_of=A, mask_stride=3), -1),
    (dict(vocab=(1 << 20) + 1, logits_stride=1 << 21, out_stride=1 << 21), -5), (dict(rows=65536), -5),
    (dict(requests=1 << 31), -5), (dict(history_stride=(1 << 20) + 1), -5),
    (dict(biases=(1 << 20) + 1, bias_ids=A, bias_values=A), -5), (dict(first_row=0x7fffffff), -5),
    (dict(mask_rows=1 << 31, masks=A, mask_of=A, mask_stride=4), -5)])
def test_rules_refusals(kw, code):
    refused(lambda: logits.apply_rules(rules(**kw)), code)


@pytest.mark.parametrize("kw, code", [
    (dict(logits=None), -1), (dict(tokens=None), -1), (dict(vocab=0), -1), (dict(logits_stride=99), -1),
    (dict(numbers=None), -1), (dict(requests=0), -1), (dict(vocab=(1 << 20) + 1, logits_stride=1 << 21), -5),
    (dict(rows=65536), -5), (dict(requests=1 << 31), -5)])
def test_draw_refusals(kw, code):
    refused(lambda: logits.draw(drawing(**kw), A, 1 << 40), code)
    assert logits.draw_workspace_bytes(drawing(**kw)) == 0


@pytest.mark.parametrize("kw", [{}, dict(drawings=None, numbers=None), dict(request=None), dict(vocab=1, logits_stride=1),
                                dict(vocab=1 << 20, logits_stride=1 << 20, rows=65535)])
def test_draw_workspace_of_a_valid_call_is_checked(kw):
    size = logits.draw_workspace_bytes(drawing(**kw))
    assert size > 0
    refused(lambda: logits.draw(drawing(**kw), A, size - 1), -5)
    refused(lambda: logits.draw(drawing(**kw), None, size), -1)
    refused(lambda: logits.draw(drawing(**kw), A + 4, size), -1)


def test_no_rows_is_no_work():
    logits.apply_rules(rules(rows=0))
    logits.draw(drawing(rows=0), None, 0)


def test_null_structs_are_refused():
    L, n = logits._lib(), C.c_uint64(0)
    assert L.iris_logits_rules(None, None) == -1
    assert L.iris_logits_draw(None, A, n, None) == -1
    assert L.iris_logits_draw_workspace_bytes(None) == 0
    M, h = adapters._lib(), C.c_void_p()
    assert M.iris_adapters_create(64, None, 1, 1, 1, C.byref(h)) == -1
    assert M.iris_adapters_load(None, 0, 0, A, 0, A, 0, 1) == -1
    assert M.iris_adapters_apply(None, None, A, n, None) == -1
    assert M.iris_adapters_workspace_bytes(None, 5) == 0 and M.iris_adapters_device_bytes(None) == 0
    M.iris_adapters_free(None)


@pytest.mark.parametrize("cols, parts, slots, rank, code", [
    (0, [(4, 0, 1)], 1, 1, -1), (48, [(4, 0, 1)], 1, 1, -1), (64, [], 1, 1, -1), (64, [(4, 0, 1)] * 4, 1, 1, -1),
    (64, [(4, 0, 1)], 0, 1, -1), (64, [(4, 0, 1)], 1, 0, -1), (64, [(0, 0, 1)], 1, 1, -1), (64, [(4, 0, 0)], 1, 1, -1),
    (65536, [(4, 0, 1)], 1, 1, -5), (64, [(4, 0, 1)], 65536, 1, -5), (64, [(4, 0, 1)], 1, 257, -5),
    (64, [(4, 1 << 24, 1)], 1, 1, -5), (64, [(1 << 24, 0, 2)], 1, 1, -5),
    (64, [(4, 0, 1), (4, 3, 1)], 1, 1, -1), (64, [(4, 0, 2), (9, 1, 3)], 1, 1, -1), (64, [(3, 8, 1), (1, 10, 1)], 1, 1, -1)])
def test_bank_refusals(cols, parts, slots, rank, code):
    refused(lambda: adapters.AdapterBank(cols, parts, slots, rank), code)


TYPES = {C.c_void_p: "*", C.c_uint32: "uint32_t", C.c_int32: "int32_t"}
RUST = {"const int32_t*": "*const i32", "int32_t*": "*mut i32", "uint32_t": "u32", "int32_t": "i32",
        "const uint32_t*": "*const u32", "int64_t*": "*mut i64", "const IrisTokenRule*": "*const IrisTokenRule",
        "const IrisDrawing*": "*const IrisDrawing"}


@pytest.mark.parametrize("module, name", [(adapters, "AdapterPart"), (adapters, "AdapterRows"), (logits, "TokenRule"),
                                          (logits, "LogitsRules"), (logits, "Drawing"), (logits, "LogitsDraw")])
def test_structs_match_the_header(module, name):
    text = re.sub(r"/\*.*?\*/", "", open(native.HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct Iris%s \{(.*?)\} Iris%s;" % (name, name), text, flags=re.S).group(1)
    want = []
    for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
        m = re.match(r"((?:const )?\w+\*?) (.*)", decl)
        want += [(n.strip(), m.group(1)) for n in m.group(2).split(",")]
    assert [(n, TYPES[t]) for n, t in getattr(module, name)._fields_] == [(n, "*" if "*" in t else t) for n, t in want]
    ffi = os.path.join(os.path.dirname(os.path.dirname(native.HEADER)), "crates", "iris-hip", "src", "ffi.rs")
    body = re.search(r"pub struct Iris%s \{(.*?)\n\}" % name, open(ffi).read(), flags=re.S).group(1)
    assert re.findall(r"pub (\w+): ([^,]+),", body) == [(n, RUST[t]) for n, t in want]


def test_bounds_match_the_header():
    text = open(native.HEADER).read()
    for name, value in (("PARTS", adapters.MAX_PARTS), ("RANK", adapters.MAX_RANK), ("WEIGHT", adapters.MAX_WEIGHT),
                        ("BITS", adapters.MAX_BITS)):
        assert re.search(r"#define IRIS_ADAPTER_%s %d\n" % (name, value), text)


@pytest.mark.parametrize("scale", [1e-6, 0.003, 0.4, 0.9999, 1.0, 17.3, 32639.0])
def test_weights_to_fixed(scale):
    rng = np.random.default_rng(4)
    w = rng.uniform(-1, 1, (7, 33)) * scale
    w[0, 0] = scale
    q, bits = adapters.to_fixed(w)
    assert q.dtype == np.int16 and np.abs(q.astype(int)).max() <= adapters.MAX_WEIGHT and 0 <= bits <= adapters.MAX_BITS
    # Half a step of the last bit.
    assert np.abs(q / 2.0 ** bits - w).max() <= 0.5 / 2 ** bits
    # One bit more would not fit.
    assert bits == adapters.MAX_BITS or np.rint(scale * 2.0 ** (bits + 1)) > adapters.MAX_WEIGHT


def test_weights_to_fixed_edges():
    q, bits = adapters.to_fixed(np.zeros((2, 3)))
    assert not q.any() and bits == adapters.MAX_BITS
    for bad in (np.inf, np.nan, 32640.0):
        with pytest.raises(ValueError):
            adapters.to_fixed(np.array([[bad]]))


def test_drawing_records():
    d = logits.drawing(0.5, 40, 0.95, 0.05)
    assert (d.inverse_temperature, d.top_k, d.top_p) == (1 << 17, 40, round(0.95 * 2 ** 32))
    assert d.max_gap == round(-math.log(0.05) * 65536)
    d = logits.drawing()
    assert (d.inverse_temperature, d.top_k, d.top_p, d.max_gap) == (65536, 0, 0, 0)
    assert logits.drawing(0).inverse_temperature == 0
    # Neither end of the temperatures turns into the first maximum.
    assert logits.drawing(1e9).inverse_temperature == 1
    assert logits.drawing(1e-9).inverse_temperature == (1 << 31) - 1
    assert logits.drawing(top_p=1e-12).top_p == 1 and logits.drawing(min_p=1.0).max_gap == 1
    for bad in (dict(temperature=-1), dict(top_p=0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=2), dict(top_k=-1),
                dict(temperature=math.nan)):
        with pytest.raises(ValueError):
            logits.drawing(**bad)
    assert logits.fixed(1.5) == 98304
    with pytest.raises(ValueError):
        logits.fixed(32768)


def test_reference_draw():
    # Two tokens of equal weight: the lower index takes the lower half of the numbers.
    l = np.array([5, 9, 9, ref.LOWEST], np.int32) * 1
    one = 1 << 32
    far = (1 << 16, 2, 0, 0)
    assert ref.draw(l, far, 0) == (1, one, 2 * one) and ref.draw(l, far, (1 << 31) - 1) == (1, one, 2 * one)
    assert ref.draw(l, far, 1 << 31)[0] == 2 and ref.draw(l, None, 7) == (1, one, one)
    assert ref.draw(np.full(3, ref.LOWEST, np.int32), far, 5) == (-1, 0, 0)


@pytest.mark.parametrize("scale", [5e-324, 1e-310, 1e-300, 1e-20, 2.0 ** -41, 2.0 ** -40, 2.0 ** -26, 2.0 ** -25])
def test_tiny_weights_to_fixed(scale):
    # The smallest overflowed in the number of bits.
    w = np.array([[scale, -scale, 0.0]])
    q, bits = adapters.to_fixed(w)
    assert bits == (adapters.MAX_BITS if scale < 2.0 ** -25 else 39)
    assert np.array_equal(q, np.rint(w * 2.0 ** bits))
