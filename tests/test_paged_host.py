"""The paged-cache operators' argument checks (no GPU: a refused call runs
nothing), and their structs against the header's."""
import re

import pytest

from iris_amd import native, paged

A = 1 << 20  # an aligned address that nothing reads: every call here is refused


def cache(**kw):
    return paged.PagedKv(**{**dict(k=A, v=A, pages=4, page_size=16, kv_heads=2, head_dim=64), **kw})


def plan(**kw):
    return paged.PagedPlan(**{**dict(lengths=A, added=A, parents=None, held=A, held_out=A, table=A, ring=A, ring_state=A,
                                     ring_state_out=A, row_start=A, slots=A, positions=None, status=A, requests=3,
                                     table_stride=4, pages=8, page_size=16, max_rows=9), **kw})


def packed(**kw):
    return paged.PackedAttention(**{**dict(q=A, k=A, v=A, out=A, row_start=A, status=None, q_stride=256, k_stride=128,
                                           v_stride=128, out_stride=256, sequences=2, rows=9, max_length=9, heads=4,
                                           kv_heads=2, head_dim=64, window=0, scaled=1, scale_q32=1 << 29), **kw})


def tree(**kw):
    return paged.TreeAttention(**{**dict(q=A, out=A, row_start=A, lengths=A, parents=None, table=A, status=None,
                                         q_stride=256, out_stride=256, requests=2, rows=9, table_stride=4, max_nodes=5,
                                         max_positions=64, heads=4, window=0, scaled=1, scale_q32=1 << 29), **kw})


def refused(call, code):
    with pytest.raises(native.IrisError) as e:
        call()
    assert e.value.code == code


@pytest.mark.parametrize("kw, code", [
    (dict(lengths=None), -1), (dict(added=None), -1), (dict(held=None), -1), (dict(held_out=None), -1),
    (dict(table=None), -1), (dict(ring=None), -1), (dict(ring_state=None), -1), (dict(ring_state_out=None), -1),
    (dict(row_start=None), -1), (dict(slots=None), -1), (dict(status=None), -1), (dict(requests=0), -1),
    (dict(table_stride=0), -1), (dict(pages=0), -1), (dict(page_size=0), -1), (dict(page_size=2), -1),
    (dict(page_size=24), -1), (dict(page_size=2048), -1), (dict(requests=4097), -5), (dict(pages=1 << 27), -5),
    (dict(table_stride=1 << 27), -5), (dict(max_rows=1 << 31), -5)])
def test_plan_refusals(kw, code):
    refused(lambda: paged.plan(plan(**kw)), code)


BAD_CACHES = [(dict(k=None), -1), (dict(v=None), -1), (dict(k=A + 4), -1), (dict(v=A + 8), -1), (dict(pages=0), -1),
              (dict(page_size=3), -1), (dict(page_size=2048), -1), (dict(kv_heads=0), -1), (dict(head_dim=0), -1),
              (dict(head_dim=66), -1), (dict(head_dim=516), -1), (dict(pages=1 << 27), -5)]


@pytest.mark.parametrize("kw, code", BAD_CACHES)
def test_cache_refusals(kw, code):
    refused(lambda: paged.store(cache(**kw), A, 128, A, 128, A, 1), code)
    refused(lambda: paged.attend_tree(cache(**kw), tree(), A, 1 << 40), code)
    assert paged.tree_workspace_bytes(cache(**kw), tree()) == 0


@pytest.mark.parametrize("args", [(None, 128, A, 128, A), (A, 128, None, 128, A), (A, 128, A, 128, None),
                                  (A + 4, 128, A, 128, A), (A, 128, A + 4, 128, A), (A, 130, A, 128, A),
                                  (A, 128, A, 130, A), (A, 124, A, 128, A), (A, 128, A, 124, A)])
def test_store_refusals(args):
    refused(lambda: paged.store(cache(), *args, 3), -1)


def test_store_of_too_many_rows():
    refused(lambda: paged.store(cache(), A, 128, A, 128, A, 1 << 24), -5)
    paged.store(cache(), A, 128, A, 128, A, 0)


@pytest.mark.parametrize("kw, code", [
    (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1), (dict(row_start=None), -1),
    (dict(q=A + 4), -1), (dict(k=A + 4), -1), (dict(v=A + 4), -1), (dict(out=A + 4), -1), (dict(q_stride=258), -1),
    (dict(k_stride=130), -1), (dict(v_stride=130), -1), (dict(out_stride=258), -1), (dict(q_stride=252), -1),
    (dict(k_stride=124), -1), (dict(v_stride=124), -1), (dict(out_stride=252), -1), (dict(heads=0), -1),
    (dict(kv_heads=0), -1), (dict(heads=3), -1), (dict(head_dim=0), -1), (dict(head_dim=66), -1),
    (dict(head_dim=516, q_stride=4096, k_stride=4096, v_stride=4096, out_stride=4096), -1), (dict(max_length=0), -1),
    (dict(max_length=65536), -5), (dict(rows=1 << 31), -5), (dict(rows=(1 << 24) + 1), -5),
    (dict(rows=1 << 20, heads=64, kv_heads=64, q_stride=4096, k_stride=4096, v_stride=4096, out_stride=4096), -5)])
def test_packed_refusals(kw, code):
    refused(lambda: paged.attend_packed(packed(**kw), A, 1 << 40), code)
    assert paged.packed_workspace_bytes(packed(**kw)) == 0


def test_packed_workspace():
    size = paged.packed_workspace_bytes(packed())
    assert size > 0
    refused(lambda: paged.attend_packed(packed(), A, size - 1), -5)
    refused(lambda: paged.attend_packed(packed(), None, size), -1)
    refused(lambda: paged.attend_packed(packed(), A + 4, size), -1)
    # Nothing to do: nothing runs.
    paged.attend_packed(packed(rows=0), None, 0)
    paged.attend_packed(packed(sequences=0), None, 0)


@pytest.mark.parametrize("kw, code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(row_start=None), -1), (dict(lengths=None), -1),
    (dict(table=None), -1), (dict(q=A + 4), -1), (dict(out=A + 4), -1), (dict(q_stride=258), -1),
    (dict(out_stride=258), -1), (dict(q_stride=252), -1), (dict(out_stride=252), -1), (dict(heads=0), -1),
    (dict(heads=3), -1), (dict(table_stride=0), -1), (dict(max_nodes=0), -1), (dict(max_positions=0), -1),
    (dict(max_nodes=65), -5), (dict(max_positions=(1 << 20) + 1), -5), (dict(rows=1 << 31), -5),
    (dict(requests=65536), -5), (dict(heads=2050, max_nodes=64, q_stride=1 << 18, out_stride=1 << 18), -5)])
def test_tree_refusals(kw, code):
    refused(lambda: paged.attend_tree(cache(), tree(**kw), A, 1 << 40), code)
    assert paged.tree_workspace_bytes(cache(), tree(**kw)) == 0


def test_tree_workspace():
    size = paged.tree_workspace_bytes(cache(), tree())
    if size:
        refused(lambda: paged.attend_tree(cache(), tree(), A, size - 1), -5)
        refused(lambda: paged.attend_tree(cache(), tree(), None, size), -1)
        refused(lambda: paged.attend_tree(cache(), tree(), A + 4, size), -1)
    paged.attend_tree(cache(), tree(rows=0), None, 0)
    paged.attend_tree(cache(), tree(requests=0), None, 0)


@pytest.mark.parametrize("kw", [{}, dict(requests=1, rows=1, max_nodes=1, max_positions=1), dict(window=5),
                                dict(requests=64, max_positions=9000, table_stride=600),
                                dict(heads=32, q_stride=2048, out_stride=2048, max_nodes=64, rows=128)])
def test_tree_workspace_of_a_valid_call_is_checked(kw):
    size = paged.tree_workspace_bytes(cache(), tree(**kw))
    assert size > 0
    refused(lambda: paged.attend_tree(cache(), tree(**kw), A, size - 1), -5)
    refused(lambda: paged.attend_tree(cache(), tree(**kw), None, size), -1)
    refused(lambda: paged.attend_tree(cache(), tree(**kw), A + 4, size), -1)


C_TYPES = {paged._P: "*", paged._U: "uint32_t", paged._I: "int32_t"}


@pytest.mark.parametrize("name", ["PagedKv", "PagedPlan", "PackedAttention", "TreeAttention"])
def test_structs_match_the_header(name):
    text = re.sub(r"/\*.*?\*/", "", open(native.HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct Iris%s \{(.*?)\} Iris%s;" % (name, name), text, flags=re.S).group(1)
    want = []
    for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
        m = re.match(r"((?:const )?\w+\*?) (.*)", decl)
        want += [(n.strip(), "*" if "*" in m.group(1) else m.group(1)) for n in m.group(2).split(",")]
    assert [(n, C_TYPES[t]) for n, t in getattr(paged, name)._fields_] == want


@pytest.mark.parametrize("name", ["IrisPagedKv", "IrisPagedPlan", "IrisPackedAttention", "IrisTreeAttention"])
def test_rust_structs_match_the_header(name):
    import os
    ffi = os.path.join(os.path.dirname(os.path.dirname(native.HEADER)), "crates", "iris-hip", "src", "ffi.rs")
    text = re.sub(r"/\*.*?\*/", "", open(native.HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    rust = {"const int32_t*": "*const i32", "int32_t*": "*mut i32", "uint32_t": "u32", "int32_t": "i32"}
    want = []
    for decl in filter(None, (" ".join(d.split()) for d in body.split(";"))):
        m = re.match(r"((?:const )?\w+\*?) (.*)", decl)
        want += [(n.strip(), rust[m.group(1)]) for n in m.group(2).split(",")]
    body = re.search(r"pub struct %s \{(.*?)\n\}" % name, open(ffi).read(), flags=re.S).group(1)
    assert re.findall(r"pub (\w+): ([^,]+),", body) == want


def test_batch_refuses_null_handles():
    import ctypes as C
    from iris_amd import direct
    L, h, n = direct._declare(), C.c_void_p(), C.c_uint32()
    assert L.iris_batch_create(None, 1, 1, 16, 16, 16, C.byref(h)) == -1
    assert L.iris_batch_prefill(None, A, A, A) == -1
    assert L.iris_batch_step(None, A, None, A, A, A) == -1
    assert L.iris_batch_release(None, 0) == -1
    assert L.iris_batch_length(None, 0, C.byref(n)) == -1
    L.iris_batch_free(None)


def test_ids_refused_refuses_null_handles():
    import ctypes as C
    from iris_amd import direct
    assert direct._declare().iris_model_ids_refused(None, A, 1, C.byref(C.c_uint32())) == -1
