"""GPU: block tables and slot maps (iris_paged_plan) and the store of rows into
their pages (iris_paged_store), against plain implementations."""
import random

import numpy as np
import pytest
import torch

from iris_amd import native, paged
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


def dev(a):
    return torch.tensor(np.asarray(a, dtype=np.int32), device="cuda")


class Plan:
    """A plan's device arrays; `in_place` writes held and ring_state over."""

    def __init__(self, lengths, added, held, table, ring, ring_state, pages, page, max_rows, parents=None,
                 in_place=False, positions=True):
        n, stride = table.shape
        self.t = dict(lengths=dev(lengths), added=dev(added), held=dev(held), table=dev(table), ring=dev(ring),
                      ring_state=dev(ring_state), row_start=dev([7] * (n + 1)), slots=dev([7] * max(max_rows, 1)),
                      status=dev([7]))
        self.t["held_out"] = self.t["held"] if in_place else dev([7] * n)
        self.t["ring_state_out"] = self.t["ring_state"] if in_place else dev([7, 7])
        if positions:
            self.t["positions"] = dev([7] * max(max_rows, 1))
        if parents is not None:
            self.t["parents"] = dev(list(parents) or [0])
        self.d = paged.PagedPlan(**{k: v.data_ptr() for k, v in self.t.items()}, requests=n, table_stride=stride,
                                 pages=pages, page_size=page, max_rows=max_rows)

    def run(self, stream=None):
        paged.plan(self.d, stream)

    def got(self):
        torch.cuda.synchronize()
        names = ("table", "held_out", "ring", "ring_state_out", "row_start", "slots", "positions", "status")
        return [self.t[x].cpu().numpy() for x in names if x in self.t]


def state(rng, requests, page, longest, rows, spare=5):
    """Random lengths, rows to add, pages held (some requests done, some with
    pages to return) and a ring that wraps around."""
    lengths = [rng.choice([0, 1, page, rng.randrange(longest + 1)]) for _ in range(requests)]
    held = [-(-x // page) + rng.choice([0, 0, 0, 2]) for x in lengths]
    added = [0] * requests
    for _ in range(rows):
        added[rng.randrange(requests)] += 1
    for i in range(0, requests, 5):
        lengths[i] = 0
    need = [-(-(x + a) // page) for x, a in zip(lengths, added)]
    pages = sum(max(a, b) for a, b in zip(need, held)) + spare
    order = list(range(pages))
    rng.shuffle(order)
    table, at = np.full((requests, max(max(need), max(held)) + 2), -1, np.int32), 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    head, ring = rng.randrange(pages), [-1] * pages
    for i, p in enumerate(order[at:]):
        ring[(head + i) % pages] = p
    return lengths, added, held, table, ring, [head, pages - at], pages


def check(plan, want):
    got = plan.got()
    names = ["table", "held", "ring", "ring_state", "row_start", "slots", "positions", "status"]
    if len(got) == 7:
        want, names = want[:6] + want[7:], names[:6] + names[7:]
    for name, g, w in zip(names, got, want):
        assert np.array_equal(g.reshape(np.shape(w)), w), name


@pytest.mark.parametrize("requests, page, longest, rows, tail", [
    (1, 16, 40, 1, 0), (1, 4, 0, 1, 3), (3, 8, 30, 0, 4), (8, 16, 300, 8, 0), (17, 4, 50, 200, 11),
    (64, 128, 900, 64, 1), (257, 16, 100, 3000, 0), (300, 16, 200, 9001, 70), (1000, 32, 64, 5000, 0),
    (4096, 8, 20, 20011, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(requests, page, longest, rows, tail, in_place):
    rng = random.Random(requests * 31 + rows)
    lengths, added, held, table, ring, rs, pages = state(rng, requests, page, longest, rows)
    p = Plan(lengths, added, held, table, ring, rs, pages, page, rows + tail, in_place=in_place)
    p.run()
    check(p, ref.plan(lengths, added, None, held, table, ring, rs, pages, page, rows + tail))


@pytest.mark.parametrize("requests, most", [(1, 1), (5, 64), (70, 20), (400, 33)])
def test_plan_positions_of_trees(requests, most):
    rng = random.Random(requests)
    lengths, _, held, table, ring, rs, pages = state(rng, requests, 16, 100, 0, spare=64 * requests)
    table = np.concatenate([table, np.full((requests, 6), -1, np.int32)], axis=1)
    added = [rng.randrange(0, most + 1) for _ in range(requests)]
    added[0] = most
    # chains, bushes, several roots, and values that name no earlier row
    parents = [rng.choice([i - 1, max(0, i - 7), -1, -5, i, 99, rng.randrange(i) if i else -1]) for a in added
               for i in range(a)]
    p = Plan(lengths, added, held, table, ring, rs, pages, 16, sum(added) + 2, parents=parents)
    p.run()
    check(p, ref.plan(lengths, added, parents, held, table, ring, rs, pages, 16, sum(added) + 2))


def test_plan_of_a_deep_chain_and_no_positions():
    p = Plan([5], [64], [1], np.array([[3, -1, -1, -1, -1, -1]]), [9, 8, 7, 6, 5, 4, 2, 1, 0, -1], [0, 9], 10, 16, 64,
             parents=list(range(-1, 63)))
    p.run()
    assert np.array_equal(p.got()[6], np.arange(5, 69))
    q = Plan([5], [64], [1], np.array([[3, -1, -1, -1, -1, -1]]), [9, 8, 7, 6, 5, 4, 2, 1, 0, -1], [0, 9], 10, 16, 64,
             positions=False)
    q.run()
    for a, b in zip(p.got()[:6], q.got()[:6]):
        assert np.array_equal(a, b)


def test_plan_all_pages_return_and_are_taken_again():
    rng = random.Random(3)
    lengths, added, held, table, ring, rs, pages = state(rng, 9, 8, 100, 60)
    p = Plan(lengths, added, held, table, ring, rs, pages, 8, 60, in_place=True)
    p.run()
    p.t["lengths"].zero_()
    p.t["added"].zero_()
    p.run()
    _, held_now, ring_now, state_now, starts, slots, _, status = p.got()
    assert status[0] == 0 and not held_now.any() and state_now[1] == pages and not starts.any() and (slots == -1).all()
    assert sorted(ring_now) == list(range(pages))


@pytest.mark.parametrize("change, code", [
    (dict(max_rows=5), -5), (dict(ring_state=[0, 0]), -5), (dict(lengths=[-1, 3]), -1), (dict(added=[-2, 30]), -1),
    (dict(held=[-1, 1]), -1), (dict(held=[99, 1]), -1), (dict(held=[0, 1]), -1), (dict(added=[500, 3]), -5),
    (dict(ring_state=[-1, 4]), -1), (dict(ring_state=[0, 99]), -1), (dict(ring_state=[8, 4]), -1),
    (dict(added=[2 ** 31 - 1, 2 ** 31 - 1], max_rows=2 ** 31 - 1), None), (dict(lengths=[2 ** 31 - 1, 0]), -1),
    (dict(added=[0, 30], held=[4, 1], ring_state=[0, 8]), -1)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_that_cannot_be(change, code, in_place):
    s = dict(lengths=[17, 3], added=[20, 14], held=[2, 1], ring_state=[0, 4], max_rows=40)
    s.update(change)
    table = np.array([[6, 5, -1, -1], [7, -1, -1, -1]], np.int32)
    ring = [0, 1, 2, 3, -1, -1, -1, -1]
    max_rows = min(s["max_rows"], 40)
    p = Plan(s["lengths"], s["added"], s["held"], table, ring, s["ring_state"], 8, 16, max_rows, in_place=in_place)
    p.run()
    want = ref.plan(s["lengths"], s["added"], None, s["held"], table, ring, s["ring_state"], 8, 16, max_rows)
    assert want[-1] == (code if code is not None else -5)
    check(p, want)


def test_plan_with_a_bad_page_gives_no_slot():
    p = Plan([3, 4], [2, 1], [1, 1], np.array([[8, 0], [-3, 0]]), [1, 2, 3, 4, 5, 6, 7, 0], [0, 8], 8, 16, 3)
    p.run()
    assert np.array_equal(p.got()[5], [-1, -1, -1]) and np.array_equal(p.got()[6], [3, 4, 4])


def test_plan_captured_and_replayed():
    # In place, several workgroups: each replay grows every request by a row.
    rng = random.Random(11)
    n, page = 64, 4
    held = [1] * n
    table = np.full((n, 40), -1, np.int32)
    table[:, 0] = np.arange(n)
    pages = n * 40
    ring = list(range(n, pages)) + [-1] * n
    lengths, added = [rng.randrange(5) for _ in range(n)], [rng.randrange(1, 12) for _ in range(n)]
    p = Plan(lengths, added, held, table, ring, [0, pages - n], pages, page, 8192, in_place=True)
    want = (table, held, ring, [0, pages - n])
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        p.run(torch.cuda.current_stream().cuda_stream)
        p.t["lengths"].add_(p.t["added"])
    for _ in range(4):
        out = ref.plan(lengths, added, None, want[1], want[0], want[2], want[3], pages, page, 8192)
        g.replay()
        check(p, out)
        lengths = [x + a for x, a in zip(lengths, added)]
        want = out[:4]


# ------------------------------------------------------------------ store


@pytest.mark.parametrize("rows, kv_heads, hd, page, extra", [
    (1, 1, 4, 4, 0), (3, 2, 64, 16, 0), (8, 8, 128, 16, 4), (70, 1, 256, 64, 8), (33, 3, 80, 8, 12), (9, 2, 512, 1024, 0),
    (257, 5, 20, 32, 4)])
def test_store(rows, kv_heads, hd, page, extra):
    g = torch.Generator(device="cuda").manual_seed(rows)
    width, pages = kv_heads * hd, -(-rows // page) + 2

    def ints(*shape):
        return torch.randint(-2 ** 31, 2 ** 31, shape, dtype=torch.int64, device="cuda", generator=g).to(torch.int32)

    k, v = ints(rows, width + extra), ints(rows, width + 2 * extra)
    kp, vp = ints(pages, kv_heads, page, hd), ints(pages, kv_heads, page, hd)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:rows].to(torch.int32)
    # rows that are skipped: behind the last, past either end of the cache
    for i, bad in enumerate((-1, pages * page, 2 ** 31 - 1, -2 ** 31)):
        if i + 1 < rows:
            slots[i + 1] = bad
    want_k, want_v, s = kp.cpu().numpy(), vp.cpu().numpy(), slots.tolist()
    for r, slot in enumerate(s):
        if 0 <= slot < pages * page:
            want_k[slot // page, :, slot % page] = k[r, :width].cpu().numpy().reshape(kv_heads, hd)
            want_v[slot // page, :, slot % page] = v[r, :width].cpu().numpy().reshape(kv_heads, hd)
    c = paged.PagedKv(k=kp.data_ptr(), v=vp.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads, head_dim=hd)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    paged.store(c, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), slots.data_ptr(), rows, stream.cuda_stream)
    stream.synchronize()
    assert np.array_equal(kp.cpu().numpy(), want_k) and np.array_equal(vp.cpu().numpy(), want_v)
    paged.store(c, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), slots.data_ptr(), 0)  # no rows: nothing


def test_store_past_four_gigabytes():
    # 2^20 + slots of 1024 values: offsets past 2^32 bytes in each array.
    kv_heads, hd, page = 8, 128, 1024
    pages = 1100
    kp = torch.zeros(pages, kv_heads, page, hd, dtype=torch.int32, device="cuda")
    vp = torch.zeros_like(kp)
    rows = 5
    k = torch.arange(rows * 1024, dtype=torch.int32, device="cuda").reshape(rows, 1024)
    slots = dev([pages * page - 1, 0, 1 << 20, (1 << 20) + 1, pages * page - 7])
    c = paged.PagedKv(k=kp.data_ptr(), v=vp.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads, head_dim=hd)
    paged.store(c, k.data_ptr(), 1024, (k + 1).data_ptr(), 1024, slots.data_ptr(), rows)
    torch.cuda.synchronize()
    for r, s in enumerate(slots.tolist()):
        assert torch.equal(kp[s // page, :, s % page].reshape(-1), k[r])
    assert int((kp != 0).sum()) == rows * 1024 - 1


def test_store_of_two_rows_of_one_slot():
    # The slot's contents are not specified, every other value is.
    kv_heads, hd, page, pages, rows = 2, 64, 16, 4, 40
    rng = np.random.default_rng(30)
    k, v = (rng.integers(-2 ** 31, 2 ** 31, (rows, kv_heads * hd)).astype(np.int32) for _ in range(2))
    slots = rng.permutation(pages * page)[:rows].astype(np.int32)
    slots[[7, 30]] = slots[3]
    margin, left = 4096, 123456789
    big = [torch.full((2 * margin + pages * kv_heads * page * hd,), left, dtype=torch.int32, device="cuda") for _ in range(2)]
    kp, vp = (b[margin:-margin].view(pages, kv_heads, page, hd) for b in big)
    c = paged.PagedKv(k=kp.data_ptr(), v=vp.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads, head_dim=hd)
    tk, tv, ts = dev(k), dev(v), dev(slots)
    paged.store(c, tk.data_ptr(), kv_heads * hd, tv.data_ptr(), kv_heads * hd, ts.data_ptr(), rows)
    torch.cuda.synchronize()
    for b, cache, x in zip(big, (kp, vp), (k, v)):
        got, want = cache.cpu().numpy(), np.full(cache.shape, left, np.int32)
        for r, s in enumerate(slots.tolist()):
            want[s // page, :, s % page] = x[r].reshape(kv_heads, hd)
        s = int(slots[3])
        got[s // page, :, s % page] = want[s // page, :, s % page] = 0
        assert np.array_equal(got, want)
        assert bool((b[:margin] == left).all()) and bool((b[-margin:] == left).all())
