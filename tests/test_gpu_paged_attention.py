"""GPU: attention over packed prompts and of drafted trees over a paged cache,
bit for bit against a plain 64-bit implementation with the oracle's softmax."""
import random

import numpy as np
import pytest
import torch

from iris_amd import native, paged, scalars
from oracle import cpu
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

LEFT = 123456789  # what rows that a call leaves hold


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


def values(rng, shape, kind):
    """Q16.16 values: "normal" (three digits), "wide" (every int32), "mixed"
    (normal with some of four and five digits), "sharp" (large, so that scores
    differ by thousands), "ends" (the ends of the range), "same" (all equal)."""
    if kind == "wide":
        return rng.integers(-2 ** 31, 2 ** 31, shape, dtype=np.int64).astype(np.int32)
    if kind == "ends":
        return rng.choice(np.array([-2 ** 31, -2 ** 31 + 1, 2 ** 31 - 1, 0, 1, -1, -2 ** 23, 2 ** 23 - 1, 8355711, 8355712,
                                    -8421504, -8421505], np.int64), shape).astype(np.int32)
    if kind == "same":
        return np.full(shape, 40000, np.int32)
    x = rng.normal(0, 65536 * (16 if kind == "sharp" else 1), shape).round().astype(np.int64)
    if kind == "mixed":
        at = rng.random(shape) < 0.002
        x = np.where(at, rng.integers(-2 ** 31, 2 ** 31, shape), x)
    return x.astype(np.int32)


def dev(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def padded(a, extra):
    """The rows of `a` at a stride of `extra` more values."""
    out = torch.full((a.shape[0], a.shape[1] + extra), 77, dtype=torch.int32, device="cuda")
    out[:, :a.shape[1]] = dev(a)
    return out


def scale_of(hd, scaled):
    return scalars.attention_scale_q32(hd) if scaled else 0


class Packed:
    def __init__(self, rng, lens, heads, kv_heads, hd, window=0, scaled=True, kinds=("normal", "normal", "normal"),
                 extra=(0, 0, 0, 0), behind=0, max_length=None):
        self.starts = np.concatenate([[0], np.cumsum(lens)]).astype(np.int32)
        rows = int(self.starts[-1]) + behind
        self.heads, self.kv_heads, self.hd, self.window, self.scale = heads, kv_heads, hd, window, scale_of(hd, scaled)
        self.q, self.k, self.v = (values(rng, (rows, n * hd), kind)
                                  for n, kind in zip((heads, kv_heads, kv_heads), kinds))
        self.t = [padded(x, e) for x, e in zip((self.q, self.k, self.v), extra)]
        self.out = torch.full((rows, heads * hd + extra[3]), LEFT, dtype=torch.int32, device="cuda")
        self.row_start, self.status = dev(self.starts), dev([0])
        q, k, v = self.t
        self.d = paged.PackedAttention(
            q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=self.out.data_ptr(), row_start=self.row_start.data_ptr(),
            status=self.status.data_ptr(), q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0),
            out_stride=self.out.stride(0), sequences=len(lens), rows=rows, max_length=max_length or max(max(lens), 1),
            heads=heads, kv_heads=kv_heads, head_dim=hd, window=window, scaled=int(scaled), scale_q32=self.scale)
        self.size = paged.packed_workspace_bytes(self.d)
        self.space = torch.full((max(self.size, 16),), 0xA5, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        paged.attend_packed(self.d, self.space.data_ptr(), self.size, stream)

    def want(self):
        out = np.full(self.out.shape, LEFT, np.int32)
        ref.packed(self.q, self.k, self.v, self.starts.tolist(), self.heads, self.kv_heads, self.hd, self.window,
                   self.scale, out)
        return out

    def check(self):
        torch.cuda.synchronize()
        assert np.array_equal(self.out.cpu().numpy(), self.want())
        assert self.status.item() == 0


@pytest.mark.parametrize("heads, kv_heads, hd", [(1, 1, 4), (2, 1, 20), (4, 2, 64), (6, 2, 80), (8, 2, 128), (5, 5, 64),
                                                 (8, 1, 256), (7, 1, 128), (2, 1, 512), (4, 4, 132)])
@pytest.mark.parametrize("scaled", [True, False])
def test_packed_heads(heads, kv_heads, hd, scaled):
    rng = np.random.default_rng(hd + heads)
    p = Packed(rng, [1, 17, 0, 64, 3, 66], heads, kv_heads, hd, scaled=scaled, extra=(4, 8, 12, 16), behind=3)
    p.run()
    p.check()


@pytest.mark.parametrize("lens", [[1], [2], [15], [16], [17], [63], [64], [65], [129], [1] * 40, [0, 0, 5, 0], [100, 1, 1, 200],
                                  [31, 33, 48, 16, 5, 250]])
@pytest.mark.parametrize("window", [0, 1, 7, 64, 100])
def test_packed_lengths_and_windows(lens, window):
    rng = np.random.default_rng(sum(lens) + window)
    p = Packed(rng, lens, 4, 2, 64, window=window)
    p.run()
    p.check()


@pytest.mark.parametrize("kinds", [("wide", "wide", "wide"), ("normal", "wide", "normal"), ("wide", "normal", "normal"),
                                   ("normal", "normal", "wide"), ("mixed", "mixed", "mixed"), ("ends", "ends", "ends"),
                                   ("sharp", "sharp", "sharp"), ("same", "same", "ends"), ("normal", "normal", "ends"),
                                   ("sharp", "normal", "mixed")])
@pytest.mark.parametrize("heads, kv_heads, hd, scaled", [(4, 2, 64, True), (2, 2, 128, False), (4, 1, 256, False),
                                                         (3, 1, 80, True), (2, 1, 512, True)])
def test_packed_values(kinds, heads, kv_heads, hd, scaled):
    rng = np.random.default_rng(hd)
    p = Packed(rng, [37, 90, 16], heads, kv_heads, hd, scaled=scaled, kinds=kinds)
    p.run()
    p.check()


@pytest.mark.parametrize("lens, window, hd", [([2700], 0, 64), ([700, 2400, 90], 0, 64), ([5000], 900, 128), ([1300, 1200], 0, 256),
                                              ([1900], 0, 512)])
def test_packed_long(lens, window, hd):
    # Few heads; the rows that are compared: each sequence's ends and some between.
    rng = np.random.default_rng(sum(lens))
    p = Packed(rng, lens, 2, 1, hd, window=window, kinds=("sharp", "normal", "normal"))
    p.run()
    torch.cuda.synchronize()
    got = p.out.cpu().numpy()
    for a, b in zip(p.starts[:-1], p.starts[1:]):
        n = b - a
        rows = sorted({0, 1, n // 2, n - 17, n - 2, n - 1} | set(rng.integers(0, n, 10).tolist()))
        at = np.arange(n)
        seen = np.stack([(at <= r) & ((r - at < window) if window else True) for r in rows])
        for h in range(2):
            cols = slice(h * hd, h * hd + hd)
            want = ref.attend(p.q[a:b][rows][:, cols], p.k[a:b], p.v[a:b], seen, p.scale)
            assert np.array_equal(got[a:b][rows][:, cols], want)


def check_some_rows(p, rng):
    """Each sequence's ends and some rows between, three heads."""
    torch.cuda.synchronize()
    got = p.out.cpu().numpy()
    group = p.heads // p.kv_heads
    for a, b in zip(p.starts[:-1], p.starts[1:]):
        n = int(b - a)
        rows = sorted({0, n - 1} | set(rng.integers(0, n, 5).tolist()))
        at = np.arange(n)
        seen = np.stack([(at <= r) & ((r - at < p.window) if p.window else True) for r in rows])
        for h in sorted({0, p.heads // 2, p.heads - 1}):
            cols, kv = slice(h * p.hd, h * p.hd + p.hd), slice(h // group * p.hd, h // group * p.hd + p.hd)
            want = ref.attend(p.q[a:b][rows][:, cols], p.k[a:b, kv], p.v[a:b, kv], seen, p.scale)
            assert np.array_equal(got[a:b][rows][:, cols], want)
    assert p.status.item() == 0


@pytest.mark.parametrize("hd, kv_heads", [(64, 4), (128, 2), (256, 1), (80, 4)])
@pytest.mark.parametrize("lens, heads", [([300, 77, 250], 16), ([90, 200], 16), ([700, 130, 90], 8), ([1000], 4), ([1400], 32),
                                         ([2700], 4)])
def test_packed_launch_shapes(lens, heads, hd, kv_heads):
    # Four, eight and sixteen waves a tile, scores in LDS and behind it.
    rng = np.random.default_rng(hd + heads + lens[0])
    p = Packed(rng, lens, heads, min(kv_heads, heads), hd, kinds=("sharp", "mixed", "mixed"))
    p.run()
    check_some_rows(p, rng)


def tied_difference(n):
    """A score difference d for which n - 1 keys that far below the largest
    have weights within 2^-17 of a rounding tie, and the weight before rounding."""
    term = cpu.lib().dn_softmax_exp_term
    for d in range(1, 700000):
        e = term(-d * 65536)
        total = (1 << 32) + (n - 1) * e
        if abs((e * 65536) % total - total // 2) < total >> 17 and e * 65536 // total:
            return d
    raise AssertionError("no such difference")


@pytest.mark.parametrize("n", [100, 333])
def test_packed_weights_near_ties(n):
    # The last row of every sequence: all its weights but one are near a tie.
    rng = np.random.default_rng(n)
    p = Packed(rng, [n] * 9, 2, 1, 64, scaled=False)
    d = tied_difference(n)
    for t, x in zip(p.t, (p.q, p.k)):
        x[:] = 0
        x[:, ::64] = 65536
    p.k[:] = 0
    p.k[p.starts[1:] - 1, 0] = d
    for t, x in zip(p.t, (p.q, p.k)):
        t.copy_(dev(x))
    p.run()
    p.check()


def test_packed_rows_deeper_than_max_length_are_left():
    rng = np.random.default_rng(5)
    p = Packed(rng, [40, 90, 20], 4, 2, 64, max_length=50)
    p.run()
    torch.cuda.synchronize()
    got, want = p.out.cpu().numpy(), p.want()
    want[40 + 50:130] = LEFT
    assert np.array_equal(got, want) and p.status.item() == -5


def test_packed_starts_that_cannot_be_stay_in_bounds():
    # Every row's first row is clamped to what lies before it.
    rng = np.random.default_rng(6)
    p = Packed(rng, [30, 30, 30], 2, 1, 64)
    for starts in ([0, -5, 30, 90], [50, 40, 30, 90], [0, 30, 200, 300], [0, 0, 0, -4], [-9, 2 ** 31 - 1, -2 ** 31, 90]):
        p.row_start.copy_(dev(starts))
        p.run()
        torch.cuda.synchronize()


@pytest.mark.parametrize("first, lens", [(1, [30]), (5, [20, 33]), (16, [1, 64]), (70, [3, 100, 20])])
@pytest.mark.parametrize("window", [0, 9])
def test_packed_rows_before_the_first_start_are_left(first, lens, window):
    rng = np.random.default_rng(first)
    p = Packed(rng, lens, 4, 2, 64, window=window, behind=first + 3)
    p.starts += first
    p.row_start.copy_(dev(p.starts))
    p.run()
    p.check()


def test_packed_result_is_the_same_beside_other_sequences():
    rng = np.random.default_rng(8)
    p = Packed(rng, [70, 200, 33], 4, 2, 128)
    p.run()
    torch.cuda.synchronize()
    a, b = 70, 270
    alone = Packed(rng, [200], 4, 2, 128)
    for t, x in zip(alone.t, p.t):
        t.copy_(x[a:b])
    alone.run()
    torch.cuda.synchronize()
    assert torch.equal(alone.out, p.out[a:b])


def replays(p, change):
    """Two captured graphs of one call, replayed in turns with eager runs and
    other inputs between."""
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            p.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    for i in range(4):
        change(i)
        p.out.fill_(LEFT)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = p.out.clone()
        p.out.fill_(LEFT)
        p.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(got, p.out)
        if i in (0, 3):
            p.check()


def test_packed_captured_and_replayed():
    rng = np.random.default_rng(12)
    p = Packed(rng, [50, 1, 80], 4, 2, 64)

    def change(i):
        p.q = values(rng, p.q.shape, "wide" if i == 2 else "normal")
        p.t[0].copy_(dev(p.q))

    replays(p, change)


def test_packed_calls_at_once_on_two_streams():
    rng = np.random.default_rng(13)
    calls = [Packed(rng, lens, 8, 2, 128) for lens in ([300, 20], [17, 400])]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(calls, streams):
            c.run(s.cuda_stream)
    for c in calls:
        c.check()


# ------------------------------------------------------------------ trees


class Tree:
    def __init__(self, rng, lengths, nodes, heads, kv_heads, hd, window=0, scaled=True, page=16, parents="random",
                 kinds=("normal", "normal", "normal"), extra=(0, 0), behind=0, max_nodes=None, max_positions=None,
                 spare_pages=2):
        r = random.Random(int(rng.integers(1 << 30)))
        n = len(lengths)
        self.lengths, self.starts = list(lengths), [0] + list(np.cumsum(nodes))
        rows = self.starts[-1] + behind
        self.heads, self.window, self.scale = heads, window, scale_of(hd, scaled)
        held = [-(-(x + m) // page) for x, m in zip(lengths, nodes)]
        pages = sum(held) + spare_pages
        order = list(range(pages))
        r.shuffle(order)
        self.table, at = np.full((n, max(max(held), 1) + 1), -1, np.int32), 0
        for i, h in enumerate(held):
            self.table[i, :h] = order[at:at + h]
            at += h
        if parents == "random":
            parents = [r.choice([i - 1, r.randrange(i) if i else -1, max(i - 3, -1), -1, i + 1, -9]) for m in nodes
                       for i in range(m)]
        self.parents = parents
        self.q = values(rng, (rows, heads * hd), kinds[0])
        self.kp, self.vp = (values(rng, (pages, kv_heads, page, hd), kind) for kind in kinds[1:])
        self.tq, self.tk, self.tv = padded(self.q, extra[0]), dev(self.kp), dev(self.vp)
        self.out = torch.full((rows, heads * hd + extra[1]), LEFT, dtype=torch.int32, device="cuda")
        self.t = dict(row_start=dev(self.starts), lengths=dev(lengths), table=dev(self.table), status=dev([0]))
        if parents is not None:
            self.t["parents"] = dev(list(parents) or [0])
        self.c = paged.PagedKv(k=self.tk.data_ptr(), v=self.tv.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads,
                               head_dim=hd)
        self.d = paged.TreeAttention(
            q=self.tq.data_ptr(), out=self.out.data_ptr(), **{k: v.data_ptr() for k, v in self.t.items()},
            q_stride=self.tq.stride(0), out_stride=self.out.stride(0), requests=n, rows=rows,
            table_stride=self.table.shape[1], max_nodes=max_nodes or max(max(nodes), 1),
            max_positions=max_positions or max(max(x + m for x, m in zip(lengths, nodes)), 1), heads=heads, window=window,
            scaled=int(scaled), scale_q32=self.scale)
        self.size = paged.tree_workspace_bytes(self.c, self.d)
        self.space = torch.full((max(self.size, 16),), 0xA5, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        paged.attend_tree(self.c, self.d, self.space.data_ptr(), self.size, stream)

    def want(self):
        out = np.full(self.out.shape, LEFT, np.int32)
        return ref.tree(self.q, self.kp, self.vp, self.table, self.starts, self.lengths, self.parents, self.heads,
                        self.window, self.scale, out)

    def check(self, status=0):
        torch.cuda.synchronize()
        assert np.array_equal(self.out.cpu().numpy(), self.want())
        assert self.t["status"].item() == status


HEADS = [(1, 1, 4), (2, 1, 20), (4, 2, 64), (6, 2, 80), (8, 2, 128), (5, 5, 64), (8, 1, 256), (7, 1, 128), (2, 1, 512),
         (4, 4, 132), (32, 2, 64)]


@pytest.mark.parametrize("heads, kv_heads, hd", HEADS)
@pytest.mark.parametrize("scaled", [True, False])
def test_tree_heads(heads, kv_heads, hd, scaled):
    rng = np.random.default_rng(hd + heads)
    t = Tree(rng, [0, 40, 7, 130], [3, 1, 0, 9], heads, kv_heads, hd, scaled=scaled, extra=(4, 8), behind=2)
    t.run()
    t.check()


@pytest.mark.parametrize("lengths, nodes", [([0], [1]), ([1], [1]), ([15], [1]), ([16], [1]), ([63], [1]), ([64], [1]),
                                            ([200], [64]), ([0], [64]), ([5, 0, 900], [0, 0, 2]), ([300] * 5, [1] * 5),
                                            ([1, 2, 3, 70, 129, 400], [17, 33, 5, 16, 64, 2])])
@pytest.mark.parametrize("window", [0, 1, 3, 65, 300])
@pytest.mark.parametrize("page", [4, 16, 128])
def test_tree_lengths_windows_and_pages(lengths, nodes, window, page):
    rng = np.random.default_rng(sum(lengths) + window + page)
    t = Tree(rng, lengths, nodes, 4, 2, 64, window=window, page=page)
    t.run()
    t.check()


@pytest.mark.parametrize("kinds", [("wide", "wide", "wide"), ("normal", "wide", "normal"), ("wide", "normal", "normal"),
                                   ("normal", "normal", "wide"), ("mixed", "mixed", "mixed"), ("ends", "ends", "ends"),
                                   ("sharp", "sharp", "sharp"), ("same", "same", "ends")])
@pytest.mark.parametrize("heads, kv_heads, hd, scaled", [(4, 2, 64, True), (2, 2, 128, False), (4, 1, 256, False),
                                                         (3, 1, 80, True), (2, 1, 512, True)])
def test_tree_values(kinds, heads, kv_heads, hd, scaled):
    rng = np.random.default_rng(hd)
    t = Tree(rng, [150, 20], [9, 21], heads, kv_heads, hd, scaled=scaled, kinds=kinds, page=32)
    t.run()
    t.check()


@pytest.mark.parametrize("length, nodes, heads, kv_heads, hd, page, window", [
    (9000, 2, 2, 1, 64, 64, 0), (3000, 1, 4, 1, 128, 16, 0), (20000, 1, 1, 1, 64, 256, 0), (6000, 5, 2, 2, 256, 32, 2500),
    (4100, 7, 2, 1, 512, 16, 0)])
def test_tree_long_contexts(length, nodes, heads, kv_heads, hd, page, window):
    rng = np.random.default_rng(length)
    t = Tree(rng, [length, 33], [nodes, 1], heads, kv_heads, hd, page=page, window=window,
             kinds=("sharp", "normal", "normal"))
    t.run()
    t.check()


# Bounds on the positions that are far from what is held: the same rows by the
# kernels for long spans, in chunks of several sizes.
LONG = [2600, 30000, 300000]


@pytest.mark.parametrize("heads, kv_heads, hd", HEADS)
@pytest.mark.parametrize("max_positions", LONG)
def test_tree_heads_in_long_spans(heads, kv_heads, hd, max_positions):
    rng = np.random.default_rng(hd + heads)
    t = Tree(rng, [0, 40, 7, 130], [3, 1, 0, 9], heads, kv_heads, hd, extra=(4, 8), behind=2, max_positions=max_positions)
    t.run()
    t.check()


@pytest.mark.parametrize("kinds", [("wide", "wide", "wide"), ("normal", "wide", "normal"), ("normal", "normal", "wide"),
                                   ("mixed", "mixed", "mixed"), ("ends", "ends", "ends"), ("sharp", "sharp", "sharp"),
                                   ("same", "same", "ends")])
@pytest.mark.parametrize("heads, kv_heads, hd, scaled", [(4, 2, 64, True), (2, 2, 128, False), (12, 1, 256, False),
                                                         (9, 1, 80, True), (6, 1, 512, True), (32, 2, 128, True)])
@pytest.mark.parametrize("max_positions", [2600, 300000])
def test_tree_values_in_long_spans(kinds, heads, kv_heads, hd, scaled, max_positions):
    rng = np.random.default_rng(hd)
    t = Tree(rng, [150, 20], [9, 5], heads, kv_heads, hd, scaled=scaled, kinds=kinds, page=32, max_positions=max_positions)
    t.run()
    t.check()


@pytest.mark.parametrize("lengths, nodes", [([0], [1]), ([63], [1]), ([64], [1]), ([200], [64]), ([5, 0, 900], [0, 0, 2]),
                                            ([1, 2, 3, 70, 129, 400], [17, 33, 5, 16, 64, 2])])
@pytest.mark.parametrize("window", [0, 3, 65])
@pytest.mark.parametrize("heads", [2, 16])
def test_tree_lengths_in_long_spans(lengths, nodes, window, heads):
    rng = np.random.default_rng(sum(lengths) + window)
    t = Tree(rng, lengths, nodes, heads, 2, 64, window=window, page=4 if heads == 2 else 64, max_positions=5000,
             kinds=("sharp", "normal", "mixed"))
    t.run()
    t.check()


@pytest.mark.parametrize("requests, heads, kv_heads, hd", [(70, 8, 4, 64), (40, 8, 2, 256), (300, 2, 1, 128)])
def test_tree_of_many_requests(requests, heads, kv_heads, hd):
    # Short spans, but more workgroups than the card holds at once.
    rng = np.random.default_rng(requests)
    t = Tree(rng, rng.integers(0, 150, requests).tolist(), rng.integers(0, 3, requests).tolist(), heads, kv_heads, hd)
    t.run()
    t.check()


@pytest.mark.parametrize("n", [101, 700])
@pytest.mark.parametrize("heads", [1, 40])
@pytest.mark.parametrize("max_positions", [None, 2600, 300000])
def test_tree_weights_near_ties(n, heads, max_positions):
    # Every row's own key is its largest, all others' weights are near a tie.
    rng = np.random.default_rng(n)
    t = Tree(rng, [n - 1], [3], heads, 1, 64, scaled=False, parents=[-1] * 3, max_positions=max_positions)
    t.q[:], t.kp[:] = 0, 0
    t.q[:, ::64] = 65536
    d = tied_difference(n)
    for i in range(3):
        at = n - 1 + i
        t.kp[t.table[0, at // 16], 0, at % 16, 0] = d
    t.tq.copy_(dev(t.q))
    t.tk.copy_(dev(t.kp))
    t.run()
    t.check()


def test_tree_of_null_parents_is_a_chain():
    rng = np.random.default_rng(3)
    t = Tree(rng, [77, 3], [12, 40], 4, 2, 64, parents=None)
    t.run()
    t.check()


def test_tree_rows_equal_single_tokens():
    # Row i of a chain, and one token over the cache that holds the rows before it.
    rng = np.random.default_rng(4)
    t = Tree(rng, [100], [6], 8, 2, 128, parents=None)
    t.run()
    torch.cuda.synchronize()
    for i in range(6):
        one = Tree(rng, [100 + i], [1], 8, 2, 128, parents=None)
        one.c, one.t["table"] = t.c, t.t["table"]
        one.d.table, one.d.table_stride = t.t["table"].data_ptr(), t.table.shape[1]
        one.tq.copy_(t.tq[i:i + 1])
        one.run()
        torch.cuda.synchronize()
        assert torch.equal(one.out[0], t.out[i])


@pytest.mark.parametrize("length", [60, 3000])
def test_tree_bad_pages_read_as_zeros(length):
    rng = np.random.default_rng(9)
    t = Tree(rng, [length, 30], [5, 2], 4, 2, 64)
    for col, page in ((0, -1), (2, t.c.pages), (length // 16, 2 ** 31 - 1)):
        t.table[0, col] = page
    t.t["table"].copy_(dev(t.table))
    t.run()
    t.check(status=-1)


@pytest.mark.parametrize("name, value, rows_left", [
    ("lengths", -1, 1), ("lengths", 2 ** 31 - 1, 1), ("lengths", 57, 1), ("max_nodes", 3, 1), ("rows", 7, 2),
    ("max_positions", 40, 1), ("table_stride", 3, 1)])
def test_tree_requests_that_do_not_fit_are_left(name, value, rows_left):
    # Request 1 of three passes a bound; the others are computed.
    rng = np.random.default_rng(10)
    t = Tree(rng, [20, 45, 9], [2, 5, 1], 4, 2, 64, max_positions=60)
    want = t.want()
    want[2:7] = LEFT
    if name == "lengths":
        t.t["lengths"][1] = value
    elif name == "rows":
        # the last request's rows pass the end of q and out
        t.d.rows = value
        want = t.want()
        want[7:] = LEFT
    elif name == "table_stride":
        t.t["table"] = dev(t.table[:, :3])
        t.d.table, t.d.table_stride = t.t["table"].data_ptr(), 3
    else:
        setattr(t.d, name, value)
    t.run()
    torch.cuda.synchronize()
    assert np.array_equal(t.out.cpu().numpy(), want)
    assert t.t["status"].item() == -5


def test_tree_row_starts_that_cannot_be():
    rng = np.random.default_rng(11)
    t = Tree(rng, [20, 45, 9], [2, 5, 1], 4, 2, 64)
    for starts in ([0, -3, 2, 4], [5, 2, 1, 0], [-1, 2, 7, 900], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 8]):
        t.t["row_start"].copy_(dev(starts))
        t.run()
        torch.cuda.synchronize()


def test_tree_captured_and_replayed():
    rng = np.random.default_rng(14)
    t = Tree(rng, [500, 40], [9, 3], 4, 2, 64, max_positions=520)

    def change(i):
        t.q = values(rng, t.q.shape, "wide" if i == 1 else "normal")
        t.tq.copy_(dev(t.q))
        t.lengths[1] = 40 + i  # the last rows' keys are others now, and still in the request's pages
        t.t["lengths"].copy_(dev(t.lengths))

    replays(t, change)


def test_tree_calls_at_once_on_two_streams():
    rng = np.random.default_rng(15)
    calls = [Tree(rng, [700, 30], [4, 9], 8, 2, 128), Tree(rng, [90, 2100], [1, 2], 8, 2, 128)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(calls, streams):
            c.run(s.cuda_stream)
    for c in calls:
        c.check()


def test_tree_cache_past_four_gigabytes():
    # Pages at the far end of 4.3 GB of keys.
    kv_heads, hd, page, pages = 8, 128, 1024, 1050
    rng = np.random.default_rng(16)
    t = Tree(rng, [1500], [3], 8, 8, hd, page=page)
    kp = torch.zeros(pages, kv_heads, page, hd, dtype=torch.int32, device="cuda")
    vp = torch.zeros_like(kp)
    for col in range(2):
        kp[pages - 1 - col] = t.tk[int(t.table[0, col])]
        vp[pages - 1 - col] = t.tv[int(t.table[0, col])]
    t.t["table"][0, :2] = dev([pages - 1, pages - 2])
    t.c = paged.PagedKv(k=kp.data_ptr(), v=vp.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads, head_dim=hd)
    t.run()
    t.check()


# ------------------------------------- pages of more positions than a chunk's


def chunk_of(t):
    """Positions per chunk, as the launch rule has them (no window)."""
    want = max(1, 1024 // (len(t.lengths) * t.c.kv_heads))
    return min(1024, max(64, -(-(-(-t.d.max_positions // want)) // 64) * 64))


# A chunk that starts inside a page meets one page more than its length fills:
# (requests, kv_heads, longest, page, chunk).
CHUNKS_INSIDE_PAGES = [(64, 8, 340, 256, 192), (64, 8, 1400, 1024, 704), (4, 8, 4200, 512, 192), (4, 8, 14000, 256, 448),
                       (8, 8, 11200, 512, 704), (16, 4, 2200, 256, 192)]


@pytest.mark.parametrize("requests, kv_heads, longest, page, chunk", CHUNKS_INSIDE_PAGES)
@pytest.mark.parametrize("group, nodes, hd", [(1, 1, 64), (3, 9, 20)])
def test_tree_chunks_that_start_inside_a_page(requests, kv_heads, longest, page, chunk, group, nodes, hd):
    # One row tile and several; the last shape is the short form's.
    rng = np.random.default_rng(longest + page)
    some = requests if nodes == 1 else min(requests, 8)  # the others have no rows
    lengths = rng.integers(longest // 2, longest - nodes, requests)
    lengths[0] = longest - nodes
    t = Tree(rng, lengths.tolist(), [nodes] * some + [0] * (requests - some), group * kv_heads, kv_heads, hd, page=page)
    assert chunk_of(t) == chunk
    t.run()
    t.check()


@pytest.mark.parametrize("heads, nodes", [(1, 1), (3, 9)])
def test_tree_bad_page_behind_a_chunk_that_starts_inside_a_page(heads, nodes):
    # 512 requests of two chunks of 192: page 1 lies in the second chunk's end.
    rng = np.random.default_rng(21)
    t = Tree(rng, [340] + [0] * 511, [nodes] + [0] * 511, heads, 1, 64, page=256)
    assert chunk_of(t) == 192
    t.table[0, 1] = t.c.pages
    t.t["table"].copy_(dev(t.table))
    t.run()
    t.check(status=-1)


# ------------------------------------------------- the ends of the ranges


@pytest.mark.parametrize("kinds", [("sharp", "normal", "normal"), ("same", "same", "ends"), ("wide", "wide", "wide")])
@pytest.mark.parametrize("hd", [4, 68])
def test_packed_longest_sequence(kinds, hd):
    rng = np.random.default_rng(hd)
    p = Packed(rng, [65535, 1], 1, 1, hd, kinds=kinds, extra=(4, 0, 0, 0))
    p.run()
    torch.cuda.synchronize()
    got = p.out.cpu().numpy()
    rows = [0, 1, 32767, 43690, 65518, 65519, 65533, 65534]
    seen = np.arange(65535)[None, :] <= np.array(rows)[:, None]
    want = ref.attend(p.q[rows], p.k[:65535], p.v[:65535], seen, p.scale)
    assert np.array_equal(got[rows, :hd], want)
    assert np.array_equal(got[65535, :hd], ref.attend(p.q[65535:], p.k[65535:], p.v[65535:], np.ones((1, 1), bool), p.scale)[0])
    assert p.status.item() == 0


@pytest.mark.parametrize("kinds", [("sharp", "normal", "normal"), ("same", "same", "ends"), ("wide", "wide", "wide")])
@pytest.mark.parametrize("page, nodes", [(1024, 1), (256, 2), (4, 33)])
def test_tree_most_positions(kinds, page, nodes):
    rng = np.random.default_rng(page)
    t = Tree(rng, [(1 << 20) - nodes], [nodes], 1, 1, 4, page=page, kinds=kinds, parents=None)
    t.run()
    torch.cuda.synchronize()
    n, at = nodes - 1, np.arange(1 << 20)
    ids = t.table[0][at // page]
    k, v = t.kp[ids, 0, at % page], t.vp[ids, 0, at % page]
    for i in {0, n // 2, n}:
        seen = (at <= (1 << 20) - nodes + i)[None, :]
        assert np.array_equal(t.out[i].cpu().numpy(), ref.attend(t.q[i:i + 1], k, v, seen, t.scale)[0])
    assert t.t["status"].item() == 0


@pytest.mark.parametrize("scale", [1, 1 << 16, (1 << 31) + 12345, (1 << 32) - 1])
@pytest.mark.parametrize("kind", ["normal", "mixed", "ends"])
def test_scales(scale, kind):
    rng = np.random.default_rng(scale % 1000)
    p = Packed(rng, [40, 3], 4, 2, 64, kinds=(kind,) * 3)
    t = Tree(rng, [70, 5], [3, 9], 4, 2, 64, kinds=(kind,) * 3)
    for c in (p, t):
        c.scale = c.d.scale_q32 = scale
        c.run()
        c.check()


@pytest.mark.parametrize("window", [2 ** 31, 2 ** 32 - 1])
def test_windows_past_every_position(window):
    rng = np.random.default_rng(40)
    p = Packed(rng, [90, 40], 4, 2, 64)
    t = Tree(rng, [200, 5], [3, 9], 4, 2, 64, max_positions=2600)
    want = p.want(), t.want()
    for c, w in zip((p, t), want):
        c.d.window = window
        c.size = paged.packed_workspace_bytes(c.d) if c is p else paged.tree_workspace_bytes(c.c, c.d)
        c.space = torch.full((c.size,), 0xA5, dtype=torch.uint8, device="cuda")
        c.run()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), w)


def test_packed_rows_past_four_giga_values():
    # 1.1 million rows of 32 heads of 128: queries, outputs and digit planes
    # with offsets past 2^32 values; the rows that are looked at lie at both ends.
    rows, heads, kv_heads, hd, n = 1_100_003, 32, 1, 128, 300
    g = torch.Generator(device="cuda").manual_seed(50)
    q, k, v = (torch.randint(-200000, 200000, (rows, x * hd), dtype=torch.int32, device="cuda", generator=g)
               for x in (heads, kv_heads, kv_heads))
    out = torch.full((rows, heads * hd), LEFT, dtype=torch.int32, device="cuda")
    starts = torch.tensor(list(range(0, rows - 50, n)) + [rows - 1], dtype=torch.int32, device="cuda")
    status = dev([0])
    d = paged.PackedAttention(
        q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(), row_start=starts.data_ptr(),
        status=status.data_ptr(), q_stride=heads * hd, k_stride=hd, v_stride=hd, out_stride=heads * hd,
        sequences=len(starts) - 1, rows=rows, max_length=n + 50, heads=heads, kv_heads=kv_heads, head_dim=hd, window=0,
        scaled=1, scale_q32=scale_of(hd, True))
    size = paged.packed_workspace_bytes(d)
    assert size > 1 << 34
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    paged.attend_packed(d, space.data_ptr(), size)
    torch.cuda.synchronize()
    assert status.item() == 0 and bool((out[-1] == LEFT).all())
    for i in (0, len(starts) // 2, len(starts) - 2):
        a, b = int(starts[i]), int(starts[i + 1])
        qs, ks, vs, got = (x[a:b].cpu().numpy() for x in (q, k, v, out))
        pick = [0, 1, b - a - 17, b - a - 1]
        seen = np.arange(b - a)[None, :] <= np.array(pick)[:, None]
        for h in (0, 17, heads - 1):
            cols = slice(h * hd, h * hd + hd)
            assert np.array_equal(got[pick, cols], ref.attend(qs[pick][:, cols], ks, vs, seen, d.scale_q32))


def test_tree_work_space_past_four_gigabytes():
    # 64 trees of 64 rows at up to 12000 positions: 6.4 GB of scores.
    requests, nodes, heads, kv_heads, hd, page, longest = 64, 64, 32, 8, 64, 128, 12000
    g = torch.Generator(device="cuda").manual_seed(51)
    held = -(-(longest + nodes) // page)
    pages = requests * held
    kp, vp = (torch.randint(-300000, 300000, (pages, kv_heads, page, hd), dtype=torch.int32, device="cuda", generator=g)
              for _ in range(2))
    q = torch.randint(-300000, 300000, (requests * nodes, heads * hd), dtype=torch.int32, device="cuda", generator=g)
    table = torch.randperm(pages, device="cuda", generator=g).to(torch.int32).reshape(requests, held)
    r = random.Random(52)
    lengths = [longest - r.randrange(3000) for _ in range(requests - 1)] + [longest]
    parents = [r.randrange(-1, i) if i else -1 for _ in range(requests) for i in range(nodes)]
    out = torch.full_like(q, LEFT)
    t = dict(row_start=dev(range(0, requests * nodes + 1, nodes)), lengths=dev(lengths), parents=dev(parents), table=table,
             status=dev([0]))
    c = paged.PagedKv(k=kp.data_ptr(), v=vp.data_ptr(), pages=pages, page_size=page, kv_heads=kv_heads, head_dim=hd)
    d = paged.TreeAttention(
        q=q.data_ptr(), out=out.data_ptr(), **{n: x.data_ptr() for n, x in t.items()}, q_stride=heads * hd,
        out_stride=heads * hd, requests=requests, rows=requests * nodes, table_stride=held, max_nodes=nodes,
        max_positions=longest + nodes, heads=heads, window=0, scaled=1, scale_q32=scale_of(hd, True))
    size = paged.tree_workspace_bytes(c, d)
    assert size > 6 << 30
    space = torch.empty(size, dtype=torch.uint8, device="cuda")
    paged.attend_tree(c, d, space.data_ptr(), size)
    torch.cuda.synchronize()
    assert t["status"].item() == 0
    for b in (0, requests - 1):
        seen, _ = ref.tree_mask(lengths[b], parents[b * nodes:b * nodes + nodes], 0)
        at = np.arange(seen.shape[1])
        ids, rows = table[b].cpu().numpy()[at // page], slice(b * nodes, b * nodes + nodes)
        qs, got, pick = q[rows].cpu().numpy(), out[rows].cpu().numpy(), [0, 30, 63]
        own = torch.from_numpy(ids).long().cuda()
        for h in (0, heads - 1):
            cols, kv = slice(h * hd, h * hd + hd), h // (heads // kv_heads)
            ks, vs = (x[own, kv, torch.from_numpy(at % page).cuda()].cpu().numpy() for x in (kp, vp))
            assert np.array_equal(got[pick, cols], ref.attend(qs[pick][:, cols], ks, vs, seen[pick], d.scale_q32))


@pytest.mark.parametrize("heads, kv_heads", [(3000, 3000), (3000, 3), (1200, 600)])
def test_many_heads(heads, kv_heads):
    rng = np.random.default_rng(heads + kv_heads)
    p = Packed(rng, [3, 18], heads, kv_heads, 4)
    t = Tree(rng, [20, 3], [1, 2], heads, kv_heads, 4)
    for c in (p, t):
        c.run()
        c.check()


def test_tree_requests_that_share_pages():
    # Three requests over the pages of one prompt, their newest rows in pages of their own.
    rng = np.random.default_rng(53)
    t = Tree(rng, [64, 64, 64], [3, 1, 5], 4, 2, 64)
    t.table[1:, :4] = t.table[0, :4]
    t.t["table"].copy_(dev(t.table))
    t.d.status = t.d.parents = None
    t.parents = None
    t.run()
    t.check()
