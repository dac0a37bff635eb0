"""GPU: rules on logits and the draw of tokens, bit for bit against plain 64-bit
implementations with the oracle's exp terms."""
import numpy as np
import pytest
import torch

from iris_amd import logits, native
from tests import requests_reference as ref
from tests.test_gpu_paged_attention import dev

pytestmark = pytest.mark.gpu

LEFT = 123456789
MARGIN = 1 << 14
ONE = 1 << 16


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


def words(a):
    """Unsigned 32-bit values on the device."""
    return torch.from_numpy(np.ascontiguousarray(np.asarray(a, np.int64).astype(np.uint32)).view(np.int32)).cuda()


def padded(a, stride):
    out = torch.full((a.shape[0], stride), 77, dtype=torch.int32, device="cuda")
    out[:, :a.shape[1]] = dev(a)
    return out


def some_logits(rng, shape, kind):
    if kind == "wide":
        return rng.integers(-2 ** 31, 2 ** 31, shape, dtype=np.int64).astype(np.int32)
    if kind == "ends":
        return rng.choice(np.array([-2 ** 31, -2 ** 31 + 1, 2 ** 31 - 1, 2 ** 31 - 2, 0, 1, -1, 65536], np.int64),
                          shape).astype(np.int32)
    if kind == "same":
        return np.full(shape, -70000, np.int32)
    if kind == "two":
        return rng.choice(np.array([5 * ONE, 4 * ONE], np.int32), shape)
    if kind == "flat":
        return rng.integers(-40, 40, shape).astype(np.int32)
    x = rng.normal(0, 2.5 * ONE, shape)
    return np.round(x).astype(np.int32)


# ------------------------------------------------------------------ rules


class Rules:
    """Rows of logits, their requests' rules and texts; drafted rows where `nodes`."""

    def __init__(self, rng, vocab, lengths, nodes=None, trees=True, kind="normal", masks=0, biases=0, extra=(0, 0),
                 in_place=False, rules=None, first_row=0, request=None, history=True, window=None):
        n = len(lengths)
        self.starts = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32) if nodes else None
        request = [i for i, c in enumerate(nodes) for _ in range(c)] if nodes else request if request is not None else range(n)
        self.request = np.asarray(list(request), np.int32)[first_row:]
        self.first_row, self.vocab, rows = first_row, vocab, len(self.request)
        self.logits = some_logits(rng, (rows, vocab), kind)
        self.lengths = np.asarray(lengths, np.int32)
        self.stride = max(int(self.lengths.max()), 1) + 3
        # Few different tokens, so that they repeat; some outside the vocabulary.
        self.history = rng.integers(-1, min(vocab, 40) + 1, (n, self.stride)).astype(np.int32)
        self.history[:, ::3] = rng.integers(0, vocab, self.history[:, ::3].shape)
        if not history:
            self.history = None
        self.ids = self.parents = None
        if nodes:
            total = int(self.starts[-1])
            self.ids = rng.integers(0, min(vocab, 20), total).astype(np.int32)
            if trees:
                self.parents = np.concatenate([[int(rng.integers(-1, i)) if i else -1 for i in range(c)] for c in nodes
                                               if c]).astype(np.int32)
        self.bias_ids = rng.integers(-2, vocab + 2, biases * n).astype(np.int32)
        if biases:
            self.bias_ids[:biases // 2] = self.bias_ids[0]  # the same token again and again
        self.bias_values = rng.integers(-200 * ONE, 200 * ONE, biases * n).astype(np.int32)
        self.rule = np.array(rules if rules is not None else
                             [[int(rng.choice([1.0, 1.2, 0.7, 30.0]) * ONE), int(rng.integers(-ONE, ONE)), int(rng.integers(-ONE, ONE)),
                               int(rng.choice([0, 0, 1, 2, 7, 1000])) if window is None else window, i * biases,
                               biases if i != 1 else 0] for i in range(n)], np.int64)
        self.masks = self.mask_of = None
        if masks:
            self.stride_words = (vocab + 31) // 32 + 1
            self.masks = rng.integers(0, 2 ** 32, (masks, self.stride_words), dtype=np.int64).astype(np.uint32)
            self.masks[0] = 0
            self.mask_of = rng.integers(-1, masks, rows).astype(np.int32)
        self.extra, self.in_place = extra, in_place
        self.status = dev([0])
        out_stride = vocab + extra[1 if not in_place else 0]
        self.guard = torch.full((2 * MARGIN + rows * out_stride,), LEFT, dtype=torch.int32, device="cuda")
        self.out = self.guard[MARGIN:-MARGIN].view(rows, out_stride)
        t = dict(logits=padded(self.logits, vocab + extra[0]), request=dev(self.request), rules=words(self.rule),
                 lengths=dev(self.lengths), bias_ids=dev(self.bias_ids), bias_values=dev(self.bias_values))
        for name in ("history", "ids", "parents", "mask_of"):
            if getattr(self, name) is not None:
                t[name] = dev(getattr(self, name))
        if self.starts is not None:
            t["row_start"] = dev(self.starts)
        if masks:
            t["masks"] = words(self.masks)
        self.t = t
        p = {k: v.data_ptr() for k, v in t.items()}
        if in_place:
            p["logits"] = self.out.data_ptr()
        if not biases:
            p["bias_ids"] = p["bias_values"] = None
        self.d = logits.LogitsRules(out=self.out.data_ptr(), status=self.status.data_ptr(), rows=rows, first_row=first_row,
                                    vocab=vocab, logits_stride=out_stride if in_place else vocab + extra[0], out_stride=out_stride,
                                    requests=n, history_stride=self.stride, biases=biases * n, mask_rows=masks,
                                    mask_stride=self.stride_words if masks else 0, **p)

    def fill(self):
        self.out.fill_(LEFT)
        if self.in_place:
            self.out[:, :self.vocab] = dev(self.logits)

    def want(self, request=None, mask_of=None):
        want = ref.rules(self.logits, self.request if request is None else request, self.rule, self.history, self.lengths,
                         self.starts, self.ids, self.parents, self.bias_ids, self.bias_values, self.masks,
                         self.mask_of if mask_of is None else mask_of, self.first_row)
        out = np.full(self.out.shape, LEFT, np.int32)
        out[:, :self.vocab] = want
        return out

    def check(self, status=0, want=None):
        self.fill()
        logits.apply_rules(self.d)
        got = self.out.cpu().numpy()
        assert np.array_equal(got, self.want() if want is None else want)
        assert self.status.item() == status
        assert bool((self.guard[:MARGIN] == LEFT).all()) and bool((self.guard[-MARGIN:] == LEFT).all())


@pytest.mark.parametrize("vocab", [1, 2, 31, 32, 33, 1000, 4095, 4096, 4097, 8191, 9001])
@pytest.mark.parametrize("masks, biases", [(0, 0), (3, 0), (0, 9), (2, 70)])
def test_rules(vocab, masks, biases):
    rng = np.random.default_rng(vocab)
    Rules(rng, vocab, [0, 1, 17, 300], masks=masks, biases=biases).check()


@pytest.mark.parametrize("kind", ["normal", "wide", "ends", "same"])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules_values(kind, in_place):
    rng = np.random.default_rng(3)
    extremes = [[ONE, 0, 0, 0, 0, 5], [1, 2 ** 31 - 1, 2 ** 31 - 1, 0, 5, 5], [2 ** 31 - 1, -2 ** 31, -2 ** 31, 0, 10, 5],
                [3, 1, -1, 0, 15, 5], [65537, 5, 7, 3, 0, 20], [2, -1, 1, 9, 20, 5]]
    for extra in ((0, 0), (3, 1)):
        Rules(rng, 700, [200, 90, 90, 400, 64, 5], kind=kind, biases=5, masks=2, rules=extremes, in_place=in_place,
              extra=extra).check()


def test_division_by_the_repetition_rounds_to_even():
    # Every remainder of small divisors, and quotients of 47 bits.
    rng = np.random.default_rng(4)
    rules = [[rep, 0, 0, 0, 0, 0] for rep in (1, 2, 3, 4, 6, 131072, 196608, 98304, 2 ** 31 - 1, 65535)]
    c = Rules(rng, 4000, [4000] * len(rules), kind="wide", rules=rules)
    c.history[:, :4000] = np.arange(4000)
    c.t["history"].copy_(dev(c.history))
    c.logits[:, :2000] = np.arange(2000)
    c.logits[:, 2000:2050] = 2 ** 31 - 1 - np.arange(50)
    c.t["logits"].copy_(dev(c.logits))
    c.check()


@pytest.mark.parametrize("nodes", [[1, 1, 1], [9, 0, 3, 64], [64, 64], [2, 33]])
@pytest.mark.parametrize("trees", [True, False])
@pytest.mark.parametrize("window", [None, 1, 2, 5, 40])
def test_rules_of_drafted_rows(nodes, trees, window):
    rng = np.random.default_rng(len(nodes))
    Rules(rng, 300, [int(rng.integers(0, 30)) for _ in nodes], nodes=nodes, trees=trees, window=window, masks=3, biases=4).check()


@pytest.mark.parametrize("vocab, biases", [(600, 3000), (5000, 9000), (9001, 1500)])
def test_rules_of_many_biases(vocab, biases):
    # More biased tokens than the sums that a workgroup keeps; each several times.
    rng = np.random.default_rng(biases)
    Rules(rng, vocab, [40, 3, 900], biases=biases).check()
    Rules(rng, vocab, [40, 3], biases=biases, rules=[[ONE, 0, 0, 0, 0, biases], [ONE, 0, 1, 0, biases // 2, biases]], masks=2).check()


def test_rules_of_a_part_of_a_pass():
    rng = np.random.default_rng(2)
    for first in (1, 5, 9):
        Rules(rng, 200, [3, 20, 8], nodes=[4, 5, 7], first_row=first, biases=3).check()
    Rules(rng, 200, [3, 20], nodes=[4, 5], history=False, window=3).check()


def test_rules_of_parents_that_cannot_be():
    # Such a row has no parent: its path begins with it.
    rng = np.random.default_rng(12)
    c = Rules(rng, 100, [5, 5], nodes=[6, 6])
    c.parents[:] = [-1, 1, 99, -7, 2 ** 31 - 1, 3, 0, -2 ** 31, 1, 2, 4, 5]
    c.t["parents"].copy_(dev(c.parents))
    c.check()


def test_rules_without_requests():
    rng = np.random.default_rng(5)
    c = Rules(rng, 300, [4, 4, 4], masks=2, request=[-1, -1, 2])
    c.check()
    c.d.rules = c.d.request = None
    c.check(want=c.want(request=[-1, -1, -1]))
    c = Rules(rng, 300, [4, 4], kind="ends", request=[-1, 0, -1, 1])
    c.check()


@pytest.mark.parametrize("change, status, dropped", [
    (dict(request=(1, 3)), -1, [1]), (dict(request=(0, -2)), -1, [0]), (dict(request=(2, 2 ** 31 - 1)), -1, [2]),
    (dict(rules=(1, 0, 0)), -1, [1]), (dict(rules=(1, 0, -5)), -1, [1]), (dict(rules=(2, 4, 100)), -1, [2]),
    (dict(rules=(2, 5, 100)), -1, [2]), (dict(rules=(2, 4, -1)), -1, [2]), (dict(lengths=(0, -1)), -5, [0]),
    (dict(lengths=(1, 1 << 20)), -5, [1]), (dict(row_start=(0, -1)), -5, [0]), (dict(row_start=(1, 9)), -5, [1]),
    (dict(row_start=(3, 2)), -5, [2]), (dict(row_start=(1, -2 ** 31)), -5, [0, 1])])
def test_rules_report_what_cannot_be(change, status, dropped):
    rng = np.random.default_rng(7)
    c = Rules(rng, 200, [9, 9, 9], nodes=[1, 1, 1], biases=3, masks=2)
    for name, at in change.items():
        t = c.t[name]
        if len(at) == 3:
            t.view(3, 6)[at[0], at[1]] = at[2]
        else:
            t[at[0]] = at[1]
    request = c.request.copy()
    request[dropped] = -1
    c.check(status=status, want=c.want(request=request))


def test_rules_report_masks_that_cannot_be():
    rng = np.random.default_rng(8)
    for bad in (2, -2, 2 ** 31 - 1):
        c = Rules(rng, 200, [9, 9, 9], masks=2)
        mask_of = c.mask_of.copy()
        c.t["mask_of"][1] = bad
        mask_of[1] = -1
        c.check(status=-1, want=c.want(mask_of=mask_of))


def test_rules_captured_and_on_another_stream():
    rng = np.random.default_rng(9)
    c = Rules(rng, 5000, [50, 60, 70], nodes=[3, 1, 5], masks=3, biases=6)
    side = torch.cuda.Stream()
    want = c.want()
    c.fill()
    torch.cuda.synchronize()
    logits.apply_rules(c.d, side.cuda_stream)
    side.synchronize()
    assert np.array_equal(c.out.cpu().numpy(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits.apply_rules(c.d, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        c.logits[:] = some_logits(rng, c.logits.shape, "normal")
        c.t["logits"].copy_(dev(c.logits))
        c.lengths[:] = rng.integers(0, 50, 3)
        c.t["lengths"].copy_(dev(c.lengths))
        c.fill()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), c.want())


# ------------------------------------------------------------------ draw


class Draw:
    def __init__(self, x, drawings, numbers, extra=0, request=None, mass=True):
        self.x, (rows, vocab) = x, x.shape
        self.request = np.arange(rows) if request is None else np.asarray(request)
        self.drawings, self.numbers = np.asarray(drawings, np.int64), np.asarray(numbers, np.int64)
        self.t = dict(logits=padded(x, vocab + extra), drawings=words(self.drawings), numbers=words(self.numbers))
        if request is not None:
            self.t["request"] = dev(self.request)
        self.tokens = torch.full((2 * MARGIN + rows,), LEFT, dtype=torch.int32, device="cuda")
        self.mass = torch.full((2 * MARGIN + 2 * rows,), LEFT, dtype=torch.int64, device="cuda")
        self.status = dev([0])
        self.d = logits.LogitsDraw(tokens=self.tokens[MARGIN:].data_ptr(), mass=self.mass[MARGIN:].data_ptr() if mass else None,
                                   status=self.status.data_ptr(), rows=rows, vocab=vocab, logits_stride=vocab + extra,
                                   requests=len(self.drawings), **{k: v.data_ptr() for k, v in self.t.items()})
        self.size = logits.draw_workspace_bytes(self.d)
        self.space = torch.full((2 * MARGIN + self.size,), 0xA5, dtype=torch.uint8, device="cuda")

    def run(self, stream=None):
        logits.draw(self.d, self.space[MARGIN:].data_ptr(), self.size, stream)

    def got(self):
        rows = len(self.x)
        return [(t, *m) for t, m in zip(self.tokens[MARGIN:MARGIN + rows].tolist(),
                                        self.mass[MARGIN:MARGIN + 2 * rows].view(rows, 2).tolist())]

    def want(self):
        n = len(self.drawings)
        return [ref.draw(l, self.drawings[q] if 0 <= q < n else None, u) for l, q, u in zip(self.x, self.request, self.numbers)]

    def check(self, status=0):
        self.run()
        torch.cuda.synchronize()
        assert self.got() == self.want()
        assert self.status.item() == status
        for t, v in ((self.tokens, LEFT), (self.mass, LEFT), (self.space, 0xA5)):
            assert bool((t[:MARGIN] == v).all()) and bool((t[-MARGIN:] == v).all())


def some_drawings(rng, n):
    return [[int(rng.choice([0, 1 << 15, ONE, 100000, 1 << 18])), int(rng.choice([0, 0, 1, 3, 40, 1000])),
             int(rng.choice([0, 0, 1, 1 << 30, 4080218931, 2 ** 32 - 1])), int(rng.choice([0, 0, 1, ONE, 3 * ONE, 1 << 20]))]
            for _ in range(n)]


def some_numbers(rng, n):
    u = rng.integers(0, 2 ** 32, n)
    u[::5], u[1::5] = 0, 2 ** 32 - 1
    return u


@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 511, 4095, 4096, 4097, 9001, 32003])
@pytest.mark.parametrize("kind", ["normal", "flat", "same", "two"])
def test_draw(vocab, kind):
    rng = np.random.default_rng(vocab)
    rows = 24 if vocab < 5000 else 8
    x = some_logits(rng, (rows, vocab), kind)
    Draw(x, some_drawings(rng, rows), some_numbers(rng, rows)).check()
    x[rng.random(x.shape) < 0.7] = ref.LOWEST
    x[0] = ref.LOWEST
    Draw(x, some_drawings(rng, rows), some_numbers(rng, rows), extra=5).check()


@pytest.mark.parametrize("kind", ["wide", "ends", "normal"])
def test_draw_at_the_ends_of_temperature(kind):
    rng = np.random.default_rng(11)
    betas = [1, 2, 3, 2 ** 31 - 1, 2 ** 31 - 2, 1 << 30, 65535, 65537, 12345, -1, -2 ** 31, 16, 33, 524287]
    for k, p, far in ((0, 0, 0), (7, 0, 0), (0, 3 << 30, 0), (0, 0, 1), (900, 1 << 31, 2), (0, 0, 2 ** 32 - 1), (0, 0, 4095)):
        x = some_logits(rng, (len(betas), 2500), kind)
        Draw(x, [[b, k, p, far] for b in betas], some_numbers(rng, len(betas))).check()


def test_draw_of_crowded_gaps():
    # Thousands of equal logits around each bound: the index decides.
    rng = np.random.default_rng(12)
    vocab = 30011
    x = np.full((12, vocab), -3 * ONE, np.int32)
    x[:, rng.permutation(vocab)[:9000]] = 0
    x[4:8] += rng.integers(0, 3, (4, vocab)).astype(np.int32)
    x[8:, 77] = 9 * ONE
    draws = [[ONE, 0, 0, 0], [ONE, 8999, 0, 0], [ONE, 9001, 0, 0], [ONE, 20000, 3 << 30, 0]] * 3
    Draw(x, draws, some_numbers(rng, 12)).check()
    Draw(x, [[3, *d[1:]] for d in draws], some_numbers(rng, 12)).check()


def test_draw_reaches_every_token():
    # All 2^32 numbers are too many: those at the border of each token's part.
    rng = np.random.default_rng(13)
    l = some_logits(rng, (1, 40), "normal")[0]
    drawing = [ONE, 0, 0, 0]
    order = np.lexsort((np.arange(40), -l))
    w = [int(ref.terms()[min(int(l[order[0]]) - int(l[i]), (1 << 20) - 1)]) for i in order]
    whole, at, numbers = sum(w), 0, []
    for e in w:
        at += e
        edge = -(-(at << 32) // whole)  # the first number past it
        numbers += [edge - 1] + ([edge] if edge < 2 ** 32 else [])
    Draw(np.repeat(l[None], len(numbers), 0), [drawing] * len(numbers), numbers).check()


@pytest.mark.parametrize("kind", ["normal", "same"])
def test_draw_of_a_large_vocabulary(kind):
    rng = np.random.default_rng(14)
    x = some_logits(rng, (5, 256000), kind)
    draws = [[ONE, 0, 0, 0], [ONE, 50, 0, 0], [78643, 0, 4080218931, 0], [ONE, 70000, 3865470566, 0], [ONE, 0, 0, 2 * ONE]]
    Draw(x, draws, some_numbers(rng, 5)).check()


def test_draw_of_the_largest_vocabulary():
    rng = np.random.default_rng(15)
    x = np.full((2, 1 << 20), 7, np.int32)
    x[1] = rng.integers(-3, 3, 1 << 20)
    Draw(x, [[ONE, 0, 0, 0], [ONE, 1 << 19, 0, 0]], [2 ** 32 - 1, 1 << 31]).check()


def test_draw_by_requests():
    rng = np.random.default_rng(16)
    x = some_logits(rng, (9, 700), "normal")
    draws = some_drawings(rng, 3)
    Draw(x, draws, some_numbers(rng, 9), request=[2, 2, 0, -1, 1, 1, 1, 0, -1]).check()
    for bad in (3, -2, 2 ** 31 - 1):
        Draw(x, draws, some_numbers(rng, 9), request=[2, 2, 0, -1, 1, bad, 1, 0, -1]).check(status=-1)
    c = Draw(x, draws * 3, some_numbers(rng, 9), mass=False)
    c.run()
    assert [t for t, _, _ in c.got()] == [t for t, _, _ in c.want()]
    # No records: first maxima, and rows past the requests have none.
    c = Draw(x, draws, some_numbers(rng, 9))
    c.d.drawings = c.d.numbers = None
    c.run()
    assert c.got() == [ref.draw(l, None, 0) for l in x]


def test_draw_captured_and_on_another_stream():
    rng = np.random.default_rng(17)
    rows = 6
    c = Draw(some_logits(rng, (rows, 9000), "normal"), some_drawings(rng, rows), some_numbers(rng, rows))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    c.run(side.cuda_stream)
    side.synchronize()
    assert c.got() == c.want()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        c.x[:] = some_logits(rng, c.x.shape, "normal")
        c.t["logits"].copy_(dev(c.x))
        c.drawings[:] = some_drawings(rng, rows)
        c.t["drawings"].copy_(words(c.drawings))
        graph.replay()
        torch.cuda.synchronize()
        assert c.got() == c.want()
        c.run()
        torch.cuda.synchronize()
        assert c.got() == c.want()


def test_two_draws_at_once():
    rng = np.random.default_rng(18)
    calls = [Draw(some_logits(rng, (n, 6000), "normal"), some_drawings(rng, n), some_numbers(rng, n)) for n in (1, 40)]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s in zip(calls, streams):
            c.run(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        assert c.got() == c.want()


def test_rules_then_draw():
    # As a server calls them: rules in place, then the draw, drafted rows of a tree.
    rng = np.random.default_rng(19)
    r = Rules(rng, 4500, [30, 0, 12], nodes=[5, 1, 7], masks=4, biases=8, in_place=True)
    r.fill()
    rows = len(r.request)
    d = Draw(r.logits, some_drawings(rng, 3), some_numbers(rng, rows), request=r.request)
    d.d.logits, d.d.logits_stride = r.out.data_ptr(), r.out.stride(0)
    logits.apply_rules(r.d)
    d.run()
    torch.cuda.synchronize()
    d.x = r.want()[:, :4500]
    assert d.got() == d.want()


@pytest.mark.parametrize("kind", ["normal", "same", "two"])
def test_captured_draws_of_long_rows(kind):
    # Rows whose tokens are gathered by pieces, and crowded ones.
    rng = np.random.default_rng(24)
    draws = [[ONE, 0, 0, 0], [ONE, 50, 0, 0], [1 << 18, 0, 4080218931, 0], [30000, 6000, 1 << 31, 0]]
    c = Draw(some_logits(rng, (4, 70001), kind), draws, some_numbers(rng, 4), extra=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        c.x[:] = some_logits(rng, c.x.shape, kind)
        c.x[rng.random(c.x.shape) < 0.2] = ref.LOWEST
        c.t["logits"][:, :70001].copy_(dev(c.x))
        c.numbers[:] = rng.integers(0, 2 ** 32, 4)
        c.t["numbers"].copy_(words(c.numbers))
        graph.replay()
        torch.cuda.synchronize()
        want = c.want()
        assert c.got() == want
        c.run()
        torch.cuda.synchronize()
        assert c.got() == want


@pytest.mark.parametrize("vocab", [65535, 65536, 65537, 66000])
def test_draw_about_the_longest_row_of_one_workgroup(vocab):
    rng = np.random.default_rng(vocab)
    Draw(some_logits(rng, (6, vocab), "normal"), some_drawings(rng, 6), some_numbers(rng, 6)).check()


@pytest.mark.parametrize("vocab", [513, 1025, 5000, 40001])
@pytest.mark.parametrize("in_place", [False, True])
def test_rules_of_a_bias_on_every_token(vocab, in_place):
    # Lists that no piece has room for, beside short and empty ones.
    rng = np.random.default_rng(vocab)
    ids = np.concatenate([rng.permutation(vocab + 4) - 2, rng.integers(0, vocab, vocab)]).astype(np.int32)
    rules = [[int(1.3 * ONE), ONE, 0, 0, 0, len(ids)], [ONE, 0, 0, 0, 0, vocab], [int(1.3 * ONE), 5, 9, 0, 7, 3], [ONE, 0, 0, 0, 0, 0]]
    for extra in ((0, 0), (3, 5)):
        c = Rules(rng, vocab, [60, 5, 9, 0], rules=rules, masks=2, extra=extra, in_place=in_place, biases=len(ids) // 4)
        values = rng.integers(-2 ** 31, 2 ** 31, len(ids), dtype=np.int64).astype(np.int32)
        c.bias_ids, c.bias_values = ids, values
        c.t["bias_ids"], c.t["bias_values"] = dev(ids), dev(values)
        c.d.bias_ids, c.d.bias_values, c.d.biases = c.t["bias_ids"].data_ptr(), c.t["bias_values"].data_ptr(), len(ids)
        c.check()


def test_rules_of_a_token_with_thousands_of_biases():
    # Beside as many others as there is room for, one fewer and one more.
    rng = np.random.default_rng(25)
    for others in (1, 255, 510, 511, 512, 900):
        ids = np.concatenate([np.full(7000, 77), 100 + np.arange(others)]).astype(np.int32)
        ids = ids[rng.permutation(len(ids))]
        c = Rules(rng, 1024, [30, 4], rules=[[ONE, 9, 0, 0, 0, len(ids)], [2 * ONE, 0, 0, 0, 5000, 2000]], biases=len(ids) // 2)
        c.bias_ids, c.bias_values = ids, rng.integers(-2 ** 31, 2 ** 31, len(ids), dtype=np.int64).astype(np.int32)
        c.t["bias_ids"], c.t["bias_values"] = dev(c.bias_ids), dev(c.bias_values)
        c.d.bias_ids, c.d.bias_values, c.d.biases = c.t["bias_ids"].data_ptr(), c.t["bias_values"].data_ptr(), len(ids)
        c.check()


def test_the_time_of_a_bias_on_every_token():
    # A pass over the list for each part of a piece, not for each of its tokens:
    # that took 101 ms here.
    rng = np.random.default_rng(26)
    n = 1 << 18
    t = dict(logits=dev(rng.integers(-9 * ONE, 9 * ONE, (1, n)).astype(np.int32)), out=torch.zeros(n, dtype=torch.int32, device="cuda"),
             request=dev([0]), rules=words([[ONE, 0, 0, 0, 0, n]]), bias_ids=dev(rng.permutation(n).astype(np.int32)),
             bias_values=dev(np.full(n, 5, np.int32)))
    d = logits.LogitsRules(rows=1, vocab=n, logits_stride=n, out_stride=n, requests=1, biases=n, **{k: v.data_ptr() for k, v in t.items()})
    stream, times = torch.cuda.current_stream().cuda_stream, []
    for _ in range(4):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        begin.record()
        logits.apply_rules(d, stream)
        end.record()
        end.synchronize()
        times.append(begin.elapsed_time(end))
    assert torch.equal(t["out"], t["logits"][0] + 5)
    assert min(times) < 10, times
