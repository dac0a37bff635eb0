"""GPU: low-rank adapters of many requests beside one product, bit for bit
against a plain 64-bit implementation."""
import numpy as np
import pytest
import torch

from iris_amd import adapters, native
from tests import requests_reference as ref
from tests.test_gpu_paged_attention import dev, values

pytestmark = pytest.mark.gpu

LEFT = 123456789  # what columns and rows that a call leaves hold
MARGIN = 1 << 14

QKV = [(64, 0, 1), (32, 64, 1), (32, 96, 1)]
GATED = [(150, 0, 2), (150, 1, 2)]
PAIRS = [(152, 0, 2), (152, 1, 2)]
TURNED = [(60, 5, 2), (60, 4, 2)]
ODD = [(77, 0, 1), (131, 80, 1)]
ONE = [(40, 3, 1)]


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


class Call:
    """A bank, its weights on the host, and a call's buffers between margins."""

    def __init__(self, rng, cols, parts, ranks, rows, slots, kind="normal", bits=(18, 16), weights="normal", extra=(0, 0, 0),
                 in_place=False, y_kind="normal"):
        self.parts, self.cols, self.rows = parts, cols, rows
        most = max(1, max(max(r) for r in ranks))
        self.bank = adapters.AdapterBank(cols, parts, len(ranks), most)
        self.weights = []
        for s, slot in enumerate(ranks):
            self.weights.append([])
            for p, rank in enumerate(slot):
                if not rank:
                    self.weights[-1].append(None)
                    continue
                self.weights[-1].append((self.some(rng, (rank, cols), weights), bits[0],
                                         self.some(rng, (parts[p][0], rank), weights), bits[1]))
                a, a_bits, b, b_bits = self.weights[-1][-1]
                self.bank.load(s, p, a, a_bits, b, b_bits)
        self.width = max(first + (n - 1) * step for n, first, step in parts) + 1
        self.x, self.y = values(rng, (rows, cols), kind), values(rng, (rows, self.width), y_kind)
        self.slots = np.asarray(slots, np.int32)
        xs, ys, os = cols + extra[0], self.width + extra[1], self.width + (extra[1] if in_place else extra[2])
        self.d_x, self.d_y = self.strided(self.x, xs), self.strided(self.y, ys)
        self.guard = torch.full((2 * MARGIN + rows * os,), LEFT, dtype=torch.int32, device="cuda")
        self.out = self.guard[MARGIN:-MARGIN].view(rows, os)
        self.in_place = in_place
        self.d_slots, self.status = dev(self.slots), dev([0])
        self.size = self.bank.workspace_bytes(rows)
        self.space = torch.full((2 * MARGIN + self.size,), 0xA5, dtype=torch.uint8, device="cuda")
        self.d = adapters.AdapterRows(x=self.d_x.data_ptr(), y=self.out.data_ptr() if in_place else self.d_y.data_ptr(),
                                      out=self.out.data_ptr(), slots=self.d_slots.data_ptr(), status=self.status.data_ptr(),
                                      x_stride=xs, y_stride=os if in_place else ys, out_stride=os, rows=rows)

    @staticmethod
    def some(rng, shape, kind):
        if kind == "ends":
            return rng.choice(np.array([-32639, 32639, 0, 1, -1, 127, 128, -128, -129, 255, -256, 32512], np.int16), shape)
        if kind == "top":
            return np.full(shape, 32639, np.int16)
        if kind == "uniform":
            return rng.integers(-32639, 32640, shape).astype(np.int16)
        return np.clip(rng.normal(0, 4000, shape), -32639, 32639).astype(np.int16)

    @staticmethod
    def strided(a, stride):
        out = torch.full((a.shape[0], stride), 77, dtype=torch.int32, device="cuda")
        out[:, :a.shape[1]] = dev(a)
        return out

    def run(self, stream=None):
        self.bank.apply(self.d, self.space[MARGIN:].data_ptr(), self.size, stream)

    def fill(self):
        self.out.fill_(LEFT)
        if self.in_place:
            self.out[:, :self.width] = dev(self.y)

    def want(self):
        slots = np.where((self.slots >= 0) & (self.slots < len(self.weights)), self.slots, -1)
        want = ref.adapters(self.x, self.y, slots, self.parts, self.weights)
        covered = np.zeros(self.width, bool)
        for n, first, step in self.parts:
            covered[first:first + n * step:step] = True
        out = np.full(self.out.shape, LEFT, np.int32)
        out[:, :self.width] = np.where(covered, want, self.y if self.in_place else LEFT)
        return out

    def check(self, want=None, status=0):
        self.fill()
        self.run()
        got = self.out.cpu().numpy()
        assert np.array_equal(got, self.want() if want is None else want)
        assert self.status.item() == status
        for t, v in ((self.guard, LEFT), (self.space, 0xA5)):
            assert bool((t[:MARGIN] == v).all()) and bool((t[-MARGIN:] == v).all())


@pytest.mark.parametrize("rows", [1, 2, 5, 15, 16, 17, 33, 70, 129, 256, 257, 300, 417])
@pytest.mark.parametrize("parts", [QKV, GATED, PAIRS, TURNED, ODD, ONE], ids=["qkv", "gated", "pairs", "turned", "odd", "one"])
def test_rows_of_many_adapters(rows, parts):
    rng = np.random.default_rng(rows)
    n = len(parts)
    ranks = [[16] * n, [5] * n, [1] * n, [33] + [8] * (n - 1), [40] + [0] * (n - 1)]
    Call(rng, 128, parts, ranks, rows, rng.integers(-1, 5, rows)).check()
    Call(rng, 128, parts, [[0] * (n - 1) + [7], [70] * n], rows, rng.integers(-1, 2, rows), in_place=rows % 2 == 0,
         extra=(4, 4, 8)).check()


@pytest.mark.parametrize("in_place", [False, True])
def test_a_tile_of_many_adapters(in_place):
    # Every row its own adapter, a few without, some parts empty.
    rng = np.random.default_rng(21)
    ranks = [[int(rng.integers(0, 20)) for _ in QKV] for _ in range(90)]
    for rows in (100, 300):
        Call(rng, 160, QKV, ranks, rows, np.arange(rows) % 91 - 1, in_place=in_place).check()
        Call(rng, 160, QKV, ranks, rows, rng.integers(-1, 7, rows), in_place=in_place, kind="mixed").check()
        Call(rng, 160, PAIRS, [r[:2] for r in ranks], rows, np.arange(rows) % 91 - 1, in_place=in_place).check()


@pytest.mark.parametrize("rank", [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 128, 129, 255, 256])
@pytest.mark.parametrize("rows", [1, 40, 75])
def test_ranks(rank, rows):
    rng = np.random.default_rng(rank)
    Call(rng, 96, QKV, [[rank] * 3, [max(1, rank // 2), rank, 0]], rows, rng.integers(0, 2, rows)).check()


@pytest.mark.parametrize("cols", [32, 64, 96, 224, 416, 1024, 2080, 14336, 65504])
@pytest.mark.parametrize("rows", [1, 3, 35, 260])
def test_columns(cols, rows):
    rng = np.random.default_rng(cols)
    Call(rng, cols, ODD, [[9, 16], [16, 3]], rows, np.arange(rows) % 2).check()


@pytest.mark.parametrize("kind", ["normal", "wide", "mixed", "sharp", "ends", "same"])
@pytest.mark.parametrize("weights", ["normal", "ends", "top", "uniform"])
@pytest.mark.parametrize("rows", [3, 40, 83])
@pytest.mark.parametrize("parts", [QKV, PAIRS], ids=["qkv", "pairs"])
def test_values(kind, weights, rows, parts):
    # Every digit of the values and both clamps.
    rng = np.random.default_rng(5)
    for bits in ((18, 16), (0, 0), (40, 40), (1, 33)):
        for ranks in ([[20, 3, 16], [16, 16, 70]], [[8, 200, 1], [130, 256, 9]]):
            Call(rng, 160, parts, [r[:len(parts)] for r in ranks], rows, rng.integers(-1, 2, rows), kind=kind, weights=weights,
                 bits=bits, y_kind=kind).check()


def test_the_largest_sums():
    # 65504 products of 2^31 and 32639, without and with shifts, of either sign.
    rng = np.random.default_rng(1)
    for bits in ((0, 0), (40, 40), (38, 20)):
        for rows in (2, 40, 261):
            c = Call(rng, 65504, ONE, [[3]], rows, [0] * rows, weights="top", bits=bits)
            c.x[:] = np.where(np.arange(rows) % 2, -2 ** 31, 2 ** 31 - 1)[:, None]
            c.d_x.copy_(Call.strided(c.x, 65504))
            c.check()


@pytest.mark.parametrize("rows", [41, 95, 301])
def test_ties_round_to_even(rows):
    # One column of one, weights of halves: sums at every tie of two bits.
    c = Call(np.random.default_rng(0), 32, ONE, [[1]], rows, [0] * rows, bits=(2, 1))
    a = np.zeros((1, 32), np.int16)
    a[0, 5] = 1
    b = np.arange(-20, 20).astype(np.int16).reshape(40, 1)
    c.bank.load(0, 0, a, 2, b, 1)
    c.weights = [[(a, 2, b, 1)]]
    c.x[:] = 0
    c.x[:, 5] = np.arange(rows) - rows // 2
    c.d_x.copy_(Call.strided(c.x, 32))
    c.check()


@pytest.mark.parametrize("rows", [1, 5, 40, 200])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_places(rows, in_place):
    rng = np.random.default_rng(rows)
    for extra in ((0, 0, 0), (4, 1, 3), (12, 7, 0)):
        Call(rng, 128, ODD, [[16, 7], [0, 40]], rows, rng.integers(-1, 2, rows), extra=extra, in_place=in_place).check()


@pytest.mark.parametrize("rows", [1, 20, 300])
@pytest.mark.parametrize("in_place", [False, True])
def test_no_row_has_an_adapter(rows, in_place):
    rng = np.random.default_rng(2)
    Call(rng, 64, QKV, [[4, 4, 4]], rows, [-1] * rows, in_place=in_place).check()
    Call(rng, 64, QKV, [[0, 0, 0], [4, 4, 4]], rows, [0] * rows, in_place=in_place).check()


@pytest.mark.parametrize("rows", [3, 40, 290])
def test_slots_outside_the_bank_are_reported(rows):
    rng = np.random.default_rng(3)
    for bad in (-2, 2, 65535, 2 ** 31 - 1, -2 ** 31):
        slots = rng.integers(-1, 2, rows)
        slots[1] = bad
        Call(rng, 64, QKV, [[4, 4, 4], [9, 2, 0]], rows, slots).check(status=-1)


@pytest.mark.parametrize("rows", [37, 270])
def test_slots_load_again_and_empty(rows):
    rng = np.random.default_rng(8)
    c = Call(rng, 96, QKV, [[16, 16, 16], [8, 8, 8]], rows, rng.integers(-1, 2, rows))
    c.check()
    a, b = Call.some(rng, (5, 96), "uniform"), Call.some(rng, (32, 5), "uniform")
    c.bank.load(0, 1, a, 20, b, 14)
    c.weights[0][1] = (a, 20, b, 14)
    c.check()
    c.bank.load(0, 0, None)
    c.weights[0][0] = None
    c.check()
    # What is refused leaves the part as it was.
    for kw in (dict(a=np.full((5, 96), -32640, np.int16)), dict(b=np.full((32, 5), 32640, np.int16)), dict(a_bits=41),
               dict(a=np.zeros((17, 96), np.int16), b=np.zeros((32, 17), np.int16))):
        with pytest.raises(native.IrisError) as e:
            c.bank.load(0, 1, **{**dict(a=a, a_bits=20, b=b, b_bits=14), **kw})
        assert e.value.code == -5
    for slot, part in ((2, 1), (0, 3)):
        with pytest.raises(native.IrisError):
            c.bank.load(slot, part, a, 20, b, 14)
    c.check()


def test_refused_calls_run_nothing():
    c = Call(np.random.default_rng(1), 64, QKV, [[4, 4, 4]], 3, [0] * 3)
    c.fill()

    def refused(code, space=None, size=None, **kw):
        d = adapters.AdapterRows.from_buffer_copy(c.d)
        for k, v in kw.items():
            setattr(d, k, v)
        with pytest.raises(native.IrisError) as e:
            c.bank.apply(d, c.space[MARGIN:].data_ptr() if space is None else space, c.size if size is None else size)
        assert e.value.code == code

    for k in ("x", "y", "out", "slots"):
        refused(-1, **{k: None})
    refused(-1, x=c.d.x + 4), refused(-1, x_stride=66), refused(-1, x_stride=60), refused(-1, y_stride=127)
    refused(-1, out_stride=127), refused(-1, out=c.d.y, out_stride=130), refused(-5, rows=65536)
    refused(-5, size=c.size - 1), refused(-1, space=0), refused(-1, space=c.space[MARGIN:].data_ptr() + 4)
    c.bank.apply(adapters.AdapterRows(rows=0), None, 0)
    assert c.bank.workspace_bytes(0) == 0 and c.bank.workspace_bytes(65536) == 0
    torch.cuda.synchronize()
    assert bool((c.out == LEFT).all()) and c.bank.device_bytes() > 0


def test_rows_do_not_depend_on_the_rows_beside_them():
    rng = np.random.default_rng(6)
    ranks = [[16, 8, 8], [3, 40, 0]]
    c = Call(rng, 256, QKV, ranks, 290, rng.integers(-1, 2, 290))
    c.fill()
    c.run()
    whole = c.out.cpu().numpy()
    for r in (0, 17, 289):
        d = adapters.AdapterRows.from_buffer_copy(c.d)
        d.x, d.y, d.out = (v + 4 * r * s for v, s in ((d.x, d.x_stride), (d.y, d.y_stride), (d.out, d.out_stride)))
        d.slots, d.rows = d.slots + 4 * r, 1
        c.out.fill_(LEFT)
        c.bank.apply(d, c.space[MARGIN:].data_ptr(), c.size)
        assert np.array_equal(c.out.cpu().numpy()[r], whole[r])


@pytest.mark.parametrize("rows", [2, 60, 270])
def test_captured_calls_and_other_streams(rows):
    rng = np.random.default_rng(7)
    c = Call(rng, 224, GATED, [[16, 8], [5, 33]], rows, rng.integers(-1, 2, rows))
    want = c.want()
    side = torch.cuda.Stream()
    c.fill()
    torch.cuda.synchronize()
    c.run(side.cuda_stream)
    side.synchronize()
    assert np.array_equal(c.out.cpu().numpy(), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        x = values(rng, (rows, 224), "mixed")
        c.x[:] = x
        c.d_x.copy_(dev(x))
        c.fill()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), c.want())


def test_two_calls_at_once():
    rng = np.random.default_rng(9)
    calls = [Call(rng, 512, QKV, [[16, 8, 8], [64, 5, 0]], n, rng.integers(-1, 2, n)) for n in (3, 130)]
    streams = [torch.cuda.Stream() for _ in calls]
    for c in calls:
        c.fill()
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.run(s.cuda_stream)
    torch.cuda.synchronize()
    for c in calls:
        assert np.array_equal(c.out.cpu().numpy(), c.want())


@pytest.mark.parametrize("rows", [3, 40, 257, 300])
@pytest.mark.parametrize("parts", [[(1300, 0, 1), (513, 1300, 1), (40, 1813, 1)], [(40, 0, 1), (1024, 40, 1), (511, 1064, 1)],
                                   [(1028, 0, 2), (1028, 1, 2)], [(1028, 1, 2), (1028, 0, 2)], [(700, 3, 2), (1200, 2, 2)]],
                         ids=["falling", "rising", "pairs", "turned", "uneven"])
def test_parts_of_several_chunks(rows, parts):
    rng = np.random.default_rng(rows)
    n = len(parts)
    ranks = [[20] * n, [16] * (n - 1) + [0], [0] * (n - 1) + [3]]
    for in_place in (False, True):
        Call(rng, 64, parts, ranks, rows, rng.integers(-1, 3, rows), in_place=in_place).check()


@pytest.mark.parametrize("parts", [QKV, PAIRS, TURNED], ids=["qkv", "pairs", "turned"])
def test_captured_calls_beside_eager_ones(parts):
    rng = np.random.default_rng(23)
    rows = 290
    c = Call(rng, 192, parts, [[16] * len(parts), [65, 7, 30][:len(parts)]], rows, rng.integers(-1, 2, rows), in_place=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for _ in range(4):
        c.slots[:] = rng.integers(-1, 2, rows)
        c.d_slots.copy_(dev(c.slots))
        c.fill()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), c.want())
        c.check()


def in_larger_bank(c, max_rank):
    """The call's adapters in a bank that may hold larger ones."""
    c.bank = adapters.AdapterBank(c.cols, c.parts, len(c.weights), max_rank)
    for s, slot in enumerate(c.weights):
        for p, pair in enumerate(slot):
            if pair is not None:
                c.bank.load(s, p, *pair)
    c.size = c.bank.workspace_bytes(c.rows)
    c.space = torch.full((2 * MARGIN + c.size,), 0xA5, dtype=torch.uint8, device="cuda")
    return c


@pytest.mark.parametrize("rows", [1, 17, 70, 256, 257])
@pytest.mark.parametrize("parts", [QKV, PAIRS, ODD], ids=["qkv", "pairs", "odd"])
def test_a_bank_that_may_hold_larger_ranks(rows, parts):
    rng = np.random.default_rng(31)
    n = len(parts)
    ranks = [[16] * n, [5] * n, [1] * (n - 1) + [0], [8] * n]
    for max_rank in (17, 64, 256):
        c = Call(rng, 160, parts, ranks, rows, rng.integers(-1, 4, rows), in_place=max_rank == 64)
        in_larger_bank(c, max_rank).check()
    # None loaded, and the largest one emptied.
    c = in_larger_bank(Call(rng, 160, parts, [[0] * n, [0] * n], rows, rng.integers(-1, 2, rows)), 256)
    c.check()
    a, b = Call.some(rng, (200, 160), "normal"), Call.some(rng, (parts[0][0], 200), "normal")
    c.bank.load(1, 0, a, 18, b, 16)
    c.weights[1][0] = (a, 18, b, 16)
    c.check()
    c.bank.load(1, 0, None)
    c.weights[1][0] = None
    c.check()


@pytest.mark.parametrize("rows", [1, 20, 300])
def test_a_captured_call_takes_larger_ranks_loaded_since(rows):
    rng = np.random.default_rng(32)
    c = in_larger_bank(Call(rng, 224, QKV, [[0, 0, 0], [3, 9, 0]], rows, rng.integers(-1, 2, rows), in_place=True), 130)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(torch.cuda.current_stream().cuda_stream)
    for rank in (2, 9, 10, 19, 64, 130, 1):
        for slot, part in ((0, 0), (1, 2)):
            a, b = Call.some(rng, (rank, 224), "uniform"), Call.some(rng, (QKV[part][0], rank), "uniform")
            c.bank.load(slot, part, a, 20, b, 14)
            c.weights[slot][part] = (a, 20, b, 14)
        c.fill()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(c.out.cpu().numpy(), c.want())
        c.check()


def test_the_time_goes_by_the_ranks_that_are_loaded():
    # 256 rows of 40 adapters of rank 16 took 30 us where the bank could hold
    # such ranks, and 193 where it could hold ranks of 256.
    rng = np.random.default_rng(33)
    parts, rows, best = [(4096, 0, 1), (1024, 4096, 1), (1024, 5120, 1)], 256, []
    c = Call(rng, 4096, parts, [[16] * 3] * 40, rows, np.arange(rows) % 40)
    for max_rank in (16, 256):
        in_larger_bank(c, max_rank)
        times = []
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            stream = torch.cuda.current_stream().cuda_stream
            begin.record()
            for _ in range(20):
                c.run(stream)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        best.append(min(times))
    assert best[1] < 3 * best[0], best


def test_the_largest_sums_in_one_piece():
    # So many tiles and ranks that the columns are not divided: every digit at
    # its end in each of 65504 products, with a sum of either sign.
    rng, rows = np.random.default_rng(34), 700
    parts = [(2, 0, 1), (2, 2, 1), (2, 4, 1)]
    for x in (-2 ** 31, 2 ** 31 - 1, -(128 << 16 | 128 << 8 | 128), 127 << 16 | 127 << 8 | 127):
        c = Call(rng, 65504, parts, [[2, 1, 1]], rows, [0] * rows, weights="top", bits=(33, 15))
        for p, pair in enumerate(c.weights[0]):
            c.weights[0][p] = (np.full_like(pair[0], (127 * 257, -32639, -126 * 256 - 128)[p]), *pair[1:])
        in_larger_bank(c, 256)
        c.x[:] = x
        c.x[::3] = -1 - x
        c.d_x.copy_(Call.strided(c.x, 65504))
        c.check()
