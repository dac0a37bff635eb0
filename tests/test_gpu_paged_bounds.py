"""GPU: what the operators over a paged cache must leave alone. Outputs and
work spaces lie between margins of a known value, which every call leaves; row
starts that cannot be leave the rows that no sequence has."""
import numpy as np
import pytest
import torch

from iris_amd import native
from tests.test_gpu_paged_attention import LEFT, Packed, Tree, dev

pytestmark = pytest.mark.gpu

MARGIN = 1 << 16  # bytes or values on either side


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


class Guarded:
    """The call's output and work space moved between margins."""

    def __init__(self, call, size):
        self.call, rows, stride = call, call.out.shape[0], call.out.stride(0)
        self.out = torch.full((2 * MARGIN + rows * stride,), LEFT, dtype=torch.int32, device="cuda")
        call.out = self.out[MARGIN:-MARGIN].view(rows, stride)
        call.d.out = call.out.data_ptr()
        self.space = torch.full((2 * MARGIN + size,), 0xA5, dtype=torch.uint8, device="cuda")
        call.space = self.space[MARGIN:MARGIN + size]
        assert call.out.data_ptr() % 16 == 0 and call.space.data_ptr() % 16 == 0

    def run(self):
        self.call.out.fill_(LEFT)
        self.call.run()
        torch.cuda.synchronize()
        for t, value in ((self.out, LEFT), (self.space, 0xA5)):
            assert bool((t[:MARGIN] == value).all()) and bool((t[-MARGIN:] == value).all())
        return self.call.out.cpu().numpy()


@pytest.mark.parametrize("lens, heads, kv_heads, hd, window", [
    ([1], 4, 2, 64, 0), ([17, 3, 90], 4, 2, 80, 0), ([300, 250], 8, 1, 256, 100), ([2700], 2, 1, 64, 0), ([700], 2, 2, 512, 0)])
def test_packed_margins(lens, heads, kv_heads, hd, window):
    rng = np.random.default_rng(hd)
    p = Packed(rng, lens, heads, kv_heads, hd, window=window, extra=(4, 8, 12, 0), kinds=("sharp", "mixed", "mixed"))
    g = Guarded(p, p.size)
    g.run()
    if sum(lens) < 1000:
        p.check()


@pytest.mark.parametrize("lengths, nodes, heads, kv_heads, hd, max_positions", [
    ([0], [1], 4, 2, 64, None), ([700, 40], [1, 9], 8, 2, 128, None), ([300, 5], [30, 1], 8, 1, 80, 5000),
    ([2600], [2], 2, 1, 512, 30000), ([90] * 40, [2] * 40, 8, 2, 256, None)])
def test_tree_margins(lengths, nodes, heads, kv_heads, hd, max_positions):
    rng = np.random.default_rng(hd)
    t = Tree(rng, lengths, nodes, heads, kv_heads, hd, max_positions=max_positions, kinds=("sharp", "mixed", "mixed"))
    g = Guarded(t, t.size)
    g.run()
    t.check()


@pytest.mark.parametrize("starts, left", [
    ([0, -5, 30, 90], []), ([50, 40, 30, 90], list(range(50))), ([0, 30, 200, 300], []), ([0, 0, 0, -4], list(range(90))),
    ([-9, 2 ** 31 - 1, -2 ** 31, 90], []), ([200, 300, 400, 500], list(range(90))), ([0, 10, 20, 30], list(range(30, 90)))])
def test_packed_starts_that_cannot_be_leave_rows_of_no_sequence(starts, left):
    rng = np.random.default_rng(6)
    p = Packed(rng, [30, 30, 30], 2, 1, 64)
    g = Guarded(p, p.size)
    p.row_start.copy_(dev(starts))
    got = g.run()
    assert (got[left] == LEFT).all()
    assert p.status.item() in (0, -5)


@pytest.mark.parametrize("starts", [[0, -3, 2, 4], [5, 2, 1, 0], [-1, 2, 7, 900], [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1, 8],
                                    [8, 8, 8, 9], [0, 2, 7, 8]])
@pytest.mark.parametrize("max_positions", [None, 5000])
def test_tree_row_starts_that_cannot_be_leave_those_requests(starts, max_positions):
    # A request's rows are computed where they lie in [0, rows) and fit its
    # bounds, whatever the others' starts are.
    rng = np.random.default_rng(11)
    t = Tree(rng, [20, 45, 9], [2, 5, 1], 4, 2, 64, max_positions=max_positions or 60)
    g = Guarded(t, t.size)
    t.t["row_start"].copy_(dev(starts))
    got, want, bad = g.run(), np.full(t.out.shape, LEFT, np.int32), False
    for i, (a, b) in enumerate(zip(starts[:-1], starts[1:])):
        if b <= a:
            continue
        if a < 0 or b > 8 or b - a > t.d.max_nodes:
            bad = True
            continue
        one = Tree.__new__(Tree)
        one.__dict__.update(t.__dict__)
        one.starts, one.lengths, one.table = [a, b], t.lengths[i:i + 1], t.table[i:i + 1]
        own = one.want()
        want[a:b] = own[a:b]
    assert np.array_equal(got, want)
    assert t.t["status"].item() == (-5 if bad else 0)
