"""GPU: the calls of perf/more_operators.py give what its plain forms give, bit
for bit, at small sizes of each kind."""
import pytest
import torch

from iris_amd import native
from perf import more_operators as measured

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


CASES = [dict(op="adapters", product=product, requests=min(5, rows), rows=rows, rank=12, slots=4, mix=3)
         for product in sorted(measured.PRODUCTS) for rows in (1, 7, 350)] + \
        [dict(op="rules", vocab=vocab, requests=5, nodes=nodes, longest=80, masks=masks, biases=30, mix=4)
         for vocab, nodes, masks in ((100, 1, 0), (4099, 6, 3))] + \
        [dict(op="draw", vocab=vocab, rows=9, kind=kind, closed=closed, mix=5)
         for vocab, kind, closed in ((101, "mixed", 1), (5000, "both", 0), (70003, "mixed", 1))]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "_".join(str(v) for v in c.values()))
def test_calls_give_what_the_plain_forms_give(case, monkeypatch):
    monkeypatch.setattr(measured, "own", True)
    state = measured.prepare(case, 17)
    for _ in range(2):  # the second finds the first one's outputs in its buffers
        got = measured.run(state)
    monkeypatch.setattr(measured, "own", False)
    want = measured.run(state)
    torch.cuda.synchronize()
    if not isinstance(got, dict):
        got, want = dict(out=got), dict(out=want)
    assert got.keys() == want.keys()
    for k in want:
        assert torch.equal(got[k], want[k]), k
