"""GPU: several requests at a time over one paged cache, against the session
that runs one (its tokens are the oracle's, tests/test_gpu_direct.py): prompts
packed, single tokens, chains and trees of drafts, pages that come and go."""
import random

import numpy as np
import pytest

from iris_amd import native, synth
from iris_amd.direct import Batch, DeviceModel, Session
from oracle import cpu

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


def parity_gemma(eos=()):
    return synth.gemma_model(synth.parity_gemma_shape(), 256, seed=5, eos_token_ids=eos)


MODELS = {
    "mistral": lambda: synth.mistral_model(128, 2, 4, 2, 32, 256, 512, seed=21, per_row_scale=False),
    "mistral wide heads": lambda: synth.mistral_model(256, 3, 6, 2, 128, 512, 512, seed=22),
    "mistral odd heads": lambda: synth.mistral_model(96, 2, 3, 3, 32, 160, 320, seed=23, per_row_scale=False, tied_head=True),
    "gemma": lambda: synth.tiny_gemma(),
    "gemma windows": parity_gemma,
    "gemma two head sizes": lambda: synth.gemma4_e2b_scaled(),
    "no layers": lambda: synth.mistral_model(128, 0, 4, 2, 32, 256, 512, seed=24),
}
_made = {}


def made(name):
    """The model on the device and its single-request session's tokens."""
    if name not in _made:
        dm = DeviceModel(MODELS[name]())
        _made[name] = dm, Session(dm, 256, 160), {}
    return _made[name]


def alone(name, prompt, tokens):
    dm, s, known = made(name)
    key = (tuple(int(i) for i in prompt), tokens)
    if key not in known:
        known[key] = s.generate(prompt, tokens)
    return known[key]


def prompts(name, lens, seed=1):
    vocab = made(name)[0].model.vocab
    return [synth.token_ids(seed + i, n, vocab).astype(np.int32) for i, n in enumerate(lens)]


def drafter(name, ps, tokens, seed, tree):
    """Proposals that hold the true continuation or parts of it, and others."""
    r, vocab = random.Random(seed), made(name)[0].model.vocab

    def draft(p, ids):
        true = alone(name, ps[p], tokens).token_ids[len(ids) - len(ps[p]):]
        good = true[:r.randrange(0, 9)]
        if not tree:
            ids = good + [r.randrange(vocab) for _ in range(r.randrange(3))]
            return (ids, None) if r.random() < 0.8 else (ids, list(range(-1, len(ids) - 1)))
        out, above, spine = [], [], -1
        for t in good:
            for _ in range(r.randrange(3)):  # others beside the true one, and below each other
                out.append(r.randrange(vocab))
                above.append(r.choice([spine, spine, len(out) - 2, -1]))
            out.append(t)
            above.append(spine)
            spine = len(out) - 1
        for _ in range(r.randrange(3)):
            out.append(r.randrange(vocab))
            above.append(spine)
        return out[:63], above[:63]

    return draft


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("how", ["plain", "chain", "tree"])
def test_batch_generates_what_a_session_does(name, how):
    tokens, lens = 24, [5, 1, 37, 64, 12, 3, 90, 17]
    ps = prompts(name, lens)
    want = [alone(name, p, tokens) for p in ps]
    b = Batch(made(name)[0], 5, 60, 16, 256, 160)
    draft = None if how == "plain" else drafter(name, ps, tokens, 7, how == "tree")
    for _ in range(2):  # and over pages that others have left
        got = b.generate(ps, tokens, draft)
        assert [g.token_ids for g in got] == [w.token_ids for w in want]
        assert [g.stop_reason for g in got] == [w.stop_reason for w in want]


def test_batch_tokens_are_the_oracles():
    m = MODELS["mistral"]()
    ps = [synth.token_ids(40 + i, n, 512).astype(np.int32) for i, n in enumerate((9, 2, 21))]
    got = Batch(DeviceModel(m), 3, 30, 4, 64, 64).generate(ps, 8)
    for p, g in zip(ps, got):
        assert g.token_ids == cpu.OracleRun(m, 64).generate(list(p), 8, keep_logits=True)[0]


def test_selected_tokens_vary():
    # So that a wrong row, position or page would show in the tokens.
    seen = {t for n in ("mistral", "gemma windows", "gemma two head sizes") for p in prompts(n, [5, 37, 64, 12, 90, 17])
            for t in alone(n, p, 24).token_ids}
    assert len(seen) > 20


@pytest.mark.parametrize("name", ["mistral wide heads", "gemma windows"])
def test_batch_stops_at_end_ids(name):
    ps = prompts(name, [5, 37, 64, 12])
    free = [alone(name, p, 24).token_ids for p in ps]
    m = MODELS[name]()
    m.eos_token_ids = (free[0][3], free[2][7])
    dm = DeviceModel(m)
    s = Session(dm, 256, 160)
    want = [s.generate(p, 24) for p in ps]
    assert {w.stop_reason for w in want} >= {"eos"}
    for tree in (False, True):
        got = Batch(dm, 3, 40, 16, 256, 160).generate(ps, 24, drafter(name, ps, 24, 3, tree))
        assert [g.token_ids for g in got] == [w.token_ids for w in want]
        assert [g.stop_reason for g in got] == [w.stop_reason for w in want]


@pytest.mark.parametrize("requests, pages, page, rows", [(1, 8, 16, 96), (8, 9, 16, 90), (4, 30, 4, 90), (6, 2, 128, 128),
                                                         (3, 200, 4, 91)])
def test_batch_of_few_pages_and_rows(requests, pages, page, rows):
    name, tokens = "mistral", 20
    ps = prompts(name, [90, 3, 40, 40, 2, 61, 8], seed=60)
    b = Batch(made(name)[0], requests, pages, page, 256, rows)
    got = b.generate(ps, tokens, drafter(name, ps, tokens, 9, True))
    assert [g.token_ids for g in got] == [alone(name, p, tokens).token_ids for p in ps]
    assert all(b.length(i) == 0 for i in range(requests))


@pytest.mark.parametrize("name", ["mistral", "gemma two head sizes"])
def test_step_keeps_the_path_of_the_selections(name):
    ps = prompts(name, [30, 7], seed=80)
    true = [alone(name, p, 12).token_ids for p in ps]
    b = Batch(made(name)[0], 4, 20, 16, 128, 64)
    assert b.prefill({1: ps[0], 3: ps[1]}) == {1: true[0][0], 3: true[1][0]}
    assert [b.length(i) for i in range(4)] == [0, 30, 0, 7]
    # Request 1: the true tokens at rows 2, 5 and 6 among others; a second copy
    # of a true token stands behind the first. Request 3 is a single token.
    wrong = (true[0][1] + 1) % made(name)[0].model.vocab
    rows = [true[0][0], wrong, true[0][1], true[0][1], wrong, true[0][2], true[0][3], wrong]
    parents = [-1, 0, 0, 0, 1, 2, 5, 6]
    got = b.step({1: rows, 3: [true[1][0]]}, {1: parents})
    assert got == {1: true[0][1:5], 3: [true[1][1]]}
    assert [b.length(i) for i in range(4)] == [0, 34, 0, 8]
    for j in range(5, 8):
        got = b.step({1: [true[0][j - 1]], 3: [true[1][j - 4], true[1][j - 4]]})
        assert got[1] == [true[0][j]] and got[3][0] == true[1][j - 3]
        b_len = b.length(3)
        if len(got[3]) == 2:  # the repeated token was the model's choice too
            break
    b.release(1)
    assert b.length(1) == 0 and b.length(3) == b_len
    again = b.prefill({1: ps[0], 0: ps[0]})
    assert again == {0: true[0][0], 1: true[0][0]}


def refused(code, call):
    with pytest.raises(native.IrisError) as e:
        call()
    assert e.value.code == code


def test_batch_refusals_change_nothing():
    name = "mistral"
    dm = made(name)[0]
    b = Batch(dm, 2, 4, 16, 48, 40)
    p = prompts(name, [20, 30], seed=90)
    true = alone(name, p[0], 8).token_ids
    refused(-1, lambda: b.prefill({0: [512]}))
    refused(-1, lambda: b.prefill({0: [-1]}))
    refused(-5, lambda: b.prefill({0: [1] * 41}))                # rows
    refused(-5, lambda: Batch(dm, 2, 2, 16, 48, 64).prefill({0: [1] * 20, 1: [1] * 20}))  # pages
    refused(-5, lambda: Batch(dm, 2, 9, 16, 48, 64).prefill({0: [1] * 49}))  # positions
    refused(-4, lambda: b.step({0: [1]}))                        # nothing held
    assert b.prefill({0: p[0]}) == {0: true[0]}
    refused(-4, lambda: b.prefill({0: p[1]}))                    # holds positions
    refused(-4, lambda: b.generate([p[1]], 2))
    refused(-5, lambda: b.step({0: [true[0]] * 29}))             # positions
    refused(-5, lambda: b.prefill({1: [1] * 40}))                # pages
    refused(-1, lambda: b.step({0: [true[0], 512]}))
    assert b.length(0) == 20
    for j in range(1, 8):
        assert b.step({0: [true[j - 1]]}) == {0: [true[j]]}
    with pytest.raises(ValueError):
        b.step({2: [1]})
    with pytest.raises(ValueError):
        b.step({0: [1, 2]}, {0: [-1]})


def test_batch_of_too_many_rows_of_a_request():
    b = Batch(made("mistral")[0], 1, 99, 16, 400, 200)
    first = b.prefill({0: [1, 2, 3]})[0]
    refused(-5, lambda: b.step({0: [first] * 65}))
    assert len(b.step({0: [first] * 64})[0]) >= 1


@pytest.mark.parametrize("kw, code", [
    (dict(requests=0), -1), (dict(pages=0), -1), (dict(page_size=0), -1), (dict(page_size=24), -1), (dict(page_size=2048), -1),
    (dict(max_positions=0), -1), (dict(max_rows=0), -1), (dict(requests=4097), -5), (dict(max_positions=(1 << 20) + 1), -5),
    (dict(max_rows=65536), -5), (dict(pages=1 << 27), -5)])
def test_batch_create_refusals(kw, code):
    args = dict(requests=2, pages=4, page_size=16, max_positions=64, max_rows=32)
    refused(code, lambda: Batch(made("mistral")[0], **{**args, **kw}))


def test_two_batches_and_a_session_in_turns():
    name = "gemma windows"
    ps = prompts(name, [25, 6], seed=95)
    true = [alone(name, p, 10).token_ids for p in ps]
    dm, s, _ = made(name)
    bs = [Batch(dm, 2, 20, 16, 64, 64) for _ in ps]
    for b, p, t in zip(bs, ps, true):
        assert b.prefill({1: p}) == {1: t[0]}
    for j in range(1, 10):
        for b, t in zip(bs, true):
            assert b.step({1: [t[j - 1]]}) == {1: [t[j]]}
        assert s.generate(ps[j % 2], 10).token_ids == true[j % 2]


def test_step_of_more_rows_than_logits_are_held_for():
    # 3 requests of 41 rows: the last token and the 40 that follow it.
    name = "mistral wide heads"
    ps = prompts(name, [9, 30, 2], seed=110)
    true = [alone(name, p, 43).token_ids for p in ps]
    b = Batch(made(name)[0], 3, 40, 16, 128, 130)
    b.prefill(dict(enumerate(ps)))
    got = b.step({i: t[:41] for i, t in enumerate(true)})
    assert got == {i: t[1:42] for i, t in enumerate(true)}
    assert b.step({i: [t[41]] for i, t in enumerate(true)}) == {i: [t[42]] for i, t in enumerate(true)}


@pytest.mark.parametrize("name", ["mistral", "gemma windows"])
def test_batch_of_one_row(name):
    b = Batch(made(name)[0], 2, 9, 4, 32, 1)
    ps = [np.array([5], np.int32), np.array([300], np.int32)]
    assert [g.token_ids for g in b.generate(ps, 9)] == [alone(name, p, 9).token_ids for p in ps]


def test_batch_refuses_a_row_without_finite_scales():
    m = synth.mistral_model(128, 1, 4, 2, 32, 256, 512, seed=25, per_row_scale=False)
    raw = m.tensors["model.language_model.embed_tokens.weight"].copy()
    raw[7, 35] = 0x7C  # the second block's scale
    m.tensors["model.language_model.embed_tokens.weight"] = raw
    b = Batch(DeviceModel(m), 2, 8, 16, 64, 32)
    refused(-2, lambda: b.prefill({0: [1, 7]}))
    token = b.prefill({0: [1, 6]})[0]
    refused(-2, lambda: b.step({0: [token, 7]}))
    assert len(b.step({0: [token]})[0]) == 1


def test_generate_after_a_draft_that_fails():
    name = "mistral"
    ps = prompts(name, [12, 30], seed=120)
    b = Batch(made(name)[0], 2, 8, 16, 64, 64)
    for bad, error in ((lambda p, ids: 1 / 0, ZeroDivisionError), (lambda p, ids: ([3, 4], [-1]), ValueError),
                       (lambda p, ids: ([512], None), native.IrisError)):
        with pytest.raises(error):
            b.generate(ps, 9, bad)
        assert [b.length(0), b.length(1)] == [0, 0]
    assert [g.token_ids for g in b.generate(ps, 9)] == [alone(name, p, 9).token_ids for p in ps]


def test_batch_of_long_requests():
    # Positions past the short form's, pages of more positions than a chunk's
    # length divides, a work space that grows from call to call.
    name = "mistral wide heads"
    dm = made(name)[0]
    lens, tokens = [1400, 1351, 700, 90], 40
    ps = [synth.token_ids(130 + i, n, dm.model.vocab).astype(np.int32) for i, n in enumerate(lens)]
    s = Session(dm, 2048, 1400)
    want = [s.generate(p, tokens).token_ids for p in ps]

    def draft(p, ids):  # the true next two of every third place, else a wrong one
        at = len(ids) - lens[p]
        return (want[p][at:at + 2] if at % 3 == 0 else [(want[p][at] + 1) % dm.model.vocab]), None

    for page, requests in ((256, 64), (1024, 64), (16, 4)):
        b = Batch(dm, requests, 8192 // page, page, 2048, 3600)
        for d in (None, draft):
            assert [g.token_ids for g in b.generate(ps, tokens, d)] == want


def test_calls_after_a_batch_that_the_device_cannot_hold():
    # 2^31 - 16 positions of 64 key values in two layers: over two terabytes.
    name = "mistral"
    ps = prompts(name, [12, 30], seed=145)
    want = [alone(name, p, 9).token_ids for p in ps]
    dm, s, _ = made(name)
    b = Batch(dm, 2, 8, 16, 64, 64)
    for _ in range(2):
        refused(2, lambda: Batch(dm, 2, (1 << 27) - 1, 16, 64, 64))  # hipErrorOutOfMemory
        assert s.generate(ps[0], 9, use_graph=False).token_ids == want[0]
        refused(2, lambda: Batch(dm, 2, (1 << 27) - 1, 16, 64, 64))
        assert [g.token_ids for g in b.generate(ps, 9)] == want


def test_batch_pass_without_work_space_changes_nothing():
    # Trees of 64 rows for each of 4096 requests over 16000 positions would
    # take hundreds of gigabytes: refused before the pass, and single rows go on.
    m = synth.mistral_model(128, 1, 32, 1, 4, 64, 64, seed=26, per_row_scale=False)
    dm, n = DeviceModel(m), 16000
    p = synth.token_ids(140, n, 64).astype(np.int32)
    want = Session(dm, n + 8, n).generate(p, 4).token_ids
    b = Batch(dm, 4096, 40, 1024, n + 100, n)
    assert b.prefill({7: p}) == {7: want[0]}
    for j in range(1, 4):
        refused(2, lambda: b.step({7: [want[j - 1]] * 64}))  # hipErrorOutOfMemory
        assert b.length(7) == n + j - 1
        assert b.step({7: [want[j - 1]]}) == {7: [want[j]]}


def without_embedding(name, token):
    """The model, with no finite scale in the token's row of the embedding (its
    selections are the other model's while none embeds that row)."""
    m = MODELS[name]()
    raw = m.tensors["model.language_model.embed_tokens.weight"].copy()
    raw[token, 35] = 0x7C  # the second block's scale
    m.tensors["model.language_model.embed_tokens.weight"] = raw
    return DeviceModel(m)


def test_generate_ends_only_the_prompt_whose_selection_is_refused():
    name, tokens = "mistral wide heads", 12
    ps = prompts(name, [5, 37, 20, 12], seed=150)
    want = [alone(name, p, tokens).token_ids for p in ps]
    others = {int(t) for p in ps for t in p} | {t for w in (want[0], want[2], want[3]) for t in w}
    at, token = next((i, t) for i, t in enumerate(want[1][:-1]) if t not in others)
    dm = without_embedding(name, token)
    refused(-2, lambda: Session(dm, 256, 160).generate(ps[1], tokens))
    for draft in (None, drafter(name, ps, tokens, 5, True)):
        b = Batch(dm, 2, 20, 16, 256, 160)
        with pytest.raises(native.IrisError) as e:
            b.generate(ps, tokens, draft)
        assert e.value.code == -2
        assert [r and r.token_ids for r in e.value.results] == [want[0], None, want[2], want[3]]
        assert [b.length(0), b.length(1)] == [0, 0]
        # Selected last it is not embedded.
        assert [r.token_ids for r in b.generate(ps, at + 1, draft)] == [w[:at + 1] for w in want]


@pytest.mark.parametrize("tree", [False, True])
def test_generate_does_not_depend_on_drafts_that_cannot_be_embedded(tree):
    name, tokens = "mistral wide heads", 12
    ps = prompts(name, [5, 37, 20], seed=160)
    want = [alone(name, p, tokens).token_ids for p in ps]
    token = next(t for t in range(512) if t not in {int(t) for p in ps for t in p} | {t for w in want for t in w})

    def draft(p, ids):
        true = want[p][len(ids) - len(ps[p]):]
        if not tree:
            return true[:2] + [token] + true[2:], None
        # The refused row first, rows under it, and true ones beside them.
        return [token, 3, true[0], token, 4] + true[1:2], [-1, 0, -1, 2, 3] + [2] * len(true[1:2])

    b = Batch(without_embedding(name, token), 2, 20, 16, 256, 160)
    assert [r.token_ids for r in b.generate(ps, tokens, draft)] == want


def test_generate_refuses_a_prompt_before_any_pass():
    name = "mistral wide heads"
    ps = prompts(name, [5, 37, 20], seed=170)
    dm = without_embedding(name, int(ps[2][7]))
    b, calls = Batch(dm, 1, 20, 16, 256, 160), []
    refused(-2, lambda: b.generate(ps, 5, lambda p, ids: calls.append(p)))
    refused(-1, lambda: b.generate([ps[0], [3, 512]], 5, lambda p, ids: calls.append(p)))
    assert not calls and b.length(0) == 0


def test_ids_refused():
    dm = without_embedding("mistral", 7)
    for ids, want in (([], (0, 0)), ([1, 2, 511], (0, 3)), ([1, 7, 512], (-2, 1)), ([0, 512, 7], (-1, 1)), ([-1], (-1, 0))):
        assert dm.ids_refused(ids) == want
    m = parity_gemma()
    raw = m.tensors["model.language_model.embed_tokens_per_layer.weight"].copy()
    raw[9, 1] = 0x7C  # the first block's scale
    m.tensors["model.language_model.embed_tokens_per_layer.weight"] = raw
    assert DeviceModel(m).ids_refused([8, 9]) == (-2, 1)


def test_trees_without_the_rows_that_cannot_be_embedded():
    b = Batch(without_embedding("mistral", 7), 1, 2, 16, 16, 16)
    for given, want in (
            (([1, 2], None), ([1, 2], None)), (([1, 7, 2], None), ([1], None)), (([7], None), ([], None)),
            (([1, 2, 3], [-1, 0, 1]), ([1, 2, 3], [-1, 0, 1])),
            (([7, 2, 3], [-1, 0, -1]), ([3], [-1])),
            (([1, 7, 3, 4, 5, 6], [-1, -1, 1, 2, 0, 4]), ([1, 5, 6], [-1, 0, 1])),
            (([7, 1, 2], [-1, 9, 1]), ([1, 2], [-2, 0])), (([512, 7], [-1, 0]), ([512, 7], [-1, 0]))):
        assert b._embedded(*given) == want
    with pytest.raises(ValueError):
        b._embedded([1, 7], [-1])


def test_generate_without_work_space_for_its_drafts():
    m = synth.mistral_model(128, 1, 32, 1, 4, 64, 64, seed=26, per_row_scale=False)
    dm, n = DeviceModel(m), 16000
    p = synth.token_ids(140, n, 64).astype(np.int32)
    want = Session(dm, n + 100, n).generate(p, 90).token_ids
    b, asked = Batch(dm, 4096, 40, 1024, n + 100, n), []

    def draft(index, ids):  # 63 rows at the first step, then one
        asked.append(len(ids))
        return ([1] * 63 if len(asked) == 1 else [want[len(ids) - n]]), None

    assert b.generate([p], 90, draft)[0].token_ids == want
    assert asked[:2] == [n + 1, n + 2]  # the first pass kept its last token's row only


def test_two_batches_at_once():
    # Each on a thread of its own, over one model.
    from concurrent.futures import ThreadPoolExecutor
    name, tokens = "mistral wide heads", 24
    sets = [prompts(name, [5, 37, 64], seed=180), prompts(name, [90, 12], seed=190)]
    want = [[alone(name, p, tokens).token_ids for p in ps] for ps in sets]
    bs = [Batch(made(name)[0], 2, 30, 16, 256, 160) for _ in sets]
    drafts = [drafter(name, sets[0], tokens, 3, True), None]
    with ThreadPoolExecutor(2) as pool:
        for _ in range(3):
            runs = [pool.submit(b.generate, ps, tokens, d) for b, ps, d in zip(bs, sets, drafts)]
            assert [[g.token_ids for g in r.result()] for r in runs] == want


def test_generate_after_an_interrupt():
    ps = prompts("mistral", [12, 30], seed=200)
    b = Batch(made("mistral")[0], 2, 8, 16, 64, 64)

    def interrupted(p, ids):
        raise KeyboardInterrupt

    with pytest.raises(KeyboardInterrupt):
        b.generate(ps, 9, interrupted)
    assert [b.length(0), b.length(1)] == [0, 0]
    assert [g.token_ids for g in b.generate(ps, 9)] == [alone("mistral", p, 9).token_ids for p in ps]
