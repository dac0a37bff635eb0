"""GPU: requests of one batch with adapters, rules, masks and draws of their own,
token for token against the oracle's pieces run one request at a time."""
import random

import numpy as np
import pytest

from iris_amd import logits, native, synth
from iris_amd.direct import Batch, DeviceModel, ModelAdapters, RequestOptions, Session
from tests.requests_forward import Forward

pytestmark = pytest.mark.gpu

ONE = 1 << 16
MODELS = {
    "mistral": lambda: synth.mistral_model(128, 2, 4, 2, 32, 256, 512, seed=21, per_row_scale=False),
    "mistral odd": lambda: synth.mistral_model(96, 2, 3, 3, 32, 160, 320, seed=23, per_row_scale=False, tied_head=True),
    "mistral rows": lambda: synth.mistral_model(256, 1, 4, 1, 64, 512, 777, seed=25),
    "gemma": lambda: synth.tiny_gemma(),
    "gemma windows": lambda: synth.gemma_model(synth.parity_gemma_shape(), 256, seed=5),
}
_made = {}


@pytest.fixture(scope="module", autouse=True)
def device():
    native.check(native.lib().q8gpu_init(), "q8gpu_init")


def made(name):
    if name not in _made:
        _made[name] = DeviceModel(MODELS[name]())
    return _made[name]


def some_adapter(rng, model, names, rank):
    """{tensor name: pair}, large enough that tokens change."""
    out = {}
    for layer in range(model.num_layers):
        for part in names:
            if rng.random() < 0.85:
                name = model.layer_name(layer, part + ".weight")
                w = model.q8(name)
                r = max(1, int(rank * rng.choice([1, 1, 0.5])))
                a = np.clip(rng.normal(0, 3000, (r, w.shape[1] // 34 * 32)), -32639, 32639).astype(np.int16)
                b = np.clip(rng.normal(0, 3000, (w.shape[0], r)), -32639, 32639).astype(np.int16)
                out[name] = (a, 15, b, 15)
    return out


def loaded(dm, adapters, max_rank):
    s = ModelAdapters(dm, len(adapters), max_rank)
    for i, pairs in enumerate(adapters):
        for name, pair in pairs.items():
            s.load(i, name, *pair)
    return s


def prompts(dm, lens, seed=1):
    return [synth.token_ids(seed + i, n, dm.model.vocab).astype(np.int32) for i, n in enumerate(lens)]


def mask_of(seed, vocab):
    """A mask that depends on the ids so far: mostly half of the tokens, at
    times all (None)."""
    def mask(ids):
        r = np.random.default_rng([seed, *[int(i) for i in ids[-3:]], len(ids)])
        return None if r.random() < 0.2 else r.random(vocab) < 0.5
    return mask


def drafter(known, vocab, seed):
    """Proposals: parts of the true continuation, among others."""
    r = random.Random(seed)

    def draft(p, ids):
        true = known[p][len(ids):len(ids) + 4]
        if r.random() < 0.5:
            return [t if r.random() < 0.8 else r.randrange(vocab) for t in true], None
        out, parents = [], []
        for t in true:
            out += [r.randrange(vocab), t]
            parents += [len(out) - 3 if len(out) > 2 else -1] * 2
        return out, parents
    return draft


def wanted(model, p, tokens, o, adapters):
    rule = None
    if o is not None and (o.rule is not None or o.biases):
        rule = (o.rule.repetition, o.rule.frequency, o.rule.presence, o.rule.window) if o.rule is not None else (ONE, 0, 0, 0)
    if o is None:
        return Forward(model).generate(p, tokens)
    d = o.drawing
    return Forward(model, adapters[o.adapter] if o.adapter >= 0 else None).generate(
        p, tokens, rule, list(o.biases.items()) if isinstance(o.biases, dict) else list(o.biases or ()),
        (d.inverse_temperature, d.top_k, d.top_p, d.max_gap) if d is not None else None, o.numbers, o.mask)


def run_and_check(name, lens, tokens, options, adapters=(), max_rank=16, drafts=True, requests=None):
    dm = made(name)
    ps = prompts(dm, lens)
    want = [wanted(dm.model, p, tokens, o, adapters) for p, o in zip(ps, options)]
    known = [p.tolist() + w[0] for p, w in zip(ps, want)]
    b = Batch(dm, requests or len(lens), 60, 4, 64, 96)
    if adapters:
        b.adapters(loaded(dm, adapters, max_rank))
    for draft in (None, drafter(known, dm.model.vocab, 3), drafter(known, dm.model.vocab, 4)) if drafts else (None,):
        got = b.generate(ps, tokens, draft=draft, options=options)
        assert [(r.token_ids, r.stop_reason) for r in got] == want
    return want


ALL = ModelAdapters.PRODUCTS


@pytest.mark.parametrize("name", list(MODELS))
@pytest.mark.parametrize("names", [ALL, ("self_attn.q_proj", "self_attn.v_proj"), ("mlp.gate_proj", "mlp.up_proj"),
                                   ("mlp.down_proj", "self_attn.o_proj")], ids=["all", "qv", "gate up", "down o"])
def test_adapters_of_several_requests(name, names):
    model, rng = made(name).model, np.random.default_rng(7)
    adapters = [some_adapter(rng, model, names, r) for r in (16, 5, 8)]
    lens, tokens = [5, 9, 1, 12], 4
    # First maxima, and draws at a high temperature, which small changes of the
    # logits change too.
    for hot in (False, True):
        options = [RequestOptions(adapter=i, drawing=logits.drawing(40.0) if hot else None,
                                  numbers=rng.integers(0, 2 ** 32, tokens)) for i in (2, -1, 0, 1)]
        got = run_and_check(name, lens, tokens, options, adapters)
    for o in options:
        o.adapter = -1
    plain = [wanted(model, p, tokens, o, ()) for p, o in zip(prompts(made(name), lens), options)]
    assert got[1] == plain[1] and all(got[i] != plain[i] for i in (0, 2, 3))


def test_adapters_of_many_rows():
    # Past the rows and ranks of the single-row kernels, and one row alone.
    name = "mistral rows"
    rng = np.random.default_rng(8)
    adapters = [some_adapter(rng, made(name).model, ALL, r) for r in (40, 3)]
    run_and_check(name, [60, 30], 2, [RequestOptions(adapter=1), RequestOptions(adapter=0)], adapters, max_rank=64, drafts=False)
    run_and_check(name, [1], 3, [RequestOptions(adapter=1)], adapters, max_rank=64)


RULE = logits.TokenRule(repetition=int(1.4 * ONE), frequency=ONE // 3, presence=ONE // 4, window=0)


@pytest.mark.parametrize("name", ["mistral", "mistral odd", "gemma"])
def test_rules_of_several_requests(name):
    vocab = made(name).model.vocab
    plain = [wanted(made(name).model, p, 1, None, ())[0][0] for p in prompts(made(name), [7, 3, 1, 10])]
    options = [RequestOptions(rule=RULE), RequestOptions(rule=logits.TokenRule(repetition=ONE, frequency=5 * ONE, window=3)),
               RequestOptions(biases={plain[2]: -100 * ONE, 5: 2 * ONE}),
               RequestOptions(rule=RULE, biases=[(1, ONE), (1, ONE), (vocab + 3, ONE)], mask=mask_of(2, vocab))]
    got = run_and_check(name, [7, 3, 1, 10], 6, options)
    assert got[2][0][0] != plain[2]


@pytest.mark.parametrize("name", ["mistral", "gemma windows"])
def test_masks_of_several_requests(name):
    vocab = made(name).model.vocab

    def narrow(ids):  # two tokens, then none
        m = np.zeros(vocab, bool)
        m[[3, 4]] = len(ids) < 9
        return m
    options = [RequestOptions(mask=mask_of(1, vocab)), None, RequestOptions(mask=narrow), RequestOptions(mask=mask_of(5, vocab))]
    got = run_and_check(name, [6, 4, 7, 2], 5, options)
    assert got[2][1] == "closed" and len(got[2][0]) == 2 and set(got[2][0]) <= {3, 4}


@pytest.mark.parametrize("name", ["mistral", "mistral odd", "gemma"])
def test_draws_of_several_requests(name):
    rng = np.random.default_rng(5)
    hot = [logits.drawing(30.0), logits.drawing(20.0, top_k=7), logits.drawing(25.0, top_p=0.6), logits.drawing(20.0, min_p=0.3)]
    options = [RequestOptions(drawing=d, numbers=rng.integers(0, 2 ** 32, 6)) for d in hot] + [None]
    got = run_and_check(name, [7, 3, 1, 10, 4], 6, options)
    # The same numbers draw the same tokens, others others.
    options[0] = RequestOptions(drawing=hot[0], numbers=rng.integers(0, 2 ** 32, 6))
    assert run_and_check(name, [7, 3, 1, 10, 4], 6, options, drafts=False)[0] != got[0]


@pytest.mark.parametrize("name", ["mistral", "gemma"])
def test_all_of_them_with_fewer_requests_than_prompts(name):
    model, rng = made(name).model, np.random.default_rng(9)
    vocab = model.vocab
    adapters = [some_adapter(rng, model, ALL, r) for r in (9, 16)]
    options = [RequestOptions(adapter=1, rule=RULE, drawing=logits.drawing(20.0, top_k=50), numbers=rng.integers(0, 2 ** 32, 5)),
               None, RequestOptions(adapter=0, mask=mask_of(4, vocab)), RequestOptions(rule=RULE), None,
               RequestOptions(adapter=1, drawing=logits.drawing(15.0, top_p=0.9), numbers=rng.integers(0, 2 ** 32, 5),
                              mask=mask_of(6, vocab))]
    run_and_check(name, [5, 8, 3, 11, 2, 6], 5, options, adapters, requests=2)


def test_settings_end_with_their_request():
    # A released request runs as ever, and so do those beside requests with settings.
    name = "mistral"
    dm = made(name)
    rng = np.random.default_rng(10)
    ps = prompts(dm, [5, 6])
    alone = [Session(dm, 64, 16).generate(p, 5).token_ids for p in ps]
    b = Batch(dm, 2, 40, 4, 64, 64)
    b.adapters(loaded(dm, [some_adapter(rng, dm.model, ALL, 8)], 8))
    b.adapter(0, 0)
    b.rule(0, RULE, {1: ONE})
    b.drawing(0, logits.drawing(30.0), rng.integers(0, 2 ** 32, 64))
    first = b.prefill({0: ps[0], 1: ps[1]})
    assert first[1] == alone[1][0]
    b.release(0)
    out = [b.prefill({0: ps[0]})[0]]
    for _ in range(4):
        out.append(b.step({0: [out[-1]]})[0][0])
    assert out == alone[0]
    # Settings taken back one by one.
    b.release(0)
    b.rule(0, RULE)
    b.rule(0, None)
    b.drawing(0, logits.drawing(30.0), [1, 2, 3])
    b.drawing(0, None)
    b.adapter(0, 0)
    b.adapter(0, -1)
    b.masks(np.zeros((1, dm.model.vocab), bool), [0] * 5)
    b.masks(None)
    assert b.prefill({0: ps[0]})[0] == alone[0][0]


def test_a_rule_set_late_counts_the_whole_text():
    name = "mistral odd"
    dm = made(name)
    p, = prompts(dm, [9])
    want = Forward(dm.model).generate(p, 3)[0]
    f = Forward(dm.model)
    rule = (int(1.4 * ONE), ONE // 3, ONE // 4, 0)
    for _ in range(3):
        want += f.generate(list(p) + want, 1, rule)[0]
    b = Batch(dm, 3, 40, 4, 64, 64)
    got = [b.prefill({1: p})[1]]
    got += b.step({1: [got[-1]]})[1]
    got += b.step({1: [got[-1], 0, 5]}, {1: [-1, 0, 0]})[1][:1]
    while b.length(1) < 11:
        got += b.step({1: [got[-1]]})[1]
    got = got[:3]
    b.rule(1, RULE)
    for _ in range(3):
        got += b.step({1: [got[-1]]})[1]
    assert got == want


def test_refusals_change_nothing():
    name = "mistral"
    dm = made(name)
    rng = np.random.default_rng(11)
    ps = prompts(dm, [5])
    alone = Session(dm, 64, 16).generate(ps[0], 3).token_ids
    b = Batch(dm, 2, 40, 4, 64, 64)

    def refused(call, code):
        with pytest.raises(native.IrisError) as e:
            call()
        assert e.value.code == code

    refused(lambda: b.adapter(0, 0), -4)
    s = loaded(dm, [some_adapter(rng, dm.model, ALL, 4)], 4)
    b.adapters(s)
    for slot in (1, -2):
        refused(lambda: b.adapter(0, slot), -1)
    refused(lambda: b.adapter(2, 0), -1)
    refused(lambda: b.rule(2, RULE), -1)
    refused(lambda: b.rule(0, logits.TokenRule(repetition=0)), -1)
    refused(lambda: b.rule(0, RULE, [(0, 1)] * ((1 << 20) + 1)), -5)
    refused(lambda: b.drawing(2, logits.drawing()), -1)
    refused(lambda: b.drawing(0, logits.drawing(), [0] * 65), -5)
    vocab = dm.model.vocab
    refused(lambda: b.masks(np.ones((1, vocab), bool), [0, 1]), -1)
    refused(lambda: b.masks(np.ones((1, vocab), bool), [-2]), -1)
    refused(lambda: b.masks(np.ones((3, vocab), bool), [0, 1]), -5)
    refused(lambda: b.masks(np.ones((65, vocab), bool), [0] * 65), -5)
    with pytest.raises(ValueError):
        b.masks(np.ones((1, vocab - 1), bool), [0])
    # Masks of another number of rows, and numbers that do not reach, refuse the pass.
    b.masks(np.ones((1, vocab), bool), [0] * 4)
    refused(lambda: b.prefill({0: ps[0]}), -1)
    b.masks(None)
    b.drawing(0, logits.drawing(), [0] * 4)
    refused(lambda: b.prefill({0: ps[0]}), -5)
    b.drawing(0, logits.drawing(), [0] * 4, 5)
    refused(lambda: b.prefill({0: ps[0]}), -5)
    b.drawing(0, None)
    assert b.length(0) == 0
    out = [b.prefill({0: ps[0]})[0]]
    for _ in range(2):
        out.append(b.step({0: [out[-1]]})[0][0])
    assert out == alone
    # Adapters of another model; matrices that it lacks.
    other = ModelAdapters(made("mistral odd"), 1, 4)
    refused(lambda: b.adapters(other), -1)
    for bad in ("model.language_model.layers.9.mlp.up_proj.weight", "model.language_model.layers.0.mlp.other.weight", "x"):
        with pytest.raises((native.IrisError, KeyError)):
            s.load(0, bad, np.zeros((1, 128), np.int16), 0, np.zeros((256, 1), np.int16), 0)
    L = native.lib()
    a = np.zeros((1, 128), np.int16)
    assert L.iris_model_adapters_load(s.handle, 0, b"model.language_model.layers.9.mlp.up_proj.weight", a.ctypes.data, 0,
                                      a.ctypes.data, 0, 1) == -1
    assert L.iris_model_adapters_load(s.handle, 1, b"model.language_model.layers.0.mlp.up_proj.weight", a.ctypes.data, 0,
                                      a.ctypes.data, 0, 1) == -1
    b.release(0)
    with pytest.raises(ValueError):
        b.generate(ps, 3, options=[])
    with pytest.raises(ValueError):
        b.generate(ps, 3, options=[RequestOptions(drawing=logits.drawing(), numbers=[1, 2])])


def test_real_weights_and_cleared_slots():
    name = "mistral"
    dm = made(name)
    rng = np.random.default_rng(12)
    s = ModelAdapters(dm, 2, 8)
    assert s.device_bytes() == 0
    q = dm.model.layer_name(0, "self_attn.q_proj.weight")
    a, w = rng.normal(0, 0.1, (8, 128)), rng.normal(0, 0.1, (128, 8))
    s.load_real(1, q, a, w, scale=2.0)
    assert s.device_bytes() >= 2 * 2 * 8 * (128 + 128)
    from iris_amd.adapters import to_fixed
    pair = (*to_fixed(a), *to_fixed(w * 2.0))
    p, = prompts(dm, [6])
    b = Batch(dm, 1, 20, 4, 64, 64)
    b.adapters(s)
    assert b.generate([p], 4, options=[RequestOptions(adapter=1)])[0].token_ids == Forward(dm.model, {q: pair}).generate(p, 4)[0]
    s.clear(1)
    assert b.generate([p], 4, options=[RequestOptions(adapter=1)])[0].token_ids == Forward(dm.model).generate(p, 4)[0]
    b.adapters(None)
    assert b.generate([p], 4)[0].token_ids == Forward(dm.model).generate(p, 4)[0]


def test_two_batches_of_one_set_in_turn():
    name, tokens = list(MODELS)[0], 5
    dm, rng = made(name), np.random.default_rng(31)
    adapters = [some_adapter(rng, dm.model, ALL, r) for r in (8, 16)]
    shared = loaded(dm, adapters, 16)
    ps = prompts(dm, [7, 11])
    options = [RequestOptions(adapter=i, rule=logits.TokenRule(repetition=80000, frequency=3000),
                              drawing=logits.drawing(30.0, top_k=200), numbers=rng.integers(0, 2 ** 32, tokens)) for i in (1, 0)]
    want = [wanted(dm.model, p, tokens, o, adapters)[0] for p, o in zip(ps, options)]
    batches, got = [], []
    for p, o in zip(ps, options):
        b = Batch(dm, 2, 20, 4, 64, 32)
        b.adapters(shared)
        b.adapter(1, o.adapter)
        b.rule(1, o.rule)
        b.drawing(1, o.drawing, o.numbers, p.size - 1)
        batches.append(b)
        got.append([b.prefill({1: p})[1]])
    for _ in range(tokens - 1):
        for b, out in zip(batches, got):
            out += b.step({1: [out[-1]]})[1]
    assert [g[:len(w)] for g, w in zip(got, want)] == want  # (an end token stops `want`)


def test_generation_begins_without_earlier_settings():
    dm, rng = made("mistral"), np.random.default_rng(41)
    ps = prompts(dm, [6, 9])
    want = Batch(dm, 2, 40, 4, 64, 64).generate(ps, 4)
    b = Batch(dm, 2, 40, 4, 64, 64)
    s = loaded(dm, [some_adapter(rng, dm.model, ALL, 8)], 8)
    b.adapters(s)
    for request in (0, 1):
        b.adapter(request, 0)
        b.rule(request, logits.TokenRule(repetition=1 << 20), {int(t): 1 << 28 for t in range(9)})
        b.drawing(request, logits.drawing(50.0), rng.integers(0, 2 ** 32, 64))
    b.masks(np.zeros((1, dm.model.vocab), bool), [0])
    got = b.generate(ps, 4, options=[None, RequestOptions()])
    assert [r.token_ids for r in got] == [r.token_ids for r in want]


def test_names_that_are_no_layers_are_refused():
    dm = made("mistral")
    s = ModelAdapters(dm, 1, 4)
    a = np.zeros((1, 256), np.int16)
    load = native.lib().iris_model_adapters_load
    at = b"model.language_model.layers.%s.self_attn.o_proj.weight"
    assert load(s.handle, 0, at % b"1", a.ctypes.data, 0, a.ctypes.data, 0, 1) == 0
    held = s.device_bytes()
    for layer in (b"x", b"", b"00", b" 1", b"+1", b"1x", b"-0", b"4294967296", b"2"):
        assert load(s.handle, 0, at % layer, a.ctypes.data, 0, a.ctypes.data, 0, 1) == -1
    assert load(s.handle, 0, at % b"1" + b".x", a.ctypes.data, 0, a.ctypes.data, 0, 1) == -1
    assert s.device_bytes() == held


def test_rules_and_draws_of_a_larger_vocabulary_are_refused():
    # The operators on logits take 2^20 tokens; such a model generates greedily
    # as ever, with adapters too.
    model = synth.mistral_model(32, 1, 1, 1, 32, 64, (1 << 20) + 32, seed=27)
    dm, rng = DeviceModel(model), np.random.default_rng(42)
    p, = prompts(dm, [5])
    want = Session(dm, 16, 8).generate(p, 3).token_ids
    b = Batch(dm, 1, 8, 4, 32, 16)
    for call in (lambda: b.rule(0, RULE), lambda: b.drawing(0, logits.drawing(), [0] * 9),
                 lambda: b.masks(np.ones((1, model.vocab), bool), [0] * 5)):
        with pytest.raises(native.IrisError) as e:
            call()
        assert e.value.code == -5
    b.rule(0, None)
    b.drawing(0, None)
    b.masks(None)
    assert b.generate([p], 3)[0].token_ids == want
    pairs = some_adapter(rng, model, ALL, 8)
    b.adapters(loaded(dm, [pairs], 8))
    assert b.generate([p], 3, options=[RequestOptions(adapter=0)])[0].token_ids == \
        Forward(model, pairs).generate(p, 3)[0]


def test_requests_keep_their_slots_when_the_set_is_given_again():
    name = "mistral"
    dm, rng = made(name), np.random.default_rng(43)
    adapters = [some_adapter(rng, dm.model, ALL, 8) for _ in range(4)]
    first, second = loaded(dm, adapters[:2], 8), loaded(dm, adapters[2:], 8)
    p, = prompts(dm, [6])
    numbers = rng.integers(0, 2 ** 32, 64)

    def tokens(pairs):
        return Forward(dm.model, pairs).generate(p, 1, drawing=(logits.drawing(40.0).inverse_temperature, 0, 0, 0),
                                                 numbers=numbers[p.size - 1:])[0]
    want = [tokens(a) for a in adapters] + [tokens(None)]
    assert len({t[0] for t in want}) > 3
    b = Batch(dm, 2, 20, 4, 64, 32)

    def got(slot):
        b.drawing(0, logits.drawing(40.0), numbers)
        out = [b.prefill({0: p})[0]]
        b.release(0)
        b.adapter(0, slot)  # (a released request has none)
        return out

    b.adapters(first)
    b.adapter(0, 1)
    b.adapters(first)
    assert got(1) == want[1]
    b.adapters(second)  # the slot of the other set
    assert got(1) == want[3]
    # A set without a request's slot is refused and changes nothing.
    small = loaded(dm, adapters[:1], 8)
    with pytest.raises(native.IrisError) as e:
        b.adapters(small)
    assert e.value.code == -1
    assert got(0) == want[3]
    b.adapters(small)
    assert got(0) == want[0]
    b.adapters(None)
    assert got(-1) == want[4]
    b.adapters(first)
    assert got(-1) == want[4]


def test_options_that_cannot_be_are_refused_before_any_pass():
    dm, rng = made("mistral"), np.random.default_rng(44)
    ps = prompts(dm, [5, 7, 4])
    want = [r.token_ids for r in Batch(dm, 1, 20, 4, 64, 32).generate(ps, 3)]
    b, passes = Batch(dm, 1, 20, 4, 64, 32), []  # one request: the last prompt's turn comes late
    prefill = b.prefill
    b.prefill = lambda rows: passes.append(rows) or prefill(rows)

    def refused(error, code=None, **kw):
        with pytest.raises(error) as e:
            b.generate(ps, 3, options=[None, None, RequestOptions(**kw)])
        assert code is None or e.value.code == code
        assert not passes and b.length(0) == 0

    refused(native.IrisError, -4, adapter=0)
    b.adapters(loaded(dm, [some_adapter(rng, dm.model, ALL, 4)] * 2, 4))
    for slot in (2, -2, 1 << 20):
        refused(native.IrisError, -1, adapter=slot)
    for repetition in (0, -5):
        refused(native.IrisError, -1, rule=logits.TokenRule(repetition=repetition))
    refused(native.IrisError, -5, biases=np.zeros(((1 << 20) + 1, 2), np.int32))
    refused(OverflowError, biases={1: 1 << 31})
    refused(OverflowError, biases=np.array([[1 << 31, 0]]))
    refused(ValueError, biases=np.zeros((4, 3), np.int32))
    refused(OverflowError, drawing=logits.drawing(), numbers=[1, 1 << 32, 2])
    refused(ValueError, drawing=logits.drawing(), numbers=[1, 2])
    assert [r.token_ids for r in b.generate(ps, 3, options=[None, RequestOptions(), None])] == want


def test_biases_as_an_array():
    dm = made("mistral")
    p, = prompts(dm, [6])
    b = Batch(dm, 1, 20, 4, 64, 32)
    plain = b.generate([p], 3)[0].token_ids
    pairs = [(int(plain[0]), -100 * ONE), (5, ONE), (5, ONE)]
    want = wanted(dm.model, p, 3, RequestOptions(biases=pairs), ())[0]
    assert want != plain
    for biases in (pairs, np.array(pairs), np.array(pairs, np.int32)):
        assert b.generate([p], 3, options=[RequestOptions(biases=biases)])[0].token_ids == want
        b.rule(0, None, biases)
        assert b.prefill({0: p})[0] == want[0]
        b.release(0)
    for none in (None, {}, [], np.zeros((0, 2), np.int32)):
        assert b.generate([p], 3, options=[RequestOptions(biases=none)])[0].token_ids == plain


def test_prompts_whose_options_find_no_room_leave_the_others_results():
    dm = made("mistral")
    ps = prompts(dm, [5, 7, 4])
    plain = Batch(dm, 3, 40, 4, 64, 64).generate(ps, 4)
    # Two requests' biases together pass the most that all may have.
    many = np.zeros((700000, 2), np.int32)
    many[:, 0] = dm.model.vocab  # (outside the vocabulary: no token changes)
    options = [None, RequestOptions(biases=many), RequestOptions(biases=many)]
    b = Batch(dm, 3, 40, 4, 64, 64)
    with pytest.raises(native.IrisError) as e:
        b.generate(ps, 4, options=options)
    assert e.value.code == -5 and "prompt 2" in str(e.value)
    assert [r and r.token_ids for r in e.value.results] == [plain[0].token_ids, plain[1].token_ids, None]
    assert [b.length(i) for i in range(3)] == [0, 0, 0]
    # One after the other they fit.
    got = Batch(dm, 1, 40, 4, 64, 64).generate(ps, 4, options=options)
    assert [r.token_ids for r in got] == [r.token_ids for r in plain]


def own_of(rng, i, vocab, tokens):
    """Options that differ from request to request in all that is kept by row."""
    return RequestOptions(rule=logits.TokenRule(repetition=ONE + 3000 * i, frequency=200 * i, presence=0, window=i % 5) if i % 3 else None,
                          biases={int(t): 3 * ONE for t in rng.integers(0, vocab, i % 4)},
                          mask=mask_of(i, vocab) if i % 4 != 1 else None,
                          drawing=logits.drawing(20.0 + i, top_k=(0, 9, 100)[i % 3]) if i % 5 else None,
                          numbers=rng.integers(0, 2 ** 32, tokens))


@pytest.mark.parametrize("name", ["mistral", "gemma"])
def test_drafts_of_more_rows_than_logits_are_held_for(name):
    # Up to 120 rows a pass, a request's on both sides of the 64th.
    dm, rng = made(name), np.random.default_rng(51)
    n, tokens, vocab = 20, 6, dm.model.vocab
    options = [own_of(rng, i, vocab, tokens) for i in range(n)]
    ps = prompts(dm, [3 + i % 5 for i in range(n)])
    want = [wanted(dm.model, p, tokens, o, ()) for p, o in zip(ps, options)]
    known = [p.tolist() + w[0] for p, w in zip(ps, want)]
    b, most = Batch(dm, n, 100, 4, 64, 120), []
    step = b.step
    b.step = lambda rows, parents=None: most.append(sum(len(r) for r in rows.values())) or step(rows, parents)
    for seed in range(3):
        got = b.generate(ps, tokens, draft=drafter(known, vocab, seed), options=options)
        assert [(r.token_ids, r.stop_reason) for r in got] == want
    assert max(most) > 64


def test_more_prompts_than_logits_are_held_for():
    dm, rng = made("mistral odd"), np.random.default_rng(52)
    n, tokens, vocab = 70, 2, dm.model.vocab
    options = [own_of(rng, i, vocab, tokens) for i in range(n)]
    ps = prompts(dm, [1 + i % 3 for i in range(n)])
    want = [wanted(dm.model, p, tokens, o, ()) for p, o in zip(ps, options)]
    b, most = Batch(dm, n, 2 * n, 4, 64, 150), []
    prefill = b.prefill
    b.prefill = lambda rows: most.append(len(rows)) or prefill(rows)
    got = b.generate(ps, tokens, options=options)
    assert [(r.token_ids, r.stop_reason) for r in got] == want
    assert max(most) == n
