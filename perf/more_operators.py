"""The measured cases of the operators that give each request of a batch its own
fine-tuning, its own rules and its own way of drawing a token.

Three kinds of call:

- ``adapters``: low-rank adapters beside a product whose rows belong to
  different requests: row r with adapter s gets out = y + B_s (A_s x). A and B
  are 16-bit integers with one number of fraction bits a matrix; the product
  may have up to three parts (q, k and v; gate and up, whose rows alternate)
  with an adapter each.
- ``rules``: penalties for repeated tokens, biases and grammar masks on rows of
  logits; drafted rows count the drafted tokens above them too.
- ``draw``: a token for each row of logits: the first maximum, or drawn with a
  temperature and bounds on their number (top-k), their share (top-p) and their
  distance from the first, from a random number that is an input.

All values are Q16.16 integers, and every result is an integer that the
arithmetic fixes bit for bit: sums are exact, each rounding goes to the nearest
and to even at ties, results that leave 32 bits are clamped, and tokens of equal
logits are ordered by their index. The draw's weights are the attention's exp
terms in 32 fraction bits.

``run`` takes what ``prepare`` made; with ``own`` false it computes the
operators with elementary torch operations. The adapters' products there are in
float64 and exact: |x| stays below 2^21, the weights below 2^15 and the columns
at 2^14, so a sum stays below 2^50.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

ONE = 1 << 16
LN2 = 2977044472  # ln 2 in 32 fraction bits
LOWEST, HIGHEST = -(1 << 31), (1 << 31) - 1
WEIGHT = 32639  # the largest weight of an adapter

# A product's columns, and its parts: rows, first output, step between outputs.
# The benchmark's two models' products, and a smaller one of odd sizes.
PRODUCTS = {
    "qkv_4096": (4096, [(4096, 0, 1), (1024, 4096, 1), (1024, 5120, 1)]),
    "gate_up_4096": (4096, [(14336, 0, 2), (14336, 1, 2)]),
    "down_14336": (14336, [(4096, 0, 1)]),
    "qkv_2048": (2048, [(2048, 0, 1), (256, 2048, 1), (256, 2304, 1)]),
    "gate_up_2048": (2048, [(16384, 0, 2), (16384, 1, 2)]),
    "down_16384": (16384, [(2048, 0, 1)]),
    "odd_416": (416, [(77, 0, 1), (131, 80, 1)]),
}


def listed():
    return [
        # A decode step of one request with an adapter on q, k and v.
        dict(name="adapters_1row_qkv", op="adapters", product="qkv_4096", requests=1, rows=1, rank=16, slots=8, mix=1),
        # A decode step of a busy server: a row each, many adapters, some requests without.
        dict(name="adapters_32rows_gate_up", op="adapters", product="gate_up_2048", requests=32, rows=32, rank=8, slots=24,
             mix=2),
        # Ragged prompts of a dozen adapters, packed.
        dict(name="adapters_19seqs_2309rows_qkv", op="adapters", product="qkv_4096", requests=19, rows=2309, rank=64, slots=12,
             mix=3),
        # Long prompts on one adapter of the widest product.
        dict(name="adapters_4096rows_down", op="adapters", product="down_14336", requests=3, rows=4096, rank=32, slots=1,
             mix=4),
        # One request's penalties.
        dict(name="rules_1row_32000", op="rules", vocab=32000, requests=1, nodes=1, longest=700, masks=0, biases=0, mix=5),
        # Drafted trees under grammars, with biases.
        dict(name="rules_12x9_256000", op="rules", vocab=256000, requests=12, nodes=9, longest=2100, masks=64, biases=40,
             mix=6),
        # A token each of many requests late in long texts.
        dict(name="rules_64rows_32000", op="rules", vocab=32000, requests=64, nodes=1, longest=32700, masks=3, biases=300,
             mix=7),
        # One request's draw.
        dict(name="draw_1row_32000", op="draw", vocab=32000, rows=1, kind="both", closed=0, mix=8),
        # A few requests, temperature alone.
        dict(name="draw_9rows_256000", op="draw", vocab=256000, rows=9, kind="plain", closed=0, mix=9),
        # Rows under grammar masks, each with bounds of its own.
        dict(name="draw_33rows_32003", op="draw", vocab=32003, rows=33, kind="mixed", closed=1, mix=10),
        # The rows of many requests' drafted trees.
        dict(name="draw_108rows_256000", op="draw", vocab=256000, rows=108, kind="mixed", closed=0, mix=11),
    ]


def _log(rng, lo, hi):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v))))


def draw(rng):
    op = rng.choice(["adapters", "rules", "draw"])
    mix = rng.randrange(1, 1 << 30)
    if op == "adapters":
        product = rng.choice(sorted(PRODUCTS))
        cols, parts = PRODUCTS[product]
        # At most the values and the products of the largest listed case.
        rank, outputs = _log(rng, 1, 128), sum(p[0] for p in parts)
        most = min(4096, 4096 * (14336 + 2 * 4096) // (cols + 2 * outputs),
                   4096 * 32 * (14336 + 4096) // (rank * (cols + outputs)))
        rows = _log(rng, 1, most)
        return dict(op=op, product=product, requests=_log(rng, 1, min(64, rows)), rows=rows, rank=rank,
                    slots=_log(rng, 1, 48), mix=mix)
    vocab = rng.choice([32000, 256000, _log(rng, 100, 256000)])
    if op == "rules":
        requests, nodes = _log(rng, 1, 64), rng.choice([1, 1, _log(rng, 1, 64)])
        nodes = max(1, min(nodes, 108 * 256000 // (requests * vocab)))
        return dict(op=op, vocab=vocab, requests=requests, nodes=nodes, longest=_log(rng, 1, 32700),
                    masks=rng.choice([0, _log(rng, 1, 64)]), biases=rng.choice([0, _log(rng, 1, 1000)]), mix=mix)
    rows = _log(rng, 1, min(108, 108 * 256000 // vocab))
    return dict(op=op, vocab=vocab, rows=rows, kind=rng.choice(["plain", "top_k", "top_p", "both", "mixed"]),
                closed=rng.choice([0, 1]), mix=mix)


# ------------------------------------------------------------------ inputs


def _gen(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed((seed * 1000003 + salt * 7919 + 1) & 0x7FFFFFFFFFFF)
    return g


def _rows(seed, salt, shape, sigma):
    """Q16.16 values, Gaussian of the given standard deviation, below 2^21."""
    x = torch.randn(shape, device="cuda", generator=_gen(seed, salt)) * (sigma * ONE)
    return torch.round(x).clamp(1 - (1 << 21), (1 << 21) - 1).to(torch.int32)


def _parts(total, count, mix):
    """`total` in `count` ragged parts of at least one."""
    r = random.Random(mix)
    w = [r.lognormvariate(0, 1) for _ in range(count)]
    s = sum(w)
    parts = [1 + int((total - count) * x / s) for x in w]
    parts[0] += total - sum(parts)
    return parts


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _bits(sigma):
    """Fraction bits with which Gaussian weights of this deviation reach 15 bits at five of it."""
    return int(math.floor(math.log2(WEIGHT / (5 * sigma))))


def _request_slots(case):
    """Each request's adapter (-1: none, one request in eight where there are several)."""
    r = random.Random(case["mix"] + 1)
    n = case["requests"]
    return [-1 if n > 3 and r.random() < 0.125 else r.randrange(case["slots"]) for _ in range(n)]


def _ranks(case):
    """[slot][part]: the case's rank, of some adapters half of it, of some parts none."""
    r = random.Random(case["mix"] + 2)
    ranks = []
    for _ in range(case["slots"]):
        rank = case["rank"] if r.random() < 0.7 else max(1, case["rank"] // 2)
        ranks.append([rank if r.random() < 0.9 or p == 0 else 0 for p in range(len(PRODUCTS[case["product"]][1]))])
    return ranks


def _prepare_adapters(case, seed):
    cols, parts = PRODUCTS[case["product"]]
    rows = case["rows"]
    counts = _parts(rows, case["requests"], case["mix"])
    slots = _request_slots(case)
    order = list(range(len(slots)))
    random.Random(seed).shuffle(order)
    counts, slots = [counts[i] for i in order], [slots[i] for i in order]
    width = max(first + (n - 1) * step for n, first, step in parts) + 1
    width = -(-width // 4) * 4
    a_bits, b_bits = _bits(1 / math.sqrt(cols)), _bits(0.1)
    weights = []
    for s, ranks in enumerate(_ranks(case)):
        weights.append([])
        for p, rank in enumerate(ranks):
            g = _gen(seed, 100 + 10 * s + p)
            a = torch.randn((rank, cols), device="cuda", generator=g) * (2.0 ** a_bits / math.sqrt(cols))
            b = torch.randn((parts[p][0], rank), device="cuda", generator=g) * (2.0 ** b_bits * 0.1)
            weights[-1].append(tuple(torch.round(w).clamp(-WEIGHT, WEIGHT).to(torch.int16) for w in (a, b)))
    per_row = [s for s, c in zip(slots, counts) for _ in range(c)]
    s = dict(case=case, x=_rows(seed, 1, (rows, cols), 1.0), y=_rows(seed, 2, (rows, width), 2.0), slots=_ints(per_row),
             weights=weights, a_bits=a_bits, b_bits=b_bits,
             by_slot=[(t, [i for i, u in enumerate(per_row) if u == t]) for t in sorted(set(per_row)) if t >= 0])
    s["out"] = torch.zeros_like(s["y"])
    if own:
        from iris_amd import adapters
        # (A call leaves the columns of no part as they are.)
        s["between"] = width > sum(n for n, _, _ in parts)
        bank = adapters.AdapterBank(cols, parts, slots=case["slots"], max_rank=case["rank"])
        for t, ws in enumerate(weights):
            for p, (a, b) in enumerate(ws):
                if a.shape[0]:
                    bank.load(t, p, a.cpu().numpy(), a_bits, b.cpu().numpy(), b_bits)
        call = adapters.AdapterRows(x=s["x"].data_ptr(), y=s["y"].data_ptr(), out=s["out"].data_ptr(),
                                    slots=s["slots"].data_ptr(), status=None, x_stride=cols, y_stride=width, out_stride=width,
                                    rows=rows)
        size = bank.workspace_bytes(rows)
        s["call"] = (bank, call, torch.empty(max(size, 16), dtype=torch.uint8, device="cuda"), size)
    return s


def _lengths_and_nodes(case):
    """Each request's positions so far and drafted rows: the first the longest of each."""
    r = random.Random(case["mix"])
    lengths, nodes = [case["longest"]], [case["nodes"]]
    for _ in range(case["requests"] - 1):
        lengths.append(_log(r, max(1, case["longest"] // 16), case["longest"]))
        nodes.append(r.randrange(1, case["nodes"] + 1))
    return lengths, nodes


def _prepare_rules(case, seed):
    vocab = case["vocab"]
    lengths, nodes = _lengths_and_nodes(case)
    order = list(range(len(lengths)))
    random.Random(seed).shuffle(order)
    lengths, nodes = [lengths[i] for i in order], [nodes[i] for i in order]
    n, rows, most = len(lengths), sum(nodes), max(lengths)
    r = random.Random(seed + 1)
    # Some tokens are far more usual than others.
    text = torch.rand((n, most), device="cuda", generator=_gen(seed, 1)) ** 4
    drafted = torch.rand(rows, device="cuda", generator=_gen(seed, 2)) ** 4
    rules, ids, values = [], [], []
    for _ in range(n):
        count = r.randrange(case["biases"] + 1) if case["biases"] and n > 1 else case["biases"]
        rules.append([int(r.choice([1.0, 1.1, 1.3]) * ONE), int(r.choice([0.0, 0.1, 0.5]) * ONE),
                      int(r.choice([0.0, 0.2, 0.6]) * ONE), r.choice([0, 0, 64, 1024]), len(ids), count])
        ids += [r.randrange(vocab) for _ in range(count)]
        values += [int(r.choice([-100.0, r.uniform(-5, 5)]) * ONE) for _ in range(count)]
    if n == 1:
        rules[0][:4] = [int(1.1 * ONE), ONE // 10, ONE // 5, 0]
    words = -(-vocab // 32)
    mask_rows = case["masks"]
    # Grammars: some leave a handful of tokens, some close a few.
    open_share = [r.choice([0.002, 0.3, 0.98]) for _ in range(mask_rows)]
    bits = torch.zeros((mask_rows, words * 32), dtype=torch.int64, device="cuda")
    for i, share in enumerate(open_share):
        bits[i] = torch.rand(words * 32, device="cuda", generator=_gen(seed, 10 + i)) < share
    packed = (bits.view(mask_rows, words, 32) << torch.arange(32, device="cuda")).sum(-1) if mask_rows else bits[:, :words]
    starts = [0] + list(np.cumsum(nodes))
    s = dict(case=case, logits=_rows(seed, 3, (rows, vocab), 2.5),
             request=_ints([i for i, c in enumerate(nodes) for _ in range(c)]),
             rules=_ints(rules).view(n, 6), history=(text * vocab).to(torch.int32).clamp(max=vocab - 1), lengths=_ints(lengths),
             ids=(drafted * vocab).to(torch.int32).clamp(max=vocab - 1), row_start=_ints(starts),
             parents=_ints([r.randrange(max(0, i - 6), i) if i else -1 for c in nodes for i in range(c)]),
             bias_ids=_ints(ids or [0]), bias_values=_ints(values or [0]), biases=len(ids),
             masks=torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32),
             mask_of=_ints([r.randrange(-1, mask_rows) if mask_rows else -1 for _ in range(rows)]))
    s["out"] = torch.zeros_like(s["logits"])
    if own:
        from iris_amd import logits
        p = {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
        s["call"] = (logits, logits.LogitsRules(
            logits=p["logits"], out=p["out"], request=p["request"], rules=p["rules"], history=p["history"],
            lengths=p["lengths"], row_start=p["row_start"], ids=p["ids"], parents=p["parents"], bias_ids=p["bias_ids"],
            bias_values=p["bias_values"], masks=p["masks"] if mask_rows else None, mask_of=p["mask_of"] if mask_rows else None,
            status=None, rows=rows, first_row=0, vocab=vocab, logits_stride=vocab, out_stride=vocab, requests=n,
            history_stride=most, biases=len(ids), mask_rows=mask_rows, mask_stride=words))
    return s


def _drawings(case):
    """[row]: inverse temperature, k, p, the largest distance from the first (0: any)."""
    r = random.Random(case["mix"])
    out = []
    for _ in range(case["rows"]):
        kind = case["kind"] if case["kind"] != "mixed" else r.choice(["greedy", "plain", "top_k", "top_p", "both", "gap"])
        beta = 0 if kind == "greedy" else int(ONE / r.choice([0.3, 0.7, 0.8, 1.0, 1.5]))
        k = r.choice([1, 5, 40, 50, 1000]) if kind in ("top_k", "both") else 0
        p = int(r.choice([0.1, 0.5, 0.9, 0.95, 0.999]) * 2 ** 32) if kind in ("top_p", "both") else 0
        if case["kind"] == "both":
            k, p = 40, int(0.95 * 2 ** 32)
        # A distance of -ln(0.05) keeps tokens of at least a twentieth of the first's weight.
        out.append([beta, k, p, int(-math.log(r.choice([0.01, 0.05, 0.2])) * ONE) if kind == "gap" else 0])
    return out


def _words32(values):
    """Values of 32 bits without sign as the int32 of their bits."""
    return torch.from_numpy(np.array(values, dtype=np.int64).astype(np.uint32).view(np.int32)).cuda()


def _prepare_draw(case, seed):
    rows, vocab = case["rows"], case["vocab"]
    drawings = _drawings(case)
    random.Random(seed).shuffle(drawings)
    x = torch.randn((rows, vocab), device="cuda", generator=_gen(seed, 1)) * 2.0
    # A text's logits: most tokens unlikely, a few stand out, on some rows one far.
    lift = torch.rand((rows, 12), device="cuda", generator=_gen(seed, 2)) * 8 + 2
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 12), device="cuda", generator=_gen(seed, 3)), lift)
    logits = torch.round(x * ONE).to(torch.int32)
    if case["closed"]:
        share = torch.rand((rows, 1), device="cuda", generator=_gen(seed, 4)) ** 3
        logits[torch.rand((rows, vocab), device="cuda", generator=_gen(seed, 5)) > share + 2.0 / vocab] = LOWEST
    r = random.Random(seed + 1)
    s = dict(case=case, logits=logits, drawings=_words32(drawings).view(rows, 4), request=_ints(list(range(rows))),
             numbers=_words32([r.getrandbits(32) for _ in range(rows)]), tokens=_ints([0] * rows),
             mass=torch.zeros((rows, 2), dtype=torch.int64, device="cuda"))
    if own:
        from iris_amd import logits as calls
        d = calls.LogitsDraw(logits=s["logits"].data_ptr(), request=s["request"].data_ptr(),
                             drawings=s["drawings"].data_ptr(), numbers=s["numbers"].data_ptr(),
                             tokens=s["tokens"].data_ptr(), mass=s["mass"].data_ptr(), status=None, rows=rows, vocab=vocab,
                             logits_stride=vocab, requests=rows)
        size = calls.draw_workspace_bytes(d)
        s["call"] = (calls, d, torch.empty(size, dtype=torch.uint8, device="cuda"), size)
    return s


def prepare(case, seed):
    return {"adapters": _prepare_adapters, "rules": _prepare_rules, "draw": _prepare_draw}[case["op"]](case, seed)


# ------------------------------------------------------------------ the plain forms


def _rte(x, shift):
    """x / 2^shift, ties to even."""
    if shift == 0:
        return x
    low = x >> shift
    return low + ((x & ((1 << shift) - 1)) + (low & 1) > (1 << (shift - 1)))


def _div(x, n):
    """x / n for n > 0, ties to even."""
    q = torch.div(x, n, rounding_mode="floor")
    twice = (x - q * n) * 2
    return q + ((twice > n) | ((twice == n) & ((q & 1) == 1)))


def _plain_adapters(s):
    _, parts = PRODUCTS[s["case"]["product"]]
    out = s["y"].clone()
    for slot, rows in s["by_slot"]:
        at = torch.tensor(rows, device="cuda")
        x = s["x"][at].double()
        for (n, first, step), (a, b) in zip(parts, s["weights"][slot]):
            if not a.shape[0]:
                continue
            t = _rte((x @ a.double().T).to(torch.int64), s["a_bits"]).clamp(LOWEST, HIGHEST)
            u = _rte((t.double() @ b.double().T).to(torch.int64), s["b_bits"]).clamp(LOWEST, HIGHEST)
            columns = slice(first, first + (n - 1) * step + 1, step)
            out[at, columns] = (out[at, columns].long() + u).clamp(LOWEST, HIGHEST).int()
    return out


def _plain_rules(s):
    c = s["case"]
    vocab, rows, n = c["vocab"], s["logits"].shape[0], c["requests"]
    q = s["request"].long()
    rep, freq, pres, window, b0, bn = (s["rules"][:, i].long() for i in range(6))
    start, length = s["row_start"].long(), s["lengths"].long()
    row = torch.arange(rows, device="cuda")
    # Each row's ancestors, from itself up: their ids, and its own depth.
    up, paths = row, []
    for _ in range(c["nodes"]):
        paths.append(up)
        parent = torch.where(up >= 0, s["parents"].long()[up.clamp(min=0)], -1)
        up = torch.where(parent >= 0, start[q] + parent, -1)
    paths = torch.stack(paths, 1)
    depth = (paths >= 0).sum(1) - 1
    last = length[q] + depth  # the row's own position
    oldest = torch.where(window[q] > 0, last - window[q] + 1, 0)
    count = torch.zeros((rows, vocab + 1), dtype=torch.int64, device="cuda")
    at = torch.arange(s["history"].shape[1], device="cuda")
    seen = (at[None, :] < length[q][:, None]) & (at[None, :] >= oldest[:, None])
    ids = torch.where(seen, s["history"][q].long(), vocab)
    count.scatter_add_(1, ids, torch.ones_like(ids))
    place = last[:, None] - torch.arange(c["nodes"], device="cuda")
    seen = (paths >= 0) & (place >= oldest[:, None])
    ids = torch.where(seen, s["ids"].long()[paths.clamp(min=0)], vocab)
    count.scatter_add_(1, ids, torch.ones_like(ids))
    count = count[:, :vocab]
    l = s["logits"].long()
    rep = rep[q][:, None]
    l = torch.where(count > 0, torch.where(l > 0, _div(l << 16, rep), _rte(l * rep, 16)), l)
    l = l - count * freq[q][:, None] - (count > 0) * pres[q][:, None]
    if s["biases"]:
        entry = torch.arange(s["biases"], device="cuda")
        of = torch.searchsorted(b0 + bn, entry, right=True)
        bias = torch.zeros((n, vocab), dtype=torch.int64, device="cuda")
        bias.view(-1).scatter_add_(0, of * vocab + s["bias_ids"].long(), s["bias_values"].long())
        l = l + bias[q]
    l = l.clamp(LOWEST + 1, HIGHEST)
    if c["masks"]:
        v = torch.arange(vocab, device="cuda")
        is_open = ((s["masks"].long()[:, v // 32] >> (v % 32)) & 1) == 1
        of = s["mask_of"].long()
        l = torch.where((of < 0)[:, None] | is_open[of.clamp(min=0)], l, LOWEST)
    return l.int()


def _exp(diff):
    """exp of -diff / 2^16 in 32 fraction bits."""
    d = diff.clamp(max=1 << 20) << 16
    k = torch.div(d, LN2, rounding_mode="floor")
    r = d - k * LN2
    r2 = _rte(r * r, 32)
    r3 = _rte(r2 * r, 32)
    r4 = _rte(r3 * r, 32)
    e = (1 << 32) - r + _div(r2, 2) - _div(r3, 6) + _div(r4, 24) - _div(_rte(r4 * r, 32), 120)
    low = e >> k
    half = (1 << k) >> 1
    e = low + ((e - (low << k)) + (low & 1) > half) * (k > 0)
    return e * (diff < (1 << 20))


def _scaled_floor(value, share):
    """value share / 2^32, rounded down, and whether anything was cut off; value below 2^52."""
    high, low = (value >> 32) * share, (value & 0xFFFFFFFF) * (share >> 16)
    rest = (value & 0xFFFFFFFF) * (share & 0xFFFF)
    total = low + (rest >> 16)
    return high + (total >> 16), ((total & 0xFFFF) | (rest & 0xFFFF)) != 0


def _plain_draw(s):
    beta, k, p, most = (s["drawings"][:, i].long() & 0xFFFFFFFF for i in range(4))
    number = s["numbers"].long() & 0xFFFFFFFF
    l, index = torch.sort(s["logits"].long(), dim=1, descending=True, stable=True)
    is_open = l > LOWEST
    gap = l[:, :1] - l
    gap = _rte(torch.minimum(gap, torch.full_like(gap, (1 << 31) - 1)) * beta[:, None], 16).clamp(max=1 << 20)
    e = _exp(gap) * is_open * ((most == 0)[:, None] | (gap <= most[:, None]))
    place = torch.arange(l.shape[1], device="cuda")[None, :]
    e = e * ((k == 0)[:, None] | (place < k[:, None]))
    total = e.cumsum(1)
    whole, cut = _scaled_floor(total[:, -1], p)
    before = total - e
    e = e * ((p == 0)[:, None] | (before < (whole + cut)[:, None]))
    total = e.cumsum(1)
    target, _ = _scaled_floor(total[:, -1], number)
    at = (total > target[:, None]).to(torch.int8).argmax(1)
    at = torch.where(beta == 0, 0, at)[:, None]
    some = is_open[:, 0]
    token = torch.where(some, index.gather(1, at)[:, 0], -1).int()
    full = torch.full_like(beta, 1 << 32)
    mass = torch.stack([torch.where(beta == 0, full, e.gather(1, at)[:, 0]), torch.where(beta == 0, full, total[:, -1])], 1)
    return {"tokens": token, "mass": mass * some[:, None]}


# ------------------------------------------------------------------ the framework's calls


def _own(s):
    stream = torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "adapters":
        bank, call, space, size = s["call"]
        if s["between"]:
            s["out"].copy_(s["y"])
        bank.apply(call, space.data_ptr(), size, stream)
        return s["out"]
    if op == "rules":
        calls, call = s["call"]
        calls.apply_rules(call, stream)
        return s["out"]
    calls, call, space, size = s["call"]
    calls.draw(call, space.data_ptr(), size, stream)
    return {"tokens": s["tokens"], "mass": s["mass"]}


def run(state):
    if own:
        return _own(state)
    return {"adapters": _plain_adapters, "rules": _plain_rules, "draw": _plain_draw}[state["case"]["op"]](state)


def work(case):
    if case["op"] == "adapters":
        cols, parts = PRODUCTS[case["product"]]
        counts, slots, ranks = _parts(case["rows"], case["requests"], case["mix"]), _request_slots(case), _ranks(case)
        width = -(-(max(first + (n - 1) * step for n, first, step in parts) + 1) // 4) * 4
        weights = sum(2 * rank * (cols + p[0]) for t in set(slots) if t >= 0 for rank, p in zip(ranks[t], parts))
        macs = sum(c * rank * (cols + p[0]) for c, t in zip(counts, slots) if t >= 0 for rank, p in zip(ranks[t], parts))
        adapted = sum(c for c, t in zip(counts, slots) if t >= 0)
        return {"bytes": 4 * adapted * cols + 8 * case["rows"] * width + 4 * case["rows"] + weights, "flops": 2 * macs}
    if case["op"] == "rules":
        lengths, nodes = _lengths_and_nodes(case)
        rows = sum(nodes)
        return {"bytes": 8 * rows * case["vocab"] + case["masks"] * case["vocab"] // 8 + 4 * sum(lengths), "flops": 0}
    return {"bytes": 4 * case["rows"] * case["vocab"] + 44 * case["rows"], "flops": 0}


# ------------------------------------------------------------------ 64 bits


def _nearest(num, den):
    """num / den to the nearest integer, ties to even, for den > 0 (numpy int64)."""
    q = num // den
    over = 2 * (num - q * den) - den
    return q + ((over > 0) | ((over == 0) & (q % 2 != 0)))


def _clip32(x):
    return np.clip(x, LOWEST, HIGHEST)


def _products(x, w):
    """Exact integer products x w^T (int64 tensors) from the halves of x."""
    high, low = (x >> 12).double(), (x & 4095).double()
    w = w.double().T.contiguous()
    return ((high @ w).to(torch.int64) * 4096 + (low @ w).to(torch.int64)).cpu().numpy()


def _exact_adapters(s):
    _, parts = PRODUCTS[s["case"]["product"]]
    out = s["y"].cpu().numpy().astype(np.int64)
    for r0 in range(0, out.shape[0], 512):
        slots = s["slots"][r0:r0 + 512].cpu().numpy()
        for t in range(s["case"]["slots"]):
            at = r0 + np.nonzero(slots == t)[0]
            if not at.size:
                continue
            x = s["x"][torch.from_numpy(at).cuda()].long()
            for (n, first, step), (a, b) in zip(parts, s["weights"][t]):
                if a.shape[0]:
                    low = _clip32(_nearest(_products(x, a.long()), 2 ** s["a_bits"]))
                    add = _clip32(_nearest(_products(torch.from_numpy(low).cuda(), b.long()), 2 ** s["b_bits"]))
                    for_part = first + step * np.arange(n)
                    out[at[:, None], for_part] = _clip32(out[at[:, None], for_part] + add)
    return out.astype(np.int32)


def _exact_rules(s):
    vocab = s["case"]["vocab"]
    logits = s["logits"].cpu().numpy().astype(np.int64)
    rules, history, lengths, starts, ids, parents, of, words = (
        s[k].cpu().numpy() for k in ("rules", "history", "lengths", "row_start", "ids", "parents", "mask_of", "masks"))
    b_ids, b_values = s["bias_ids"].cpu().numpy(), s["bias_values"].cpu().numpy()
    for q in range(len(lengths)):
        rep, freq, pres, window, b0, bn = (int(v) for v in rules[q])
        for i in range(starts[q], starts[q + 1]):
            path, at = [], i - starts[q]
            while at >= 0:
                path.append(ids[starts[q] + at])
                at = parents[starts[q] + at]
            text = np.concatenate([history[q, :lengths[q]], np.array(path[::-1], dtype=np.int32)])
            if window:
                text = text[-window:]
            token, count = np.unique(text, return_counts=True)
            v = logits[i, token]
            v = np.where(v > 0, _nearest(v * 65536, rep), _nearest(v * rep, 65536))
            logits[i, token] = v - count * freq - pres
            np.add.at(logits[i], b_ids[b0:b0 + bn], b_values[b0:b0 + bn])
            logits[i] = np.clip(logits[i], LOWEST + 1, HIGHEST)
            if of[i] >= 0:
                is_open = np.unpackbits(words[of[i]].view(np.uint8), bitorder="little")[:vocab]
                logits[i, is_open == 0] = LOWEST
    return logits.astype(np.int32)


def _exact_term(gap):
    """exp(-gap / 2^16) in 32 fraction bits, gap below 2^20 (numpy int64)."""
    wide = gap * 65536
    octave, r = wide // LN2, (wide % LN2).astype(np.uint64)
    power = [r]
    for _ in range(4):
        # power r / 2^32 of two values below 2^32: the product fits 64 bits without sign
        prod = power[-1] * r
        q, rest = prod >> np.uint64(32), prod & np.uint64(0xFFFFFFFF)
        half = np.uint64(1 << 31)
        power.append(q + ((rest > half) | ((rest == half) & (q % np.uint64(2) == 1))))
    _, r2, r3, r4, r5 = (v.astype(np.int64) for v in power)
    e = 2 ** 32 - r.astype(np.int64) + _nearest(r2, 2) - _nearest(r3, 6) + _nearest(r4, 24) - _nearest(r5, 120)
    return _nearest(e, 2 ** octave)


def _exact_draw(s):
    logits = s["logits"].cpu().numpy().astype(np.int64)
    drawings = s["drawings"].cpu().numpy().view(np.uint32)
    numbers = s["numbers"].cpu().numpy().view(np.uint32)
    tokens, mass = [], []
    for i, l in enumerate(logits):
        beta, k, p, most = (int(v) for v in drawings[i])
        order = np.lexsort((np.arange(l.size), -l))
        order = order[l[order] > LOWEST]
        if not order.size:
            tokens.append(-1)
            mass.append((0, 0))
            continue
        if beta == 0:
            tokens.append(int(order[0]))
            mass.append((1 << 32, 1 << 32))
            continue
        if k:
            order = order[:k]
        gap = _nearest((l[order[0]] - l[order]) * beta, 65536)
        gap = gap[gap <= (most or HIGHEST)]
        gap = gap[gap < 1 << 20]
        terms = _exact_term(gap)
        if p:
            need = -(-p * int(terms.sum()) >> 32)
            terms = terms[:np.searchsorted(np.cumsum(terms), need) + 1]
        whole = int(terms.sum())
        at = int(np.searchsorted(np.cumsum(terms), whole * int(numbers[i]) >> 32, side="right"))
        tokens.append(int(order[at]))
        mass.append((int(terms[at]), whole))
    return {"tokens": np.array(tokens, dtype=np.int32), "mass": np.array(mass, dtype=np.int64)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"adapters": _exact_adapters, "rules": _exact_rules, "draw": _exact_draw}[case["op"]](s)
