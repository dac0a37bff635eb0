"""The measured cases of the operators that serve several requests over one
paged cache of keys and values.

Four kinds of call:

- ``plan``: the block tables, slot map, row starts and positions of a pass,
  from the requests' lengths and the rows each adds.
- ``store``: a pass's keys and values into their pages, by the slot map.
- ``packed``: causal attention over whole prompts of different lengths, packed
  row after row.
- ``tree``: attention of each request's drafted tokens (a tree of them, or the
  one token of a decode step) over its cached positions and over the drafted
  tokens above it in its tree.

All values are Q16.16 integers, and every result is an integer that the
arithmetic fixes bit for bit: wrapping 64-bit dot products, scores rounded to
even, exponentials in 32 fraction bits from a five-term series rounded at each
step, weights rounded to even, and what the weights lack of one on the first
largest score.

``run`` takes what ``prepare`` made; with ``own`` false it computes the
operators with elementary torch operations. Products of the matrices there are
in float64 and exact: |q| and |k| stay below 2^21 and |v| below 2^21, so a sum
over 512 dimensions or over weights that add to about 2^16 stays below 2^53.
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

# (query heads, key heads, head size, scaled): the benchmark's two models, a
# small head, one that is not a power of two, and the widest head.
HEADS = [(32, 8, 128, True), (8, 1, 256, False), (4, 2, 64, True), (12, 4, 80, True), (8, 2, 512, False)]


def listed():
    m = dict(heads=32, kv_heads=8, head_dim=128, scaled=True)
    g = dict(heads=8, kv_heads=1, head_dim=256, scaled=False)
    return [
        # Before a decode step of a few requests: one row each.
        dict(name="plan_8_decode", op="plan", requests=8, rows=8, longest=900, page=16, mix=1),
        # Before the prompts of a full server: ragged rows, some requests done.
        dict(name="plan_2048_ragged", op="plan", requests=2048, rows=60011, longest=8000, page=16, mix=2),
        # A decode step's keys and values of one layer.
        dict(name="store_8rows", op="store", rows=8, kv_heads=8, head_dim=128, page=16, mix=3),
        # A large packed pass's keys and values of one layer.
        dict(name="store_6007rows", op="store", rows=6007, kv_heads=8, head_dim=128, page=64, mix=4),
        # One very short prompt.
        dict(name="packed_13rows", op="packed", seqs=1, rows=13, window=0, mix=5, **m),
        # A few prompts through a sliding-window layer of wide heads.
        dict(name="packed_9seqs_1501rows_window", op="packed", seqs=9, rows=1501, window=512, mix=6, **g),
        # A ragged set of prompts, some of a few tokens.
        dict(name="packed_19seqs_2309rows", op="packed", seqs=19, rows=2309, window=0, mix=7, **m),
        # One long prompt.
        dict(name="packed_4096rows", op="packed", seqs=1, rows=4096, window=0, mix=8, **m),
        # One token of one request: a decode step's latency.
        dict(name="tree_1x1_at_700", op="tree", requests=1, nodes=1, longest=700, window=0, page=16, mix=9, **m),
        # Drafted trees of a dozen requests, sliding window, wide heads.
        dict(name="tree_12x9_at_2100_window", op="tree", requests=12, nodes=9, longest=2100, window=1024, page=32,
             mix=10, **g),
        # One token each of a few requests late in long texts.
        dict(name="tree_4x1_at_32700", op="tree", requests=4, nodes=1, longest=32700, window=0, page=64, mix=11, **m),
        # Drafted trees of many requests.
        dict(name="tree_32x25_at_8000", op="tree", requests=32, nodes=25, longest=8000, window=0, page=16, mix=12, **m),
    ]


def _log(rng, lo, hi):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(round(v))))


def draw(rng):
    op = rng.choice(["plan", "store", "packed", "packed", "packed", "tree", "tree", "tree"])
    mix = rng.randrange(1, 1 << 30)
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "plan":
        requests = _log(rng, 1, 2048)
        return dict(op=op, requests=requests, rows=_log(rng, requests, max(requests, 60000)),
                    longest=_log(rng, 16, 8000), page=page, mix=mix)
    heads, kv_heads, head_dim, scaled = rng.choice(HEADS)
    if op == "store":
        return dict(op=op, rows=_log(rng, 1, 6000), kv_heads=kv_heads, head_dim=head_dim, page=page, mix=mix)
    h = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, scaled=scaled)
    window = 0 if rng.random() < 0.6 else _log(rng, 16, 2048)
    if op == "packed":
        rows = _log(rng, 1, 3500)
        return dict(op=op, seqs=_log(rng, 1, min(64, rows)), rows=rows, window=window, mix=mix, **h)
    requests, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
    # At most as many scores and cached positions as the largest listed case.
    most = min(32768, 32 * 25 * 8000 * 32 // (requests * nodes * heads), 32 * 8000 * 1024 // (requests * kv_heads * head_dim))
    return dict(op=op, requests=requests, nodes=nodes, longest=_log(rng, 1, max(1, most)), window=window, page=page,
                mix=mix, **h)


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


def _trees(case):
    """Each request's cached length and drafted tokens: the first the longest
    of each, the others ragged."""
    r = random.Random(case["mix"])
    lengths, nodes = [case["longest"]], [case["nodes"]]
    for _ in range(case["requests"] - 1):
        lengths.append(_log(r, max(1, case["longest"] // 16), case["longest"]))
        nodes.append(r.randrange(1, case["nodes"] + 1))
    return lengths, nodes


def _shuffled(seed, *lists):
    """The lists in one new order, which another seed makes another."""
    order = list(range(len(lists[0])))
    random.Random(seed).shuffle(order)
    return [[x[i] for i in order] for x in lists]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(counts):
    return _ints([0] + list(np.cumsum(counts)))


def _plan_inputs(case, seed):
    """Lengths, rows added, pages held, the table, the ring of free pages."""
    r = random.Random(case["mix"])
    n, page = case["requests"], case["page"]
    added = _parts(case["rows"], n, case["mix"])
    lengths = [_log(r, 1, case["longest"]) for _ in range(n)]
    held = [-(-x // page) for x in lengths]
    if case["rows"] > 4 * n:  # prompts: most requests are new, some are done
        for i in range(n):
            if r.random() < 0.8:
                lengths[i] = held[i] = 0
            elif r.random() < 0.2:
                held[i] += 3
        for i in range(1, n, 7):
            added[0] += added[i]
            lengths[i] = added[i] = 0
    lengths, added, held = _shuffled(seed, lengths, added, held)
    need = [-(-(x + a) // page) for x, a in zip(lengths, added)]
    pages = sum(max(a, b) for a, b in zip(need, held)) * 9 // 8 + 4
    stride = max(max(need), max(held)) + 1
    order = list(range(pages))
    random.Random(seed + 1).shuffle(order)
    table, at = np.full((n, stride), -1, dtype=np.int32), 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    free = order[at:]
    head = random.Random(seed + 2).randrange(pages)
    ring = np.zeros(pages, dtype=np.int32)
    for i, p in enumerate(free):
        ring[(head + i) % pages] = p
    return lengths, added, held, table, ring, head, len(free), pages, stride


def prepare(case, seed):
    s = dict(case=case)
    if case["op"] == "plan":
        lengths, added, held, table, ring, head, free, pages, stride = _plan_inputs(case, seed)
        rows = sum(added)
        s.update(lengths=_ints(lengths), added=_ints(added), held=_ints(held), table=torch.from_numpy(table).cuda(),
                 ring=torch.from_numpy(ring).cuda(), ring_state=_ints([head, free]), pages=pages, stride=stride,
                 max_rows=rows + 5, held_out=_ints([0] * len(held)), ring_state_out=_ints([0, 0]),
                 row_start=_ints([0] * (len(held) + 1)), slots=_ints([0] * (rows + 5)),
                 positions=_ints([0] * (rows + 5)), status=_ints([0]))
        return s
    if case["op"] == "store":
        rows, page, width = case["rows"], case["page"], case["kv_heads"] * case["head_dim"]
        pages = -(-rows // page) * 5 // 4 + 3
        slots = list(range(pages * page))
        random.Random(seed).shuffle(slots)
        shape = (pages, case["kv_heads"], page, case["head_dim"])
        s.update(k=_rows(seed, 1, (rows, width), 1.0), v=_rows(seed, 2, (rows, width), 1.0), slots=_ints(slots[:rows]),
                 k_pages=_rows(seed, 3, shape, 1.0), v_pages=_rows(seed, 4, shape, 1.0), pages=pages)
        return s
    heads, kv_heads, hd = case["heads"], case["kv_heads"], case["head_dim"]
    # Scores of standard deviation two.
    q_sigma = 2.0 if case["scaled"] else 2.0 / math.sqrt(hd)
    s["scale"] = math.isqrt((1 << 64) // hd) if case["scaled"] else 0  # 2^32 / sqrt(head size)
    if case["op"] == "packed":
        rows = case["rows"]
        counts, = _shuffled(seed, _parts(rows, case["seqs"], case["mix"]))
        s.update(q=_rows(seed, 1, (rows, heads * hd), q_sigma), k=_rows(seed, 2, (rows, kv_heads * hd), 1.0),
                 v=_rows(seed, 3, (rows, kv_heads * hd), 1.0), row_start=_starts(counts), longest=max(counts))
    else:
        lengths, nodes = _shuffled(seed, *_trees(case))
        rows, page = sum(nodes), case["page"]
        held = [-(-(x + n) // page) for x, n in zip(lengths, nodes)]
        pages = sum(held) * 9 // 8 + 2
        order = list(range(pages))
        random.Random(seed + 1).shuffle(order)
        table, at = np.zeros((len(held), max(held) + 1), dtype=np.int32), 0
        for i, h in enumerate(held):
            table[i, :h] = order[at:at + h]
            at += h
        r = random.Random(seed + 2)
        parents = [r.randrange(max(0, i - 6), i) if i else -1 for n in nodes for i in range(n)]
        shape = (pages, kv_heads, page, hd)
        s.update(q=_rows(seed, 1, (rows, heads * hd), q_sigma), k_pages=_rows(seed, 2, shape, 1.0),
                 v_pages=_rows(seed, 3, shape, 1.0), table=torch.from_numpy(table).cuda(), lengths=_ints(lengths),
                 row_start=_starts(nodes), parents=_ints(parents), pages=pages,
                 longest=max(x + n for x, n in zip(lengths, nodes)))
    s["out"] = torch.zeros((rows, heads * hd), dtype=torch.int32, device="cuda")
    return s


# ------------------------------------------------------------------ the plain forms


def _rte(x, shift):
    """x / 2^shift, ties to even."""
    low = x >> shift
    return low + ((x & ((1 << shift) - 1)) + (low & 1) > (1 << (shift - 1)))


def _div(x, n):
    """x / n for x >= 0, ties to even."""
    q = torch.div(x, n, rounding_mode="floor")
    twice = (x - q * n) * 2
    return q + ((twice > n) | ((twice == n) & ((q & 1) == 1)))


def _score(dot, scale):
    """The scores of float64 dot products that are whole."""
    s = dot.to(torch.int64)
    if scale:
        s = (s >> 32) * scale + (((s & 0xFFFFFFFF) * scale) >> 32)
    return _rte(s, 16).clamp_(LOWEST, HIGHEST)


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


def _weights(score, visible):
    """Softmax weights in 16 fraction bits along the last axis; a row that
    sees nothing has none."""
    top = torch.where(visible, score, LOWEST - 1).amax(-1, keepdim=True)
    e = _exp((top - score).clamp_(min=0)) * visible
    total = e.sum(-1, keepdim=True).clamp_(min=1)
    # (e << 32) / total in two steps of 16 bits, then ties to even twice
    q = torch.div(e << 16, total, rounding_mode="floor")
    rest = ((e << 16) - q * total) << 16
    low = torch.div(rest, total, rounding_mode="floor")
    q = (q << 16) + low
    twice = (rest - low * total) * 2
    w = _rte(q + ((twice > total) | ((twice == total) & ((q & 1) == 1))), 16)
    first = (visible & (score == top)).to(torch.int8).argmax(-1, keepdim=True)
    return w.scatter_add(-1, first, ONE - w.sum(-1, keepdim=True)) * visible


def _context(weights, values):
    """Weighted values, ties to even; a key head's rows by a batched product."""
    return _rte((weights.double() @ values).to(torch.int64), 16).clamp_(LOWEST, HIGHEST).to(torch.int32)


def _plain_plan(s):
    page, pages, stride = s["case"]["page"], s["pages"], s["stride"]
    length, add, held = s["lengths"].long(), s["added"].long(), s["held"].long()
    need = (length + add + page - 1) // page
    grow, back = (need - held).clamp(min=0), (held - need).clamp(min=0)
    head, free = s["ring_state"][0].long(), s["ring_state"][1].long()
    starts = torch.cat([add.new_zeros(1), add.cumsum(0)])
    ok = (starts[-1] <= s["max_rows"]) & (need.amax() <= stride) & (grow.sum() <= free)
    col = torch.arange(stride, device="cuda")[None, :]
    pop = (grow.cumsum(0) - grow)[:, None] + col - held[:, None]
    fresh = (col >= held[:, None]) & (col < need[:, None]) & ok
    table = torch.where(fresh, s["ring"][(head + pop) % pages], s["table"])
    push = (head + free + (back.cumsum(0) - back)[:, None] + col - need[:, None]) % pages
    put = torch.where((col >= need[:, None]) & (col < held[:, None]) & ok, push, pages)
    ring = torch.cat([s["ring"], s["ring"].new_zeros(1)]).scatter(0, put.reshape(-1), s["table"].reshape(-1))[:pages]
    row = torch.arange(s["max_rows"], device="cuda")
    b = (torch.searchsorted(starts, row, right=True) - 1).clamp(max=length.numel() - 1)
    pos = length[b] + row - starts[b]
    slot = table[b, (pos // page).clamp(max=stride - 1)].long() * page + pos % page
    used = (row < starts[-1]) & ok
    state = torch.stack([(head + grow.sum()) % pages, free - grow.sum() + back.sum()])
    return {"table": table, "held": torch.where(ok, need, held).int(), "ring": ring,
            "ring_state": torch.where(ok, state, torch.stack([head, free])).int(),
            "row_start": torch.where(ok, starts, 0).int(), "slots": torch.where(used, slot, -1).int(),
            "positions": torch.where(used, pos, -1).int(), "status": torch.where(ok, 0, -5).int().reshape(1)}


def _plain_store(s):
    c = s["case"]
    slot = s["slots"].long()
    shape = (c["rows"], c["kv_heads"], c["head_dim"])
    s["k_pages"][slot // c["page"], :, slot % c["page"]] = s["k"].view(shape)
    s["v_pages"][slot // c["page"], :, slot % c["page"]] = s["v"].view(shape)
    return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_packed(s):
    c = s["case"]
    rows, heads, kv_heads, hd = c["rows"], c["heads"], c["kv_heads"], c["head_dim"]
    group = heads // kv_heads
    at = torch.arange(rows, device="cuda")
    start = s["row_start"].long()[torch.searchsorted(s["row_start"].long(), at, right=True) - 1]
    lowest = torch.maximum(start, at + 1 - c["window"]) if c["window"] else start
    seen = (at[None, :] >= lowest[:, None]) & (at[None, :] <= at[:, None])
    q = s["q"].view(rows, kv_heads, group, hd).permute(1, 2, 0, 3).double().reshape(kv_heads, group * rows, hd)
    k = s["k"].view(rows, kv_heads, hd).permute(1, 2, 0).double().contiguous()
    v = s["v"].view(rows, kv_heads, hd).permute(1, 0, 2).double().contiguous()
    score = _score(q @ k, s["scale"]).view(kv_heads, group, rows, rows)
    w = _weights(score, seen).view(kv_heads, group * rows, rows)
    return _context(w, v).view(heads, rows, hd).permute(1, 0, 2).reshape(rows, heads * hd)


def _plain_tree(s):
    c = s["case"]
    n, heads, kv_heads, hd, most = c["requests"], c["heads"], c["kv_heads"], c["head_dim"], c["nodes"]
    group, rows = heads // kv_heads, s["q"].shape[0]
    starts, length = s["row_start"].long(), s["lengths"].long()
    count = starts[1:] - starts[:-1]
    node = torch.arange(most, device="cuda")
    row = (starts[:-1, None] + node).clamp(max=rows - 1)  # [request][node]
    parent = torch.where(node < count[:, None], s["parents"].long()[row], -1)
    # A node's ancestors and itself: the paths of I + (child -> parent).
    step = torch.eye(most, device="cuda", dtype=torch.float64) + (parent[:, :, None] == node)
    above = torch.linalg.matrix_power(step, 63) > 0
    place = length[:, None] + above.sum(-1) - 1
    key = torch.arange(s["table"].shape[1] * c["page"], device="cuda")
    drafted = key[None, :] - length[:, None]
    up = torch.gather(above, 2, drafted.clamp(0, most - 1)[:, None, :].expand(-1, most, -1))
    # The position a key stands for: its own, or its node's place in the tree.
    at = torch.where(drafted < 0, key[None, :], torch.gather(place, 1, drafted.clamp(0, most - 1)))
    seen = torch.where((drafted < 0)[:, None, :], True, up & (drafted < count[:, None])[:, None, :])
    if c["window"]:
        seen = seen & (at[:, None, :] + c["window"] > place[:, :, None])
    q = s["q"].view(rows, kv_heads, group, hd)[row].permute(0, 2, 1, 3, 4).double().reshape(n, kv_heads, most * group, hd)
    pages = s["table"].long()
    k = s["k_pages"][pages].permute(0, 2, 4, 1, 3).double().reshape(n, kv_heads, hd, -1)
    score = _score(q @ k, s["scale"])
    seen = seen[:, None, :, None, :].expand(-1, 1, -1, group, -1).reshape(n, 1, most * group, -1)
    w = _weights(score, seen)
    v = s["v_pages"][pages].permute(0, 2, 1, 3, 4).double().reshape(n, kv_heads, -1, hd)
    ctx = _context(w, v).view(n, kv_heads, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n * most, heads * hd)
    b = torch.searchsorted(starts, torch.arange(rows, device="cuda"), right=True) - 1
    return ctx[b * most + torch.arange(rows, device="cuda") - starts[b]]


# ------------------------------------------------------------------ the framework's calls


def _call(s):
    """The descriptors and the work space that a program makes once."""
    from iris_amd import paged
    c, p = s["case"], {k: v.data_ptr() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if c["op"] == "plan":
        return paged, paged.PagedPlan(
            lengths=p["lengths"], added=p["added"], parents=None, held=p["held"], held_out=p["held_out"],
            table=p["table"], ring=p["ring"], ring_state=p["ring_state"], ring_state_out=p["ring_state_out"],
            row_start=p["row_start"], slots=p["slots"], positions=p["positions"], status=p["status"],
            requests=c["requests"], table_stride=s["stride"], pages=s["pages"], page_size=c["page"],
            max_rows=s["max_rows"])
    if c["op"] == "packed":
        width = c["kv_heads"] * c["head_dim"]
        a = paged.PackedAttention(
            q=p["q"], k=p["k"], v=p["v"], out=p["out"], row_start=p["row_start"], status=None,
            q_stride=c["heads"] * c["head_dim"], k_stride=width, v_stride=width, out_stride=c["heads"] * c["head_dim"],
            sequences=c["seqs"], rows=c["rows"], max_length=s["longest"], heads=c["heads"], kv_heads=c["kv_heads"],
            head_dim=c["head_dim"], window=c["window"], scaled=int(c["scaled"]), scale_q32=s["scale"])
        size = paged.packed_workspace_bytes(a)
        return paged, a, torch.empty(size, dtype=torch.uint8, device="cuda"), size
    cache = paged.PagedKv(k=p["k_pages"], v=p["v_pages"], pages=s["pages"], page_size=c["page"], kv_heads=c["kv_heads"],
                          head_dim=c["head_dim"])
    if c["op"] == "store":
        return paged, cache
    a = paged.TreeAttention(
        q=p["q"], out=p["out"], row_start=p["row_start"], lengths=p["lengths"], parents=p["parents"], table=p["table"],
        status=None, q_stride=c["heads"] * c["head_dim"], out_stride=c["heads"] * c["head_dim"],
        requests=c["requests"], rows=s["q"].shape[0], table_stride=s["table"].shape[1], max_nodes=c["nodes"],
        max_positions=s["longest"], heads=c["heads"], window=c["window"], scaled=int(c["scaled"]), scale_q32=s["scale"])
    size = paged.tree_workspace_bytes(cache, a)
    return paged, cache, a, torch.empty(size, dtype=torch.uint8, device="cuda"), size


def _own(s):
    if "call" not in s:
        s["call"] = _call(s)
    paged, *call = s["call"]
    stream = torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "plan":
        paged.plan(call[0], stream)
        return {"table": s["table"], "held": s["held_out"], "ring": s["ring"], "ring_state": s["ring_state_out"],
                "row_start": s["row_start"], "slots": s["slots"], "positions": s["positions"], "status": s["status"]}
    if op == "store":
        width = s["k"].shape[1]
        paged.store(call[0], s["k"].data_ptr(), width, s["v"].data_ptr(), width, s["slots"].data_ptr(),
                    s["k"].shape[0], stream)
        return {"k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    if op == "packed":
        a, space, size = call
        paged.attend_packed(a, space.data_ptr(), size, stream)
    else:
        cache, a, space, size = call
        paged.attend_tree(cache, a, space.data_ptr(), size, stream)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "plan":
        return _plain_plan(state)
    if op == "store":
        return _plain_store(state)
    return _plain_packed(state) if op == "packed" else _plain_tree(state)


def work(case):
    if case["op"] == "plan":
        lengths, added, held, table, _, _, _, _, _ = _plan_inputs(case, 0)
        need = [-(-(x + a) // case["page"]) for x, a in zip(lengths, added)]
        moved = sum(abs(a - b) for a, b in zip(need, held))
        return {"bytes": 4 * (5 * len(held) + 2 * moved + 2 * sum(added)), "flops": 0}
    if case["op"] == "store":
        return {"bytes": case["rows"] * (16 * case["kv_heads"] * case["head_dim"] + 4), "flops": 0}
    width, kv = case["heads"] * case["head_dim"], case["kv_heads"] * case["head_dim"]
    window = case["window"] or 1 << 30
    if case["op"] == "packed":
        pairs = 0
        for n in _parts(case["rows"], case["seqs"], case["mix"]):
            m = min(n, window)
            pairs += m * (m + 1) // 2 + (n - m) * m
        return {"bytes": 8 * case["rows"] * (width + kv), "flops": 4 * pairs * width}
    lengths, nodes = _trees(case)
    # A drafted row sees its context and, of its tree, its ancestors (a few; itself counted).
    pairs = sum(n * min(x + 1, window) for x, n in zip(lengths, nodes))
    keys = sum(min(x, window) + n for x, n in zip(lengths, nodes))
    return {"bytes": 8 * keys * kv + 8 * sum(nodes) * width, "flops": 4 * pairs * width}


# ------------------------------------------------------------------ 64 bits


def _even(num, den):
    """num / den to the nearest integer, ties to even, for num >= 0 < den."""
    q = num // den
    over = 2 * (num - q * den) - den
    return torch.where(over > 0, q + 1, torch.where((over == 0) & (q % 2 == 1), q + 1, q))


def _dots(q, k):
    """Exact integer products [rows][keys] from 16-bit halves of the keys."""
    high, low = (k >> 16).double(), (k & 65535).double()
    q = q.double()
    return (q @ high.T).to(torch.int64) * 65536 + (q @ low.T).to(torch.int64)


def _exact_rows(q, k, v, seen, scale):
    """Attention of the rows [n][hd] over keys [m][hd], from the definition."""
    dot = _dots(q, k)
    if scale:
        # floor(dot * scale / 2^32) in three 16-bit pieces of the dot product
        a, b, c = dot >> 32, (dot >> 16) & 65535, dot & 65535
        dot = a * scale + ((b * scale * 65536 + c * scale) >> 32)
    whole, part = dot >> 16, dot & 65535
    score = whole + torch.where((part > 32768) | ((part == 32768) & (whole % 2 != 0)), 1, 0)
    score = score.clamp(LOWEST, HIGHEST)
    hidden = ~seen
    top = score.masked_fill(hidden, LOWEST - 1).max(dim=1, keepdim=True).values
    gap = (top - score).masked_fill(hidden, 1 << 20).clamp(max=1 << 20) * 65536
    octave = gap // LN2
    r = gap % LN2
    power = [None, r]
    for _ in range(4):
        power.append(_even(power[-1] * r, 1 << 32) if r.numel() else r)
    e = (1 << 32) - r + _even(power[2], 2) - _even(power[3], 6) + _even(power[4], 24) - _even(power[5], 120)
    e = _even(e, 2 ** octave).masked_fill(gap >= 1 << 36, 0)
    total = e.sum(dim=1, keepdim=True)
    # 2^32 e / total bit group by bit group: eight bits at a time
    quotient, rest = e // total, e % total
    for _ in range(4):
        quotient = quotient * 256 + rest * 256 // total
        rest = rest * 256 % total
    quotient = quotient + torch.where((2 * rest > total) | ((2 * rest == total) & (quotient % 2 == 1)), 1, 0)
    w = _even(quotient, 65536)
    best = (score == top) & seen
    best = best & (best.cumsum(dim=1) == 1)
    w = w + best * (65536 - w.sum(dim=1, keepdim=True))
    high, low = (v >> 16).double(), (v & 65535).double()
    total = (w.double() @ high).to(torch.int64) * 65536 + (w.double() @ low).to(torch.int64)
    whole, part = total >> 16, total & 65535
    out = whole + torch.where((part > 32768) | ((part == 32768) & (whole % 2 != 0)), 1, 0)
    return out.clamp(LOWEST, HIGHEST).to(torch.int32)


def _exact_plan(s):
    page, pages = s["case"]["page"], s["pages"]
    lengths, added, held = (s[k].tolist() for k in ("lengths", "added", "held"))
    table, ring = s["table"].cpu().numpy().copy(), s["ring"].tolist()
    head, free = s["ring_state"].tolist()
    slots, positions, starts, out = [], [], [0], []
    taken, given = 0, []
    for i, (x, a, h) in enumerate(zip(lengths, added, held)):
        need = -(-(x + a) // page)
        for j in range(h, need):
            table[i, j] = ring[(head + taken) % pages]
            taken += 1
        given += [int(table[i, j]) for j in range(need, h)]
        for p in range(x, x + a):
            slots.append(int(table[i, p // page]) * page + p % page)
            positions.append(p)
        starts.append(starts[-1] + a)
        out.append(need)
    for j, p in enumerate(given):
        ring[(head + free + j) % pages] = p
    fill = [-1] * (s["max_rows"] - len(slots))
    return {"table": torch.from_numpy(table), "held": _ints(out), "ring": _ints(ring),
            "ring_state": _ints([(head + taken) % pages, free - taken + len(given)]), "row_start": _ints(starts),
            "slots": _ints(slots + fill), "positions": _ints(positions + fill), "status": _ints([0])}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return _exact_plan(s)
    if case["op"] == "store":
        got = {}
        for name in ("k", "v"):
            pages = s[name + "_pages"].cpu().numpy().transpose(0, 2, 1, 3).copy()  # [page][place][head][dim]
            flat = pages.reshape(-1, case["kv_heads"] * case["head_dim"])
            flat[s["slots"].cpu().numpy()] = s[name].cpu().numpy()
            got[name + "_pages"] = np.ascontiguousarray(flat.reshape(pages.shape).transpose(0, 2, 1, 3))
        return got
    heads, kv_heads, hd, window = case["heads"], case["kv_heads"], case["head_dim"], case["window"] or 1 << 30
    starts = s["row_start"].tolist()
    out = torch.zeros_like(s["out"])
    for i in range(len(starts) - 1):
        a, b = starts[i], starts[i + 1]
        n = b - a
        if case["op"] == "packed":
            k, v = (s[x][a:b].view(n, kv_heads, hd).long() for x in ("k", "v"))
            at = torch.arange(n, device="cuda")
            seen = (at[None, :] <= at[:, None]) & (at[:, None] - at[None, :] < window)
        else:
            x = int(s["lengths"][i])
            m = x + n
            pos = torch.arange(m, device="cuda")
            page = s["table"][i].long()[pos // case["page"]]
            k, v = (s[y][page, :, pos % case["page"]].long() for y in ("k_pages", "v_pages"))
            parents, place, rows = s["parents"][a:b].tolist(), [], []
            for j, p in enumerate(parents):
                rows.append((rows[p] if p >= 0 else set()) | {j})
                place.append(x + len(rows[j]) - 1)
            see = np.zeros((n, m), dtype=bool)
            for j in range(n):
                see[j, max(0, place[j] + 1 - window):x] = True
                for y in rows[j]:
                    see[j, x + y] = place[j] - place[y] < window
            seen = torch.from_numpy(see).cuda()
        for h in range(heads):
            g = h // (heads // kv_heads)
            out[a:b, h * hd:(h + 1) * hd] = _exact_rows(s["q"][a:b, h * hd:(h + 1) * hd].long(), k[:, g], v[:, g], seen,
                                                        s["scale"])
    return out
