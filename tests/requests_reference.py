"""Plain 64-bit implementations of the operators that give requests their own
adapters, rules and draws, for their tests: numpy integers, the exp terms of the
oracle (det-num in C)."""
import functools

import numpy as np

from oracle import cpu
from tests.paged_reference import ancestors

LOWEST, HIGHEST = -(1 << 31), (1 << 31) - 1


def nearest(num, den):
    """num / den to the nearest integer, ties to even, den > 0 (Python integers
    or int64 arrays that hold 2 num)."""
    q = num // den
    over = 2 * (num - q * den) - den
    return q + ((over > 0) | ((over == 0) & (q % 2 != 0)))


def clip32(x):
    return np.clip(x, LOWEST, HIGHEST)


def shifted(sums, bits):
    """sums / 2^bits, rounded and clamped; sums below 2^62 in magnitude."""
    low = sums >> bits
    rest = sums - (low << bits)
    half = (1 << bits) >> 1
    up = ((rest > half) | ((rest == half) & (low % 2 != 0))) if bits else np.zeros(sums.shape, bool)
    return clip32(low + up)


def adapters(x, y, slots, parts, weights):
    """weights[slot][part]: (a, a_bits, b, b_bits) or None. Integer products in
    int64: at most 65504 2^31 2^15 < 2^62."""
    out = y.astype(np.int64)
    for r, s in enumerate(slots):
        if s < 0:
            continue
        for (rows, first, step), part in zip(parts, weights[s]):
            if part is None:
                continue
            a, a_bits, b, b_bits = part
            t = shifted(a.astype(np.int64) @ x[r].astype(np.int64), a_bits)
            u = shifted(b.astype(np.int64) @ t, b_bits)
            at = first + step * np.arange(rows)
            out[r, at] = clip32(out[r, at] + u)
    return out.astype(np.int32)


def rules(logits, request, rule, history, lengths, row_start=None, ids=None, parents=None, bias_ids=(), bias_values=(),
          masks=None, mask_of=None, first_row=0):
    """rule: (repetition, frequency, presence, window, bias start, bias count)
    each request; masks: [rows][words]. Python integers throughout."""
    rows, vocab = logits.shape
    out = np.empty_like(logits)
    for r in range(rows):
        l = [int(v) for v in logits[r]]
        closed = {v for v in range(vocab) if l[v] == LOWEST}
        q = -1 if request is None else int(request[r])
        if q >= 0:
            rep, freq, pres, window, b0, bn = (int(v) for v in rule[q])
            text = [int(t) for t in history[q][:lengths[q]]] if history is not None else []
            if ids is not None:
                a = int(row_start[q])
                up = parents[a:first_row + r + 1] if parents is not None else np.arange(-1, first_row + r - a)
                text += [int(ids[a + i]) for i in sorted(ancestors([int(p) for p in up])[first_row + r - a])]
            if window:
                text = text[-window:]
            count = {}
            for t in text:
                if 0 <= t < vocab:
                    count[t] = count.get(t, 0) + 1
            for t, c in count.items():
                v = nearest(l[t] << 16, rep) if l[t] > 0 else nearest(l[t] * rep, 1 << 16)
                l[t] = v - c * freq - pres
            for t, v in zip(bias_ids[b0:b0 + bn], bias_values[b0:b0 + bn]):
                if 0 <= t < vocab:
                    l[t] += int(v)
        out[r] = [min(max(v, LOWEST + 1), HIGHEST) for v in l]
        out[r, sorted(closed)] = LOWEST
        if masks is not None and mask_of[r] >= 0:
            words = np.ascontiguousarray(masks[mask_of[r]]).view(np.uint8)
            out[r, np.unpackbits(words, bitorder="little")[:vocab] == 0] = LOWEST
    return out


@functools.lru_cache(maxsize=None)
def terms():
    """The exp term of every gap below 2^20."""
    f = cpu.lib().dn_softmax_exp_term
    return np.array([f(-g << 16) for g in range(1 << 20)], dtype=np.int64)


def draw(l, drawing, number):
    """One row's (token, weight, sum); drawing: (inverse temperature, top_k,
    top_p, max_gap) or None."""
    order = np.lexsort((np.arange(l.size), -l.astype(np.int64)))
    order = order[l[order] > LOWEST]
    if not order.size:
        return -1, 0, 0
    if drawing is None or drawing[0] <= 0:
        return int(order[0]), 1 << 32, 1 << 32
    beta, k, p, far = (int(v) for v in drawing)
    gap = [nearest((int(l[order[0]]) - int(v)) * beta, 1 << 16) for v in l[order[:k] if k else order]]
    w = [int(terms()[g]) if g < 1 << 20 and not (far and g > far) else 0 for g in gap]
    if p:
        whole, have, kept = sum(w), 0, 0
        while have << 32 < p * whole:
            have += w[kept]
            kept += 1
        w = w[:kept]
    target, have, at = sum(w) * int(number) >> 32, 0, 0
    while have + w[at] <= target:
        have += w[at]
        at += 1
    return int(order[at]), w[at], sum(w)
