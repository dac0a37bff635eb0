"""A model's tokens for one prompt with an adapter, rules, masks and a drawing of
its own, from the oracle's pieces: every pass over the whole text anew, adapters
as tests/requests_reference.py has them."""
import numpy as np

from oracle import cpu
from tests import paged_reference as paged
from tests import requests_reference as ref


def each(f, *arrays):
    """f of the values of int32 arrays of one shape."""
    out = np.empty(arrays[0].shape, np.int32)
    for i in np.ndindex(out.shape):
        out[i] = f(*(int(a[i]) for a in arrays))
    return out


def add(a, b):
    return ref.clip32(a.astype(np.int64) + b).astype(np.int32)


def mul(a, b):
    return ref.shifted(a.astype(np.int64) * b, 16).astype(np.int32)


class Forward:
    """adapter: {tensor name: (a, a_bits, b, b_bits)}, or None."""

    def __init__(self, model, adapter=None, max_positions=256):
        self.m, self.s, self.adapter = model, model.shape, adapter or {}
        self.oracle = cpu.OracleRun(model, max_positions)

    def name(self, layer, part):
        return self.m.layer_name(layer, part + ".weight")

    def values(self, layer, part):
        return self.m.values(self.name(layer, part))

    def linear(self, layer, part, x):
        """(the product, the adapter's pair of it)"""
        return cpu.linear_q8(x, self.m.q8(self.name(layer, part))), self.adapter.get(self.name(layer, part))

    def adapted(self, y, x, pair):
        if pair is None:
            return y
        return ref.adapters(x, y, [0] * len(x), [(y.shape[1], 0, 1)], [[pair]])

    def project(self, layer, part, x):
        y, pair = self.linear(layer, part, x)
        return self.adapted(y, x, pair)

    def norm(self, x, w):
        return np.stack([cpu.rms_norm(r, w, self.s.norm_eps) for r in x])

    def mistral_layer(self, layer, x):
        s, n = self.s, len(x)
        heads, kv, hd = s.num_attention_heads, s.num_key_value_heads, s.head_dim
        h = self.norm(x, self.values(layer, "input_layernorm"))
        q, k, v = (self.project(layer, f"self_attn.{c}_proj", h) for c in "qkv")
        for a, count in ((q, heads), (k, kv)):
            for pos in range(n):
                for i in range(count):
                    a[pos, i * hd:(i + 1) * hd] = cpu.rotate_consecutive_pairs(a[pos, i * hd:(i + 1) * hd],
                                                                               s.rope_inverse_frequencies, pos)
        ctx = paged.packed(q, k, v, [0, n], heads, kv, hd, 0, s.attention_scale_q32, np.zeros_like(q))
        # The layer adds the residual in the product; the adapter's part comes behind.
        y, pair = self.linear(layer, "self_attn.o_proj", ctx)
        attended = self.adapted(add(y, x), ctx, pair)
        f = self.norm(attended, self.values(layer, "pre_feedforward_layernorm"))
        gate, up = self.project(layer, "mlp.gate_proj", f), self.project(layer, "mlp.up_proj", f)
        gated = mul(cpu.silu_many(gate).reshape(gate.shape), up)
        y, pair = self.linear(layer, "mlp.down_proj", gated)
        return self.adapted(add(y, attended), gated, pair)

    def gemma_layer(self, layer, x, ple, caches):
        m, s, n, L = self.m, self.s, len(x), cpu.lib()
        heads, kv, hd = s.num_attention_heads, s.num_key_value_heads, m.head_dim_at(layer)
        base, rotary, fbd = m.rope_at(layer)
        h = self.norm(x, self.values(layer, "input_layernorm"))
        q, k, v = (self.project(layer, f"self_attn.{c}_proj", h) for c in "qkv")
        for a, count, w in ((q, heads, "q_norm"), (k, kv, "k_norm")):
            for pos in range(n):
                for i in range(count):
                    at = slice(i * hd, (i + 1) * hd)
                    a[pos, at] = cpu.rope_rotate_pairs(cpu.rms_norm(a[pos, at], self.values(layer, "self_attn." + w), s.norm_eps),
                                                       rotary, fbd, base, pos)
        for pos in range(n):
            for i in range(kv):
                row = np.ascontiguousarray(v[pos, i * hd:(i + 1) * hd])
                L.dn_value_rms_norm(row, hd, s.norm_eps)
                v[pos, i * hd:(i + 1) * hd] = row
        caches[layer] = (k, v)
        donor = m.kv_donor_layer(layer)
        k, v = caches[layer if donor < 0 else donor]
        ctx = paged.packed(q, k, v, [0, n], heads, kv, hd, m.sliding_window_at(layer), 0, np.zeros_like(q))
        resid = add(self.norm(self.project(layer, "self_attn.o_proj", ctx), self.values(layer, "post_attention_layernorm")), x)
        f = self.norm(resid, self.values(layer, "pre_feedforward_layernorm"))
        gate, up = self.project(layer, "mlp.gate_proj", f), self.project(layer, "mlp.up_proj", f)
        gated = mul(each(L.dn_gelu, gate), up)
        xs = add(self.norm(self.project(layer, "mlp.down_proj", gated), self.values(layer, "post_feedforward_layernorm")), resid)
        g = mul(each(L.dn_gelu, cpu.linear_i32(xs, self.values(layer, "per_layer_input_gate").reshape(-1, s.hidden_size))), ple)
        p = s.hidden_size_per_layer_input
        out = add(self.norm(cpu.linear_i32(g, self.values(layer, "per_layer_projection").reshape(-1, p)),
                            self.values(layer, "post_per_layer_input_norm")), xs)
        scalar = m.layer_scalar(layer)
        return mul(out, np.full_like(out, scalar)) if scalar else out

    def logits(self, ids):
        """The logits behind the last of the ids."""
        x = seed = self.oracle.embed(ids)
        caches = {}
        for layer in range(self.m.num_layers):
            if self.m.family == "mistral-dense":
                x = self.mistral_layer(layer, x)
            else:
                x = self.gemma_layer(layer, x, self.oracle._ple_rows(layer, ids, seed), caches)
        return self.oracle.logits(x[-1])

    def generate(self, prompt, tokens, rule=None, biases=(), drawing=None, numbers=(), mask=None):
        """(token ids, stop reason)"""
        ids, eos = [int(i) for i in prompt], self.m.eos_token_ids
        for t in range(tokens):
            l = self.logits(ids)[None]
            words, of = None, None
            if mask is not None and mask(ids) is not None:
                bits = np.zeros(-(-l.shape[1] // 32) * 32, np.uint8)
                bits[:l.shape[1]] = mask(ids)
                words, of = np.packbits(bits, bitorder="little").view(np.uint32)[None], [0]
            record = [(*rule, 0, len(biases))] if rule is not None else None
            l = ref.rules(l, [0] if rule is not None else None, record, [ids], [len(ids)], bias_ids=[t for t, _ in biases],
                          bias_values=[v for _, v in biases], masks=words, mask_of=of)
            token = ref.draw(l[0], drawing, int(numbers[t]) if drawing is not None else 0)[0]
            if token < 0:
                return ids[len(prompt):], "closed"
            ids.append(token)
            if token in eos:
                return ids[len(prompt):], "eos"
        return ids[len(prompt):], "max_new_tokens"
