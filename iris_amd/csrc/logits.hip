// Rows of logits to tokens, each request in its own way: penalties for repeated
// tokens, biases and grammar masks (iris_logits_rules), and the draw of a token
// (iris_logits_draw).
#include <algorithm>

#include "detnum_dev.h"
#include "paged.h"
#include "softmax_double.h"
#include "wave_ops.h"

namespace {

constexpr uint32_t MAX_VOCAB = 1u << 20, MAX_ROWS = 65535, MAX_HISTORY = 1u << 20, MAX_BIASES = 1u << 20;

// ------------------------------------------------------------------ rules

// Tokens a workgroup takes: their counts and biases in LDS.
constexpr uint32_t MIN_RULE_PIECE = 1024, MAX_RULE_PIECE = 4096, RULE_GROUPS = 2048;
// Texts from here on: larger pieces, since each reads the text (64 rows of 32000
// behind texts of up to 32700: 21.6 us with pieces of 4096, 29 with 1024).
constexpr uint32_t LONG_TEXT = 4096;
constexpr uint32_t BIAS_PLACES = 512;  // sums of biases at a time; a crowded piece has more biased tokens
constexpr uint32_t COUNT_BITS = 21;    // of a text's 2^20 tokens and a path's 64
static_assert((BIAS_PLACES + 1) << COUNT_BITS >> COUNT_BITS == BIAS_PLACES + 1 && (1u << COUNT_BITS) > MAX_HISTORY + TREE_MAX_NODES,
              "a count and a place in a word");

// x / 2^16 of repetition, rounded to even: l 2^16 / rep for l > 0 and rep > 0.
// The quotient in double is within one of the exact one (below 2^47), and its
// remainder exact; a step by it gives the nearest, of two the even one.
__device__ __forceinline__ int64_t divided(int32_t l, int32_t rep, double inverse) {
    const double n = (double)l * 65536.0;
    const double q = rint(n * inverse);
    const int64_t r = (int64_t)fma(-q, (double)rep, n);  // exact: |n| and |q rep| below 2^48
    const int64_t up = 2 * r - rep, down = 2 * r + rep;
    int64_t w = (int64_t)q;
    if (up > 0 || (up == 0 && (w & 1))) w++;
    else if (down < 0 || (down == 0 && (w & 1))) w--;
    return w;
}

__device__ __forceinline__ void report(const IrisLogitsRules& a, int32_t code) {
    if (a.status) *a.status = code;
}

// Pieces of one row, in turn: the text's tokens in the piece are counted and the
// biases summed in LDS, then the piece's logits pass once, four to a thread and
// turn where the rows allow it. (Biased tokens are few, so their sums have places
// of their own: a sum for every token would leave three workgroups a CU, 50 us
// against 40 for 63 rows of 256000. A piece with more biased tokens than places, or
// nearly as many where threads that meet a token at once each take one, is done by
// parts that have a sum for every token, with a pass over the list each: a bias on
// each token of one row of 32000 takes 85 us, of 2^20 2.1 ms, of 16 rows of 256000
// 1.1 ms.) The rule's loads are a chain of four (request,
// rule, parents, ids), which a workgroup of several pieces pays once. It is what
// one row of 32000 costs (6.5 us with the launch); 63 rows of 256000 of drafted trees
// take 38.5 us, 131 MB read and written at 3.4 TB/s, the counts and the barriers
// around them between the loads and the stores (vector units issue in 45% of the
// cycles, and waves wait 65% of their time).
template <bool VEC>
__global__ __launch_bounds__(256) void rules_kernel(const IrisLogitsRules a, const uint32_t piece) {
    // A token's occurrences, and above COUNT_BITS the place of its biases' sum.
    __shared__ uint32_t s_count[MAX_RULE_PIECE];
    __shared__ uint64_t s_bias[BIAS_PLACES];
    __shared__ uint32_t s_places;
    const uint32_t row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const bool first = blockIdx.x == 0 && tid == 0;
    const int32_t* in = a.logits + (size_t)row * a.logits_stride;
    int32_t* out = a.out + (size_t)row * a.out_stride;

    int32_t mask = a.masks && a.mask_of ? a.mask_of[row] : -1;
    int32_t q = a.rules ? a.request[row] : -1;
    if (mask < -1 || mask >= (int32_t)a.mask_rows) {
        if (first) report(a, IRIS_E_INVALID);
        mask = -1;
    }
    if (q < -1 || q >= (int32_t)a.requests) {
        if (first) report(a, IRIS_E_INVALID);
        q = -1;
    }
    IrisTokenRule rule{};
    int64_t length = 0;
    int32_t start = 0, own = -1;
    if (q >= 0) {
        rule = a.rules[q];
        length = a.history ? a.lengths[q] : 0;
        int32_t bad = 0;
        if (rule.repetition <= 0 || rule.bias_start > a.biases || rule.bias_count > a.biases - rule.bias_start) bad = IRIS_E_INVALID;
        else if (length < 0 || length > a.history_stride) bad = IRIS_E_RANGE;
        if (a.ids && !bad) {
            const int64_t r = (int64_t)a.first_row + row;
            start = a.row_start[q];
            own = (int32_t)(r - start);
            if (start < 0 || r < start || r >= a.row_start[q + 1] || r - start >= TREE_MAX_NODES) bad = IRIS_E_RANGE;
        }
        if (bad) {
            if (first) report(a, bad);
            q = -1;
        }
    }
    // A rule that changes nothing needs no counts.
    const bool counted = q >= 0 && (rule.repetition != dn::ONE_ACT || rule.frequency || rule.presence);
    const bool biased = q >= 0 && rule.bias_count;
    const int32_t* text = a.history + (size_t)max(q, 0) * a.history_stride;  // its part that counts: `words` tokens
    uint32_t words = 0;
    int32_t drafted = -1;  // this lane's row of the path behind it
    if (counted) {
        uint64_t path = 0;  // the drafted rows from the root to this one
        if (own >= 0) {
            const uint64_t above = tree_ancestors(a.parents ? a.parents + start : nullptr, own + 1, lane);
            path = readlane64(above, __builtin_amdgcn_readfirstlane(own));
        }
        const int64_t whole = length + __popcll(path);
        const int64_t from = rule.window && whole > rule.window ? whole - rule.window : 0;
        words = from < length ? (uint32_t)(length - from) : 0;
        text += from;
        // The path's row of lane l is its place in the path behind the history.
        if (tid < 64 && (path >> lane & 1) && length + __popcll(path & ((1ull << lane) - 1)) >= from) drafted = a.ids[start + lane];
    }
    constexpr uint32_t HELD = 8;  // the text's first tokens stay in registers from piece to piece
    int32_t held[HELD];
#pragma unroll
    for (uint32_t j = 0; j < HELD; j++) held[j] = tid + 256 * j < words ? text[tid + 256 * j] : -1;
    const uint32_t* bits = a.masks + (size_t)max(mask, 0) * a.mask_stride;
    const double inverse = 1.0 / rule.repetition;
    // A token with its occurrences and its biases' sum.
    auto with_bias = [&](int32_t logit, uint32_t count, int64_t bias) {
        int64_t l = logit;
        if (count) {
            l = l > 0 ? divided((int32_t)l, rule.repetition, inverse) : dn::rshift_rte(l * rule.repetition, 16);
            l -= (int64_t)count * rule.frequency + rule.presence;
        }
        l += bias;
        return logit == INT32_MIN ? INT32_MIN : l < INT32_MIN + 1 ? INT32_MIN + 1 : l > INT32_MAX ? INT32_MAX : (int32_t)l;
    };
    // A token that the text or a bias names.
    auto ruled = [&](int32_t logit, uint32_t word) {
        const uint32_t place = word >> COUNT_BITS;
        return with_bias(logit, word & ((1u << COUNT_BITS) - 1), place ? (int64_t)s_bias[place - 1] : 0);
    };
    auto open = [&](uint32_t v) { return mask < 0 || (bits[v / 32] >> (v % 32) & 1); };

#pragma unroll 1
    for (uint32_t v0 = blockIdx.x * piece; v0 < a.vocab; v0 += gridDim.x * piece) {
        const uint32_t v1 = min(v0 + piece, a.vocab), fours = VEC ? v0 + ((v1 - v0) & ~3u) : v0;  // where whole fours end
        constexpr uint32_t TURNS = MAX_RULE_PIECE / 1024;
        int4 x[TURNS];
        uint32_t word[TURNS];
        if constexpr (VEC) {
            // (v0 is a multiple of 32: the four tokens' bits are in one word.)
#pragma unroll
            for (uint32_t i = 0; i < TURNS; i++) {
                const uint32_t v = v0 + 4 * tid + 1024 * i;
                if (v < fours) x[i] = *(const int4*)(in + v), word[i] = mask >= 0 ? bits[v / 32] >> (v % 32) : 15;
            }
        }
        const bool named = counted || biased;
        if (named) {
            for (uint32_t i = 4 * tid; i < piece; i += 1024) *(uint4*)&s_count[i] = uint4{};
            if (biased)
                for (uint32_t i = tid; i < BIAS_PLACES; i += 256) s_bias[i] = 0;
            if (tid == 0) s_places = 0;
            __syncthreads();
        }
        if (counted) {
            auto count = [&](int32_t token) {
                const uint32_t v = (uint32_t)token - v0;
                if (v < v1 - v0) atomicAdd(&s_count[v], 1u);
            };
#pragma unroll
            for (uint32_t j = 0; j < HELD; j++) count(held[j]);
            // (Eight loads ahead: each piece reads the rest of the text.)
#pragma unroll 1
            for (uint32_t i = tid + HELD * 256; i < words; i += 8 * 256) {
                int32_t token[8];
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) token[j] = i + 256 * j < words ? text[i + 256 * j] : -1;
#pragma unroll
                for (uint32_t j = 0; j < 8; j++) count(token[j]);
            }
            count(drafted);
        }
        if (biased) {
            if (counted) __syncthreads();  // (a count that changes would cost a place)
            for (uint32_t i = tid; i < rule.bias_count; i += 256) {
                const uint32_t v = (uint32_t)a.bias_ids[rule.bias_start + i] - v0;
                if (v >= v1 - v0) continue;
                uint32_t word = s_count[v];
                while (!(word >> COUNT_BITS)) {  // one of a token's entries takes its place
                    const uint32_t taken = word | (min(atomicAdd(&s_places, 1u), BIAS_PLACES) + 1) << COUNT_BITS;
                    const uint32_t old = atomicCAS(&s_count[v], word, taken);
                    word = old == word ? taken : old;
                }
                const uint32_t place = word >> COUNT_BITS;
                if (place > BIAS_PLACES) break;  // (the piece is crowded)
                atomicAdd((unsigned long long*)&s_bias[place - 1], (unsigned long long)(int64_t)a.bias_values[rule.bias_start + i]);
            }
        }
        if (named) __syncthreads();
        const bool crowded = biased && s_places > BIAS_PLACES;
        if (crowded) {
            // A sum for every token, BIAS_PLACES of them at a time, each time by a
            // pass over the list, eight loads ahead.
#pragma unroll 1
            for (uint32_t u0 = v0; u0 < v1; u0 += BIAS_PLACES) {
                const uint32_t n = min(BIAS_PLACES, v1 - u0);
                for (uint32_t i = tid; i < BIAS_PLACES; i += 256) s_bias[i] = 0;
                __syncthreads();
#pragma unroll 1
                for (uint32_t i = tid; i < rule.bias_count; i += 8 * 256) {
                    int32_t id[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8; j++) id[j] = i + 256 * j < rule.bias_count ? a.bias_ids[rule.bias_start + i + 256 * j] : -1;
#pragma unroll
                    for (uint32_t j = 0; j < 8; j++) {
                        const uint32_t k = (uint32_t)id[j] - u0;
                        if (k < n)
                            atomicAdd((unsigned long long*)&s_bias[k],
                                      (unsigned long long)(int64_t)a.bias_values[rule.bias_start + i + 256 * j]);
                    }
                }
                __syncthreads();
                for (uint32_t v = u0 + tid; v < u0 + n; v += 256)
                    out[v] = open(v) ? with_bias(in[v], s_count[v - v0] & ((1u << COUNT_BITS) - 1), (int64_t)s_bias[v - u0]) : INT32_MIN;
                __syncthreads();  // before the next tokens' sums
            }
            continue;
        }
        if constexpr (VEC) {
#pragma unroll
            for (uint32_t i = 0; i < TURNS; i++) {
                const uint32_t v = v0 + 4 * tid + 1024 * i, k = v - v0;
                if (v >= fours) continue;
                const uint4 c = named ? *(const uint4*)&s_count[k] : uint4{};
                int4 l = x[i];
                // Few tokens are named, so most waves of a large vocabulary have none.
                if (c.x | c.y | c.z | c.w) {
#pragma unroll 1
                    for (uint32_t j = 0; j < 4; j++) {
                        const int32_t y = ruled(j == 0 ? l.x : j == 1 ? l.y : j == 2 ? l.z : l.w,
                                                j == 0 ? c.x : j == 1 ? c.y : j == 2 ? c.z : c.w);
                        l.x = j == 0 ? y : l.x, l.y = j == 1 ? y : l.y, l.z = j == 2 ? y : l.z, l.w = j == 3 ? y : l.w;
                    }
                }
                *(int4*)(out + v) = make_int4(word[i] & 1 ? l.x : INT32_MIN, word[i] & 2 ? l.y : INT32_MIN,
                                              word[i] & 4 ? l.z : INT32_MIN, word[i] & 8 ? l.w : INT32_MIN);
            }
        }
        for (uint32_t v = fours + tid; v < v1; v += 256)
            out[v] = open(v) ? ruled(in[v], named ? s_count[v - v0] : 0) : INT32_MIN;
        if (named) __syncthreads();  // before the next piece's counts
    }
}

// ------------------------------------------------------------------ draw
//
// All bounds keep a run from the front of the row's order (falling logits, of
// equal ones the smaller index first), and the draw picks the place where a
// running sum passes a number: each is the place in that order where a count
// or a sum of weights is reached. So a histogram over the gap to the maximum,
// with each bucket's count and sum, narrows every one of them to a bucket, and
// only that bucket's tokens are put in order.
//
// Three launches: the row's maximum by pieces; the histogram; the places, by one
// workgroup, which reads the row once more for the tokens of the buckets where
// they can lie. Of long rows a launch in between gathers those, by pieces: one
// workgroup has too little in flight (256000 tokens: 30 us). Sums of weights are
// whole numbers, so their order does not matter.
//
// All is short work between barriers: one row of 32000 takes 3.4 + 4.3 + 16.7 us,
// the last one workgroup's chain, nine rows of 256000 3.9 + 15.9 + 12.2 + 9.4. 108
// rows of 256000 read 110 MB three times, from the last-level cache after the
// first: 18 us (6.1 TB/s), 39.6 (the terms' arithmetic and atomics, vector units
// issue in 70% of the cycles), 29.6 (3.7 TB/s) and 14.1.

// Enough that few tokens share a bucket of a dense row: with 1024 the gathered
// tokens of some rows passed GATHER, 97 to 196 us for 108 rows by their numbers.
constexpr uint32_t BUCKETS = 2048;
constexpr uint32_t PICK_THREADS = 512;
constexpr uint32_t LIST = 512;        // tokens put in order at a time
constexpr uint32_t GATHER = 4096;     // tokens held in LDS
constexpr uint32_t SUB_BITS = 9;      // a crowded bucket's parts
constexpr uint32_t INDEX_BITS = 20;   // of a token's index
constexpr uint32_t SUM_BITS = 47;     // of a piece's sum of weights, its count above them
// Rows past this are gathered by pieces, a launch more. Gathered and not, for 1 and
// 108 rows: 32000 tokens 27 and 42 us against 21 and 34, 65536 the same within 1 us,
// 128000 29 and 73 against 36 and 82, 256000 31 and 110 against 58 and 135.
constexpr uint32_t LONG_ROW = 65536;
constexpr uint32_t GATHER_PIECE = 16384, PIECE_LIST = 512;  // tokens of a piece, of them held in LDS
constexpr uint32_t MAX_PIECE = 16384;  // tokens of a piece: their weights of 2^32 add to at most 2^46

// A logit and its index as one key, above 0: larger for a larger logit, of equal
// ones for the smaller index.
__device__ __forceinline__ uint64_t draw_key(int32_t v, uint32_t i) { return (uint64_t)((uint32_t)v ^ 0x80000000u) << 32 | (uint32_t)~i; }
__device__ __forceinline__ int32_t key_logit(uint64_t k) { return (int32_t)((uint32_t)(k >> 32) ^ 0x80000000u); }

// f(four logits, first index) for v0 .. v1 of a row, by a workgroup of THREADS: 16
// bytes at a time, DEPTH loads ahead, where the rows allow it (v0 is a multiple
// of 4), else one and three closed places. Short code
// where f is long: a workgroup or two run it cold, and each 64 bytes of it are a
// fetch.
template <uint32_t THREADS, uint32_t DEPTH, class F>
__device__ __forceinline__ void each_logit(const int32_t* row, uint32_t v0, uint32_t v1, bool vec, F&& f) {
    const uint32_t whole = vec ? v0 + ((v1 - v0) & ~3u) : v0;
#pragma unroll 1
    for (uint32_t v = v0 + 4 * threadIdx.x; v < whole; v += 4 * DEPTH * THREADS) {
        int4 x[DEPTH];
#pragma unroll
        for (uint32_t i = 0; i < DEPTH; i++)
            if (v + 4 * i * THREADS < whole) x[i] = *(const int4*)(row + v + 4 * i * THREADS);
#pragma unroll
        for (uint32_t i = 0; i < DEPTH; i++)
            if (v + 4 * i * THREADS < whole) f(x[i], v + 4 * i * THREADS);
    }
#pragma unroll 1
    for (uint32_t v = whole + threadIdx.x; v < v1; v += THREADS) f(make_int4(row[v], INT32_MIN, INT32_MIN, INT32_MIN), v);
}

// How a row draws. Gaps from `end` on have no weight; bucket b holds the gaps
// from b << shift on.
struct RowDraw {
    int64_t beta;
    uint32_t top_k, top_p;
    uint64_t end;
    uint32_t shift, pad;
    // Few tokens are kept: their weights are formed when they are gathered,
    // and the histogram only counts.
    __device__ __forceinline__ bool counts_only() const { return top_k && top_k <= LIST; }
};

// Work space of a row: how it draws, the histogram, and the tokens gathered from a
// long row.
struct DrawRow {
    RowDraw draw;
    uint32_t count[BUCKETS];
    uint64_t sum[BUCKETS];
    uint64_t key[GATHER];
    uint32_t gathered, pad[3];
    static_assert(sizeof(RowDraw) % 16 == 0, "aligned counts and sums");
};

// The weight of a gap below `end`.
__device__ __forceinline__ uint64_t weight_of(const RowDraw& d, uint32_t gap) {
    uint32_t kept;
    return (uint64_t)softmax_term((uint32_t)dn::rshift_rte((int64_t)gap * d.beta, 16), &kept);
}

__device__ __forceinline__ RowDraw row_draw(const IrisLogitsDraw& a, uint32_t row) {
    RowDraw d{};
    if (!a.drawings) return d;
    const int32_t q = a.request ? a.request[row] : (int32_t)row;
    if (q < 0 || q >= (int32_t)a.requests) {
        if (q != -1 && a.status) *a.status = IRIS_E_INVALID;
        return d;
    }
    const IrisDrawing w = a.drawings[q];
    if (w.inverse_temperature <= 0) return d;
    d.beta = w.inverse_temperature, d.top_k = w.top_k, d.top_p = w.top_p;
    // The first scaled gap without weight, and the first gap that rounds to it:
    // gap beta / 2^16 >= none - 1/2, or past that where none is odd.
    const uint64_t none = w.max_gap && w.max_gap < 1u << 20 ? w.max_gap + 1 : 1u << 20;
    const uint64_t twice = 2 * (uint64_t)d.beta, bound = (none << 17) - (1u << 16) + (none & 1);
    d.end = min((bound + twice - 1) / twice, 1ull << 32);
    // The least shift with (end - 1) >> shift below BUCKETS.
    const uint32_t bits = 64 - __builtin_clzll(d.end - 1 | 1);
    d.shift = bits > 11 ? bits - 11 : 0;
    static_assert(BUCKETS == 1u << 11, "bits of a bucket");
    return d;
}

struct DrawPieces {
    uint32_t size, count;
    bool vec;  // rows of 16-byte aligned logits
};

// The largest key of each piece of a row; and the row's histogram cleared.
__global__ __launch_bounds__(256) void draw_top_kernel(const IrisLogitsDraw a, const DrawPieces p, uint64_t* tops, DrawRow* space) {
    __shared__ uint64_t s_best[4];
    const uint32_t row = blockIdx.y, v0 = blockIdx.x * p.size, v1 = min(v0 + p.size, a.vocab);
    uint64_t k = 0;
    each_logit<256, 4>(a.logits + (size_t)row * a.logits_stride, v0, v1, p.vec, [&](int4 l, uint32_t v) {
        // The first of the four that is as large as any.
        const int32_t most = max(max(l.x, l.y), max(l.z, l.w));
        k = max(k, draw_key(most, v + (l.x == most ? 0 : l.y == most ? 1 : l.z == most ? 2 : 3)));
    });
    k = wave_max_u64(k);
    if (threadIdx.x % 64 == 0) s_best[threadIdx.x / 64] = k;
    __syncthreads();
    if (threadIdx.x == 0) tops[(size_t)row * p.count + blockIdx.x] = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
    if (blockIdx.x == 0 && threadIdx.x == 0) space[row].draw = row_draw(a, row), space[row].gathered = 0;
    if (!a.drawings) return;
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < BUCKETS; i += p.count * 256) space[row].count[i] = 0, space[row].sum[i] = 0;
}

// The row's largest key, by a workgroup (every thread gets it).
template <uint32_t THREADS>
__device__ __forceinline__ uint64_t row_top(const uint64_t* tops, uint32_t pieces, uint64_t* s_best) {
    uint64_t k = 0;
    for (uint32_t i = threadIdx.x; i < pieces; i += THREADS) k = max(k, tops[i]);
    k = wave_max_u64(k);
    if (threadIdx.x % 64 == 0) s_best[threadIdx.x / 64] = k;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 64; w++) k = max(k, s_best[w]);
    return k;
}

// A piece's part of the row's histogram.
__global__ __launch_bounds__(256) void draw_histogram_kernel(const IrisLogitsDraw a, const DrawPieces p, const uint64_t* tops,
                                                             DrawRow* space) {
    __shared__ uint64_t s_bucket[BUCKETS];
    __shared__ uint64_t s_best[4];
    const uint32_t row = blockIdx.y, v0 = blockIdx.x * p.size, v1 = min(v0 + p.size, a.vocab);
    const RowDraw d = space[row].draw;
    if (!d.beta) return;
    for (uint32_t i = threadIdx.x; i < BUCKETS; i += 256) s_bucket[i] = 0;
    const int32_t most = key_logit(row_top<256>(tops + (size_t)row * p.count, p.count, s_best));
    if (most == INT32_MIN) return;
    const bool counts_only = d.counts_only();
    each_logit<256, 1>(a.logits + (size_t)row * a.logits_stride, v0, v1, p.vec, [&](int4 x, uint32_t) {
        const int32_t l[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t gap = (uint32_t)most - (uint32_t)l[i];
            if (l[i] != INT32_MIN && gap < d.end)
                atomicAdd((unsigned long long*)&s_bucket[gap >> d.shift],
                          (unsigned long long)(1ull << SUM_BITS | (counts_only ? 0 : weight_of(d, gap))));
        }
    });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < BUCKETS; i += 256) {
        const uint64_t x = s_bucket[i];
        if (!x) continue;
        atomicAdd(&space[row].count[i], (uint32_t)(x >> SUM_BITS));
        if (!counts_only) atomicAdd((unsigned long long*)&space[row].sum[i], (unsigned long long)(x & ((1ull << SUM_BITS) - 1)));
    }
}

// A place in the row's order: the token's key (gap 2^20 + index), its weight,
// and the tokens and weights up to it, itself included.
struct Place {
    uint64_t key, weight, count, sum;
};

// The buckets' running sums.
struct BucketSpace {
    uint64_t sum[BUCKETS];  // inclusive
    uint32_t count[BUCKETS];
    uint64_t wave[2][PICK_THREADS / 64];
    uint64_t whole;  // of all buckets
    uint32_t open, at[2], listed;
};

struct PickSpace : BucketSpace {
    uint32_t place_of[BUCKETS];  // of a wanted bucket: its place among them, and its first token's among the gathered
    union {
        // A row's gathered tokens: put in order, and their weights' running sums;
        struct {
            uint64_t token[GATHER];  // as found, then in order
            uint64_t key[GATHER], upto[GATHER];
            uint32_t part[GATHER];   // parts of the buckets: counts, then first places
            uint16_t behind[GATHER];  // of a token as found: those before it in its part
        };
        // or those of one bucket at a time: its parts, and the tokens of the last.
        struct {
            uint64_t sub_sum[1 << SUB_BITS];
            uint32_t sub_count[1 << SUB_BITS];
        };
        struct {
            uint64_t list[LIST], list_weight[LIST];
        };
    };
    uint32_t found;
    Place place;
    static_assert(LIST >= 1u << (SUB_BITS - 1) && LIST <= PICK_THREADS, "a listed token a thread");
};

// Inclusive running sums over the workgroup's threads of a pair.
template <uint32_t THREADS>
__device__ __forceinline__ void running_sums(uint64_t& x, uint64_t& y, BucketSpace& s) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_running_sum_u64(x), y = wave_running_sum_u64(y);
    if (lane == 63) s.wave[0][wave] = x, s.wave[1][wave] = y;
    __syncthreads();
    // (All waves' sums at once: a loop up to this wave's would wait for each.)
#pragma unroll
    for (uint32_t w = 0; w < THREADS / 64; w++) {
        const uint64_t a = s.wave[0][w], b = s.wave[1][w];
        x += w < wave ? a : 0, y += w < wave ? b : 0;
    }
    __syncthreads();
}

// What the places of a row are found from.
struct Pick {
    RowDraw d;
    const int32_t* in;
    uint32_t vocab;
    int32_t most;
    bool vec;

    // f(key, gap) for the row's tokens with keys from `first` on, 2^bits of
    // them, by the workgroup.
    template <class F>
    __device__ __forceinline__ void each(uint64_t first, uint32_t bits, F&& f) const {
        each_logit<PICK_THREADS, 4>(in, 0, vocab, vec, [&](int4 x, uint32_t v) {
#pragma unroll 1
            for (uint32_t i = 0; i < 4; i++) {
                const int32_t l = i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w;
                const uint32_t gap = (uint32_t)most - (uint32_t)l;
                const uint64_t key = (uint64_t)gap << INDEX_BITS | (v + i);
                if (l != INT32_MIN && gap < d.end && key - first < 1ull << bits) f(key, gap);
            }
        });
    }
};

// The first bucket whose running count reaches `value` (by_count), or whose
// running sum passes it.
__device__ __forceinline__ uint32_t bucket_of(const PickSpace& s, bool by_count, uint64_t value) {
    uint32_t low = 0, high = BUCKETS - 1;
    while (low < high) {
        const uint32_t mid = (low + high) / 2;
        if (by_count ? s.count[mid] >= value : s.sum[mid] > value) high = mid;
        else low = mid + 1;
    }
    return low;
}

// The first place where the running count reaches `value` (by_count) or the
// running sum passes it; `value` is at most the row's count, or below its sum.
// A pass over the row for each 2^9 parts of a crowded bucket, and one for the
// tokens at the place.
__device__ __forceinline__ Place find_place(const Pick& p, bool by_count, uint64_t value, PickSpace& s) {
    const uint32_t tid = threadIdx.x;
    auto reached = [&](uint64_t count, uint64_t sum) { return by_count ? count >= value : sum > value; };
    const uint32_t bucket = bucket_of(s, by_count, value);
    uint64_t count = bucket ? s.count[bucket - 1] : 0, sum = bucket ? s.sum[bucket - 1] : 0;  // before it
    uint64_t inside = s.count[bucket] - count;
    uint64_t low = (uint64_t)bucket << (p.d.shift + INDEX_BITS);  // the keys at hand: low .. low + 2^bits
    uint32_t bits = p.d.shift + INDEX_BITS;
    while (inside > LIST && bits >= SUB_BITS) {
        // A crowded range: its parts' counts and sums, and the part that reaches.
        // (Fewer bits than that hold at most LIST keys.)
        const uint32_t part_bits = bits - SUB_BITS;
        __syncthreads();
        for (uint32_t i = tid; i < 1u << SUB_BITS; i += PICK_THREADS) s.sub_sum[i] = 0, s.sub_count[i] = 0;
        if (tid == 0) s.found = (1u << SUB_BITS) - 1;
        __syncthreads();
        p.each(low, bits, [&](uint64_t key, uint32_t gap) {
            const uint32_t i = (uint32_t)((key - low) >> part_bits);
            atomicAdd(&s.sub_count[i], 1u);
            atomicAdd((unsigned long long*)&s.sub_sum[i], (unsigned long long)weight_of(p.d, gap));
        });
        __syncthreads();
        static_assert(1u << SUB_BITS == PICK_THREADS, "a part a thread");
        const uint64_t own_count = s.sub_count[tid], own_sum = s.sub_sum[tid];
        uint64_t run_count = own_count, run_sum = own_sum;
        running_sums<PICK_THREADS>(run_count, run_sum, s);
        if (reached(count + run_count, sum + run_sum)) atomicMin(&s.found, tid);
        __syncthreads();
        const uint32_t part = s.found;
        if (tid == part) s.wave[0][0] = run_count - own_count, s.wave[1][0] = run_sum - own_sum, s.listed = (uint32_t)own_count;
        __syncthreads();
        count += s.wave[0][0], sum += s.wave[1][0], inside = s.listed;
        low += (uint64_t)part << part_bits, bits = part_bits;
    }
    __syncthreads();
    if (tid == 0) s.listed = 0;
    __syncthreads();
    p.each(low, bits, [&](uint64_t key, uint32_t gap) {
        const uint32_t i = atomicAdd(&s.listed, 1u);
        if (i < LIST) s.list[i] = key, s.list_weight[i] = weight_of(p.d, gap);
    });
    __syncthreads();
    // Each token's running sums by comparing it with the others; the place is
    // the one that reaches and whose forerunner does not.
    const uint32_t n = min(s.listed, LIST);
    if (tid < n) {
        const uint64_t key = s.list[tid], weight = s.list_weight[tid];
        uint64_t c = count + 1, w = sum + weight;
        // (Both loads before the choice, or each turn would wait for two in a row.)
#pragma unroll 8
        for (uint32_t i = 0; i < n; i++) {
            const uint64_t k = s.list[i], x = s.list_weight[i];
            c += k < key ? 1 : 0, w += k < key ? x : 0;
        }
        if (reached(c, w) && !reached(c - 1, w - weight)) s.place = Place{key, weight, c, w};
    }
    __syncthreads();
    return s.place;
}

// ceil or floor of value share / 2^32, value below 2^53.
__device__ __forceinline__ uint64_t share_of(uint64_t value, uint32_t share, bool up) {
    const uint64_t high = (value >> 32) * share, low = (value & 0xffffffffull) * share;
    return high + (low >> 32) + (up && (low & 0xffffffffull) ? 1 : 0);
}

// Where a row's places can lie, by a workgroup of THREADS: each thread's buckets
// with the counts and sums before each and behind the last.
template <uint32_t THREADS>
struct Runs {
    static constexpr uint32_t OWN = BUCKETS / THREADS;
    uint32_t tokens[OWN];
    uint64_t weights[OWN], count[OWN + 1], sum[OWN + 1];
    bool by_k;          // top_k leaves tokens out
    uint32_t k_bucket;  // the k-th token's, else the last
    // Up to three runs of buckets (empty: low above high), and the tokens in them.
    uint32_t low[3], high[3], wanted_tokens, wanted_buckets;

    __device__ __forceinline__ void load(const DrawRow& row) {
#pragma unroll
        for (uint32_t i = 0; i < OWN; i += 2) {
            const uint2 c = *(const uint2*)&row.count[OWN * threadIdx.x + i];
            const ulonglong2 x = *(const ulonglong2*)&row.sum[OWN * threadIdx.x + i];
            tokens[i] = c.x, tokens[i + 1] = c.y, weights[i] = x.x, weights[i + 1] = x.y;
        }
    }

    // The running sums, in LDS too, from the counts and weights of the thread's
    // buckets.
    __device__ __forceinline__ void add_up(const uint64_t (&w)[OWN], BucketSpace& s) {
        uint64_t c = 0, x = 0;
#pragma unroll
        for (uint32_t i = 0; i < OWN; i++) c += tokens[i], x += w[i];
        uint64_t to_c = c, to_x = x;
        running_sums<THREADS>(to_c, to_x, s);
        count[0] = to_c - c, sum[0] = to_x - x;
#pragma unroll
        for (uint32_t i = 0; i < OWN; i++) {
            count[i + 1] = count[i] + tokens[i], sum[i + 1] = sum[i] + w[i];
            s.count[OWN * threadIdx.x + i] = (uint32_t)count[i + 1], s.sum[OWN * threadIdx.x + i] = sum[i + 1];
        }
        if (threadIdx.x == THREADS - 1) s.open = (uint32_t)to_c, s.whole = to_x;
        __syncthreads();
    }

    // The buckets where two queries are reached, each by its thread.
    __device__ __forceinline__ void locate(bool by_count, uint64_t first, uint64_t second, uint32_t& from, uint32_t& to,
                                           BucketSpace& s) const {
#pragma unroll
        for (uint32_t i = 0; i < OWN; i++) {
            const uint64_t x = by_count ? count[i] + 1 : sum[i], y = by_count ? count[i + 1] + 1 : sum[i + 1];
            if (x <= first && first < y) s.at[0] = OWN * threadIdx.x + i;
            if (x <= second && second < y) s.at[1] = OWN * threadIdx.x + i;
        }
        __syncthreads();
        from = s.at[0], to = s.at[1];
        __syncthreads();
    }

    __device__ __forceinline__ bool wanted(uint32_t bucket) const {
        return (bucket >= low[0] && bucket <= high[0]) || (bucket >= low[1] && bucket <= high[1]) ||
               (bucket >= low[2] && bucket <= high[2]);
    }

    // The k-th token's bucket; the share's, from what the tokens before the k-th
    // token's bucket and those up to it weigh; the draw's likewise. held and
    // buckets: the wanted tokens and buckets up to the thread's, inclusive.
    __device__ __forceinline__ void find(const RowDraw& d, uint32_t number, BucketSpace& s, uint32_t& held, uint32_t& buckets) {
        add_up(weights, s);
        const uint32_t open = s.open;
        uint64_t least = s.whole, most = least;
        auto before = [&](uint32_t bucket) { return bucket ? s.sum[bucket - 1] : 0; };
        uint32_t same;
        by_k = d.top_k && d.top_k < open, k_bucket = BUCKETS - 1;
        if (by_k) locate(true, d.top_k, d.top_k, k_bucket, same, s);
#pragma unroll
        for (int i = 0; i < 3; i++) low[i] = 1, high[i] = 0;
        if (d.counts_only()) {
            low[0] = 0, high[0] = k_bucket;
        } else {
            // (The first token is always kept and weighs 2^32.)
            if (by_k) {
                low[0] = high[0] = k_bucket;
                least = max(before(k_bucket), 1ull << 32), most = s.sum[k_bucket];
            }
            if (d.top_p) {
                locate(false, share_of(least, d.top_p, true) - 1, share_of(most, d.top_p, true) - 1, low[1], high[1], s);
                least = max(before(low[1]), 1ull << 32), most = s.sum[high[1]];
            }
            locate(false, share_of(least, number, false), share_of(most, number, false), low[2], high[2], s);
        }
        uint64_t run = 0, place = 0;
#pragma unroll
        for (uint32_t i = 0; i < OWN; i++)
            if (wanted(OWN * threadIdx.x + i)) run += tokens[i], place++;
        running_sums<THREADS>(run, place, s);
        held = (uint32_t)run, buckets = (uint32_t)place;
        if (threadIdx.x == THREADS - 1) s.at[0] = held, s.at[1] = buckets;
        __syncthreads();
        wanted_tokens = s.at[0], wanted_buckets = s.at[1];
        __syncthreads();
    }

    // Of each run, the logits lowest .. lowest + reach.
    int32_t lowest[3];
    uint32_t reach[3];
    __device__ __forceinline__ void set_logits(const RowDraw& d, int32_t top) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            lowest[i] = INT32_MIN, reach[i] = 0;  // (closed places, left out below)
            if (low[i] > high[i]) continue;
            // No gap passes that of the lowest open logit.
            const uint64_t far = min(min(((uint64_t)high[i] + 1) << d.shift, d.end) - 1, (uint64_t)((int64_t)top - INT32_MIN));
            const uint64_t near = (uint64_t)low[i] << d.shift;
            lowest[i] = (int32_t)((int64_t)top - (int64_t)far), reach[i] = (uint32_t)(far - near);
        }
    }
    __device__ __forceinline__ bool has(int32_t l) const {
        const uint32_t x = (uint32_t)l;
        return (x - (uint32_t)lowest[0] <= reach[0]) | (x - (uint32_t)lowest[1] <= reach[1]) | (x - (uint32_t)lowest[2] <= reach[2]);
    }
    // f(key, place) for the tokens of v0 .. v1 of a row in the runs, their places
    // taken from a counter in LDS, a wave's at once.
    template <uint32_t DEPTH, class F>
    __device__ __forceinline__ void each(const int32_t* in, uint32_t v0, uint32_t v1, bool vec, int32_t top, uint32_t* counter, F&& f) const {
        each_logit<THREADS, DEPTH>(in, v0, v1, vec, [&](int4 x, uint32_t v) {
            const int32_t l[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const bool found = has(l[i]) && l[i] != INT32_MIN;
                const uint64_t all = __ballot(found);
                if (!all) continue;
                const uint32_t lane = threadIdx.x & 63, first = __builtin_ctzll(all);
                uint32_t place = 0;
                if (lane == first) place = atomicAdd(counter, (uint32_t)__popcll(all));
                place = (uint32_t)__builtin_amdgcn_readlane((int)place, first) + __popcll(all & ((1ull << lane) - 1));
                if (found) f((uint64_t)((uint32_t)top - (uint32_t)l[i]) << INDEX_BITS | (v + i), place);
            }
        });
    }
};

// The tokens of a piece of a long row in the runs, behind those that other
// pieces have gathered (in any order: their keys order them).
__global__ __launch_bounds__(256) void draw_gather_kernel(const IrisLogitsDraw a, const DrawPieces p, const uint64_t* tops, DrawRow* space) {
    __shared__ BucketSpace s;
    __shared__ uint64_t s_key[PIECE_LIST];
    __shared__ uint64_t s_best[4];
    __shared__ uint32_t s_count, s_at;
    const uint32_t row = blockIdx.y, v0 = blockIdx.x * GATHER_PIECE, v1 = min(v0 + GATHER_PIECE, a.vocab);
    const RowDraw d = space[row].draw;
    if (!d.beta) return;
    if (threadIdx.x == 0) s_count = 0;
    Runs<256> runs;
    runs.load(space[row]);
    const uint32_t number = a.numbers[row];
    const int32_t top = key_logit(row_top<256>(tops + (size_t)row * p.count, p.count, s_best));
    if (top == INT32_MIN) return;
    uint32_t held, buckets;
    runs.find(d, number, s, held, buckets);
    if (runs.wanted_tokens > GATHER) return;
    runs.set_logits(d, top);
    runs.each<4>(a.logits + (size_t)row * a.logits_stride, v0, v1, p.vec, top, &s_count, [&](uint64_t key, uint32_t i) {
        if (i < PIECE_LIST) {
            s_key[i] = key;
        } else {  // (crowded)
            const uint32_t at = atomicAdd(&space[row].gathered, 1u);
            if (at < GATHER) space[row].key[at] = key;
        }
    });
    __syncthreads();
    const uint32_t n = min(s_count, PIECE_LIST);
    if (threadIdx.x == 0) s_at = n ? atomicAdd(&space[row].gathered, n) : 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < n && s_at + i < GATHER; i += 256) space[row].key[s_at + i] = s_key[i];
}

// A row's token from its histogram, and (LISTED) the tokens gathered from it.
template <bool LISTED>
__global__ __launch_bounds__(PICK_THREADS) void draw_pick_kernel(const IrisLogitsDraw a, const DrawPieces pieces, const uint64_t* tops,
                                                                 const DrawRow* space) {
    __shared__ PickSpace s;
    __shared__ uint64_t s_best[PICK_THREADS / 64];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    Pick p{};
    p.d = space[row].draw;
    p.in = a.logits + (size_t)row * a.logits_stride;
    p.vocab = a.vocab, p.vec = pieces.vec;
    const uint32_t number = a.numbers ? a.numbers[row] : 0;
    Runs<PICK_THREADS> runs;
    runs.load(space[row]);
    const uint64_t top = row_top<PICK_THREADS>(tops + (size_t)row * pieces.count, pieces.count, s_best);
    p.most = key_logit(top);
    if (p.most == INT32_MIN || !p.d.beta) {
        if (tid == 0) {
            const bool none = p.most == INT32_MIN;
            a.tokens[row] = none ? -1 : (int32_t)~(uint32_t)top;
            if (a.mass) a.mass[2 * (size_t)row] = a.mass[2 * (size_t)row + 1] = none ? 0 : 1ll << 32;
        }
        return;
    }
    const bool counts_only = p.d.counts_only();
    uint32_t held, buckets;
    runs.find(p.d, number, s, held, buckets);
    auto before = [&](uint32_t bucket) { return bucket ? s.sum[bucket - 1] : 0; };
    constexpr uint32_t MINE = Runs<PICK_THREADS>::OWN;
    const uint32_t n = runs.wanted_tokens;
    const bool gathered = n <= GATHER;
    uint32_t have = 0;  // the gathered (all n)
    auto sum_before = [&](uint32_t at) { return at ? s.upto[at - 1] : 0; };
    // The gathered tokens in order: s.token, and the running sums of their weights,
    // s.upto.
    if (gathered) {
        // Each of the thread's buckets' first place, and the place behind them.
        uint32_t first_of[MINE + 1], ordinal = buckets;
        first_of[MINE] = held;
#pragma unroll
        for (uint32_t i = MINE; i-- > 0;) {
            const bool has = runs.wanted(MINE * tid + i);
            first_of[i] = first_of[i + 1] - (has ? runs.tokens[i] : 0), ordinal -= has;
            s.place_of[MINE * tid + i] = ordinal << 16 | first_of[i];
        }
        constexpr uint32_t OWN = GATHER / PICK_THREADS;
#pragma unroll
        for (uint32_t i = 0; i < OWN; i++) s.part[tid + i * PICK_THREADS] = 0;
        if (tid == 0) s.found = 0;
        __syncthreads();
        if constexpr (LISTED) {
            have = min(n, space[row].gathered);
#pragma unroll 1
            for (uint32_t i = tid; i < have; i += PICK_THREADS) s.token[i] = space[row].key[i];
        } else {
            runs.set_logits(p.d, p.most);
            runs.each<8>(p.in, 0, p.vocab, p.vec, p.most, &s.found, [&](uint64_t key, uint32_t i) {
                if (i < GATHER) s.token[i] = key;
            });
            __syncthreads();
            have = min(s.found, n);
        }
        // By parts of the buckets, as many as there is room for, and within a
        // part by comparison: a few tokens, but all of one gap where logits are
        // equal (4000 of them in a row of 32000: 751 us, without 21.5). Weights are formed here and not
        // where the tokens are found, a few lanes of a wave at a time.
        const uint32_t fine = min(31u - __clz((int)(GATHER / max(runs.wanted_buckets, 1u))), p.d.shift + INDEX_BITS);
        auto bucket_at = [&](uint64_t key) { return min((uint32_t)(key >> (p.d.shift + INDEX_BITS)), BUCKETS - 1); };
        auto part_at = [&](uint64_t key) {
            const uint32_t inside = (uint32_t)(key >> (p.d.shift + INDEX_BITS - fine)) & ((1u << fine) - 1);
            return min((s.place_of[bucket_at(key)] >> 16 << fine) + inside, GATHER - 1);
        };
#pragma unroll 1
        for (uint32_t i = tid; i < have; i += PICK_THREADS) s.behind[i] = (uint16_t)atomicAdd(&s.part[part_at(s.token[i])], 1u);
        __syncthreads();
        static_assert(OWN == 8, "a thread's parts are two times four");
        uint4* parts = (uint4*)s.part + 2 * tid;
        const uint4 c0 = parts[0], c1 = parts[1];
        uint64_t run = c0.x + c0.y + c0.z + c0.w + c1.x + c1.y + c1.z + c1.w, sum = 0;
        const uint64_t mine = run;
        running_sums<PICK_THREADS>(run, sum, s);
        const uint32_t r0 = (uint32_t)(run - mine), r1 = r0 + c0.x + c0.y + c0.z + c0.w;
        parts[0] = make_uint4(r0, r0 + c0.x, r0 + c0.x + c0.y, r1 - c0.w);
        parts[1] = make_uint4(r1, r1 + c1.x, r1 + c1.x + c1.y, r1 + c1.x + c1.y + c1.z);
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = tid; i < have; i += PICK_THREADS) s.key[s.part[part_at(s.token[i])] + s.behind[i]] = s.token[i];
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = tid; i < have; i += PICK_THREADS) {
            const uint64_t key = s.key[i];
            const uint32_t part = part_at(key), from = s.part[part], to = part + 1 < GATHER ? s.part[part + 1] : have;
            uint32_t at = from;
#pragma unroll 4
            for (uint32_t j = from; j < to; j++) at += s.key[j] < key ? 1 : 0;
            s.token[at] = key, s.upto[at] = weight_of(p.d, (uint32_t)(key >> INDEX_BITS));
        }
        __syncthreads();
        // Neighbours in a thread, as few as there are.
        const uint32_t each = (have + PICK_THREADS - 1) / PICK_THREADS, t0 = min(tid * each, have), t1 = min(t0 + each, have);
        run = sum = 0;
#pragma unroll 1
        for (uint32_t i = t0; i < t1; i++) sum += s.upto[i];
        const uint64_t own_sum = sum;
        running_sums<PICK_THREADS>(run, sum, s);
        sum -= own_sum;
#pragma unroll 1
        for (uint32_t i = t0; i < t1; i++) s.upto[i] = sum += s.upto[i];
        __syncthreads();
        if (counts_only) {
            uint64_t of[MINE];
#pragma unroll
            for (uint32_t i = 0; i < MINE; i++) of[i] = sum_before(first_of[i + 1]) - sum_before(first_of[i]);
            runs.add_up(of, s);
        }
    } else if (counts_only) {
        // The weights of the buckets up to the k-th token's, from the row.
#pragma unroll
        for (uint32_t i = 0; i < MINE; i++) s.sum[MINE * tid + i] = 0;
        __syncthreads();
        p.each(0, 63, [&](uint64_t, uint32_t gap) {
            if (gap >> p.d.shift <= runs.k_bucket)
                atomicAdd((unsigned long long*)&s.sum[gap >> p.d.shift], (unsigned long long)weight_of(p.d, gap));
        });
        __syncthreads();
        uint64_t w[MINE];
#pragma unroll
        for (uint32_t i = 0; i < MINE; i++) w[i] = s.sum[MINE * tid + i];
        __syncthreads();
        runs.add_up(w, s);
    }

    // The weight of the tokens kept, by each bound in turn, and the token. (The
    // share's run reaches its sum: passes one less than it.)
    uint64_t sum = s.whole;
    Place at{};
#pragma unroll 1
    for (int turn = runs.by_k ? 0 : 1; turn < 3; turn++) {
        if (turn == 1 && !p.d.top_p) continue;
        const uint64_t value = turn == 0 ? p.d.top_k : turn == 1 ? share_of(sum, p.d.top_p, true) - 1 : share_of(sum, number, false);
        if (gathered) {
#pragma unroll 1
            for (uint32_t i = tid; i < have; i += PICK_THREADS) {
                const uint64_t key = s.token[i], weight = s.upto[i] - sum_before(i);
                const uint32_t bucket = min((uint32_t)(key >> (p.d.shift + INDEX_BITS)), BUCKETS - 1);
                const uint32_t start = s.place_of[bucket] & 0xffff;
                const uint64_t count = (bucket ? s.count[bucket - 1] : 0) + i - start + 1;
                const uint64_t upto = before(bucket) + s.upto[i] - sum_before(start);
                if (turn == 0 ? count == value : upto > value && upto - weight <= value) s.place = Place{key, weight, count, upto};
            }
            __syncthreads();
            at = s.place;
            __syncthreads();
        } else {
            at = find_place(p, turn == 0, value, s);
        }
        if (turn < 2) sum = at.sum;
    }
    if (tid == 0) {
        a.tokens[row] = (int32_t)(at.key & ((1u << INDEX_BITS) - 1));
        if (a.mass) a.mass[2 * (size_t)row] = (int64_t)at.weight, a.mass[2 * (size_t)row + 1] = (int64_t)sum;
    }
}

// Pieces of a row: small ones while the rows alone would leave the card idle.
DrawPieces draw_pieces(const IrisLogitsDraw& a) {
    DrawPieces p;
    p.size = 2048;
    while (p.size < MAX_PIECE && (uint64_t)a.rows * ((a.vocab + p.size - 1) / p.size) > 768) p.size *= 2;
    p.count = (a.vocab + p.size - 1) / p.size;
    p.vec = !misaligned(a.logits) && a.logits_stride % 4 == 0;
    return p;
}

int draw_check(const IrisLogitsDraw* a) {
    if (!a || !a->logits || !a->tokens || !a->vocab || a->logits_stride < a->vocab) return IRIS_E_INVALID;
    if (a->drawings && (!a->numbers || !a->requests)) return IRIS_E_INVALID;
    if (a->vocab > MAX_VOCAB || a->rows > MAX_ROWS || a->requests > INT32_MAX) return IRIS_E_RANGE;
    return 0;
}

}  // namespace

extern "C" {

int iris_logits_rules(const IrisLogitsRules* a, void* stream) {
    if (!a) return IRIS_E_INVALID;
    if (!a->rows) return 0;
    if (!a->logits || !a->out || !a->vocab || a->logits_stride < a->vocab || a->out_stride < a->vocab) return IRIS_E_INVALID;
    if (a->out == a->logits && a->out_stride != a->logits_stride) return IRIS_E_INVALID;
    if (a->rules) {
        if (!a->request || !a->requests || (a->history && !a->lengths) || (a->ids && !a->row_start)) return IRIS_E_INVALID;
        if (a->biases && (!a->bias_ids || !a->bias_values)) return IRIS_E_INVALID;
    }
    if (a->mask_rows && (!a->masks || !a->mask_of || a->mask_stride < (a->vocab + 31) / 32)) return IRIS_E_INVALID;
    if (a->vocab > MAX_VOCAB || a->rows > MAX_ROWS || a->requests > INT32_MAX || a->mask_rows > INT32_MAX ||
        a->history_stride > MAX_HISTORY || a->biases > MAX_BIASES || a->first_row > INT32_MAX - MAX_ROWS)
        return IRIS_E_RANGE;
    // Small pieces while the rows alone would leave the card idle; of many, several
    // to a workgroup.
    uint32_t piece = MIN_RULE_PIECE;
    while (piece < MAX_RULE_PIECE && (uint64_t)a->rows * ((a->vocab + piece - 1) / piece) > (a->history_stride > LONG_TEXT ? 256 : 2048)) piece *= 2;
    const uint32_t pieces = (a->vocab + piece - 1) / piece, most = std::max(1u, RULE_GROUPS / a->rows);
    const uint32_t turns = (pieces + most - 1) / most;
    const dim3 grid((pieces + turns - 1) / turns, a->rows);
    const bool vec = !misaligned(a->logits) && !misaligned(a->out) && a->logits_stride % 4 == 0 && a->out_stride % 4 == 0;
    if (vec) hipLaunchKernelGGL(rules_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, *a, piece);
    else hipLaunchKernelGGL(rules_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, *a, piece);
    return (int)hipGetLastError();
}

uint64_t iris_logits_draw_workspace_bytes(const IrisLogitsDraw* a) {
    if (draw_check(a) || !a->rows) return 0;
    return (uint64_t)a->rows * (sizeof(DrawRow) + draw_pieces(*a).count * 8);
}

int iris_logits_draw(const IrisLogitsDraw* a, void* space, uint64_t space_bytes, void* stream) {
    const int rc = draw_check(a);
    if (rc) return rc;
    if (!a->rows) return 0;
    if (!space || misaligned(space)) return IRIS_E_INVALID;
    if (space_bytes < iris_logits_draw_workspace_bytes(a)) return IRIS_E_RANGE;
    const DrawPieces pieces = draw_pieces(*a);
    DrawRow* rows = (DrawRow*)space;
    uint64_t* tops = (uint64_t*)(rows + a->rows);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(draw_top_kernel, dim3(pieces.count, a->rows), dim3(256), 0, st, *a, pieces, tops, rows);
    if (a->drawings) hipLaunchKernelGGL(draw_histogram_kernel, dim3(pieces.count, a->rows), dim3(256), 0, st, *a, pieces, tops, rows);
    if (a->drawings && a->vocab > LONG_ROW) {
        hipLaunchKernelGGL(draw_gather_kernel, dim3((a->vocab + GATHER_PIECE - 1) / GATHER_PIECE, a->rows), dim3(256), 0, st, *a, pieces,
                           tops, rows);
        hipLaunchKernelGGL(draw_pick_kernel<true>, dim3(a->rows), dim3(PICK_THREADS), 0, st, *a, pieces, tops, rows);
    } else {
        hipLaunchKernelGGL(draw_pick_kernel<false>, dim3(a->rows), dim3(PICK_THREADS), 0, st, *a, pieces, tops, rows);
    }
    return (int)hipGetLastError();
}

}  // extern "C"
