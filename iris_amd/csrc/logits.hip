// Rows of logits to tokens, each request in its own way: penalties for repeated
// tokens, biases and grammar masks (iris_logits_rules), and the draw of a token
// (iris_logits_draw).
#include <algorithm>

#include "detnum_dev.h"
#include "paged.h"
#include "softmax_double.h"

namespace {

constexpr uint32_t MAX_VOCAB = 1u << 20, MAX_ROWS = 65535, MAX_HISTORY = 1u << 20, MAX_BIASES = 1u << 20;

// ------------------------------------------------------------------ rules

constexpr uint32_t RULE_PIECE = 4096;  // tokens a workgroup takes: their counts and biases in LDS

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

// What a row's request says, read once by each workgroup.
struct RowRule {
    IrisTokenRule rule;
    const int32_t* text;   // the history
    int64_t from, length;  // of it, the part that counts
    int32_t start, own;    // the drafted rows: the first, and this one among them; own -1: none
    int32_t mask;
};

__device__ __forceinline__ void report(const IrisLogitsRules& a, int32_t code) {
    if (a.status) *a.status = code;
}

// One piece of one row: the text's tokens in the piece are counted and the
// biases summed in LDS, then the piece's logits pass once.
__global__ __launch_bounds__(256) void rules_kernel(const IrisLogitsRules a) {
    __shared__ uint32_t s_count[RULE_PIECE];
    __shared__ uint64_t s_bias[RULE_PIECE];
    const uint32_t row = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const uint32_t v0 = blockIdx.x * RULE_PIECE, v1 = min(v0 + RULE_PIECE, a.vocab);
    const bool first = blockIdx.x == 0 && tid == 0;

    int32_t mask = a.masks && a.mask_of ? a.mask_of[row] : -1;
    if (mask < -1 || mask >= (int32_t)a.mask_rows) {
        if (first) report(a, IRIS_E_INVALID);
        mask = -1;
    }
    int32_t q = a.rules ? a.request[row] : -1;
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
    const int32_t* in = a.logits + (size_t)row * a.logits_stride;
    int32_t* out = a.out + (size_t)row * a.out_stride;
    const uint32_t* bits = a.masks + (size_t)(mask < 0 ? 0 : mask) * a.mask_stride;
    if (q >= 0) {
        for (uint32_t i = tid; i < RULE_PIECE; i += 256) s_count[i] = 0, s_bias[i] = 0;
        __syncthreads();
        uint64_t path = 0;  // the drafted rows from the root to this one
        if (own >= 0) {
            const uint64_t above = tree_ancestors(a.parents ? a.parents + start : nullptr, own + 1, lane);
            path = __shfl((unsigned long long)above, own);
        }
        const int64_t whole = length + __popcll(path);
        const int64_t from = rule.window && whole > rule.window ? whole - rule.window : 0;
        const int32_t* text = a.history + (size_t)q * a.history_stride;
        for (int64_t i = from + tid; i < length; i += 256) {
            const uint32_t v = (uint32_t)text[i] - v0;
            if (v < v1 - v0) atomicAdd(&s_count[v], 1u);
        }
        // The path's row of lane l is its place in the path behind the history.
        if (tid < 64 && (path >> lane & 1) && length + __popcll(path & ((1ull << lane) - 1)) >= from) {
            const uint32_t v = (uint32_t)a.ids[start + lane] - v0;
            if (v < v1 - v0) atomicAdd(&s_count[v], 1u);
        }
        for (uint32_t i = tid; i < rule.bias_count; i += 256) {
            const uint32_t v = (uint32_t)a.bias_ids[rule.bias_start + i] - v0;
            if (v < v1 - v0) atomicAdd((unsigned long long*)&s_bias[v], (unsigned long long)(int64_t)a.bias_values[rule.bias_start + i]);
        }
        __syncthreads();
    }
    const double inverse = 1.0 / rule.repetition;
    for (uint32_t v = v0 + tid; v < v1; v += 256) {
        int64_t l = in[v];
        const bool closed = l == INT32_MIN || (mask >= 0 && !(bits[v / 32] >> (v % 32) & 1));
        if (q >= 0) {
            const int64_t c = s_count[v - v0];
            if (c) {
                l = l > 0 ? divided((int32_t)l, rule.repetition, inverse) : dn::rshift_rte(l * rule.repetition, 16);
                l -= c * rule.frequency + rule.presence;
            }
            l += (int64_t)s_bias[v - v0];
        }
        if (l < INT32_MIN + 1) l = INT32_MIN + 1;
        if (l > INT32_MAX) l = INT32_MAX;
        out[v] = closed ? INT32_MIN : (int32_t)l;
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
// Three launches: the row's maximum by pieces; the histogram; the places.

constexpr uint32_t DRAW_PIECE = 4096;
constexpr uint32_t BUCKETS = 2048;
constexpr uint32_t PICK_THREADS = 1024;
constexpr uint32_t LIST = 1024;       // tokens put in order at a time
constexpr uint32_t SUB_BITS = 10;     // a crowded bucket's parts
constexpr uint32_t INDEX_BITS = 20;   // of a token's index

// Work space of a row.
struct DrawRow {
    uint32_t count[BUCKETS];
    uint64_t sum[BUCKETS];
};

// A logit and its index as one key: larger for a larger logit, of equal ones
// for the smaller index.
__device__ __forceinline__ int64_t draw_key(int32_t v, uint32_t i) { return (int64_t)v << 32 | (uint32_t)~i; }

__device__ __forceinline__ int64_t wave_max(int64_t k) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) k = max(k, (int64_t)__shfl_xor((long long)k, off));
    return k;
}

// How a row draws. Gaps from `end` on have no weight; bucket b holds the gaps
// from b << shift on.
struct RowDraw {
    int64_t beta;
    uint32_t top_k, top_p;
    uint64_t end;
    uint32_t shift;
};

// The weight of a gap below `end`.
__device__ __forceinline__ uint64_t weight_of(const RowDraw& d, uint32_t gap) {
    uint32_t kept;
    return (uint64_t)softmax_term((uint32_t)dn::rshift_rte((int64_t)gap * d.beta, 16), &kept);
}

__device__ __forceinline__ RowDraw row_draw(const IrisLogitsDraw& a, uint32_t row, bool report) {
    RowDraw d{};
    if (!a.drawings) return d;
    const int32_t q = a.request ? a.request[row] : (int32_t)row;
    if (q < 0 || q >= (int32_t)a.requests) {
        if (q != -1 && report && a.status) *a.status = IRIS_E_INVALID;
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
    while ((d.end - 1) >> d.shift >= BUCKETS) d.shift++;
    return d;
}

// The largest key of each piece of a row; and the row's histogram cleared.
__global__ __launch_bounds__(256) void draw_top_kernel(const IrisLogitsDraw a, int64_t* tops, DrawRow* space) {
    __shared__ int64_t s_best[4];
    const uint32_t row = blockIdx.y, pieces = gridDim.x, v0 = blockIdx.x * DRAW_PIECE, v1 = min(v0 + DRAW_PIECE, a.vocab);
    const int32_t* in = a.logits + (size_t)row * a.logits_stride;
    int64_t k = INT64_MIN;
    for (uint32_t v = v0 + threadIdx.x; v < v1; v += 256) k = max(k, draw_key(in[v], v));
    k = wave_max(k);
    if (threadIdx.x % 64 == 0) s_best[threadIdx.x / 64] = k;
    __syncthreads();
    if (threadIdx.x == 0) tops[(size_t)row * pieces + blockIdx.x] = max(max(s_best[0], s_best[1]), max(s_best[2], s_best[3]));
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < BUCKETS; i += pieces * 256) space[row].count[i] = 0, space[row].sum[i] = 0;
}

// The row's largest key, by a workgroup (every thread gets it).
__device__ __forceinline__ int64_t row_top(const int64_t* tops, uint32_t pieces, int64_t* s_best) {
    int64_t k = INT64_MIN;
    for (uint32_t i = threadIdx.x; i < pieces; i += blockDim.x) k = max(k, tops[i]);
    k = wave_max(k);
    if (threadIdx.x % 64 == 0) s_best[threadIdx.x / 64] = k;
    __syncthreads();
    for (uint32_t w = 0; w < blockDim.x / 64; w++) k = max(k, s_best[w]);
    return k;
}

// A piece's part of the row's histogram.
__global__ __launch_bounds__(256) void draw_histogram_kernel(const IrisLogitsDraw a, const int64_t* tops, DrawRow* space) {
    __shared__ uint64_t s_bucket[BUCKETS];  // count 2^46 + sum: at most 4096 weights of 2^32
    __shared__ int64_t s_best[4];
    const uint32_t row = blockIdx.y, pieces = gridDim.x, v0 = blockIdx.x * DRAW_PIECE, v1 = min(v0 + DRAW_PIECE, a.vocab);
    const RowDraw d = row_draw(a, row, false);
    if (!d.beta) return;
    const int64_t top = row_top(tops + (size_t)row * pieces, pieces, s_best);
    const int32_t most = (int32_t)(top >> 32);
    if (most == INT32_MIN) return;
    for (uint32_t i = threadIdx.x; i < BUCKETS; i += 256) s_bucket[i] = 0;
    __syncthreads();
    const int32_t* in = a.logits + (size_t)row * a.logits_stride;
    for (uint32_t v = v0 + threadIdx.x; v < v1; v += 256) {
        const int32_t l = in[v];
        const uint32_t gap = (uint32_t)most - (uint32_t)l;
        if (l != INT32_MIN && gap < d.end)
            atomicAdd((unsigned long long*)&s_bucket[gap >> d.shift], (unsigned long long)(1ull << 46 | weight_of(d, gap)));
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < BUCKETS; i += 256) {
        const uint64_t x = s_bucket[i];
        if (!x) continue;
        atomicAdd(&space[row].count[i], (uint32_t)(x >> 46));
        atomicAdd((unsigned long long*)&space[row].sum[i], (unsigned long long)(x & ((1ull << 46) - 1)));
    }
}

// A place in the row's order: the token's key (gap 2^20 + index), its weight,
// and the tokens and weights up to it, itself included.
struct Place {
    uint64_t key, weight, count, sum;
};

struct PickSpace {
    uint64_t count[BUCKETS];  // running, inclusive
    uint64_t sum[BUCKETS];
    uint64_t sub_sum[1 << SUB_BITS];
    uint32_t sub_count[1 << SUB_BITS];
    uint64_t list[LIST];
    uint64_t weight[LIST];
    uint64_t wave[2][PICK_THREADS / 64];
    static_assert(LIST >= 1u << (SUB_BITS - 1) && LIST <= PICK_THREADS, "a listed token a thread");
    uint32_t listed, found;
    Place place;
};

// Inclusive running sums over the workgroup's threads of a pair.
__device__ __forceinline__ void running_sums(uint64_t& x, uint64_t& y, PickSpace& s) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint64_t px = __shfl_up((unsigned long long)x, off), py = __shfl_up((unsigned long long)y, off);
        if ((int)lane >= off) x += px, y += py;
    }
    if (lane == 63) s.wave[0][wave] = x, s.wave[1][wave] = y;
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) x += s.wave[0][w], y += s.wave[1][w];
    __syncthreads();
}

// The first place where the running count reaches `value` (by_count) or the
// running sum passes it. `value` is below the row's count + 1, or its sum.
__device__ __forceinline__ Place find_place(const IrisLogitsDraw& a, const RowDraw& d, const int32_t* in, int32_t most, bool by_count, uint64_t value,
                            PickSpace& s) {
    const uint32_t tid = threadIdx.x;
    auto reached = [&](uint64_t count, uint64_t sum) { return by_count ? count >= value : sum > value; };
    // The bucket: the first whose running sums reach it.
    if (tid == 0) s.found = BUCKETS;
    __syncthreads();
    for (uint32_t i = tid; i < BUCKETS; i += PICK_THREADS)
        if (reached(s.count[i], s.sum[i])) atomicMin(&s.found, i);
    __syncthreads();
    const uint32_t bucket = min(s.found, BUCKETS - 1);
    uint64_t count = bucket ? s.count[bucket - 1] : 0, sum = bucket ? s.sum[bucket - 1] : 0;  // before it
    uint64_t inside = s.count[bucket] - count;
    uint64_t low = (uint64_t)bucket << (d.shift + INDEX_BITS);  // the keys at hand: low .. low + 2^bits
    uint32_t bits = d.shift + INDEX_BITS;
    auto each = [&](auto&& f) {
        for (uint32_t v = tid; v < a.vocab; v += PICK_THREADS) {
            const int32_t l = in[v];
            const uint32_t gap = (uint32_t)most - (uint32_t)l;
            const uint64_t key = (uint64_t)gap << INDEX_BITS | v;
            if (l != INT32_MIN && gap < d.end && key - low < 1ull << bits) f(key, gap);
        }
    };
    while (inside > LIST && bits >= SUB_BITS) {
        // A crowded range: its parts' counts and sums, and the part that reaches.
        // (Fewer bits than that hold at most LIST keys.)
        const uint32_t part_bits = bits - SUB_BITS;
        __syncthreads();
        for (uint32_t i = tid; i < 1u << SUB_BITS; i += PICK_THREADS) s.sub_sum[i] = 0, s.sub_count[i] = 0;
        if (tid == 0) s.found = 1u << SUB_BITS;
        __syncthreads();
        each([&](uint64_t key, uint32_t gap) {
            const uint32_t i = (uint32_t)((key - low) >> part_bits);
            atomicAdd(&s.sub_count[i], 1u);
            atomicAdd((unsigned long long*)&s.sub_sum[i], (unsigned long long)weight_of(d, gap));
        });
        __syncthreads();
        static_assert(1u << SUB_BITS == PICK_THREADS, "a part a thread");
        const uint64_t own_count = s.sub_count[tid], own_sum = s.sub_sum[tid];
        uint64_t run_count = own_count, run_sum = own_sum;
        running_sums(run_count, run_sum, s);
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
    each([&](uint64_t key, uint32_t gap) {
        const uint32_t i = atomicAdd(&s.listed, 1u);
        if (i < LIST) s.list[i] = key, s.weight[i] = weight_of(d, gap);
    });
    __syncthreads();
    // Each token's running sums by comparing it with the others; the place is
    // the one that reaches and whose forerunner does not.
    const uint32_t n = min(s.listed, LIST);
    if (tid < n) {
        const uint64_t key = s.list[tid], weight = s.weight[tid];
        uint64_t c = count + 1, w = sum + weight;
        for (uint32_t i = 0; i < n; i++)
            if (s.list[i] < key) c++, w += s.weight[i];
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

// A row's token from its histogram.
__global__ __launch_bounds__(PICK_THREADS) void draw_pick_kernel(const IrisLogitsDraw a, const int64_t* tops, const DrawRow* space,
                                                                 uint32_t pieces) {
    __shared__ PickSpace s;
    __shared__ int64_t s_best[PICK_THREADS / 64];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const RowDraw d = row_draw(a, row, tid == 0);
    const int64_t top = row_top(tops + (size_t)row * pieces, pieces, s_best);
    const int32_t most = (int32_t)(top >> 32);
    if (most == INT32_MIN || !d.beta) {
        if (tid == 0) {
            const bool none = most == INT32_MIN;
            a.tokens[row] = none ? -1 : (int32_t)~(uint32_t)top;
            if (a.mass) a.mass[2 * (size_t)row] = a.mass[2 * (size_t)row + 1] = none ? 0 : 1ll << 32;
        }
        return;
    }
    const int32_t* in = a.logits + (size_t)row * a.logits_stride;
    // Running sums of the buckets, neighbours in a thread.
    {
        static_assert(BUCKETS == 2 * PICK_THREADS, "two buckets a thread");
        const uint64_t c0 = space[row].count[2 * tid], c1 = space[row].count[2 * tid + 1];
        const uint64_t w0 = space[row].sum[2 * tid], w1 = space[row].sum[2 * tid + 1];
        uint64_t c = c0 + c1, w = w0 + w1;
        running_sums(c, w, s);
        s.count[2 * tid] = c - c1, s.count[2 * tid + 1] = c;
        s.sum[2 * tid] = w - w1, s.sum[2 * tid + 1] = w;
        __syncthreads();
    }
    const uint64_t open = s.count[BUCKETS - 1];
    // The kept tokens' number and weight.
    uint64_t kept = open, sum = s.sum[BUCKETS - 1];
    if (d.top_k && d.top_k < kept) {
        const Place p = find_place(a, d, in, most, true, d.top_k, s);
        kept = p.count, sum = p.sum;
    }
    if (d.top_p) {
        // The run's sum reaches the share: passes one less than it.
        const Place p = find_place(a, d, in, most, false, share_of(sum, d.top_p, true) - 1, s);
        kept = p.count, sum = p.sum;
    }
    const Place p = find_place(a, d, in, most, false, share_of(sum, a.numbers[row], false), s);
    if (tid == 0) {
        a.tokens[row] = (int32_t)(p.key & ((1u << INDEX_BITS) - 1));
        if (a.mass) a.mass[2 * (size_t)row] = (int64_t)p.weight, a.mass[2 * (size_t)row + 1] = (int64_t)sum;
    }
}

uint32_t draw_pieces(const IrisLogitsDraw& a) { return (a.vocab + DRAW_PIECE - 1) / DRAW_PIECE; }

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
    hipLaunchKernelGGL(rules_kernel, dim3((a->vocab + RULE_PIECE - 1) / RULE_PIECE, a->rows), dim3(256), 0, (hipStream_t)stream, *a);
    return (int)hipGetLastError();
}

uint64_t iris_logits_draw_workspace_bytes(const IrisLogitsDraw* a) {
    if (draw_check(a) || !a->rows) return 0;
    return (uint64_t)a->rows * (sizeof(DrawRow) + draw_pieces(*a) * 8);
}

int iris_logits_draw(const IrisLogitsDraw* a, void* space, uint64_t space_bytes, void* stream) {
    const int rc = draw_check(a);
    if (rc) return rc;
    if (!a->rows) return 0;
    if (!space || misaligned(space)) return IRIS_E_INVALID;
    if (space_bytes < iris_logits_draw_workspace_bytes(a)) return IRIS_E_RANGE;
    const uint32_t pieces = draw_pieces(*a);
    DrawRow* rows = (DrawRow*)space;
    int64_t* tops = (int64_t*)(rows + a->rows);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(draw_top_kernel, dim3(pieces, a->rows), dim3(256), 0, st, *a, tops, rows);
    if (a->drawings) hipLaunchKernelGGL(draw_histogram_kernel, dim3(pieces, a->rows), dim3(256), 0, st, *a, tops, rows);
    hipLaunchKernelGGL(draw_pick_kernel, dim3(a->rows), dim3(PICK_THREADS), 0, st, *a, tops, rows, pieces);
    return (int)hipGetLastError();
}

}  // extern "C"
