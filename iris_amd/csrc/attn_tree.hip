// Attention of drafted trees over a paged cache, exact, on the int8 matrix
// cores.
//
// The rows of a tile are a request's (drafted row, head of one key head)
// pairs, so that each key and value is read once for all of them; keys and
// values become digit planes in registers, straight from their pages. The
// softmax is the reference's (ops.rs:233-261): first maximum, then all exp
// terms' sum, then weights. With a request's positions dealt to workgroups in
// chunks these are four launches: scores and each chunk's maxima; exp terms in
// place of the scores and each chunk's sums; weights and weighted values, a
// partial sum per chunk; the partial sums joined, with what the weights lack
// of one. All sums are integers (the exp terms' exact in double): the same
// bits however the positions are dealt.
#include <algorithm>
#include <type_traits>

#include "attn_tiles.h"

namespace {

// A place of zeros for positions whose page is outside the cache.
__device__ const int32_t g_zeros[ATTN_MAX_HEAD_DIM] = {};

constexpr uint32_t STEP = 64;  // positions of a value product

// The work space of a launch. Row tiles count a request's (drafted row, head)
// pairs by sixteens, `row_tiles` per (request, key head).
struct TreeSpace {
    uint4* scores;     // [request, key head][row tile][key tile][64] scores, then exp terms
    uint64_t* maxima;  // [..][row tile][chunk][16]: score and position, packed; 0: none seen
    double* sums;      // [..][row tile][chunk][16]
    int32_t* weights;  // [..][row tile][chunk][16] the weights' sum
    uint64_t* partial; // [..][row tile][chunk][16][HD] weighted values
    uint32_t row_tiles, chunks, chunk;  // positions per chunk, whole steps
};

// A request as a workgroup finds it.
struct Request {
    uint32_t row0, rows, length, total;  // first row, drafted rows, positions before them, all positions
    uint32_t base;                       // first position that is looked at, a multiple of STEP
    const int32_t* table;
};

__device__ __forceinline__ bool read_request(const IrisPagedKv& c, const IrisTreeAttention& a, uint32_t b, Request& r) {
    const int64_t r0 = a.row_start[b], r1 = a.row_start[b + 1], len = a.lengths[b], n = r1 - r0;
    if (n <= 0) return false;
    if (r0 < 0 || r1 > a.rows || n > a.max_nodes || len < 0 || len + n > a.max_positions ||
        len + n > (int64_t)a.table_stride * c.page_size) {
        if (a.status) *a.status = IRIS_E_RANGE;
        return false;
    }
    r.row0 = (uint32_t)r0, r.rows = (uint32_t)n, r.length = (uint32_t)len, r.total = (uint32_t)(len + n);
    const uint32_t first = a.window && r.length >= a.window ? r.length + 1 - a.window : 0;
    r.base = first & ~(STEP - 1);
    r.table = a.table + (size_t)b * a.table_stride;
    return true;
}

// What a lane's row sees: positions [lo, length) and the drafted rows of mask.
struct RowView {
    uint32_t lo, length;
    uint64_t mask;
    __device__ __forceinline__ bool sees(uint32_t key) const {
        return key < length ? key >= lo : key - length < 64 && ((mask >> (key - length)) & 1);
    }
};

// The view of (drafted row, head) pair `pair` of the request; none past the
// last. Every lane of the wave takes part.
__device__ __forceinline__ RowView row_view(const IrisTreeAttention& a, const Request& r, uint32_t pair, uint32_t group) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t mask = tree_ancestors(a.parents ? a.parents + r.row0 : nullptr, r.rows, lane);
    const uint32_t depth = __popcll(mask) - 1;
    if (a.window && a.window < TREE_MAX_NODES) {  // ancestors out of the window
        uint64_t near = 0;
        for (uint32_t j = 0; j < r.rows; j++) {
            const uint32_t d = (uint32_t)__shfl((int)depth, (int)j);
            if (((mask >> j) & 1) && depth - d < a.window) near |= 1ull << j;
        }
        mask = near;
    }
    const uint32_t node = pair / group;
    RowView v;
    v.length = r.length;
    const bool valid = node < r.rows;
    v.mask = __shfl((unsigned long long)mask, (int)min(node, 63u));
    const uint32_t pos = r.length + (uint32_t)__shfl((int)depth, (int)min(node, 63u));
    v.lo = a.window && pos >= a.window ? pos + 1 - a.window : 0;
    if (!valid) v.mask = 0, v.lo = 0xffffffffu;
    return v;
}

// The cache of one key head: where a position's values lie.
struct Places {
    const int32_t *k, *v, *table;
    uint32_t pages, page_log, place_mask, last;
    size_t page_stride;
    uint32_t hd;
    int32_t* status;
    // Positions past the last one read the last one (no row sees them).
    __device__ __forceinline__ const int32_t* at(const int32_t* base, uint32_t page, uint32_t key) const {
        return page < pages ? base + page * page_stride + (size_t)(key & place_mask) * hd : g_zeros;
    }
    __device__ __forceinline__ uint32_t page_of(uint32_t key) const { return (uint32_t)table[key >> page_log]; }
    __device__ __forceinline__ uint32_t clamped(uint32_t key) const { return min(key, last); }
};

__device__ __forceinline__ Places places(const IrisPagedKv& c, const IrisTreeAttention& a, const Request& r, uint32_t g) {
    const size_t head = (size_t)c.page_size * c.head_dim;
    return Places{c.k + g * head, c.v + g * head, r.table, c.pages, 31u - __clz((int)c.page_size), c.page_size - 1,
                  r.total - 1, c.kv_heads * head, c.head_dim, a.status};
}

__device__ __forceinline__ uint64_t pack_best(int32_t score, uint32_t key) {
    return (uint64_t)((uint32_t)score ^ 0x80000000u) << 32 | (0xffffffffu - key);
}
__device__ __forceinline__ int32_t packed_score(uint64_t p) { return (int32_t)((uint32_t)(p >> 32) ^ 0x80000000u); }
__device__ __forceinline__ uint32_t packed_key(uint64_t p) { return 0xffffffffu - (uint32_t)p; }

// A lane's four values of each 16-dimension piece of a 64-dimension step.
__device__ __forceinline__ void load_step(const int32_t* row, uint32_t ds, uint32_t hd, int4 (&v)[4]) {
    const uint32_t d0 = ds * 64 + (threadIdx.x >> 4 & 3) * 4;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t d = d0 + j * 16;
        v[j] = *(const int4*)(row + (d < hd ? d : 0));
        if (d >= hd) v[j] = make_int4(0, 0, 0, 0);
    }
}

template <int LD>
__device__ __forceinline__ void step_digits(const int4 (&v)[4], v4i (&f)[LD], uint32_t& seen) {
    uint32_t p[4][4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) split4(v[j], p[j], seen);
#pragma unroll
    for (int l = 0; l < (LD < 4 ? LD : 4); l++) f[l] = v4i{(int)p[0][l], (int)p[1][l], (int)p[2][l], (int)p[3][l]};
    if constexpr (LD == DIGITS) f[4] = v4i{(int)fifth4(v[0]), (int)fifth4(v[1]), (int)fifth4(v[2]), (int)fifth4(v[3])};
}

// The row tiles a workgroup of the scores and values launches takes: LDS and
// registers hold that many of a head size.
constexpr uint32_t row_block(uint32_t hd) { return hd <= 128 ? 4 : hd <= 256 ? 2 : 1; }

// ---- (1) scores

template <uint32_t HD, uint32_t RB>
__global__ __launch_bounds__(256, HD >= 512 ? 1 : HD >= 256 ? 2 : 3) void tree_scores_kernel(const IrisPagedKv c, const IrisTreeAttention a,
                                                                             const TreeSpace s) {
    constexpr uint32_t DS = HD / 64;
    extern __shared__ v4i s_q[];  // [RB][DS][DIGITS][64]: the rows' operand tiles
    __shared__ uint64_t s_best[4][RB][16];
    __shared__ int32_t s_wide;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, rt0 = blockIdx.y * RB, bg = blockIdx.z, b = bg / c.kv_heads, g = bg % c.kv_heads;
    const uint32_t group = a.heads / c.kv_heads;
    Request r;
    if (!read_request(c, a, b, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk, pairs = r.rows * group;
    if (key0 >= r.total || rt0 * 16 >= pairs) return;
    const uint32_t key1 = min(key0 + s.chunk, r.total), tiles = (pairs - rt0 * 16 + 15) / 16;
    const Places at = places(c, a, r, g);
    if (tid == 0) s_wide = 0;
    __syncthreads();
    uint32_t seen = 0;
    for (uint32_t i = wave; i < RB * DS; i += 4) {
        const uint32_t rt = i / DS, ds = i % DS, pair = (rt0 + rt) * 16 + (lane & 15), node = pair / group;
        if (rt >= tiles) continue;
        int4 v[4];
        v4i f[DIGITS];
        load_step(a.q + (size_t)(r.row0 + min(node, r.rows - 1)) * a.q_stride + (size_t)(g * group + pair % group) * c.head_dim, ds,
                  c.head_dim, v);
        step_digits<DIGITS>(v, f, seen);
#pragma unroll
        for (int l = 0; l < DIGITS; l++) s_q[(i * DIGITS + l) * 64 + lane] = f[l];
    }
    if (is_wide(seen) && lane == 0) s_wide = 1;
    RowView view[RB];
#pragma unroll
    for (uint32_t rt = 0; rt < RB; rt++) view[rt] = row_view(a, r, (rt0 + rt) * 16 + (lane & 15), group);
    __syncthreads();
    const bool q_wide = s_wide;

    int32_t best[RB];
    uint32_t best_key[RB];
#pragma unroll
    for (uint32_t rt = 0; rt < RB; rt++) best[rt] = INT32_MIN, best_key[rt] = 0xffffffffu;
    const uint32_t kt1 = (key1 - key0 + 15) / 16;
    uint4* out = s.scores + (((size_t)bg * s.row_tiles + rt0) * s.chunks + chunk) * (s.chunk / 16) * 64;
    const size_t rt_stride = (size_t)s.chunks * (s.chunk / 16) * 64;
    auto keep = [&](uint32_t kt, uint32_t rt, const int32_t (&sc)[4]) __attribute__((always_inline)) {
        out[rt * rt_stride + kt * 64 + lane] = make_uint4((uint32_t)sc[0], (uint32_t)sc[1], (uint32_t)sc[2], (uint32_t)sc[3]);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t key = key0 + kt * 16 + 4 * grp + i;
            const bool take = view[rt].sees(key) & ((sc[i] > best[rt]) | (best_key[rt] == 0xffffffffu));
            best[rt] = take ? sc[i] : best[rt];
            best_key[rt] = take ? key : best_key[rt];
        }
    };
    // The next tile's keys are loaded during this one's products.
    auto key_row = [&](uint32_t kt) {
        const uint32_t key = at.clamped(key0 + kt * 16 + (lane & 15)), page = at.page_of(key);
        if (page >= at.pages && at.status) *at.status = IRIS_E_INVALID;
        return at.at(at.k, page, key);
    };
    constexpr bool AHEAD = HD <= 256;
    int4 raw[AHEAD ? DS : 1][4];
    const int32_t* row = wave < kt1 ? key_row(wave) : nullptr;
    if constexpr (AHEAD)
        if (row)
#pragma unroll
            for (uint32_t ds = 0; ds < DS; ds++) load_step(row, ds, c.head_dim, raw[ds]);
#pragma unroll 1
    for (uint32_t kt = wave; kt < kt1; kt += 4) {
        v4i kf[DS][NARROW];
        uint32_t wide = 0;
        const int32_t* here = row;
#pragma unroll
        for (uint32_t ds = 0; ds < DS; ds++) {
            if constexpr (!AHEAD) load_step(here, ds, c.head_dim, raw[0]);
            step_digits<NARROW>(raw[AHEAD ? ds : 0], kf[ds], wide);
        }
        if (kt + 4 < kt1) {
            row = key_row(kt + 4);
            if constexpr (AHEAD)
#pragma unroll
                for (uint32_t ds = 0; ds < DS; ds++) load_step(row, ds, c.head_dim, raw[ds]);
        }
        if (!q_wide && !is_wide(wide)) {
#pragma unroll
            for (uint32_t rt = 0; rt < RB; rt++) {
                if (rt >= tiles) break;
                v4i acc[2 * NARROW - 1];
#pragma unroll
                for (int j = 0; j < 2 * NARROW - 1; j++) acc[j] = v4i{0, 0, 0, 0};
#pragma unroll
                for (uint32_t ds = 0; ds < DS; ds++) {
                    v4i qf[NARROW];
#pragma unroll
                    for (int l = 0; l < NARROW; l++) qf[l] = s_q[((rt * DS + ds) * DIGITS + l) * 64 + lane];
                    dot_step<NARROW>(kf[ds], qf, acc);
                }
                int32_t sc[4];
                scores_of<HD, NARROW>(acc, a.scaled, a.scale_q32, sc);
                keep(kt, rt, sc);
            }
        } else {
#pragma unroll
            for (uint32_t rt = 0; rt < RB; rt++) {
                if (rt >= tiles) break;
                v4i acc[2 * DIGITS - 1];
#pragma unroll
                for (int j = 0; j < 2 * DIGITS - 1; j++) acc[j] = v4i{0, 0, 0, 0};
#pragma unroll 1
                for (uint32_t ds = 0; ds < DS; ds++) {
                    int4 v[4];
                    v4i f[DIGITS], qf[DIGITS];
                    load_step(here, ds, c.head_dim, v);
                    step_digits<DIGITS>(v, f, wide);
#pragma unroll
                    for (int l = 0; l < DIGITS; l++) qf[l] = s_q[((rt * DS + ds) * DIGITS + l) * 64 + lane];
                    dot_step<DIGITS>(f, qf, acc);
                }
                int32_t sc[4];
                scores_of<HD, DIGITS>(acc, a.scaled, a.scale_q32, sc);
                keep(kt, rt, sc);
            }
        }
    }
#pragma unroll
    for (uint32_t rt = 0; rt < RB; rt++) {
        take_best(best[rt], best_key[rt], __shfl_xor(best[rt], 16), (uint32_t)__shfl_xor((int)best_key[rt], 16));
        take_best(best[rt], best_key[rt], __shfl_xor(best[rt], 32), (uint32_t)__shfl_xor((int)best_key[rt], 32));
        if (lane < 16) s_best[wave][rt][lane] = best_key[rt] == 0xffffffffu ? 0 : pack_best(best[rt], best_key[rt]);
    }
    __syncthreads();
    if (tid < RB * 16 && tid / 16 < tiles) {
        const uint32_t rt = tid / 16, i = tid % 16;
        const uint64_t m = max(max(s_best[0][rt][i], s_best[1][rt][i]), max(s_best[2][rt][i], s_best[3][rt][i]));
        s.maxima[(((size_t)bg * s.row_tiles + rt0 + rt) * s.chunks + chunk) * 16 + i] = m;
    }
}

// The chunks that hold positions of a request.
__device__ __forceinline__ uint32_t chunks_of(const TreeSpace& s, const Request& r) {
    return (r.total - r.base + s.chunk - 1) / s.chunk;
}

// A row's maximum over its chunks, for row lane % 16.
__device__ __forceinline__ uint64_t row_maximum(const TreeSpace& s, size_t tile, uint32_t chunks) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t m = 0;
    for (uint32_t i = lane >> 4; i < chunks; i += 4) m = max(m, s.maxima[(tile * s.chunks + i) * 16 + (lane & 15)]);
    m = max(m, (uint64_t)__shfl_xor((unsigned long long)m, 16));
    return max(m, (uint64_t)__shfl_xor((unsigned long long)m, 32));
}

// ---- (2) exp terms

__global__ __launch_bounds__(256) void tree_terms_kernel(const IrisPagedKv c, const IrisTreeAttention a, const TreeSpace s) {
    __shared__ double s_sum[4][16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, rt = blockIdx.y, bg = blockIdx.z, group = a.heads / c.kv_heads;
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk;
    if (key0 >= r.total || rt * 16 >= r.rows * group) return;
    const uint32_t kt1 = (min(s.chunk, r.total - key0) + 15) / 16;
    const size_t tile = (size_t)bg * s.row_tiles + rt;
    const uint32_t top = (uint32_t)packed_score(row_maximum(s, tile, chunks_of(s, r)));
    const RowView view = row_view(a, r, rt * 16 + (lane & 15), group);
    uint4* t = s.scores + (tile * s.chunks + chunk) * (s.chunk / 16) * 64 + lane;
    double sum = 0;  // at most 2^20 terms of 2^32: exact
#pragma unroll 2
    for (uint32_t kt = wave; kt < kt1; kt += 4) {
        const uint4 sc = t[kt * 64];
        const uint32_t v[4] = {sc.x, sc.y, sc.z, sc.w};
        uint32_t e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double x = view.sees(key0 + kt * 16 + 4 * grp + i) ? dn::softmax_exp_f64(top - v[i]) : 0.0;
            sum += x;
            e[i] = kept_term(x);
        }
        t[kt * 64] = make_uint4(e[0], e[1], e[2], e[3]);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < 16) s_sum[wave][lane] = sum;
    __syncthreads();
    if (tid < 16) s.sums[(tile * s.chunks + chunk) * 16 + tid] = s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
}

// ---- (3) weighted values

// Waves: a 64-dimension block each, `RS` halves of the row tiles, and PARTS
// of the steps.
template <uint32_t HD, uint32_t RB>
struct ValueShape {
    static constexpr uint32_t DS = HD / 64, RS = RB == 4 ? 2 : 1, WAVES = std::max(4u, DS) * RS, PARTS = WAVES / RS / DS, RW = RB / RS;
};

constexpr uint32_t BATCH = 4;  // steps whose weights are in LDS at a time

template <uint32_t HD, uint32_t RB>
__global__ __launch_bounds__((ValueShape<HD, RB>::WAVES * 64), 2) void tree_values_kernel(const IrisPagedKv c,
                                                                                       const IrisTreeAttention a,
                                                                                       const TreeSpace s) {
    using S = ValueShape<HD, RB>;
    constexpr uint32_t WAVES = S::WAVES, RW = S::RW;
    extern __shared__ uint64_t s_sums[];  // [RB][16][HD], then the weights' digits [RB][BATCH][2][64] uint4
    __shared__ int32_t s_wsum[RB][16], s_nbig[RB][16], s_big[RB][16][2];
    uint4* s_w = (uint4*)(s_sums + RB * 16 * HD);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, rt0 = blockIdx.y * RB, bg = blockIdx.z, g = bg % c.kv_heads, group = a.heads / c.kv_heads;
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk, pairs = r.rows * group;
    if (key0 >= r.total || rt0 * 16 >= pairs) return;
    const uint32_t steps = (min(s.chunk, r.total - key0) + STEP - 1) / STEP, tiles = (pairs - rt0 * 16 + 15) / 16;
    const uint32_t kt1 = (min(s.chunk, r.total - key0) + 15) / 16;
    const Places at = places(c, a, r, g);
    for (uint32_t i = tid; i < RB * 16 * HD; i += WAVES * 64) s_sums[i] = 0;
    if (tid < RB * 16) s_wsum[tid / 16][tid % 16] = 0, s_nbig[tid / 16][tid % 16] = 0;

    // The weights of (row tile, step of the batch) items, dealt to the waves.
    const size_t tile0 = (size_t)bg * s.row_tiles + rt0;
    const uint32_t chunks = chunks_of(s, r);
    auto row_sum = [&](uint32_t rt) {
        double sum = 0;
        for (uint32_t i = grp; i < chunks; i += 4) sum += s.sums[((tile0 + rt) * s.chunks + i) * 16 + (lane & 15)];
        sum += __shfl_xor(sum, 16);
        return sum + __shfl_xor(sum, 32);
    };
    // An item is always taken by a wave with the same row tile.
    const uint32_t my_rt = wave % RB;
    const bool has_rt = my_rt < tiles;
    const double sum = has_rt ? row_sum(my_rt) : 1.0;
    const bool valid = has_rt && (rt0 + my_rt) * 16 + (lane & 15) < pairs;
    const double w_scale = valid ? 65536.0 / sum : 0.0, q_scale = valid ? 4294967296.0 / sum : 0.0;
    const uint64_t total = valid ? (uint64_t)sum : 1;
    int32_t wsum = 0;

    const uint32_t block = wave % S::DS, part = wave / S::DS % S::PARTS, half = wave / S::DS / S::PARTS;
    const uint32_t d = block * 64 + 4 * (lane & 15);
    v4i acc[RW][4][NARROW + 1];
#pragma unroll
    for (uint32_t rt = 0; rt < RW; rt++)
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int j = 0; j < NARROW + 1; j++) acc[rt][t][j] = v4i{0, 0, 0, 0};
    // Four positions in a row lie in one page.
    auto load_values = [&](uint32_t step, int4 (&v)[4][4]) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) {
            const uint32_t key = key0 + step * STEP + 16 * t + 4 * grp;
            const uint32_t page = at.page_of(at.clamped(key));
#pragma unroll
            for (uint32_t i = 0; i < 4; i++)
                v[t][i] = *(const int4*)(at.at(at.v, page, at.clamped(key + i)) + (d < c.head_dim ? d : 0));
        }
    };
    __syncthreads();
#pragma unroll 1
    for (uint32_t batch = 0; batch < steps; batch += BATCH) {
        if (has_rt)
#pragma unroll 1
            for (uint32_t i = wave / RB; i < BATCH; i += WAVES / RB) {
                v4i w0 = v4i{0, 0, 0, 0}, w1 = v4i{0, 0, 0, 0};
                const uint4* t = s.scores + (((tile0 + my_rt) * s.chunks + chunk) * (s.chunk / 16) + (batch + i) * 4) * 64 + lane;
#pragma unroll
                for (uint32_t k = 0; k < 4; k++) {
                    const uint32_t kt = (batch + i) * 4 + k;
                    uint32_t low = 0, high = 0;
                    if (kt < kt1) {
                        const uint4 x = t[k * 64];
                        const uint32_t e[4] = {x.x, x.y, x.z, x.w};
                        int32_t w[4];
                        weights_of(e, total, w_scale, q_scale, w, wsum, [&](int j) {
                            const int n = atomicAdd(&s_nbig[my_rt][lane & 15], 1);
                            if (n < 2) s_big[my_rt][lane & 15][n] = (int32_t)(key0 + kt * 16 + 4 * grp + j);
                        });
                        weight_digits(w, low, high);
                    }
                    w0[k] = (int)low, w1[k] = (int)high;
                }
                s_w[((my_rt * BATCH + i) * 2) * 64 + lane] = make_uint4(w0[0], w0[1], w0[2], w0[3]);
                s_w[((my_rt * BATCH + i) * 2 + 1) * 64 + lane] = make_uint4(w1[0], w1[1], w1[2], w1[3]);
            }
        __syncthreads();
#pragma unroll 1
        for (uint32_t i = part; i < BATCH && batch + i < steps; i += S::PARTS) {
            int4 v[4][4];
            load_values(batch + i, v);
            v4i w0[RW], w1[RW];
#pragma unroll
            for (uint32_t rt = 0; rt < RW; rt++) {
                const uint4* p = s_w + (((half * RW + rt) * BATCH + i) * 2) * 64 + lane;
                const uint4 x = p[0], y = p[64];
                w0[rt] = v4i{(int)x.x, (int)x.y, (int)x.z, (int)x.w};
                w1[rt] = v4i{(int)y.x, (int)y.y, (int)y.z, (int)y.w};
            }
            auto column = [&](int k, uint32_t t) {
                auto of = [&](int4 x) { return k == 0 ? x.x : k == 1 ? x.y : k == 2 ? x.z : x.w; };
                return make_int4(of(v[t][0]), of(v[t][1]), of(v[t][2]), of(v[t][3]));
            };
            uint32_t seen = 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int4 x[4] = {column(k, 0), column(k, 1), column(k, 2), column(k, 3)};
                v4i f[NARROW];
                step_digits<NARROW>(x, f, seen);
#pragma unroll
                for (uint32_t rt = 0; rt < RW; rt++) value_step<NARROW>(w0[rt], w1[rt], f, acc[rt][k]);
            }
            // Values of more digits: the two upper planes' products, straight
            // to the sums.
            if (is_wide(seen)) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const int4 x[4] = {column(k, 0), column(k, 1), column(k, 2), column(k, 3)};
                    v4i f[DIGITS];
                    step_digits<DIGITS>(x, f, seen);
#pragma unroll 1
                    for (uint32_t rt = 0; rt < RW; rt++) {
                        if (half * RW + rt >= tiles) break;
                        const uint4* p = s_w + (((half * RW + rt) * BATCH + i) * 2) * 64 + lane;
                        const uint4 y0 = p[0], y1 = p[64];
                        const v4i a0 = v4i{(int)y0.x, (int)y0.y, (int)y0.z, (int)y0.w}, a1 = v4i{(int)y1.x, (int)y1.y, (int)y1.z, (int)y1.w};
                        const v4i upper[2] = {f[3], f[4]};
                        v4i up[3] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
                        value_step<2>(a0, a1, upper, up);
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const uint64_t t = (uint64_t)(int64_t)up[0][q] << 24;
                            const uint64_t sum3 = t + ((uint64_t)(int64_t)up[1][q] << 32) + ((uint64_t)(int64_t)up[2][q] << 40);
                            atomicAdd((unsigned long long*)&s_sums[((half * RW + rt) * 16 + 4 * grp + q) * HD + d + k], sum3);
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    wsum += __shfl_xor(wsum, 16);
    wsum += __shfl_xor(wsum, 32);
    if (has_rt && lane < 16) atomicAdd(&s_wsum[my_rt][lane], wsum);
#pragma unroll
    for (uint32_t rt = 0; rt < RW; rt++) {
        if (half * RW + rt >= tiles) break;
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int q = 0; q < 4; q++) {
                uint64_t t = 0;
#pragma unroll
                for (int j = 0; j < NARROW + 1; j++) t += (uint64_t)(int64_t)acc[rt][k][j][q] << (8 * j);
                uint64_t* to = &s_sums[((half * RW + rt) * 16 + 4 * grp + q) * HD + d + k];
                atomicAdd((unsigned long long*)to, t);
            }
    }
    __syncthreads();
    const uint32_t rows = min(RB, tiles) * 16;
    for (uint32_t i = tid; i < rows * HD; i += WAVES * 64) {
        const uint32_t row = i / HD, dim = i % HD, rt = row / 16;
        uint64_t t = s_sums[i];
        for (int j = 0; j < s_nbig[rt][row % 16]; j++) {  // at most two
            const uint32_t key = (uint32_t)s_big[rt][row % 16][j];
            if (dim < c.head_dim) t += (uint64_t)((int64_t)65536 * at.at(at.v, at.page_of(key), key)[dim]);
        }
        s.partial[(((tile0 + rt) * s.chunks + chunk) * 16 + row % 16) * HD + dim] = t;
    }
    if (tid < rows) s.weights[((tile0 + tid / 16) * s.chunks + chunk) * 16 + tid % 16] = s_wsum[tid / 16][tid % 16];
}

// ---- (4) the chunks joined: a workgroup per (drafted row, head)

__global__ __launch_bounds__(256) void tree_join_kernel(const IrisPagedKv c, const IrisTreeAttention a, const TreeSpace s,
                                                        uint32_t hd_padded) {
    __shared__ uint64_t s_part[256];
    const uint32_t tid = threadIdx.x, bg = blockIdx.y, g = bg % c.kv_heads, group = a.heads / c.kv_heads, pair = blockIdx.x;
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    if (pair >= r.rows * group) return;
    const size_t tile = (size_t)bg * s.row_tiles + pair / 16;
    const uint32_t i = pair % 16, chunks = chunks_of(s, r);
    uint64_t best = 0;
    int32_t wsum = 0;
    for (uint32_t k = 0; k < chunks; k++) {
        best = max(best, s.maxima[(tile * s.chunks + k) * 16 + i]);
        wsum += s.weights[(tile * s.chunks + k) * 16 + i];
    }
    const int64_t resid = dn::sub_sat(dn::ONE_ACT, wsum);
    const uint32_t key = packed_key(best);
    const Places at = places(c, a, r, g);
    const int32_t* v = at.at(at.v, at.page_of(key), key);
    int32_t* out = a.out + (size_t)(r.row0 + pair / group) * a.out_stride + (size_t)(g * group + pair % group) * c.head_dim;
    // Up to 256 dimensions at a time, the chunks dealt to what threads are left.
    const uint32_t width = min(hd_padded, 256u), parts = 256 / width, part = tid / width;
    for (uint32_t d0 = 0; d0 < c.head_dim; d0 += width) {
        const uint32_t d = d0 + tid % width;
        uint64_t t = 0;
        for (uint32_t k = part; k < chunks; k += parts) t += s.partial[((tile * s.chunks + k) * 16 + i) * hd_padded + d];
        s_part[tid] = t;
        __syncthreads();
        if (tid < width && d < c.head_dim) {
            for (uint32_t p = 1; p < parts; p++) t += s_part[p * width + tid];
            out[d] = dn::requantize((int64_t)(t + (uint64_t)(resid * v[d])));
        }
        __syncthreads();
    }
}

bool misaligned(const void* p) { return ((uintptr_t)p & 15) != 0; }

int tree_check(const IrisPagedKv* c, const IrisTreeAttention* a) {
    const int rc = iris_paged_check(c);
    if (rc) return rc;
    if (!a || !a->q || !a->out || !a->row_start || !a->lengths || !a->table) return IRIS_E_INVALID;
    if (misaligned(a->q) || misaligned(a->out) || (a->q_stride | a->out_stride) % 4) return IRIS_E_INVALID;
    if (!a->heads || a->heads % c->kv_heads || a->heads > 65535) return IRIS_E_INVALID;
    const uint64_t q = (uint64_t)a->heads * c->head_dim;
    if (a->q_stride < q || a->out_stride < q || !a->table_stride || !a->max_nodes || !a->max_positions)
        return IRIS_E_INVALID;
    if (a->max_nodes > TREE_MAX_NODES || a->max_positions > TREE_MAX_POSITIONS || a->rows > INT32_MAX)
        return IRIS_E_RANGE;
    if ((uint64_t)a->requests * c->kv_heads > 65535) return IRIS_E_RANGE;  // a launch's third dimension
    return 0;
}

uint32_t padded_head(uint32_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512; }

// Carves the work space (base may be null) and returns its bytes.
uint64_t tree_space(const IrisPagedKv& c, const IrisTreeAttention& a, uint8_t* base, TreeSpace* s) {
    const uint64_t hd = padded_head(c.head_dim), bg = (uint64_t)a.requests * c.kv_heads;
    const uint32_t group = a.heads / c.kv_heads;
    s->row_tiles = (a.max_nodes * group + 15) / 16;
    // Positions that a request's rows look at, from a multiple of STEP on.
    const uint64_t span = std::min<uint64_t>(a.max_positions, a.window ? (uint64_t)a.window + a.max_nodes + STEP : a.max_positions);
    const uint64_t blocks = bg * ((s->row_tiles + row_block(hd) - 1) / row_block(hd));
    const uint64_t want = std::max<uint64_t>(1, 1024 / blocks);
    s->chunk = (uint32_t)std::max<uint64_t>(128, ((span + want - 1) / want + 127) & ~127ull);
    s->chunks = (uint32_t)((span + s->chunk - 1) / s->chunk);
    uint64_t at = 0;
    auto take = [&](auto*& p, uint64_t bytes) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
        at += (bytes + 255) & ~255ull;
    };
    const uint64_t parts = bg * s->row_tiles * s->chunks;
    take(s->scores, parts * (s->chunk / 16) * TILE_BYTES);
    take(s->maxima, parts * 16 * 8);
    take(s->sums, parts * 16 * 8);
    take(s->weights, parts * 16 * 4);
    take(s->partial, parts * 16 * hd * 8);
    return at;
}

template <uint32_t HD, uint32_t RB>
int tree_launch_block(const IrisPagedKv& c, const IrisTreeAttention& a, const TreeSpace& s, hipStream_t stream) {
    const uint32_t bg = a.requests * c.kv_heads, blocks = (s.row_tiles + RB - 1) / RB;
    const size_t q_lds = RB * (HD / 64) * DIGITS * TILE_BYTES, v_lds = RB * 16 * HD * 8 + RB * BATCH * 2 * TILE_BYTES;
    hipError_t st = paged_lds_limit((const void*)tree_scores_kernel<HD, RB>, q_lds);
    if (st == hipSuccess) st = paged_lds_limit((const void*)tree_values_kernel<HD, RB>, v_lds);
    if (st != hipSuccess) return (int)st;
    hipLaunchKernelGGL((tree_scores_kernel<HD, RB>), dim3(s.chunks, blocks, bg), dim3(256), q_lds, stream, c, a, s);
    hipLaunchKernelGGL(tree_terms_kernel, dim3(s.chunks, s.row_tiles, bg), dim3(256), 0, stream, c, a, s);
    hipLaunchKernelGGL((tree_values_kernel<HD, RB>), dim3(s.chunks, blocks, bg), dim3(ValueShape<HD, RB>::WAVES * 64), v_lds,
                       stream, c, a, s);
    hipLaunchKernelGGL(tree_join_kernel, dim3(a.max_nodes * (a.heads / c.kv_heads), bg), dim3(256), 0, stream, c, a, s, HD);
    return (int)hipGetLastError();
}

template <uint32_t HD>
int tree_launch(const IrisPagedKv& c, const IrisTreeAttention& a, const TreeSpace& s, hipStream_t stream) {
    if (s.row_tiles == 1) return tree_launch_block<HD, 1>(c, a, s, stream);
    if constexpr (row_block(HD) >= 2)
        if (s.row_tiles == 2 || row_block(HD) == 2) return tree_launch_block<HD, 2>(c, a, s, stream);
    return tree_launch_block<HD, row_block(HD)>(c, a, s, stream);
}

}  // namespace

extern "C" {

uint64_t iris_attention_tree_workspace_bytes(const IrisPagedKv* c, const IrisTreeAttention* a) {
    if (tree_check(c, a) || !a->rows || !a->requests) return 0;
    TreeSpace s;
    return tree_space(*c, *a, nullptr, &s);
}

int iris_attention_tree(const IrisPagedKv* c, const IrisTreeAttention* a, void* space, uint64_t bytes, void* stream) {
    const int rc = tree_check(c, a);
    if (rc) return rc;
    if (!a->rows || !a->requests) return 0;
    if (!space || misaligned(space)) return IRIS_E_INVALID;
    TreeSpace s;
    if (bytes < tree_space(*c, *a, (uint8_t*)space, &s)) return IRIS_E_RANGE;
    switch (padded_head(c->head_dim)) {
        case 64: return tree_launch<64>(*c, *a, s, (hipStream_t)stream);
        case 128: return tree_launch<128>(*c, *a, s, (hipStream_t)stream);
        case 256: return tree_launch<256>(*c, *a, s, (hipStream_t)stream);
        default: return tree_launch<512>(*c, *a, s, (hipStream_t)stream);
    }
}

}  // extern "C"
