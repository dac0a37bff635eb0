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
// bits however the positions are dealt. Where a request's scores fit one
// workgroup's LDS and few workgroups are wanted, the last three are one launch.
//
// Few rows are bound by memory, as each key and value is read once: 4 tokens at
// up to 32700 positions (32 heads of 128, 8 key heads; 412 MB) 128 us, 3.2 TB/s.
// Trees of many rows are bound by the exact softmax and by what goes through the
// work space (four bytes per score and head, written twice and read twice): 32
// trees of 25 at up to 8000, 502 us. Short spans are bound by latency: 1 token
// at 700 positions 16.2 us.
#include <algorithm>
#include <type_traits>

#include "attn_tiles.h"
#include "tree_chunks.h"

namespace {

// Four rows of zeros for positions whose page is outside the cache.
__device__ const int32_t g_zeros[4 * ATTN_MAX_HEAD_DIM] = {};

// The work space of a launch. Row tiles count a request's (drafted row, head)
// pairs by sixteens, `row_tiles` per (request, key head).
struct TreeSpace {
    uint4* scores;      // [request, key head][row tile][chunk][key tile][64] scores, then exp terms
    int32_t* maxima;    // [..][row tile][chunk][16]
    uint32_t* firsts;   // [..][row tile][chunk][16] the first position of the row's maximum, ~0: not here
    double* sums;       // [..][row tile][chunk][16] of the exp terms
    int32_t* weights;   // [..][row tile][chunk][16] the weights' sum
    uint64_t* partial;  // [..][row tile][chunk][16][HD] weighted values
    uint32_t row_tiles, chunks, chunk;  // positions per chunk, whole steps
    uint32_t short_tiles;  // key tiles of a request where the short form is taken, else 0
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

// The cache of one key head, for positions [key0, key1) whose pages' offsets
// are in LDS. Positions past the last one read the last one (no row sees them).
struct Places {
    const int32_t *k, *v;
    const uint64_t* page;  // offsets in values, of key0's page on; ~0: outside the cache
    uint32_t page_log, place_mask, first, last, hd;
    __device__ __forceinline__ const int32_t* at(const int32_t* base, uint32_t key) const {
        key = min(key, last);
        const uint64_t p = page[(key >> page_log) - first];
        return p != ~0ull ? base + (p + (key & place_mask) * hd) : g_zeros;
    }
    // The first of four positions in a row (key a multiple of four), which
    // lie in one page; those past the last one are there, but not written.
    __device__ __forceinline__ const int32_t* four(const int32_t* base, uint32_t key) const { return at(base, min(key, last & ~3u)); }
};

// This thread's table entry of the `count` positions from key0 on, where no
// window moves them: on its way while the request is read. (0 where places()
// asks for none: from most_pages on.)
__device__ __forceinline__ uint32_t early_page(const IrisPagedKv& c, const IrisTreeAttention& a, uint32_t request, uint32_t key0,
                                               uint32_t count) {
    const uint32_t log = 31u - __clz((int)c.page_size);
    if (a.window || threadIdx.x >= most_pages(count, log)) return 0;
    const int32_t* table = a.table + (size_t)request * a.table_stride;
    return (uint32_t)load1(table + min((key0 >> log) + threadIdx.x, a.table_stride - 1));
}

// The workgroup's places; s_page has CHUNK_PAGES entries. A barrier follows.
__device__ __forceinline__ Places places(const IrisPagedKv& c, const IrisTreeAttention& a, const Request& r, uint32_t g,
                                         uint32_t key0, uint32_t key1, uint64_t* s_page, uint32_t early) {
    const size_t head = (size_t)c.page_size * c.head_dim;
    const uint32_t log = 31u - __clz((int)c.page_size), first = key0 >> log, n = ((key1 - 1) >> log) - first + 1;
    for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
        const uint32_t p = i == threadIdx.x && !a.window ? early : (uint32_t)r.table[first + i];
        s_page[i] = p < c.pages ? p * (c.kv_heads * head) : ~0ull;
        if (p >= c.pages && a.status) *a.status = IRIS_E_INVALID;
    }
    return Places{c.k + g * head, c.v + g * head, s_page, log, c.page_size - 1, first, key1 - 1, c.head_dim};
}

// A lane's four values of each 16-dimension piece of a 64-dimension step.
// FULL: the head fills its operand tiles (no dimension past it).
template <bool FULL>
__device__ __forceinline__ void load_step(const int32_t* row, uint32_t ds, uint32_t hd, int4 (&v)[4]) {
    const uint32_t d0 = (threadIdx.x >> 4 & 3) * 4;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t at = ds * 64 + j * 16;
        if constexpr (FULL) {
            v[j] = load4(row + d0 + at);
        } else {
            v[j] = load4(row + (d0 + at < hd ? d0 + at : 0));
            if (d0 + at >= hd) v[j] = make_int4(0, 0, 0, 0);
        }
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

// The row tiles of a scores workgroup: LDS holds their operands (48 KB).
constexpr uint32_t row_block(uint32_t hd) { return hd <= 128 ? 8 : 1024 / hd; }

// The chunks that hold positions of a request.
__device__ __forceinline__ uint32_t chunks_of(const TreeSpace& s, const Request& r) {
    return (r.total - r.base + s.chunk - 1) / s.chunk;
}

// ---- (1) scores and each chunk's maxima

// A wave takes 16 positions at a time, splits their keys once and meets every
// row tile's queries (digit planes in LDS) with them. 4 tokens at up to 32700:
// 65 us, 206 MB of keys at 3.2 TB/s; a workgroup's first loads depend on each
// other (request, pages, keys), and twelve waves a CU hide only a part of it
// (sixteen spill registers: 85 us). 32 trees of 25 at up to 8000: 160 us, the
// vector units issue in 42% of the cycles, the matrix cores are busy in 18%.
template <uint32_t HD, bool FULL>
__global__ __launch_bounds__(256, HD >= 512 ? 1 : HD >= 256 ? 2 : 3) void tree_scores_kernel(const IrisPagedKv c, const IrisTreeAttention a,
                                                                             const TreeSpace s) {
    constexpr uint32_t DS = HD / 64, RB = row_block(HD);
    extern __shared__ v4i s_q[];  // [tiles][DS][NARROW][64]
    __shared__ int32_t s_max[RB][64];
    __shared__ uint64_t s_mask[RB * 16];
    __shared__ uint32_t s_lo[RB * 16];
    __shared__ uint64_t s_page[CHUNK_PAGES];
    __shared__ int32_t s_wide;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index(), grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, rt0 = blockIdx.z * RB, bg = blockIdx.y, g = bg % c.kv_heads;
    const uint32_t group = a.heads / c.kv_heads;
    const uint32_t early = early_page(c, a, bg / c.kv_heads, chunk * s.chunk, s.chunk);
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk, pairs = r.rows * group;
    if (key0 >= r.total || rt0 * 16 >= pairs) return;
    const uint32_t key1 = min(key0 + s.chunk, r.total), tiles = min(RB, (pairs - rt0 * 16 + 15) / 16);
    const Places at = places(c, a, r, g, key0, key1, s_page, early);
    auto query = [&](uint32_t rt) {
        const uint32_t pair = min((rt0 + rt) * 16 + (lane & 15), pairs - 1);
        return a.q + (size_t)(r.row0 + pair / group) * a.q_stride + (size_t)(g * group + pair % group) * c.head_dim;
    };
    if (tid == 0) s_wide = 0;
    for (uint32_t i = tid; i < tiles * 64; i += 256) s_max[i / 64][i % 64] = INT32_MIN;
    __syncthreads();
    const uint32_t kt1 = (key1 - key0 + 15) / 16;
    // The next tile's keys are loaded during this one's products, the first
    // while the queries are prepared.
    constexpr bool AHEAD = HD <= 256;
    int4 raw[AHEAD ? DS : 1][4];
    // (Past the last: it again, so that no load is behind a branch, where it
    // would be waited for.)
    auto load_ahead = [&](uint32_t kt) __attribute__((always_inline)) {
        if constexpr (AHEAD) {
            const int32_t* row = at.at(at.k, key0 + min(kt, kt1 - 1) * 16 + (lane & 15));
#pragma unroll
            for (uint32_t ds = 0; ds < DS; ds++) load_step<FULL>(row, ds, c.head_dim, raw[ds]);
        }
    };
    load_ahead(wave);
    uint32_t seen = 0;
    for (uint32_t i = wave; i < tiles * DS; i += 4) {
        int4 v[4];
        v4i f[NARROW];
        load_step<FULL>(query(i / DS), i % DS, c.head_dim, v);
        step_digits<NARROW>(v, f, seen);
#pragma unroll
        for (int l = 0; l < NARROW; l++) s_q[(i * NARROW + l) * 64 + lane] = f[l];
    }
    if (is_wide(seen) && lane == 0) s_wide = 1;
    for (uint32_t rt = wave; rt < tiles; rt += 4) {
        const RowView v = row_view(a, r, (rt0 + rt) * 16 + (lane & 15), group);
        if (lane < 16) s_mask[rt * 16 + lane] = v.mask, s_lo[rt * 16 + lane] = v.lo;
    }
    __syncthreads();
    const bool q_wide = s_wide;
    // Positions [all0, length) are seen by every row.
    const uint32_t all0 = a.window && r.total > a.window ? r.total - a.window : 0;
    uint4* out = s.scores + (((size_t)bg * s.row_tiles + rt0) * s.chunks + chunk) * (s.chunk / 16) * 64;
    const size_t rt_stride = (size_t)s.chunks * (s.chunk / 16) * 64;
    auto keep = [&](uint32_t kt, uint32_t rt, const int32_t (&sc)[4]) __attribute__((always_inline)) {
        if ((rt0 + rt) * 16 + (lane & 15) < pairs)
            out[rt * rt_stride + kt * 64 + lane] = make_uint4((uint32_t)sc[0], (uint32_t)sc[1], (uint32_t)sc[2], (uint32_t)sc[3]);
        const uint32_t first = key0 + kt * 16;
        int32_t m;
        if (first >= all0 && first + 16 <= r.length) {
            m = max(max(sc[0], sc[1]), max(sc[2], sc[3]));
        } else {
            const RowView v{s_lo[rt * 16 + (lane & 15)], r.length, s_mask[rt * 16 + (lane & 15)]};
            m = INT32_MIN;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (v.sees(first + 4 * grp + i)) m = max(m, sc[i]);
        }
        atomicMax(&s_max[rt][lane], m);
    };
    uint32_t any_wide = 0;
#pragma unroll 1
    for (uint32_t kt = wave; kt < kt1; kt += 4) {
        v4i kf[DS][NARROW];
        uint32_t wide = 0;
#pragma unroll
        for (uint32_t ds = 0; ds < DS; ds++) {
            if constexpr (!AHEAD) load_step<FULL>(at.at(at.k, key0 + kt * 16 + (lane & 15)), ds, c.head_dim, raw[0]);
            step_digits<NARROW>(raw[AHEAD ? ds : 0], kf[ds], wide);
        }
        load_ahead(kt + 4);
        if (q_wide || is_wide(wide)) {  // more digits: below
            any_wide = 1;
            continue;
        }
#pragma unroll 1
        for (uint32_t rt = 0; rt < tiles; rt++) {
            v4i acc[2 * NARROW - 1];
#pragma unroll
            for (int j = 0; j < 2 * NARROW - 1; j++) acc[j] = v4i{0, 0, 0, 0};
#pragma unroll
            for (uint32_t ds = 0; ds < DS; ds++) {
                v4i qf[NARROW];
#pragma unroll
                for (int l = 0; l < NARROW; l++) qf[l] = s_q[((rt * DS + ds) * NARROW + l) * 64 + lane];
                dot_step<NARROW>(kf[ds], qf, acc);
            }
            int32_t sc[4];
            scores_of<HD, NARROW>(acc, a.scaled, a.scale_q32, sc);
            keep(kt, rt, sc);
        }
    }
    if (any_wide)
#pragma unroll 1
        for (uint32_t kt = wave; kt < kt1; kt += 4) {
            const int32_t* row = at.at(at.k, key0 + kt * 16 + (lane & 15));
            uint32_t wide = 0;
#pragma unroll 1
            for (uint32_t ds = 0; ds < DS; ds++) {
                int4 v[4];
                v4i f[NARROW];
                load_step<FULL>(row, ds, c.head_dim, v);
                step_digits<NARROW>(v, f, wide);
            }
            if (!q_wide && !is_wide(wide)) continue;  // above
#pragma unroll 1
            for (uint32_t rt = 0; rt < tiles; rt++) {
                v4i acc[2 * DIGITS - 1];
#pragma unroll
                for (int j = 0; j < 2 * DIGITS - 1; j++) acc[j] = v4i{0, 0, 0, 0};
#pragma unroll 1
                for (uint32_t ds = 0; ds < DS; ds++) {
                    int4 v[4];
                    v4i f[DIGITS], qf[DIGITS];
                    load_step<FULL>(row, ds, c.head_dim, v);
                    step_digits<DIGITS>(v, f, wide);
                    load_step<FULL>(query(rt), ds, c.head_dim, v);
                    step_digits<DIGITS>(v, qf, wide);
                    dot_step<DIGITS>(f, qf, acc);
                }
                int32_t sc[4];
                scores_of<HD, DIGITS>(acc, a.scaled, a.scale_q32, sc);
                keep(kt, rt, sc);
            }
        }
    lds_barrier();  // (keys past the last may be under way)
    if (tid < tiles * 16) {
        const uint32_t rt = tid / 16, i = tid % 16;
        s.maxima[(((size_t)bg * s.row_tiles + rt0 + rt) * s.chunks + chunk) * 16 + i] =
            max(max(s_max[rt][i], s_max[rt][16 + i]), max(s_max[rt][32 + i], s_max[rt][48 + i]));
    }
}

// Few rows in a tile leave most lanes of a wave without one: a lane then takes
// a row of `width` (a power of two, at least the rows) and one of 16 / width
// key tiles at once.
struct RowLanes {
    uint32_t width, row, sub, slot;  // slot: the row's place in a key tile
    __device__ __forceinline__ explicit RowLanes(uint32_t rows) {
        const uint32_t lane = threadIdx.x & 63;
        width = rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows > 1 ? 2 : 1;
        row = lane & (width - 1);
        sub = (lane & 15) / width;
        slot = (lane & 48) | row;
    }
};

// ---- (2) exp terms in place of the scores, each chunk's sums and first maxima.
// Bound by the vector units, 28 double operations a term: 32 trees of 25 at up
// to 8000 107 us; 4 tokens at up to 32700 11 us.

__global__ __launch_bounds__(256) void tree_terms_kernel(const IrisPagedKv c, const IrisTreeAttention a, const TreeSpace s) {
    __shared__ double s_sum[4][16];
    __shared__ uint32_t s_first[4][16];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index(), grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, rt = blockIdx.z, bg = blockIdx.y, group = a.heads / c.kv_heads;
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk, pairs = r.rows * group;
    if (key0 >= r.total || rt * 16 >= pairs) return;
    const uint32_t kt1 = (min(s.chunk, r.total - key0) + 15) / 16, rows = min(16u, pairs - rt * 16);
    const size_t tile = (size_t)bg * s.row_tiles + rt;
    const RowLanes l(rows);
    const bool valid = l.row < rows;
    // The row's maximum over its chunks.
    int32_t top = INT32_MIN;
    for (uint32_t i = lane / l.width; i < chunks_of(s, r); i += 64 / l.width)
        top = max(top, valid ? s.maxima[(tile * s.chunks + i) * 16 + l.row] : INT32_MIN);
    for (uint32_t off = l.width; off < 64; off <<= 1) top = max(top, __shfl_xor(top, (int)off));
    const RowView view = row_view(a, r, valid ? rt * 16 + l.row : 0xffffffffu, group);
    const uint32_t all0 = a.window && r.total > a.window ? r.total - a.window : 0, per = 16 / l.width;
    uint4* t = s.scores + (tile * s.chunks + chunk) * (s.chunk / 16) * 64 + l.slot;
    double sum = 0;  // at most 2^20 terms of 2^32: exact
    uint32_t found = 0xffffffffu;
#pragma unroll 2
    for (uint32_t k = wave * per; k < kt1; k += 4 * per) {
        const uint32_t kt = k + l.sub, key = key0 + kt * 16 + 4 * grp;
        const bool live = valid && kt < kt1;
        const uint4 sc = live ? t[kt * 64] : make_uint4(0, 0, 0, 0);
        const uint32_t v[4] = {sc.x, sc.y, sc.z, sc.w};
        const bool whole = key0 + k * 16 >= all0 && key0 + (k + per) * 16 <= r.length;
        uint32_t e[4];
        double x[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = softmax_term((uint32_t)top - v[i], &e[i]);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!view.sees(key + i)) x[i] = 0, e[i] = 0;
        }
        if (!live) continue;
        if (max(max(e[0], e[1]), max(e[2], e[3])) == 0xffffffffu) {  // the maximum itself
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e[i] == 0xffffffffu) found = min(found, key + i);
        }
        sum += (x[0] + x[1]) + (x[2] + x[3]);
        t[kt * 64] = make_uint4(e[0], e[1], e[2], e[3]);
    }
    for (uint32_t off = l.width; off < 64; off <<= 1) {
        sum += __shfl_xor(sum, (int)off);
        found = min(found, (uint32_t)__shfl_xor((int)found, (int)off));
    }
    if (lane < l.width) s_sum[wave][lane] = sum, s_first[wave][lane] = found;
    __syncthreads();
    if (tid < rows) {
        const size_t to = (tile * s.chunks + chunk) * 16 + tid;
        s.sums[to] = s_sum[0][tid] + s_sum[1][tid] + s_sum[2][tid] + s_sum[3][tid];
        s.firsts[to] = min(min(s_first[0][tid], s_first[1][tid]), min(s_first[2][tid], s_first[3][tid]));
    }
}

// ---- (3) weights and weighted values

// The sum of lane row `row` of tile `tile` over its chunks, the lanes of one
// row at strides of `width`.
__device__ __forceinline__ double row_sum(const TreeSpace& s, size_t tile, uint32_t chunks, uint32_t row, uint32_t width,
                                          bool valid) {
    const uint32_t lane = threadIdx.x & 63;
    double sum = 0;
    for (uint32_t i = lane / width; i < chunks; i += 64 / width) sum += valid ? s.sums[(tile * s.chunks + i) * 16 + row] : 0.0;
    for (uint32_t off = width; off < 64; off <<= 1) sum += __shfl_xor(sum, (int)off);
    return sum;
}

// A step's values for one 64-dimension block: dimensions d .. d + 3 of the
// lane's sixteen positions, four in a row at a time.
template <bool FULL>
__device__ __forceinline__ void load_values(const Places& at, uint32_t key, uint32_t d, int4 (&v)[4][4]) {
#pragma unroll
    for (uint32_t t = 0; t < 4; t++) {
        const int32_t* p = at.four(at.v, key + 16 * t) + (FULL || d < at.hd ? d : 0);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) v[t][i] = load4(p + i * at.hd);
    }
}

__device__ __forceinline__ int4 column(const int4 (&v)[4], int k) {
    auto of = [&](int4 x) { return k == 0 ? x.x : k == 1 ? x.y : k == 2 ? x.z : x.w; };
    return make_int4(of(v[0]), of(v[1]), of(v[2]), of(v[3]));
}

// What the fourth and fifth digits of the values add to a lane's four rows.
__device__ __forceinline__ void upper_values(v4i w0, v4i w1, const int4 (&x)[4], uint64_t (&add)[4]) {
    uint32_t seen = 0;
    v4i f[DIGITS];
    step_digits<DIGITS>(x, f, seen);
    const v4i upper[2] = {f[3], f[4]};
    v4i up[3] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}};
    value_step<2>(w0, w1, upper, up);
#pragma unroll
    for (int q = 0; q < 4; q++)
        add[q] = ((uint64_t)(int64_t)up[0][q] << 24) + ((uint64_t)(int64_t)up[1][q] << 32) + ((uint64_t)(int64_t)up[2][q] << 40);
}

// At most two weights of a row need a third digit: 65536 v more for each.
struct BigWeights {
    int32_t count[16];
    uint32_t key[16][2];
    __device__ __forceinline__ void add(uint32_t row, uint32_t k) {
        const int n = atomicAdd(&count[row], 1);
        if (n < 2) key[row][n] = k;
    }
};

// One row tile: a wave takes a 64-dimension block and PARTS of the steps; the
// chunk's weights, as operands, lie in LDS. Bound by memory: 4 tokens at up to
// 32700, 206 MB of values in 46 us, 4.4 TB/s.
template <uint32_t HD, bool FULL>
__global__ __launch_bounds__((HD / 64 > 4 ? HD : 256), 2) void tree_values_kernel(const IrisPagedKv c, const IrisTreeAttention a,
                                                                                const TreeSpace s) {
    constexpr uint32_t DS = HD / 64, WAVES = DS > 4 ? DS : 4, PARTS = WAVES / DS;
    extern __shared__ uint64_t s_sums[];  // [16][HD], then the weights' digits [steps][2][64] uint4
    __shared__ BigWeights s_big;
    __shared__ int32_t s_wsum[16];
    __shared__ double s_total[WAVES][16];
    __shared__ uint64_t s_page[CHUNK_PAGES];
    uint4* s_w = (uint4*)(s_sums + 16 * HD);
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index(), grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, bg = blockIdx.y, g = bg % c.kv_heads, group = a.heads / c.kv_heads;
    const uint32_t early = early_page(c, a, bg / c.kv_heads, chunk * s.chunk, s.chunk);
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk, rows = r.rows * group;
    if (key0 >= r.total) return;
    const uint32_t n = min(s.chunk, r.total - key0), steps = (n + STEP - 1) / STEP, kt1 = (n + 15) / 16;
    const Places at = places(c, a, r, g, key0, key0 + n, s_page, early);
    for (uint32_t i = tid; i < 16 * HD; i += WAVES * 64) s_sums[i] = 0;
    for (uint32_t i = tid; i < steps * 128; i += WAVES * 64) s_w[i] = make_uint4(0, 0, 0, 0);
    if (tid < 16) s_wsum[tid] = 0, s_big.count[tid] = 0;
    __syncthreads();
    const uint32_t block = wave % DS, part = wave / DS, d = block * 64 + 4 * (lane & 15);
    {
        const RowLanes l(rows);
        const bool valid = l.row < rows;
        const double total = row_sum(s, bg, chunks_of(s, r), l.row, l.width, valid);
        s_total[wave][lane & 15] = total;
        const RowScale sc(&s_total[wave][lane & 15], valid);
        const uint4* t = s.scores + ((size_t)bg * s.chunks + chunk) * (s.chunk / 16) * 64 + l.slot;
        const uint32_t per = 16 / l.width;
        int32_t wsum = 0;
        for (uint32_t k = wave * per; k < kt1; k += WAVES * per) {
            const uint32_t kt = k + l.sub;
            if (!valid || kt >= kt1) continue;
            const uint4 x = t[kt * 64];
            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
            int32_t w[4];
            weights_of(e, sc, sc.w, w, wsum, [&](int j) { s_big.add(l.row, key0 + kt * 16 + 4 * grp + j); });
            uint32_t low, high;
            weight_digits(w, low, high);
            uint32_t* to = (uint32_t*)(s_w + (size_t)(kt / 4) * 128 + l.slot) + kt % 4;
            to[0] = low;
            to[256] = high;
        }
        for (uint32_t off = l.width; off < 64; off <<= 1) wsum += __shfl_xor(wsum, (int)off);
        if (lane < l.width && valid) atomicAdd(&s_wsum[lane], wsum);
    }
    __syncthreads();
    v4i acc[4][NARROW + 1];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int j = 0; j < NARROW + 1; j++) acc[t][j] = v4i{0, 0, 0, 0};
#pragma unroll 1
    for (uint32_t step = part; step < steps; step += PARTS) {
        int4 v[4][4];
        load_values<FULL>(at, key0 + step * STEP + 4 * grp, d, v);
        const uint4 x0 = s_w[step * 128 + lane], x1 = s_w[step * 128 + 64 + lane];
        const v4i w0 = v4i{(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w}, w1 = v4i{(int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
        uint32_t seen = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int4 x[4] = {column(v[0], k), column(v[1], k), column(v[2], k), column(v[3], k)};
            v4i f[NARROW];
            step_digits<NARROW>(x, f, seen);
            value_step<NARROW>(w0, w1, f, acc[k]);
        }
        if (is_wide(seen)) {
#pragma unroll 1
            for (int k = 0; k < 4; k++) {
                int4 x[4];
#pragma unroll
                for (uint32_t t = 0; t < 4; t++) {
                    int32_t y[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++)
                        y[i] = load1(at.four(at.v, key0 + step * STEP + 4 * grp + 16 * t) + i * at.hd + (d < at.hd ? d + k : 0));
                    x[t] = make_int4(y[0], y[1], y[2], y[3]);
                }
                uint64_t add[4];
                upper_values(w0, w1, x, add);
#pragma unroll
                for (uint32_t q = 0; q < 4; q++)
                    if (4 * grp + q < rows) atomicAdd((unsigned long long*)&s_sums[(4 * grp + q) * HD + d + k], add[q]);
            }
        }
    }
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
        if (4 * grp + q >= rows) break;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint64_t t = 0;
#pragma unroll
            for (int j = 0; j < NARROW + 1; j++) t += (uint64_t)(int64_t)acc[k][j][q] << (8 * j);
            atomicAdd((unsigned long long*)&s_sums[(4 * grp + q) * HD + d + k], t);
        }
    }
    __syncthreads();
    uint64_t* out = s.partial + ((size_t)bg * s.chunks + chunk) * 16 * HD;
    for (uint32_t i = tid; i < rows * HD; i += WAVES * 64) {
        const uint32_t row = i / HD, dim = i % HD;
        uint64_t t = s_sums[i];
        if (dim < c.head_dim)
            for (int j = 0; j < s_big.count[row]; j++) t += (uint64_t)((int64_t)65536 * load1(at.at(at.v, s_big.key[row][j]) + dim));
        out[i] = t;
    }
    if (tid < rows) s.weights[((size_t)bg * s.chunks + chunk) * 16 + tid] = s_wsum[tid];
}

// Weights that an estimate leaves open (near a rounding tie, or of three
// digits): (row, position in the chunk) of each, settled after the loop over
// the steps, so that the loop keeps its registers. Past the list's end every
// position of the chunk is looked at again.
struct OpenWeights {
    static constexpr uint32_t ROOM = 64;
    uint32_t count;
    uint32_t at[ROOM];  // position << 4 | row
    int32_t add[ROOM];  // what the loop's weight lacks
    __device__ __forceinline__ void push(uint32_t row, uint32_t position) {
        const uint32_t n = atomicAdd(&count, 1u);
        if (n < ROOM) at[n] = position << 4 | row;
    }
};

// The estimate of a weight, and whether it is left open.
__device__ __forceinline__ int32_t estimate(uint32_t kept, double w_scale, bool& open) {
    const int32_t n = nearest_weight(kept, w_scale, open);
    open |= n >= BIG_WEIGHT;
    return n;
}

// Several row tiles: a workgroup takes MANY of them and 128 dimensions (64 of
// a head of 64), a wave per (row tile, 64-dimension block). Each step's values
// are split once, and its weights formed once, into LDS, a step ahead of the
// products that read them. 32 trees of 25 at up to 8000 (seven row tiles): 233
// us, of which the values' and terms' reads are the larger part (1.2 GB) and the
// start of a workgroup a quarter.
constexpr uint32_t MANY = 4;
constexpr uint32_t value_blocks(uint32_t hd) { return hd < 128 ? 1 : 2; }

template <uint32_t HD, bool FULL>
__global__ __launch_bounds__(MANY * value_blocks(HD) * 64, 4) void tree_values_many_kernel(const IrisPagedKv c,
                                                                                       const IrisTreeAttention a,
                                                                                       const TreeSpace s) {
    constexpr uint32_t BLOCKS = value_blocks(HD), WAVES = MANY * BLOCKS, VD = 64 * BLOCKS, KT = 4 / BLOCKS;
    __shared__ v4i s_v[2][BLOCKS * 4][NARROW][64];
    __shared__ uint4 s_w[2][MANY][2][64];
    __shared__ int32_t s_wsum[MANY][16];
    __shared__ uint32_t s_wide;  // a bit per step whose values need more digits
    __shared__ OpenWeights s_open[MANY];
    __shared__ double s_total[WAVES][16];
    __shared__ uint64_t s_page[CHUNK_PAGES];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index(), grp = lane >> 4;
    const uint32_t chunk = blockIdx.x, bg = blockIdx.y, g = bg % c.kv_heads, group = a.heads / c.kv_heads;
    const uint32_t dim0 = blockIdx.z % (HD / VD) * VD, rt0 = blockIdx.z / (HD / VD) * MANY;
    const uint32_t early = early_page(c, a, bg / c.kv_heads, chunk * s.chunk, s.chunk);
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t key0 = r.base + chunk * s.chunk, pairs = r.rows * group;
    if (key0 >= r.total || rt0 * 16 >= pairs) return;
    const uint32_t n = min(s.chunk, r.total - key0), steps = (n + STEP - 1) / STEP, kt1 = (n + 15) / 16;
    const Places at = places(c, a, r, g, key0, key0 + n, s_page, early);
    const uint32_t my = wave % MANY, block = wave / MANY, rt = rt0 + my, row = rt * 16 + (lane & 15);
    const bool has_rt = rt * 16 < pairs, valid = row < pairs;
    const size_t tile = (size_t)bg * s.row_tiles + (has_rt ? rt : rt0);
    if (tid == 0) s_wide = 0;
    if (tid < MANY * 16) s_wsum[tid / 16][tid % 16] = 0;
    if (tid < MANY) s_open[tid].count = 0;
    __syncthreads();

    // This wave's share of a step's values: dimensions 4 n .. of its block, at
    // positions 16 t + 4 `my` + i (lane: t and n).
    const uint32_t split_d = dim0 + block * 64 + 4 * (lane & 15);
    int4 raw[4];
    auto load_raw = [&](uint32_t step) __attribute__((always_inline)) {
        const int32_t* p = at.four(at.v, key0 + step * STEP + 16 * grp + 4 * my) + (FULL || split_d < at.hd ? split_d : 0);
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) raw[i] = load4(p + i * at.hd);
    };
    load_raw(0);
    const double total = row_sum(s, tile, chunks_of(s, r), lane & 15, 16, valid), scale = valid ? 65536.0 / total : 0.0;
    s_total[wave][lane & 15] = valid ? total : 0.0;
    // And of its weights: key tiles block * KT ..
    const uint4* t = s.scores + (tile * s.chunks + chunk) * (s.chunk / 16) * 64 + lane;
    uint4 terms[KT];
    auto load_terms = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t k = 0; k < KT; k++) terms[k] = t[min(step * 4 + block * KT + k, kt1 - 1) * 64];
    };
    load_terms(0);
    v4i acc[4][NARROW + 1];
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int j = 0; j < NARROW + 1; j++) acc[k][j] = v4i{0, 0, 0, 0};
    int32_t wsum = 0;
    uint64_t* out = s.partial + (tile * s.chunks + chunk) * 16 * HD + split_d;
#pragma unroll 1
    for (uint32_t step = 0; step < steps; step++) {
        const uint32_t buf = step & 1;
        uint32_t seen = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t p[4];
            split4(column(raw, k), p, seen);
#pragma unroll
            for (int l = 0; l < NARROW; l++) ((uint32_t*)&s_v[buf][block * 4 + k][l][my * 16 + (lane & 15)])[grp] = p[l];
        }
        if (is_wide(seen) && lane == 0) atomicOr(&s_wide, 1u << step);
        load_raw(min(step + 1, steps - 1));
#pragma unroll
        for (uint32_t k = 0; k < KT; k++) {
            const uint32_t kt = step * 4 + block * KT + k;
            const uint4 x = terms[k];
            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
            const double w_scale = kt < kt1 ? scale : 0.0;
            int32_t w[4];
            bool open[4];
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = estimate(e[i], w_scale, open[i]);
            if (__any(open[0] | open[1] | open[2] | open[3])) {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (open[i]) s_open[my].push(lane & 15, kt * 16 + 4 * grp + i);
            }
            wsum += w[0] + w[1] + w[2] + w[3];
            uint32_t low, high;
            weight_digits(w, low, high);
            ((uint32_t*)&s_w[buf][my][0][lane])[block * KT + k] = low;
            ((uint32_t*)&s_w[buf][my][1][lane])[block * KT + k] = high;
        }
        load_terms(min(step + 1, steps - 1));
        lds_barrier();
        if (!has_rt) continue;
        const uint4 x0 = s_w[buf][my][0][lane], x1 = s_w[buf][my][1][lane];
        const v4i w0 = v4i{(int)x0.x, (int)x0.y, (int)x0.z, (int)x0.w}, w1 = v4i{(int)x1.x, (int)x1.y, (int)x1.z, (int)x1.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            v4i f[NARROW];
#pragma unroll
            for (int l = 0; l < NARROW; l++) f[l] = s_v[buf][block * 4 + k][l][lane];
            value_step<NARROW>(w0, w1, f, acc[k]);
        }
    }
    // The sums so far; every (row, dimension) is one lane's own, which adds
    // what follows to its own entries.
    if (has_rt)
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
            uint64_t sum[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                sum[k] = 0;
#pragma unroll
                for (int j = 0; j < NARROW + 1; j++) sum[k] += (uint64_t)(int64_t)acc[k][j][q] << (8 * j);
            }
            if (rt * 16 + 4 * grp + q >= pairs) continue;
            uint64_t* to = out + (size_t)(4 * grp + q) * HD;
            *(ulonglong2*)to = make_ulonglong2(sum[0], sum[1]);
            *(ulonglong2*)(to + 2) = make_ulonglong2(sum[2], sum[3]);
        }
    wsum += __shfl_xor(wsum, 16);
    wsum += __shfl_xor(wsum, 32);
    if (lane < 16) atomicAdd(&s_wsum[my][lane], wsum);
    lds_barrier();

    // The open weights: what the loop's lack, a lane each (of the tile's first
    // wave), or of every position.
    const int32_t* terms0 = (const int32_t*)(s.scores + (tile * s.chunks + chunk) * (s.chunk / 16) * 64);
    auto lacking = [&](uint32_t i, uint32_t position, int32_t& off) __attribute__((always_inline)) {
        const uint32_t kept = (uint32_t)load1(terms0 + ((position / 16 * 64 + position % 16 / 4 * 16 + i) * 4 + position % 4));
        const double sum = s_total[wave][i];
        bool open;
        const int32_t n = estimate(kept, 65536.0 / sum, open), w = open ? exact_weight(kept, sum) : n;
        off = w - n;
        return w - two_digits(n);
    };
    const uint32_t open_count = s_open[my].count;
    const bool listed = open_count <= OpenWeights::ROOM;
    if (has_rt && block == 0) {
        if (listed) {
            if (lane < open_count) {
                const uint32_t x = s_open[my].at[lane];
                int32_t off;
                s_open[my].add[lane] = lacking(x & 15, x >> 4, off);
                if (off) atomicAdd(&s_wsum[my][x & 15], off);
            }
        } else if (valid) {
            int32_t all = 0;
#pragma unroll 1
            for (uint32_t k = grp; k < n; k += 4) {
                int32_t off;
                lacking(lane & 15, k, off);
                all += off;
            }
            atomicAdd(&s_wsum[my][lane & 15], all);
        }
    }
    __syncthreads();
    if (!has_rt) return;
    if (block == 0 && lane < 16 && valid && dim0 == 0) s.weights[(tile * s.chunks + chunk) * 16 + lane] = s_wsum[my][lane];
#pragma unroll 1
    for (uint32_t q = 0; q < 4; q++) {
        const uint32_t i = 4 * grp + q;
        if (rt * 16 + i >= pairs) continue;
        uint64_t* to = out + (size_t)i * HD;
#pragma unroll 1
        for (uint32_t j = 0; j < (listed ? open_count : n); j++) {
            uint32_t position = j;
            int32_t more, off;
            if (listed) {
                if ((s_open[my].at[j] & 15) != i) continue;
                position = s_open[my].at[j] >> 4, more = s_open[my].add[j];
            } else {
                more = lacking(i, j, off);
            }
            if (!more) continue;
            const int4 x = load4(at.at(at.v, key0 + position) + (split_d < at.hd ? split_d : 0));
            to[0] += (uint64_t)((int64_t)more * x.x), to[1] += (uint64_t)((int64_t)more * x.y);
            to[2] += (uint64_t)((int64_t)more * x.z), to[3] += (uint64_t)((int64_t)more * x.w);
        }
    }
    // Values of more digits: their steps' weights formed again, the upper
    // planes' products added.
    const uint32_t wide = s_wide;
#pragma unroll 1
    for (uint32_t step = 0; step < steps; step++) {
        if (!((wide >> step) & 1)) continue;
        v4i w0, w1;
#pragma unroll
        for (uint32_t k = 0; k < 4; k++) {
            const uint4 x = t[min(step * 4 + k, kt1 - 1) * 64];
            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
            int32_t w[4];
            bool open;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = estimate(e[i], step * 4 + k < kt1 ? scale : 0.0, open);
            uint32_t low, high;
            weight_digits(w, low, high);
            w0[k] = (int)low, w1[k] = (int)high;
        }
#pragma unroll 1
        for (int k = 0; k < 4; k++) {
            int4 x[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const int32_t* p = at.four(at.v, key0 + step * STEP + 4 * grp + 16 * i) + (split_d < at.hd ? split_d + k : 0);
                x[i] = make_int4(load1(p), load1(p + at.hd), load1(p + 2 * at.hd), load1(p + 3 * at.hd));
            }
            uint64_t more[4];
            upper_values(w0, w1, x, more);
#pragma unroll
            for (uint32_t q = 0; q < 4; q++)
                if (rt * 16 + 4 * grp + q < pairs) out[(size_t)(4 * grp + q) * HD + k] += more[q];
        }
    }
}

// ---- (4) the chunks joined: a wave per (drafted row, head), or four that
// share the chunks where there are many (SPLIT). Bound by memory: 32 trees of 25
// at up to 8000, 94 MB of partial sums in 17.5 us, 5.4 TB/s.

template <uint32_t HD, bool SPLIT>
__global__ __launch_bounds__(256) void tree_join_kernel(const IrisPagedKv c, const IrisTreeAttention a, const TreeSpace s) {
    constexpr uint32_t PIECES = HD > 128 ? HD / 128 : 1, PARTS = SPLIT ? 4 : 1;
    __shared__ uint64_t s_part[SPLIT ? 4 : 1][SPLIT ? HD : 1];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index();
    const uint32_t bg = blockIdx.x, g = bg % c.kv_heads, group = a.heads / c.kv_heads;
    const uint32_t pair = SPLIT ? blockIdx.y : blockIdx.y * 4 + wave, part = SPLIT ? wave : 0;
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    if (pair >= r.rows * group) return;
    const size_t tile = (size_t)bg * s.row_tiles + pair / 16;
    const uint32_t i = pair % 16, chunks = chunks_of(s, r);
    // Two dimensions per lane (HD 64: a half of the lanes has them).
    uint64_t t[PIECES][2];
#pragma unroll
    for (uint32_t p = 0; p < PIECES; p++) t[p][0] = t[p][1] = 0;
    const uint64_t* from = s.partial + (tile * s.chunks * 16 + i) * HD + (2 * lane) % HD;
#pragma unroll 4
    for (uint32_t k = part; k < chunks; k += PARTS)
#pragma unroll
        for (uint32_t p = 0; p < PIECES; p++) {
            const ulonglong2 x = *(const ulonglong2*)(from + (size_t)k * 16 * HD + p * 128);
            t[p][0] += x.x, t[p][1] += x.y;
        }
    uint32_t key = 0xffffffffu;
    int32_t wsum = 0;
    for (uint32_t k = lane; k < chunks; k += 64) {
        key = min(key, s.firsts[(tile * s.chunks + k) * 16 + i]);
        wsum += s.weights[(tile * s.chunks + k) * 16 + i];
    }
    for (int off = 1; off < 64; off <<= 1) {
        key = min(key, (uint32_t)__shfl_xor((int)key, off));
        wsum += __shfl_xor(wsum, off);
    }
    if constexpr (SPLIT) {
#pragma unroll
        for (uint32_t p = 0; p < PIECES; p++)
            if (2 * lane < HD) s_part[wave][p * 128 + 2 * lane] = t[p][0], s_part[wave][p * 128 + 2 * lane + 1] = t[p][1];
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (uint32_t p = 0; p < PIECES; p++)
#pragma unroll
            for (uint32_t w = 1; w < 4; w++)
                t[p][0] += s_part[w][p * 128 + (2 * lane) % HD], t[p][1] += s_part[w][p * 128 + (2 * lane) % HD + 1];
    }
    const int64_t resid = dn::sub_sat(dn::ONE_ACT, wsum);
    const uint32_t log = 31u - __clz((int)c.page_size), page = (uint32_t)r.table[key >> log];
    const int32_t* v = page < c.pages ? c.v + (((size_t)page * c.kv_heads + g) * c.page_size + (key & (c.page_size - 1))) * c.head_dim
                                      : g_zeros;
    int32_t* out = a.out + (size_t)(r.row0 + pair / group) * a.out_stride + (size_t)(g * group + pair % group) * c.head_dim;
#pragma unroll
    for (uint32_t p = 0; p < PIECES; p++) {
        const uint32_t d = p * 128 + 2 * lane;
        if (2 * lane < HD && d < c.head_dim)
            *(int2*)(out + d) = make_int2(dn::requantize((int64_t)(t[p][0] + (uint64_t)(resid * load1(v + d)))),
                                          dn::requantize((int64_t)(t[p][1] + (uint64_t)(resid * load1(v + d + 1)))));
    }
}

// ---- (2) to (4) in one launch, for positions whose score tiles LDS holds: a
// workgroup per (request, key head), row tile and 32 dimensions. Each forms all
// terms and weights of its rows: more arithmetic, fewer launches. Bound by
// latency: 1 token at 700 positions 11.3 us, behind 6.5 of the scores.

constexpr uint32_t SHORT_WAVES = 16;
constexpr uint32_t SHORT_DIMS = 32;
constexpr uint32_t SHORT_TILES = (160 * 1024 - 16 * SHORT_DIMS * 8 - 8192) / (TILE_BYTES + 32);

template <bool FULL>
__global__ __launch_bounds__(SHORT_WAVES * 64, 4) void tree_short_kernel(const IrisPagedKv c, const IrisTreeAttention a,
                                                                       const TreeSpace s) {
    constexpr uint32_t NW = SHORT_WAVES, DIMS = SHORT_DIMS;
    extern __shared__ uint4 s_tile[];  // score tiles, sums [16][DIMS], page offsets
    uint64_t* s_sums = (uint64_t*)(s_tile + s.short_tiles * 64);
    uint64_t* s_page = s_sums + 16 * DIMS;
    __shared__ int32_t s_wsum[16];
    __shared__ double s_sum[NW][16], s_total[16];
    __shared__ uint32_t s_first[16];
    __shared__ BigWeights s_big;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index(), grp = lane >> 4;
    const uint32_t bg = blockIdx.x, rt = blockIdx.y, g = bg % c.kv_heads, group = a.heads / c.kv_heads;
    const uint32_t early = early_page(c, a, bg / c.kv_heads, 0, s.short_tiles * 16);
    Request r;
    if (!read_request(c, a, bg / c.kv_heads, r)) return;
    const uint32_t pairs = r.rows * group;
    if (rt * 16 >= pairs) return;
    const uint32_t rows = min(16u, pairs - rt * 16), key0 = r.base, n = r.total - key0;
    const uint32_t kt1 = (n + 15) / 16, steps = (n + STEP - 1) / STEP, chunks = chunks_of(s, r);
    const Places at = places(c, a, r, g, key0, r.total, s_page, early);
    if (tid < 16) s_wsum[tid] = 0, s_first[tid] = 0xffffffffu, s_big.count[tid] = 0;
    for (uint32_t i = tid; i < 16 * DIMS; i += NW * 64) s_sums[i] = 0;
    const RowLanes l(rows);
    const bool valid = l.row < rows;
    const uint32_t per = 16 / l.width;
    const size_t tile = (size_t)bg * s.row_tiles + rt;
    int32_t top = INT32_MIN;
    for (uint32_t i = lane / l.width; i < chunks; i += 64 / l.width)
        top = max(top, valid ? s.maxima[(tile * s.chunks + i) * 16 + l.row] : INT32_MIN);
    for (uint32_t off = l.width; off < 64; off <<= 1) top = max(top, __shfl_xor(top, (int)off));
    const RowView view = row_view(a, r, valid ? rt * 16 + l.row : 0xffffffffu, group);
    const uint32_t all0 = a.window && r.total > a.window ? r.total - a.window : 0;
    // The first scores before the values: loads return in order.
    const uint4* from = s.scores + tile * s.chunks * (s.chunk / 16) * 64 + l.slot;  // chunk by chunk: tile by tile
    uint4 sc = from[min(wave * per + l.sub, kt1 - 1) * 64];
    __syncthreads();

    // A wave's first values are on their way during the softmax.
    // (Value tile k, column n: dimension 2 n + k.)
    const uint32_t d2 = 2 * (lane & 15), d = blockIdx.z * DIMS + d2;
    int2 v[4][4];
    auto load_pairs = [&](uint32_t step) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) {
            const int32_t* p = at.four(at.v, key0 + min(step, steps - 1) * STEP + 4 * grp + 16 * t) + (FULL || d < at.hd ? d : 0);
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) v[t][i] = load2(p + i * at.hd);
        }
    };
    load_pairs(wave);

    // (2) exp terms, their sum, the first maximum.
    double sum = 0;
    uint32_t found = 0xffffffffu;
#pragma unroll 1
    for (uint32_t k = wave * per; k < kt1; k += NW * per) {
        const uint32_t kt = k + l.sub, key = key0 + kt * 16 + 4 * grp;
        const bool live = valid && kt < kt1;
        const uint32_t x[4] = {sc.x, sc.y, sc.z, sc.w};
        if (k + NW * per < kt1) sc = from[min(kt + NW * per, kt1 - 1) * 64];
        uint32_t e[4];
        double t[4];
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = softmax_term((uint32_t)top - x[i], &e[i]);
        if (!(key0 + k * 16 >= all0 && key0 + (k + per) * 16 <= r.length)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!view.sees(key + i)) t[i] = 0, e[i] = 0;
        }
        if (!live) continue;
        if (max(max(e[0], e[1]), max(e[2], e[3])) == 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e[i] == 0xffffffffu) found = min(found, key + i);
        }
        sum += (t[0] + t[1]) + (t[2] + t[3]);
        s_tile[kt * 64 + l.slot] = make_uint4(e[0], e[1], e[2], e[3]);
    }
    for (uint32_t off = l.width; off < 64; off <<= 1) {
        sum += __shfl_xor(sum, (int)off);
        found = min(found, (uint32_t)__shfl_xor((int)found, (int)off));
    }
    if (lane < l.width) s_sum[wave][lane] = sum;
    if (lane < l.width && valid) atomicMin(&s_first[lane], found);
    lds_barrier();
    if (tid < 16) {
        double t = 0;
#pragma unroll
        for (uint32_t w = 0; w < NW; w++) t += s_sum[w][min(tid, l.width - 1)];
        s_total[tid] = t;
    }
    lds_barrier();

    // (3) the weights' digits in place of the terms: the low digits as dword
    // `slot` of a tile, the high ones as dword 64 + slot. A wave has read all
    // of its tiles' terms before it writes there. (Rows past the last: what
    // was there; their sums are not looked at.)
    {
        const RowScale scale(&s_total[l.row], valid);
        int32_t wsum = 0;
#pragma unroll 1
        for (uint32_t k = wave * per; k < steps * 4; k += NW * per) {
            const uint32_t kt = k + l.sub;
            const uint4 x = s_tile[min(kt, kt1 - 1) * 64 + l.slot];
            const uint32_t e[4] = {x.x, x.y, x.z, x.w};
            int32_t w[4];
            weights_of(e, scale, kt < kt1 ? scale.w : 0.0, w, wsum,
                       [&](int j) { s_big.add(l.row, key0 + kt * 16 + 4 * grp + j); });
            uint32_t low, high;
            weight_digits(w, low, high);
            if (kt < steps * 4) {
                uint32_t* to = (uint32_t*)(s_tile + kt * 64);
                to[l.slot] = low;
                to[64 + l.slot] = high;
            }
        }
        for (uint32_t off = l.width; off < 64; off <<= 1) wsum += __shfl_xor(wsum, (int)off);
        if (lane < l.width && valid) atomicAdd(&s_wsum[lane], wsum);
    }
    lds_barrier();

    // (4) weighted values: a wave takes its part of the steps. A thread
    // finishes one (row, dimension); the first maximum's value is on its way.
    static_assert(16 * DIMS <= NW * 64, "an output per thread");
    const uint32_t my_row = tid / DIMS, my_dim = blockIdx.z * DIMS + tid % DIMS;
    const bool mine = my_row < rows && my_dim < c.head_dim;
    const int32_t first_value = mine ? load1(at.at(at.v, s_first[my_row]) + my_dim) : 0;
    auto load_weights = [&](uint32_t step, v4i& w0, v4i& w1) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) {
            const uint32_t* p = (const uint32_t*)(s_tile + (step * 4 + t) * 64);
            w0[t] = (int)p[lane];
            w1[t] = (int)p[64 + lane];
        }
    };
    v4i acc[2][NARROW + 1];
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
        for (int j = 0; j < NARROW + 1; j++) acc[t][j] = v4i{0, 0, 0, 0};
    uint32_t any_wide = 0;
#pragma unroll 1
    for (uint32_t step = wave; step < steps; step += NW) {
        v4i w0, w1;
        load_weights(step, w0, w1);
#pragma unroll
        for (int k = 0; k < 2; k++) {
            int4 x[4];
#pragma unroll
            for (uint32_t t = 0; t < 4; t++)
                x[t] = k ? make_int4(v[t][0].y, v[t][1].y, v[t][2].y, v[t][3].y) : make_int4(v[t][0].x, v[t][1].x, v[t][2].x, v[t][3].x);
            v4i f[NARROW];
            step_digits<NARROW>(x, f, any_wide);
            value_step<NARROW>(w0, w1, f, acc[k]);
        }
        if (step + NW >= steps) break;
        load_pairs(step + NW);
    }
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            uint64_t t = 0;
#pragma unroll
            for (int j = 0; j < NARROW + 1; j++) t += (uint64_t)(int64_t)acc[k][j][q] << (8 * j);
            if (4 * grp + q < rows && wave < steps) atomicAdd((unsigned long long*)&s_sums[(4 * grp + q) * DIMS + d2 + k], t);
        }
    }
    if (is_wide(any_wide))
#pragma unroll 1
        for (uint32_t step = wave; step < steps; step += NW) {
            v4i w0, w1;
            load_weights(step, w0, w1);
#pragma unroll 1
            for (int k = 0; k < 2; k++) {
                int4 x[4];
#pragma unroll
                for (uint32_t t = 0; t < 4; t++) {
                    const int32_t* p = at.four(at.v, key0 + step * STEP + 4 * grp + 16 * t) + (d < at.hd ? d + k : 0);
                    x[t] = make_int4(load1(p), load1(p + at.hd), load1(p + 2 * at.hd), load1(p + 3 * at.hd));
                }
                uint64_t more[4];
                upper_values(w0, w1, x, more);
#pragma unroll
                for (uint32_t q = 0; q < 4; q++)
                    if (4 * grp + q < rows) atomicAdd((unsigned long long*)&s_sums[(4 * grp + q) * DIMS + d2 + k], more[q]);
            }
        }
    lds_barrier();
    if (!mine) return;
    uint64_t t = s_sums[tid] + (uint64_t)((int64_t)dn::sub_sat(dn::ONE_ACT, s_wsum[my_row]) * first_value);
    for (int j = 0; j < s_big.count[my_row]; j++) t += (uint64_t)((int64_t)65536 * load1(at.at(at.v, s_big.key[my_row][j]) + my_dim));
    const uint32_t pair = rt * 16 + my_row;
    a.out[(size_t)(r.row0 + pair / group) * a.out_stride + (size_t)(g * group + pair % group) * c.head_dim + my_dim] =
        dn::requantize((int64_t)t);
}

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
    // A launch's second and third dimensions.
    if ((uint64_t)a->requests * c->kv_heads > 65535 || (uint64_t)a->max_nodes * (a->heads / c->kv_heads) > 65535)
        return IRIS_E_RANGE;
    return 0;
}

// Carves the work space (base may be null) and returns its bytes.
uint64_t tree_space(const IrisPagedKv& c, const IrisTreeAttention& a, uint8_t* base, TreeSpace* s) {
    const uint64_t hd = padded_head(c.head_dim), bg = (uint64_t)a.requests * c.kv_heads;
    const uint32_t group = a.heads / c.kv_heads;
    s->row_tiles = (a.max_nodes * group + 15) / 16;
    // Positions that a request's rows look at, from a multiple of STEP on.
    const uint64_t span = std::min<uint64_t>(a.max_positions, a.window ? (uint64_t)a.window + a.max_nodes + STEP : a.max_positions);
    const uint64_t tiles = (span + STEP - 1) / STEP * 4;
    // Where its workgroups (sixteen waves: one to a CU) are there all at once.
    // us, short / long: 1 token at 700 (32 heads of 128, 32 workgroups) 17.2 /
    // 24.1, 8 at 700 (256) 19.4 / 28.2, 8 at up to 2100 (256) 29.7 / 36.1, a tree
    // of 32 at 700 (256) 32.0 / 44, 12 of 9 in a window of 1024 (heads of 256, 480)
    // 50 / 39, 32 at 700 (1024) 60 / 43.
    const uint64_t groups = bg * s->row_tiles * ((c.head_dim + SHORT_DIMS - 1) / SHORT_DIMS);
    s->short_tiles = tiles <= SHORT_TILES && groups <= 256 ? (uint32_t)tiles : 0;
    s->chunk = chunk_positions(span, bg);
    s->chunks = (uint32_t)((span + s->chunk - 1) / s->chunk);
    uint64_t at = 0;
    auto take = [&](auto*& p, uint64_t bytes) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
        at += (bytes + 255) & ~255ull;
    };
    const uint64_t parts = bg * s->row_tiles * s->chunks;
    take(s->scores, parts * (s->chunk / 16) * TILE_BYTES);
    take(s->maxima, parts * 16 * 4);
    take(s->firsts, parts * 16 * 4);
    take(s->sums, parts * 16 * 8);
    take(s->weights, parts * 16 * 4);
    if (!s->short_tiles) take(s->partial, parts * 16 * hd * 8);
    return at;
}

// Workgroups of one chunk follow each other request by request: consecutive
// ones go to the chiplets in turn, and how many chunks a request has is its own
// (with the chunks in front, one chiplet had every request's first chunk: the
// values of 32 trees at up to 8000 took twice the time).
template <uint32_t HD, bool FULL>
int tree_launch(const IrisPagedKv& c, const IrisTreeAttention& a, const TreeSpace& s, hipStream_t stream) {
    const uint32_t bg = a.requests * c.kv_heads, RB = row_block(HD), few = std::min(s.row_tiles, RB);
    const size_t q_lds = (size_t)few * (HD / 64) * NARROW * TILE_BYTES, v_lds = 16 * HD * 8 + (size_t)s.chunk / STEP * 2 * TILE_BYTES;
    hipError_t st = paged_lds_limit((const void*)tree_values_kernel<HD, FULL>, v_lds);
    if (st != hipSuccess) return (int)st;
    hipLaunchKernelGGL((tree_scores_kernel<HD, FULL>), dim3(s.chunks | 1, bg, (s.row_tiles + RB - 1) / RB), dim3(256), q_lds, stream, c,
                       a, s);
    if (s.short_tiles) {
        const size_t lds = (size_t)s.short_tiles * TILE_BYTES + 16 * SHORT_DIMS * 8 + ((size_t)s.short_tiles * 4 + 2) * 8;
        st = paged_lds_limit((const void*)tree_short_kernel<FULL>, lds);
        if (st != hipSuccess) return (int)st;
        hipLaunchKernelGGL(tree_short_kernel<FULL>, dim3(bg, s.row_tiles, (c.head_dim + SHORT_DIMS - 1) / SHORT_DIMS), dim3(SHORT_WAVES * 64), lds, stream, c, a, s);
        return (int)hipGetLastError();
    }
    hipLaunchKernelGGL(tree_terms_kernel, dim3(s.chunks | 1, bg, s.row_tiles), dim3(256), 0, stream, c, a, s);
    if (s.row_tiles == 1)
        hipLaunchKernelGGL((tree_values_kernel<HD, FULL>), dim3(s.chunks | 1, bg), dim3(HD > 256 ? HD : 256), v_lds, stream, c, a, s);
    else
        hipLaunchKernelGGL((tree_values_many_kernel<HD, FULL>),
                           dim3(s.chunks | 1, bg, (s.row_tiles + MANY - 1) / MANY * (HD / (64 * value_blocks(HD)))),
                           dim3(MANY * value_blocks(HD) * 64), 0, stream, c, a, s);
    const uint32_t pairs = a.max_nodes * (a.heads / c.kv_heads);
    // us, shared by four waves / one: 4 tokens at up to 32700 (32 chunks) 5.0 / 7.0,
    // 12 trees of 9 in a window (18) 6.0 / 6.5, 32 of 25 at up to 8000 (8) 33 / 17.
    if (s.chunks > 8) hipLaunchKernelGGL((tree_join_kernel<HD, true>), dim3(bg, pairs), dim3(256), 0, stream, c, a, s);
    else hipLaunchKernelGGL((tree_join_kernel<HD, false>), dim3(bg, (pairs + 3) / 4), dim3(256), 0, stream, c, a, s);
    return (int)hipGetLastError();
}

template <uint32_t HD>
int tree_launch_head(const IrisPagedKv& c, const IrisTreeAttention& a, const TreeSpace& s, hipStream_t stream) {
    return c.head_dim == HD ? tree_launch<HD, true>(c, a, s, stream) : tree_launch<HD, false>(c, a, s, stream);
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
    TreeSpace s;
    const uint64_t need = tree_space(*c, *a, (uint8_t*)space, &s);
    if (need && (!space || misaligned(space))) return IRIS_E_INVALID;
    if (bytes < need) return IRIS_E_RANGE;
    switch (padded_head(c->head_dim)) {
        case 64: return tree_launch_head<64>(*c, *a, s, (hipStream_t)stream);
        case 128: return tree_launch_head<128>(*c, *a, s, (hipStream_t)stream);
        case 256: return tree_launch_head<256>(*c, *a, s, (hipStream_t)stream);
        default: return tree_launch_head<512>(*c, *a, s, (hipStream_t)stream);
    }
}

}  // extern "C"
