// Causal attention over packed prompts on the int8 matrix cores.
//
// The softmax is the reference's (ops.rs:233-261): each row's first maximum
// before any exp term, the sum of all terms before any weight. So a
// workgroup takes 16 rows of one head, keeps all their scores in LDS (1 KB
// per 16 keys; the tiles past LDS in the work space), and walks them three
// times: scores and maxima, exp terms and sums, weights. The weights, as two
// digit planes in place of their terms, then meet the values: the waves share
// the keys in the first three walks and the dimensions in the last.
//
// A first launch writes the digit planes of queries, keys and values as
// operand tiles, aligned to the packed rows and not to their sequences, and
// each row's first key: a tile of rows takes the union of its rows' keys and
// each row sees its own, so short sequences share tiles. (Planes once, since
// every row tile of every head reads its keys and values again: split on the
// way they would cost each of them the splitting.)
//
// Most of its time is the exact arithmetic of the softmax on the vector units:
// of a 16 x 16 tile of scores about 395 instructions a wave, 176 of them in
// double (11 for a score, 28 for a term, 8 for a weight), beside 30 matrix
// instructions. 4096 rows of 32 heads of 128 over 8 key heads take 1.20 ms, 114
// TFLOP/s of plain products: the vector units issue in 57% of the cycles (0.68
// ms), the matrix cores are busy in 19%; the rest is waiting, at the barriers
// between the walks (15%) and for score tiles past LDS, which go through the
// work space. 2309 rows of 19 sequences, same heads: 113 us. 13 rows: 11.5 us,
// two launches and their chains of loads.
#include <algorithm>

#include "attn_tiles.h"

namespace {

// The work space of a launch.
struct PackedSpace {
    int8_t *q, *k, *v;          // digit planes, operand tiles
    size_t q_plane, kv_plane;   // bytes of one plane
    uint8_t *q_wide, *k_wide, *v_wide;  // [heads][q tiles], [kv_heads][key tiles], [kv_heads][steps][DS]
    int32_t* first;             // [rows] the first key a row sees, -1: the row is left
    uint4* spill;               // [workgroups][spill_tiles][64] score tiles past those in LDS
    uint32_t q_tiles, steps;    // 16-row tiles; 64-key steps
    uint32_t lds_tiles, spill_tiles, waves, groups;
};

// The sequence of row t: the last s[i] <= t.
__device__ __forceinline__ uint32_t sequence_of(const int32_t* s, uint32_t n, uint32_t t) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s[mid] <= (int32_t)t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Writes a 16-row tile's planes: rows row0 .. of x, HD dimensions.
template <uint32_t HD>
__device__ __forceinline__ void row_tile_planes(const int32_t* x, size_t stride, uint32_t row0, uint32_t rows, uint32_t hd,
                                                int8_t* dst, size_t plane, uint8_t* wide) {
    const uint32_t lane = threadIdx.x & 63, row = row0 + (lane & 15), d0 = (lane >> 4) * 4;
    const bool valid = row < rows;
    const int32_t* src = x + (size_t)min(row, rows - 1) * stride;
    uint32_t seen = 0;
    int4 v[HD / 64][4];
#pragma unroll
    for (uint32_t ds = 0; ds < HD / 64; ds++)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t d = ds * 64 + j * 16 + d0;
            v[ds][j] = *(const int4*)(src + (d < hd ? d : 0));
            if (!valid || d >= hd) v[ds][j] = make_int4(0, 0, 0, 0);
        }
#pragma unroll
    for (uint32_t ds = 0; ds < HD / 64; ds++) {
        uint32_t p[4][4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) split4(v[ds][j], p[j], seen);
        int8_t* at = dst + ds * TILE_BYTES + lane * 16;
#pragma unroll
        for (int l = 0; l < NARROW; l++) *(uint4*)(at + l * plane) = make_uint4(p[0][l], p[1][l], p[2][l], p[3][l]);
    }
    const bool w = is_wide(seen);
    if (lane == 0) *wide = w;
    if (!w) return;
#pragma unroll 1
    for (uint32_t ds = 0; ds < HD / 64; ds++) {
        int8_t* at = dst + ds * TILE_BYTES + lane * 16;
        uint32_t p[4][4], f[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t d = ds * 64 + j * 16 + d0;
            int4 x4 = *(const int4*)(src + (d < hd ? d : 0));
            if (!valid || d >= hd) x4 = make_int4(0, 0, 0, 0);
            split4(x4, p[j], seen);
            f[j] = fifth4(x4);
        }
        *(uint4*)(at + 3 * plane) = make_uint4(p[0][3], p[1][3], p[2][3], p[3][3]);
        *(uint4*)(at + 4 * plane) = make_uint4(f[0], f[1], f[2], f[3]);
    }
}

// Writes the four value tiles of a 64-key step and a 64-dimension block.
__device__ __forceinline__ void value_block_planes(const int32_t* x, size_t stride, uint32_t key0, uint32_t rows, uint32_t dim0,
                                                   uint32_t hd, int8_t* dst, size_t plane, uint8_t* wide) {
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, d = dim0 + 4 * (lane & 15);
    int4 v[4][4];  // [t][i]: key 16 t + 4 g + i
#pragma unroll
    for (uint32_t t = 0; t < 4; t++)
#pragma unroll
        for (uint32_t i = 0; i < 4; i++) {
            const uint32_t key = key0 + 16 * t + 4 * g + i;
            v[t][i] = *(const int4*)(x + (size_t)min(key, rows - 1) * stride + (d < hd ? d : 0));
            if (key >= rows || d >= hd) v[t][i] = make_int4(0, 0, 0, 0);
        }
    uint32_t seen = 0;
    auto column = [&](uint32_t c, uint32_t t) {  // dimension d + c of the tile's four keys
        auto of = [&](int4 x) { return c == 0 ? x.x : c == 1 ? x.y : c == 2 ? x.z : x.w; };
        return make_int4(of(v[t][0]), of(v[t][1]), of(v[t][2]), of(v[t][3]));
    };
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) {
        uint32_t p[4][4];
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) split4(column(c, t), p[t], seen);
        int8_t* at = dst + c * TILE_BYTES + lane * 16;
#pragma unroll
        for (int l = 0; l < NARROW; l++) *(uint4*)(at + l * plane) = make_uint4(p[0][l], p[1][l], p[2][l], p[3][l]);
    }
    const bool w = is_wide(seen);
    if (lane == 0) *wide = w;
    if (!w) return;
#pragma unroll
    for (uint32_t c = 0; c < 4; c++) {
        uint32_t p[4][4], f[4];
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) {
            split4(column(c, t), p[t], seen);
            f[t] = fifth4(column(c, t));
        }
        int8_t* at = dst + c * TILE_BYTES + lane * 16;
        *(uint4*)(at + 3 * plane) = make_uint4(p[0][3], p[1][3], p[2][3], p[3][3]);
        *(uint4*)(at + 4 * plane) = make_uint4(f[0], f[1], f[2], f[3]);
    }
}

// A wave per tile: keys' tiles, values' blocks, queries' tiles, and 64 rows'
// first keys. Bound by memory: four bytes read and three written per value; the
// 4096 rows above are 176 MB in 32 us, 5.4 TB/s.
template <uint32_t HD>
__global__ __launch_bounds__(256) void packed_planes_kernel(const IrisPackedAttention a, const PackedSpace s) {
    constexpr uint32_t DS = HD / 64;
    uint32_t task = blockIdx.x * 4 + wave_index();
    const uint32_t key_tiles = s.steps * 4, lane = threadIdx.x & 63;
    if (task < key_tiles * a.kv_heads) {
        const uint32_t g = task % a.kv_heads, kt = task / a.kv_heads;
        const size_t at = (size_t)g * key_tiles + kt;
        row_tile_planes<HD>(a.k + (size_t)g * a.head_dim, a.k_stride, kt * 16, a.rows, a.head_dim, s.k + at * DS * TILE_BYTES,
                            s.kv_plane, s.k_wide + at);
        return;
    }
    task -= key_tiles * a.kv_heads;
    if (task < s.steps * DS * a.kv_heads) {
        const uint32_t g = task % a.kv_heads, block = task / a.kv_heads % DS, ks = task / a.kv_heads / DS;
        const size_t at = ((size_t)g * s.steps + ks) * DS + block;
        value_block_planes(a.v + (size_t)g * a.head_dim, a.v_stride, ks * 64, a.rows, block * 64, a.head_dim,
                           s.v + at * 4 * TILE_BYTES, s.kv_plane, s.v_wide + at);
        return;
    }
    task -= s.steps * DS * a.kv_heads;
    if (task < s.q_tiles * a.heads) {
        const uint32_t h = task % a.heads, qt = task / a.heads;
        const size_t at = (size_t)h * s.q_tiles + qt;
        row_tile_planes<HD>(a.q + (size_t)h * a.head_dim, a.q_stride, qt * 16, a.rows, a.head_dim, s.q + at * DS * TILE_BYTES,
                            s.q_plane, s.q_wide + at);
        return;
    }
    task -= s.q_tiles * a.heads;
    const uint32_t t = task * 64 + lane;
    if (t >= a.rows) return;
    int32_t first = -1;
    if ((int32_t)t >= a.row_start[0] && (int32_t)t < a.row_start[a.sequences]) {
        const int32_t start = min(max(a.row_start[sequence_of(a.row_start, a.sequences, t)], 0), (int32_t)t);
        if (t - (uint32_t)start >= a.max_length) {
            if (a.status) *a.status = IRIS_E_RANGE;
        } else {
            first = a.window && t - (uint32_t)start >= a.window ? (int32_t)(t + 1 - a.window) : start;
        }
    }
    s.first[t] = first;
}

template <int NW>
struct PackedSmem {
    int32_t best[NW][16];
    double sum[NW][16], total[16];
    uint32_t first[16];
    int32_t wsum[16], nbig[16], big[16][2];
};

// The parts of the keys that the waves of one pair of dimension tiles share:
// two tiles a wave, so that a weight is read for both. (4096 rows of 32 heads of
// 128: 1318 us, with one tile a wave 1354.)
template <uint32_t HD, int NW>
constexpr uint32_t key_parts() { return NW * 32 > HD ? NW * 32 / HD : 1; }

// One (16 rows, head). NW waves; SPILL: tiles past s.lds_tiles in the work
// space (`spill`).
template <uint32_t HD, int NW, bool SPILL>
__device__ __forceinline__ void packed_rows(const IrisPackedAttention& a, const PackedSpace& s, uint32_t qt, uint32_t h,
                                            uint4* tiles, uint4* spill, PackedSmem<NW>& sm) {
    constexpr uint32_t DS = HD / 64, DT = HD / 16, PARTS = key_parts<HD, NW>(), DTW = DT * PARTS / NW;
    constexpr bool HOLD = HD <= 256;  // the queries' operands stay in registers
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = wave_index(), grp = lane >> 4;
    const uint32_t g = h / (a.heads / a.kv_heads);

    // This lane's row and the keys [first, row] it sees.
    const uint32_t row = qt * 16 + (lane & 15);
    const int32_t first = row < a.rows ? s.first[row] : -1;
    const bool valid = first >= 0;
    uint32_t lo = valid ? (uint32_t)first : 0xffffffffu, all0 = valid ? (uint32_t)first : 0;
    int32_t hi = valid ? (int32_t)row : -1;
    uint32_t all1 = valid ? row : 0xffffffffu;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
        lo = min(lo, (uint32_t)__shfl_xor((int)lo, off));
        hi = max(hi, __shfl_xor(hi, off));
        all0 = max(all0, (uint32_t)__shfl_xor((int)all0, off));
        all1 = min(all1, (uint32_t)__shfl_xor((int)all1, off));
    }
    // The same in every lane: scalars from here on. Every row sees the keys
    // [all0, all1].
    lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    all0 = (uint32_t)__builtin_amdgcn_readfirstlane((int)all0);
    all1 = (uint32_t)__builtin_amdgcn_readfirstlane((int)all1);
    if (hi < 0) return;  // no row is computed
    const uint32_t span = valid ? row - (uint32_t)first : 0;
    auto sees = [&](uint32_t key) { return valid & (key - (uint32_t)first <= span); };
    // Tiles [ta, tb) hold keys that are seen; steps are whole.
    const uint32_t ks0 = lo / 64, ks1 = (uint32_t)hi / 64 + 1, base = ks0 * 4, ta = lo / 16, tb = (uint32_t)hi / 16 + 1;
    // A tile's place: in LDS, or past it in the work space. (Two kinds of
    // access: a pointer to either would make all of them flat ones.)
    auto spilled = [&](uint32_t kt) { return SPILL && kt - base >= s.lds_tiles; };
    auto in_lds = [&](uint32_t kt) { return tiles + (kt - base) * 64; };
    typedef __attribute__((address_space(1))) v4i global_v4i;
    typedef __attribute__((address_space(1))) uint32_t global_u32;
    auto in_space = [&](uint32_t kt) { return spill + (size_t)(kt - base - s.lds_tiles) * 64; };
    auto put = [&](uint32_t kt, uint32_t x, uint32_t y, uint32_t z, uint32_t w) __attribute__((always_inline)) {
        if (spilled(kt)) *(global_v4i*)(in_space(kt) + lane) = v4i{(int)x, (int)y, (int)z, (int)w};
        else in_lds(kt)[lane] = make_uint4(x, y, z, w);
    };
    auto get = [&](uint32_t kt, uint32_t (&v)[4]) __attribute__((always_inline)) {
        if (spilled(kt)) {
            const v4i x = *(const global_v4i*)(in_space(kt) + lane);
            v[0] = (uint32_t)x[0], v[1] = (uint32_t)x[1], v[2] = (uint32_t)x[2], v[3] = (uint32_t)x[3];
        } else {
            const uint4 x = in_lds(kt)[lane];
            v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
        }
    };

    if (tid < 16) sm.wsum[tid] = 0, sm.nbig[tid] = 0, sm.first[tid] = 0xffffffffu;

    // (1) scores and the maxima.
    const int8_t* qb = s.q + ((size_t)h * s.q_tiles + qt) * DS * TILE_BYTES + lane * 16;
    const int8_t* kb = s.k + (size_t)g * s.steps * 4 * DS * TILE_BYTES + lane * 16;
    v4i qf[HOLD ? DS : 1][NARROW];
    if constexpr (HOLD)
#pragma unroll
        for (uint32_t ds = 0; ds < DS; ds++)
#pragma unroll
            for (int l = 0; l < NARROW; l++) qf[ds][l] = *(const v4i*)(qb + l * s.q_plane + ds * TILE_BYTES);
    auto whole = [&](uint32_t kt) { return kt * 16 >= all0 && kt * 16 + 15 <= all1; };
    int32_t best = INT32_MIN;
    auto keep = [&](uint32_t kt, const int32_t (&sc)[4]) __attribute__((always_inline)) {
        put(kt, (uint32_t)sc[0], (uint32_t)sc[1], (uint32_t)sc[2], (uint32_t)sc[3]);
        if (whole(kt)) {
            best = max(max(best, sc[0]), max(sc[1], max(sc[2], sc[3])));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) best = sees(kt * 16 + 4 * grp + i) ? max(best, sc[i]) : best;
        }
    };
    {
        // The next tile's keys are loaded during this one's products, where
        // the registers allow. (Past the last: it again.)
        constexpr bool AHEAD = HD <= 128;
        const uint8_t* kw = s.k_wide + (size_t)g * s.steps * 4;
        const uint32_t q_wide = s.q_wide[(size_t)h * s.q_tiles + qt];
        uint32_t any_wide = 0;
        v4i kf[AHEAD ? DS : 1][NARROW];
        uint32_t k_wide = 0;
        auto load_keys = [&](uint32_t kt) __attribute__((always_inline)) {
            k_wide = kw[kt];
            if constexpr (AHEAD)
#pragma unroll
                for (uint32_t ds = 0; ds < DS; ds++)
#pragma unroll
                    for (int l = 0; l < NARROW; l++) kf[ds][l] = *(const v4i*)(kb + l * s.kv_plane + ((size_t)kt * DS + ds) * TILE_BYTES);
        };
        load_keys(min(ta + wave, tb - 1));
#pragma unroll 1
        for (uint32_t kt = ta + wave; kt < tb; kt += NW) {
            const uint32_t wide = (uint32_t)__builtin_amdgcn_readfirstlane((int)(k_wide | q_wide));
            if (wide) {  // tiles of more digits: below
                any_wide = 1;
                load_keys(min(kt + NW, tb - 1));
                continue;
            }
            v4i acc[2 * NARROW - 1];
#pragma unroll
            for (int j = 0; j < 2 * NARROW - 1; j++) acc[j] = v4i{0, 0, 0, 0};
#pragma unroll
            for (uint32_t ds = 0; ds < DS; ds++) {
                if constexpr (AHEAD) {
                    dot_step<NARROW>(kf[ds], qf[ds], acc);
                } else {
                    v4i k[NARROW], q[NARROW];
#pragma unroll
                    for (int l = 0; l < NARROW; l++) {
                        k[l] = *(const v4i*)(kb + l * s.kv_plane + ((size_t)kt * DS + ds) * TILE_BYTES);
                        q[l] = HOLD ? qf[HOLD ? ds : 0][l] : *(const v4i*)(qb + l * s.q_plane + ds * TILE_BYTES);
                    }
                    dot_step<NARROW>(k, q, acc);
                }
            }
            load_keys(min(kt + NW, tb - 1));
            int32_t sc[4];
            scores_of<HD, NARROW>(acc, a.scaled, a.scale_q32, sc);
            keep(kt, sc);
        }
        if (any_wide)
#pragma unroll 1
            for (uint32_t kt = ta + wave; kt < tb; kt += NW) {
                // A narrow tile's upper planes were not written: its digits
                // there are zero.
                const uint32_t kwide = kw[kt];
                if (!(kwide | q_wide)) continue;
                v4i acc[2 * DIGITS - 1];
#pragma unroll
                for (int j = 0; j < 2 * DIGITS - 1; j++) acc[j] = v4i{0, 0, 0, 0};
#pragma unroll 1
                for (uint32_t ds = 0; ds < DS; ds++) {
                    v4i k[DIGITS], q[DIGITS];
#pragma unroll
                    for (int l = 0; l < DIGITS; l++) {
                        k[l] = q[l] = v4i{0, 0, 0, 0};
                        if (l < NARROW || kwide) k[l] = *(const v4i*)(kb + l * s.kv_plane + ((size_t)kt * DS + ds) * TILE_BYTES);
                        if (l < NARROW || q_wide) q[l] = *(const v4i*)(qb + l * s.q_plane + ds * TILE_BYTES);
                    }
                    dot_step<DIGITS>(k, q, acc);
                }
                int32_t sc[4];
                scores_of<HD, DIGITS>(acc, a.scaled, a.scale_q32, sc);
                keep(kt, sc);
            }
    }
    best = max(best, __shfl_xor(best, 16));
    best = max(best, __shfl_xor(best, 32));
    if (lane < 16) sm.best[wave][lane] = best;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NW; v++) best = max(best, sm.best[v][lane & 15]);

    // (2) the exp terms in place of the scores, their sum (at most 2^16 terms
    // of 2^32: exact in double, in any order), and where the maximum is first.
    double sum = 0;
    uint32_t found = 0xffffffffu;
#pragma unroll 2
    for (uint32_t kt = ta + wave; kt < tb; kt += NW) {
        uint32_t v[4], e[4];
        double x[4];
        get(kt, v);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = softmax_term((uint32_t)best - v[i], &e[i]);
        if (!whole(kt)) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (!sees(kt * 16 + 4 * grp + i)) x[i] = 0, e[i] = 0;
        }
        if (max(max(e[0], e[1]), max(e[2], e[3])) == 0xffffffffu) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (e[i] == 0xffffffffu) found = min(found, kt * 16 + 4 * grp + i);
        }
        sum += (x[0] + x[1]) + (x[2] + x[3]);
        put(kt, e[0], e[1], e[2], e[3]);
    }
    found = min(found, (uint32_t)__shfl_xor((int)found, 16));
    found = min(found, (uint32_t)__shfl_xor((int)found, 32));
    if (lane < 16) atomicMin(&sm.first[lane], found);
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (lane < 16) sm.sum[wave][lane] = sum;
    __syncthreads();
    if (tid < 16) {
        sum = sm.sum[0][tid];
#pragma unroll
        for (int v = 1; v < NW; v++) sum += sm.sum[v][tid];
        sm.total[tid] = sum;
    }
    __syncthreads();

    // (3) the weights' digits in place of the terms: the low digits of a
    // tile's four keys per lane as dword `lane`, the high ones as dword
    // 64 + lane. Tiles of the first and last step that no row sees: zeros.
    {
        const RowScale scale(&sm.total[lane & 15], valid);
        int32_t wsum = 0;
#pragma unroll 1
        for (uint32_t kt = base + wave; kt < ks1 * 4; kt += NW) {
            uint32_t low = 0, high = 0;
            if (kt >= ta && kt < tb) {
                uint32_t e[4];
                get(kt, e);
                int32_t w[4];
                weights_of(e, scale, scale.w, w, wsum, [&](int i) {
                    const int at = atomicAdd(&sm.nbig[lane & 15], 1);
                    if (at < 2) sm.big[lane & 15][at] = (int32_t)(kt * 16 + 4 * grp + i);
                });
                weight_digits(w, low, high);
            }
            if (spilled(kt)) {
                global_u32* t = (global_u32*)in_space(kt);
                t[lane] = low;
                t[64 + lane] = high;
            } else {
                uint32_t* t = (uint32_t*)in_lds(kt);
                t[lane] = low;
                t[64 + lane] = high;
            }
        }
        wsum += __shfl_xor(wsum, 16);
        wsum += __shfl_xor(wsum, 32);
        if (lane < 16) atomicAdd(&sm.wsum[lane], wsum);
    }
    if constexpr (SPILL) __threadfence_block();
    __syncthreads();

    // (4) weighted values: a wave's dimension tiles over its part of the steps.
    const uint32_t dt0 = wave % (NW / PARTS) * DTW, part = wave / (NW / PARTS);
    const int8_t* vb = s.v + (size_t)g * s.steps * DT * TILE_BYTES + lane * 16;
    const uint8_t* vw = s.v_wide + (size_t)g * s.steps * DS + dt0 / 4;
    auto load_weights = [&](uint32_t ks, v4i& w0, v4i& w1) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t t = 0; t < 4; t++) {
            if (spilled(ks * 4 + t)) {
                const global_u32* p = (const global_u32*)in_space(ks * 4 + t);
                w0[t] = (int)p[lane];
                w1[t] = (int)p[64 + lane];
            } else {
                const uint32_t* p = (const uint32_t*)in_lds(ks * 4 + t);
                w0[t] = (int)p[lane];
                w1[t] = (int)p[64 + lane];
            }
        }
    };
    v4i acc[DTW][NARROW + 1];
#pragma unroll
    for (uint32_t d = 0; d < DTW; d++)
#pragma unroll
        for (int j = 0; j < NARROW + 1; j++) acc[d][j] = v4i{0, 0, 0, 0};
    uint32_t any_wide = 0;
    auto load_values = [&](uint32_t ks, v4i (&vf)[DTW][NARROW]) __attribute__((always_inline)) {
#pragma unroll
        for (uint32_t d = 0; d < DTW; d++) {
#pragma unroll
            for (int b = 0; b < NARROW; b++)
                vf[d][b] = *(const v4i*)(vb + b * s.kv_plane + ((size_t)ks * DT + dt0 + d) * TILE_BYTES);
            if (d % 4 == 0) any_wide |= vw[ks * DS + d / 4];
        }
    };
    auto add_values = [&](uint32_t ks, const v4i (&vf)[DTW][NARROW]) __attribute__((always_inline)) {
        v4i w0, w1;
        load_weights(ks, w0, w1);
#pragma unroll
        for (uint32_t d = 0; d < DTW; d++) value_step<NARROW>(w0, w1, vf[d], acc[d]);
    };
    // A step's values are loaded during the step before, where the registers
    // allow (4096 rows: 1318 us without, 1305 with). (Past the last: it again.)
    if constexpr (DTW <= 2) {
        v4i even[DTW][NARROW], odd[DTW][NARROW];
        uint32_t ks = ks0 + part;
        if (ks < ks1) load_values(ks, even);
#pragma unroll 1
        for (; ks + PARTS < ks1; ks += 2 * PARTS) {
            load_values(ks + PARTS, odd);
            __builtin_amdgcn_sched_barrier(0);  // (the loads stay ahead of the products)
            add_values(ks, even);
            load_values(min(ks + 2 * PARTS, ks1 - 1), even);
            __builtin_amdgcn_sched_barrier(0);
            add_values(ks + PARTS, odd);
        }
        if (ks < ks1) add_values(ks, even);
    } else {
#pragma unroll 1
        for (uint32_t ks = ks0 + part; ks < ks1; ks += PARTS) {
            v4i vf[DTW][NARROW];
            load_values(ks, vf);
            add_values(ks, vf);
        }
    }
    uint64_t tot[DTW][4];
#pragma unroll
    for (uint32_t d = 0; d < DTW; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            tot[d][i] = 0;
#pragma unroll
            for (int j = 0; j < NARROW + 1; j++) tot[d][i] += (uint64_t)(int64_t)acc[d][j][i] << (8 * j);
        }
    if (__any(any_wide))  // values of more digits: the two upper planes' products
#pragma unroll 1
        for (uint32_t ks = ks0 + part; ks < ks1; ks += PARTS) {
            v4i w0, w1;
            load_weights(ks, w0, w1);
#pragma unroll
            for (uint32_t d = 0; d < DTW; d++) {
                if (!vw[ks * DS + d / 4]) continue;
                v4i up[3] = {v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}, v4i{0, 0, 0, 0}}, upper[2];
#pragma unroll
                for (int b = 0; b < 2; b++)
                    upper[b] = *(const v4i*)(vb + (NARROW + b) * s.kv_plane + ((size_t)ks * DT + dt0 + d) * TILE_BYTES);
                value_step<2>(w0, w1, upper, up);
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int j = 0; j < 3; j++) tot[d][i] += (uint64_t)(int64_t)up[j][i] << (24 + 8 * j);
            }
        }
    __syncthreads();  // the weights are read: their place takes the sums
    uint64_t* sums = (uint64_t*)tiles;  // [part][16][HD]
#pragma unroll
    for (uint32_t d = 0; d < DTW; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t dt = dt0 + d;
            sums[((size_t)part * 16 + 4 * grp + i) * HD + dt / 4 * 64 + 4 * (lane & 15) + dt % 4] = tot[d][i];
        }
    __syncthreads();

    // What the weights lack of one goes to the first maximum (ops.rs:258-260),
    // 65536 v to each weight of three digits.
    const uint32_t hd = a.head_dim, hd4 = hd / 4;
    const int32_t* v = a.v + (size_t)g * hd;
    for (uint32_t c = tid; c < 16 * hd4; c += NW * 64) {
        const uint32_t r = c / hd4, d = c % hd4 * 4, out_row = qt * 16 + r;
        if (out_row >= a.rows || s.first[out_row] < 0) continue;
        const int64_t resid = dn::sub_sat(dn::ONE_ACT, sm.wsum[r]);
        const int4 vm = *(const int4*)(v + (size_t)sm.first[r] * a.v_stride + d);
        const int32_t vv[4] = {vm.x, vm.y, vm.z, vm.w};
        uint64_t t[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            t[i] = (uint64_t)(resid * vv[i]);
#pragma unroll
            for (uint32_t p = 0; p < PARTS; p++) t[i] += sums[((size_t)p * 16 + r) * HD + d + i];
        }
        for (int j = 0; j < sm.nbig[r]; j++) {
            const int4 b = *(const int4*)(v + (size_t)sm.big[r][j] * a.v_stride + d);
            t[0] += (uint64_t)((int64_t)65536 * b.x), t[1] += (uint64_t)((int64_t)65536 * b.y);
            t[2] += (uint64_t)((int64_t)65536 * b.z), t[3] += (uint64_t)((int64_t)65536 * b.w);
        }
        *(int4*)(a.out + (size_t)out_row * a.out_stride + (size_t)h * hd + d) =
            make_int4(dn::requantize((int64_t)t[0]), dn::requantize((int64_t)t[1]), dn::requantize((int64_t)t[2]),
                      dn::requantize((int64_t)t[3]));
    }
    if constexpr (SPILL) __syncthreads();  // before the next rows' scores
}

// Workgroup index -> (row tile, head): the heads of one key head follow each
// other at a stride of kv_heads, so that with eight key heads each chiplet's
// L2 holds one head's planes; the last rows, which see the most, first.
__device__ __forceinline__ void packed_place(const IrisPackedAttention& a, const PackedSpace& s, uint32_t item, uint32_t& qt,
                                             uint32_t& h) {
    const uint32_t x = item % a.heads;
    h = x % a.kv_heads * (a.heads / a.kv_heads) + x / a.kv_heads;
    qt = s.q_tiles - 1 - item / a.heads;
}

template <uint32_t HD, int NW>
__global__ __launch_bounds__(NW * 64, HD >= 512 ? 2 : 4) void packed_lds_kernel(const IrisPackedAttention a, const PackedSpace s) {
    extern __shared__ uint4 s_tiles[];
    __shared__ PackedSmem<NW> sm;
    uint32_t qt, h;
    packed_place(a, s, blockIdx.x, qt, h);
    packed_rows<HD, NW, false>(a, s, qt, h, s_tiles, nullptr, sm);
}

// Longer sequences: a workgroup takes several (rows, head) in turn, each with
// the same part of the work space.
template <uint32_t HD, int NW>
__global__ __launch_bounds__(NW * 64, HD >= 512 ? 2 : 4) void packed_spill_kernel(const IrisPackedAttention a,
                                                                                const PackedSpace s) {
    extern __shared__ uint4 s_tiles[];
    __shared__ PackedSmem<NW> sm;
    for (uint32_t item = blockIdx.x; item < s.q_tiles * a.heads; item += gridDim.x) {
        uint32_t qt, h;
        packed_place(a, s, item, qt, h);
        packed_rows<HD, NW, true>(a, s, qt, h, s_tiles, s.spill + (size_t)blockIdx.x * s.spill_tiles * 64, sm);
    }
}

int packed_check(const IrisPackedAttention* a) {
    if (!a || !a->q || !a->k || !a->v || !a->out || !a->row_start) return IRIS_E_INVALID;
    if (misaligned(a->q) || misaligned(a->k) || misaligned(a->v) || misaligned(a->out)) return IRIS_E_INVALID;
    if (!a->heads || !a->kv_heads || a->heads % a->kv_heads || !a->head_dim || a->head_dim % 4 ||
        a->head_dim > ATTN_MAX_HEAD_DIM || a->heads > 65535)
        return IRIS_E_INVALID;
    const uint64_t q = (uint64_t)a->heads * a->head_dim, kv = (uint64_t)a->kv_heads * a->head_dim;
    if ((a->q_stride | a->k_stride | a->v_stride | a->out_stride) % 4) return IRIS_E_INVALID;
    if (a->q_stride < q || a->out_stride < q || a->k_stride < kv || a->v_stride < kv) return IRIS_E_INVALID;
    if (a->rows > INT32_MAX - 64u || a->sequences > INT32_MAX || a->max_length > ATTN_MAX_KEYS) return IRIS_E_RANGE;
    if (!a->max_length && a->rows && a->sequences) return IRIS_E_INVALID;
    // A launch has under 2^32 threads: up to 1024 for 16 rows of a head, 64 for
    // a tile of digit planes.
    if (((uint64_t)a->rows + 15) / 16 * a->heads >= 1u << 22) return IRIS_E_RANGE;
    if (((uint64_t)a->rows / 16 + 8) * (a->heads + 24ull * a->kv_heads) >= 1u << 26) return IRIS_E_RANGE;
    return 0;
}

constexpr uint32_t LDS_BYTES = 160 * 1024;
constexpr uint32_t CUS = 256;  // an MI355X

// How a launch's (rows, head) items are taken: by workgroups of `waves`, with
// `tiles` score tiles in LDS (the rest in the work space) and, where some are
// there, `groups` workgroups.
struct PackedShape {
    uint32_t waves, tiles, groups;
};

// A CU's registers hold sixteen waves of a head size up to 256, eight of 512.
// Tiles of up to a half (a quarter) of LDS: workgroups of eight (four) waves,
// so that one's waits are another's work. More than that: where the items are
// many, still two workgroups of eight waves to a CU with the tiles past 76 in
// the work space, else one of sixteen waves with 156 tiles. us, two of eight /
// one of sixteen: 4096 rows x 32 heads of 128 1349 / 1419, 2048 x 32 of 128 357
// / 371, 1300 x 32 of 128 159 / 172, 2000 x 8 of 512 256 / 307; 2300 x 8 of 256
// 175 / 161, 2000 x 4 of 64 52 / 44. Few items: sixteen waves for each, eight
// for twice as many, while there are tiles for them.
inline PackedShape packed_shape(uint32_t hd, uint32_t items, uint32_t tiles) {
    const uint32_t one = (LDS_BYTES - 4096) / TILE_BYTES, two = (LDS_BYTES / 2 - 4096) / TILE_BYTES,
                   four = (LDS_BYTES / 4 - 4096) / TILE_BYTES;
    if (tiles > two && (hd > 256 || items >= 8 * CUS)) return {8, two, 2 * CUS};
    if (hd > 256) return {8, tiles, 0};
    if (tiles > two) return {16, std::min(tiles, one), CUS};
    const uint32_t filled = items < CUS ? 16 : items < 2 * CUS ? 8 : 4;
    return {std::max(tiles > four ? 8u : 4u, std::min(filled, tiles >= 16 ? 16u : tiles >= 8 ? 8u : 4u)), tiles, 0};
}

// Carves the work space (base may be null) and returns its bytes.
uint64_t packed_space(const IrisPackedAttention& a, uint8_t* base, PackedSpace* s) {
    const uint64_t hd = padded_head(a.head_dim);
    s->q_tiles = (a.rows + 15) / 16;
    s->steps = (a.rows + 63) / 64;
    s->q_plane = (uint64_t)a.heads * s->q_tiles * 16 * hd;
    s->kv_plane = (uint64_t)a.kv_heads * s->steps * 64 * hd;
    // A tile of rows sees at most this many keys, in whole steps.
    const uint32_t span = std::min(std::min(a.max_length, a.window ? a.window : a.max_length) + 15, a.rows);
    const uint32_t tiles = std::min(((span + 126) / 64) * 4, s->steps * 4);
    const PackedShape shape = packed_shape((uint32_t)hd, s->q_tiles * a.heads, tiles);
    s->waves = shape.waves;
    s->groups = shape.groups;
    s->lds_tiles = shape.tiles;
    s->spill_tiles = tiles - s->lds_tiles;
    uint64_t at = 0;
    auto take = [&](auto*& p, uint64_t bytes) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(base + at);
        at += (bytes + 255) & ~255ull;
    };
    take(s->q, DIGITS * s->q_plane);
    take(s->k, DIGITS * s->kv_plane);
    take(s->v, DIGITS * s->kv_plane);
    take(s->q_wide, (uint64_t)a.heads * s->q_tiles);
    take(s->k_wide, (uint64_t)a.kv_heads * s->steps * 4);
    take(s->v_wide, (uint64_t)a.kv_heads * s->steps * (hd / 64));
    take(s->first, (uint64_t)a.rows * 4);
    take(s->spill, (uint64_t)s->groups * s->spill_tiles * TILE_BYTES);
    return at;
}

template <uint32_t HD, int NW>
int packed_launch_waves(const IrisPackedAttention& a, const PackedSpace& s, hipStream_t stream) {
    const uint32_t items = s.q_tiles * a.heads;
    const size_t lds = std::max<size_t>((size_t)s.lds_tiles * TILE_BYTES, (size_t)key_parts<HD, NW>() * 16 * HD * 8);
    if constexpr (NW > 4) {
        if (s.spill_tiles) {
            const hipError_t st = paged_lds_limit((const void*)packed_spill_kernel<HD, NW>, lds);
            if (st != hipSuccess) return (int)st;
            hipLaunchKernelGGL((packed_spill_kernel<HD, NW>), dim3(std::min(items, s.groups)), dim3(NW * 64), lds, stream, a, s);
            return (int)hipGetLastError();
        }
    }
    const hipError_t st = paged_lds_limit((const void*)packed_lds_kernel<HD, NW>, lds);
    if (st != hipSuccess) return (int)st;
    hipLaunchKernelGGL((packed_lds_kernel<HD, NW>), dim3(items), dim3(NW * 64), lds, stream, a, s);
    return (int)hipGetLastError();
}

template <uint32_t HD>
int packed_launch(const IrisPackedAttention& a, const PackedSpace& s, hipStream_t stream) {
    const uint32_t tasks = s.steps * 4 * a.kv_heads + s.steps * (HD / 64) * a.kv_heads + s.q_tiles * a.heads + (a.rows + 63) / 64;
    hipLaunchKernelGGL(packed_planes_kernel<HD>, dim3((tasks + 3) / 4), dim3(256), 0, stream, a, s);
    if constexpr (HD <= 256) {
        if (s.waves == 4) return packed_launch_waves<HD, 4>(a, s, stream);
        if (s.waves == 16) return packed_launch_waves<HD, 16>(a, s, stream);
    }
    return packed_launch_waves<HD, 8>(a, s, stream);
}

}  // namespace

extern "C" {

uint64_t iris_attention_packed_workspace_bytes(const IrisPackedAttention* a) {
    if (packed_check(a) || !a->rows || !a->sequences) return 0;
    PackedSpace s;
    return packed_space(*a, nullptr, &s);
}

int iris_attention_packed(const IrisPackedAttention* a, void* space, uint64_t bytes, void* stream) {
    const int rc = packed_check(a);
    if (rc) return rc;
    if (!a->rows || !a->sequences) return 0;
    if (!space || misaligned(space)) return IRIS_E_INVALID;
    PackedSpace s;
    if (bytes < packed_space(*a, (uint8_t*)space, &s)) return IRIS_E_RANGE;
    switch (padded_head(a->head_dim)) {
        case 64: return packed_launch<64>(*a, s, (hipStream_t)stream);
        case 128: return packed_launch<128>(*a, s, (hipStream_t)stream);
        case 256: return packed_launch<256>(*a, s, (hipStream_t)stream);
        default: return packed_launch<512>(*a, s, (hipStream_t)stream);
    }
}

}  // extern "C"
