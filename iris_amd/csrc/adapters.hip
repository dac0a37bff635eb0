// Low-rank adapters of many requests beside one product: row r, of adapter s,
// gets out = y + B_s (A_s x), both products exact over 16-bit weights and
// rounded once each.
//
// Two launches, since every output needs the whole of A x: the sums of A x for
// each row into the work space, then B t added to y. Few rows take a workgroup
// per value of A x and a thread per output, on the vector units; more rows tiles
// of 32 on the int8 matrix cores, a tile's adapters one after the other.
//
// A weight is kept as two signed byte digits, w = 256 high + low, in 16 bits;
// a value of x or t is up to five (three below 2^23 in magnitude, split4 in
// attn_tiles.h). Digit products of one weight 2^8s share an int32 accumulator.
#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "attn_tiles.h"
#include "runtime_internal.h"

namespace {

// One part of one slot; rank 0: empty.
struct AdapterEntry {
    const int16_t* a;  // [rank][cols]
    const int16_t* b;  // [rows][stride_of(rank)]
    uint32_t rank, a_bits, b_bits, pad;
};

// B's rows are padded with zeros to whole 16-byte pieces.
__host__ __device__ __forceinline__ uint32_t stride_of(uint32_t rank) { return (rank + 7) & ~7u; }

struct AdapterShape {
    uint32_t cols, part_count, slots, max_rank;
    IrisAdapterPart parts[IRIS_ADAPTER_PARTS];
};

// A call of up to so many rows, and rows times ranks, takes the kernels of single
// rows: they read an adapter again for each row, but a row's work does not wait
// for others'. Both kernels, q|k|v of 4096 columns: rank 16, 256 rows 26 us of 3
// or of 40 adapters, tiles 26 us for 300 rows of 3 prompts and 93 for 257 of 40;
// rank 64, 64 rows 27 us, tiles 31 for 65 rows of one adapter. The rank is the
// largest that the bank holds, not the largest that it may (of which the work
// space is): in a bank for ranks up to 256, of 40 adapters of rank 16, 256 rows take
// 30 us a call so and 193 by what it may hold.
constexpr uint32_t FEW_ROWS = 256, FEW_RANKS = 4096;
inline bool few(uint32_t rows, uint32_t rank) { return rows <= FEW_ROWS && rows * rank <= FEW_RANKS; }
constexpr uint32_t TILE_ROWS = 32;
constexpr uint32_t TILE_RANKS = 64;    // of A x a workgroup forms at a time: four 16-rank tiles
constexpr uint32_t MAX_SPLITS = 16;    // pieces of the columns, each with sums of its own
constexpr uint32_t CHUNK_OUTPUTS = 512;  // of a tile of rows that a workgroup forms

// Chunks of so many outputs that the parts have, and the part of one of them
// (chunk: its number among that part's). Parts differ in size: a grid of as many
// chunks for each would leave k's and v's to two of eight chiplets.
inline uint32_t chunks_of(const AdapterShape& s, uint32_t outputs) {
    uint32_t n = 0;
    for (uint32_t p = 0; p < s.part_count; p++) n += (s.parts[p].rows + outputs - 1) / outputs;
    return n;
}
__device__ __forceinline__ uint32_t part_of(const AdapterShape& sh, uint32_t outputs, uint32_t& chunk) {
    uint32_t part = 0;
    for (uint32_t n; chunk >= (n = (sh.parts[part].rows + outputs - 1) / outputs); part++) chunk -= n;
    return part;
}

// A weight's two digits, and the weight from them.
inline uint16_t digits_of(int16_t w) { return (uint16_t)(((w + 128) & ~255) | (w & 255)); }
__device__ __forceinline__ int32_t weight_of(uint32_t digits) {
    return (int32_t)(int16_t)digits - (int32_t)((digits & 0x80u) << 1);
}

// A sum of products as the Q16.16 value it stands for.
__device__ __forceinline__ int32_t rounded(int64_t sum, uint32_t bits) {
    return dn::clamp_i64_to_i32(dn::rshift_rte(sum, bits));
}

// The slot of a row; -1 for none and for one outside the bank.
__device__ __forceinline__ int32_t slot_of(const IrisAdapterRows& a, uint32_t slots, uint32_t row, bool report) {
    const int32_t s = a.slots[row];
    if (s >= -1 && s < (int32_t)slots) return s;
    if (report && a.status) *a.status = IRIS_E_INVALID;
    return -1;
}

__device__ __forceinline__ int64_t wave_sum(int64_t v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor((long long)v, off);
    return v;
}

// One value of t a workgroup: row blockIdx.y, value blockIdx.x of the parts'
// `ranks` each, the largest rank when the call was made (a captured call's bank may
// hold larger ones since: then every ranks-th value). 64-bit sums of products on the vector units, exact in any order.
// Bound by its chain of loads (slot, entry, weights): 3.2 us for one row of 4096
// columns with ranks of 16 and as much for 32 rows; 18 us for 256 rows, its products.
__global__ __launch_bounds__(256) void shrink_row_kernel(const IrisAdapterRows a, const AdapterShape sh,
                                                         const AdapterEntry* table, int32_t* t, uint32_t ranks) {
    __shared__ int64_t s_sum[4];
    const uint32_t row = blockIdx.y, part = blockIdx.x / ranks;
    const int32_t slot = slot_of(a, sh.slots, row, blockIdx.x == 0 && threadIdx.x == 0);
    if (slot < 0) return;
    const AdapterEntry e = table[slot * sh.part_count + part];
    const int4* x = (const int4*)(a.x + (size_t)row * a.x_stride);
    for (uint32_t j = blockIdx.x % ranks; j < e.rank; j += ranks) {
        const int4* w = (const int4*)(e.a + (size_t)j * sh.cols);
        int64_t sum = 0;
        for (uint32_t i = threadIdx.x; i < sh.cols / 8; i += 256) {
            const int4 p = w[i], x0 = x[2 * i], x1 = x[2 * i + 1];
            const int32_t q[4] = {p.x, p.y, p.z, p.w}, v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
            for (int c = 0; c < 4; c++) {
                sum += (int64_t)weight_of((uint32_t)q[c]) * v[2 * c];
                sum += (int64_t)weight_of((uint32_t)q[c] >> 16) * v[2 * c + 1];
            }
        }
        sum = wave_sum(sum);
        if (threadIdx.x % 64 == 0) s_sum[threadIdx.x / 64] = sum;
        __syncthreads();
        if (threadIdx.x == 0)
            t[((size_t)row * sh.part_count + part) * sh.max_rank + j] = rounded(s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], e.a_bits);
        if (j + ranks < e.rank) __syncthreads();  // before the next value's sums
    }
}

// One output a thread: chunk blockIdx.x of the parts' outputs, row blockIdx.y. A
// thread's weights are one row of B, 32 bytes at rank 16, and t is the same for the
// whole workgroup. Bound by the chain of loads before it: 2.9 us for one row of
// q|k|v, 5.8 us (2.9 TB/s of y, out and weights) for 32 rows of gate|up of 16384.
__global__ __launch_bounds__(256) void expand_row_kernel(const IrisAdapterRows a, const AdapterShape sh,
                                                         const AdapterEntry* table, const int32_t* t) {
    uint32_t chunk = blockIdx.x;
    const uint32_t row = blockIdx.y, part = part_of(sh, 256, chunk), i = chunk * 256 + threadIdx.x;
    const IrisAdapterPart p = sh.parts[part];
    if (i >= p.rows) return;
    const size_t column = p.first + (size_t)i * p.step;
    const int32_t slot = slot_of(a, sh.slots, row, false);
    AdapterEntry e{};
    if (slot >= 0) e = table[slot * sh.part_count + part];
    if (!e.rank && a.out == a.y) return;
    int32_t v = a.y[(size_t)row * a.y_stride + column];
    if (e.rank) {
        const int32_t* tr = t + ((size_t)row * sh.part_count + part) * sh.max_rank;
        const int32_t* w = (const int32_t*)(e.b + (size_t)i * stride_of(e.rank));
        int64_t sum = 0;
#pragma unroll 2
        for (uint32_t j = 0; j < e.rank; j += 8) {  // (the work space ends behind whole eights; weights there are zero)
            const int4 d = load4(w + j / 2);
            const uint32_t q[4] = {(uint32_t)d.x, (uint32_t)d.y, (uint32_t)d.z, (uint32_t)d.w};
#pragma unroll
            for (int c = 0; c < 4; c++) {
                sum += (int64_t)weight_of(q[c]) * tr[j + 2 * c];
                sum += (int64_t)weight_of(q[c] >> 16) * tr[j + 2 * c + 1];
            }
        }
        v = dn::add_sat(v, rounded(sum, e.b_bits));
    }
    a.out[(size_t)row * a.out_stride + column] = v;
}

// ------------------------------------------------------------------ tiles of rows

struct Tile {
    uint32_t lane, wave;
    int32_t slot;      // of row lane % 32
    uint32_t pending;  // rows whose adapter is still to come
};

__device__ __forceinline__ Tile tile_of(const IrisAdapterRows& a, const AdapterShape& sh, uint32_t row0, bool report) {
    Tile t;
    t.lane = threadIdx.x & 63, t.wave = wave_index();
    const uint32_t row = row0 + t.lane % TILE_ROWS;
    t.slot = row < a.rows ? slot_of(a, sh.slots, row, report && threadIdx.x < TILE_ROWS) : -1;
    t.pending = (uint32_t)__ballot(t.slot >= 0);
    return t;
}

// The next adapter of the tile and its rows.
__device__ __forceinline__ uint32_t next_slot(Tile& t, int32_t& slot) {
    slot = __builtin_amdgcn_readlane(t.slot, __builtin_ctz(t.pending));
    const uint32_t rows = (uint32_t)__ballot(t.slot == slot);
    t.pending &= ~rows;
    return rows;
}

// Sixteen weights' digits as two operands of the matrix cores.
__device__ __forceinline__ void split_weights(int4 p, int4 q, v4i& low, v4i& high) {
    const uint32_t d[8] = {(uint32_t)p.x, (uint32_t)p.y, (uint32_t)p.z, (uint32_t)p.w,
                           (uint32_t)q.x, (uint32_t)q.y, (uint32_t)q.z, (uint32_t)q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        low[i] = (int)__builtin_amdgcn_perm(d[2 * i + 1], d[2 * i], 0x06040200u);
        high[i] = (int)__builtin_amdgcn_perm(d[2 * i + 1], d[2 * i], 0x07050301u);
    }
}

// Three digits of sixteen values: the low three, or with HIGH the two above.
template <bool HIGH>
__device__ __forceinline__ void value_digits(const int4 (&v)[4], v4i (&digit)[3], uint32_t& seen) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t plane[4];
        split4(v[i], plane, seen);
        digit[0][i] = (int)(HIGH ? plane[3] : plane[0]);
        digit[1][i] = (int)(HIGH ? fifth4(v[i]) : plane[1]);
        digit[2][i] = HIGH ? 0 : (int)plane[2];
    }
}

// One step's products of two weight digits and DIGITS value digits.
template <int DIGITS>
__device__ __forceinline__ void digit_products(v4i low, v4i high, const v4i (&digit)[3], v4i (&acc)[4]) {
#pragma unroll
    for (int d = 0; d < DIGITS; d++) {
        acc[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(low, digit[d], acc[d], 0, 0, 0);
        acc[d + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(high, digit[d], acc[d + 1], 0, 0, 0);
    }
}

// A rank tile's place: sixteen values of A x of one part.
struct RankTile {
    const int16_t* a;  // this lane's weights row
    uint32_t at;       // of the tile's first value among the row's part_count max_rank
    uint32_t ranks;    // of the sixteen that there are
};

// The sums of A x over a piece of the columns for a tile of rows: waves take the
// piece's 64-column steps in turn, each with up to four rank tiles, and add
// their int64 sums in LDS (exact, so the order does not matter).
template <bool HIGH>
__device__ __forceinline__ bool shrink_steps(const IrisAdapterRows& a, uint32_t cols, const RankTile (&tile)[4], uint32_t tiles,
                                             uint32_t row0, uint32_t step0, uint32_t step1, const Tile& t, int64_t* s_sum) {
    v4i acc[2][4][4] = {};
    uint32_t seen = 0;
    const uint32_t n = t.lane & 15, group = t.lane >> 4;
    const int32_t* x[2];
#pragma unroll
    for (int g = 0; g < 2; g++) x[g] = a.x + (size_t)min(row0 + 16 * g + n, a.rows - 1) * a.x_stride;
    for (uint32_t step = step0 + t.wave; step < step1; step += 4) {
        const uint32_t k = step * 64 + 16 * group;
        const bool valid = k < cols;
        int4 v[2][4] = {};
        if (valid) {
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[g][i] = load4(x[g] + k + 4 * i);
        }
        v4i digit[2][3];
#pragma unroll
        for (int g = 0; g < 2; g++) value_digits<HIGH>(v[g], digit[g], seen);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (i >= (int)tiles) break;
            int4 w0{}, w1{};
            if (valid) w0 = load4((const int32_t*)(tile[i].a + k)), w1 = load4((const int32_t*)(tile[i].a + k) + 4);
            v4i low, high;
            split_weights(w0, w1, low, high);
#pragma unroll
            for (int g = 0; g < 2; g++) digit_products<HIGH ? 2 : 3>(low, high, digit[g], acc[g][i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (i >= (int)tiles) break;
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                int64_t sum = 0;
#pragma unroll
                for (int d = 3; d >= 0; d--) sum = (sum << 8) + acc[g][i][d][c];
                if (HIGH) sum <<= 24;
                atomicAdd((unsigned long long*)&s_sum[(16 * g + n) * (TILE_RANKS + 1) + 16 * i + 4 * group + c],
                          (unsigned long long)sum);
            }
    }
    return is_wide(seen);
}

// Workgroup: piece blockIdx.x of the columns, row tile blockIdx.y, and of
// blockIdx.z which of the tile's adapters and which four rank tiles of them.
// sums: [piece][row][part_count max_rank].
//
// A value's digits are split by the vector units, the larger part of a step; so a
// wave forms them once for up to four rank tiles, whose sums fill its registers.
// Neither is the bound (4096 rows of 14336 columns, rank 32: vector units issue in
// 21% of the cycles, matrix cores 4%) but the loads of x, 235 MB at 4.2 TB/s
// (56 us), with two workgroups a CU; 2309 rows of q|k|v at rank 64 take 41 us, where
// each of a tile's adapters reads x again, by three workgroups of four of its twelve
// rank tiles each. Two rank tiles a wave and the next step's
// loads ahead took 74 us there against 63 then, and 57 against 55 here.
__global__ __launch_bounds__(256, 2) void shrink_tile_kernel(const IrisAdapterRows a, const AdapterShape sh,
                                                             const AdapterEntry* table, int64_t* sums, uint32_t slot_groups) {
    __shared__ int64_t s_sum[TILE_ROWS * (TILE_RANKS + 1)];
    __shared__ uint32_t s_wide;
    const uint32_t row0 = blockIdx.y * TILE_ROWS, tid = threadIdx.x, steps = (sh.cols + 63) / 64;
    const uint32_t per = (steps + gridDim.x - 1) / gridDim.x, step0 = min(blockIdx.x * per, steps), step1 = min(step0 + per, steps);
    const uint32_t width = sh.part_count * sh.max_rank;
    const uint32_t turn = blockIdx.z % slot_groups, rank_group = blockIdx.z / slot_groups;
    Tile t = tile_of(a, sh, row0, blockIdx.x == 0 && blockIdx.z == 0);
    for (uint32_t at = 0; t.pending; at++) {
        int32_t slot;
        const uint32_t rows = next_slot(t, slot);
        if (at % slot_groups != turn) continue;
        const AdapterEntry* entry = table + (size_t)slot * sh.part_count;
        RankTile tile[4];
        uint32_t tiles = 0, skip = 4 * rank_group;
#pragma unroll
        for (uint32_t part = 0; part < IRIS_ADAPTER_PARTS; part++) {
            if (part >= sh.part_count) break;
            const AdapterEntry e = entry[part];
            const uint32_t of_part = (e.rank + 15) / 16;
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                // The part's tile that is this workgroup's i-th, if it is.
                const uint32_t at = skip + i - tiles;
                if (i < tiles || at >= of_part) continue;
                const uint32_t j = 16 * at;
                tile[i].a = e.a + (size_t)min(j + (t.lane & 15), e.rank - 1) * sh.cols;
                tile[i].at = part * sh.max_rank + j;
                tile[i].ranks = min(e.rank - j, 16u);
            }
            const uint32_t taken = min(of_part - min(skip, of_part), 4 - tiles);
            skip = skip > of_part ? skip - of_part : 0;
            tiles += taken;
        }
        if (!tiles) continue;
        __syncthreads();  // the sums before are read
        for (uint32_t i = tid; i < TILE_ROWS * (TILE_RANKS + 1); i += 256) s_sum[i] = 0;
        if (tid == 0) s_wide = 0;
        __syncthreads();
        if (shrink_steps<false>(a, sh.cols, tile, tiles, row0, step0, step1, t, s_sum) && t.lane == 0) s_wide = 1;
        __syncthreads();
        if (s_wide) {
            shrink_steps<true>(a, sh.cols, tile, tiles, row0, step0, step1, t, s_sum);
            __syncthreads();
        }
        // A row of 64 values a wave and turn.
        for (uint32_t r = t.wave; r < TILE_ROWS; r += 4) {
            if (!(rows >> r & 1)) continue;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < (int)tiles && t.lane / 16 == i && t.lane % 16 < tile[i].ranks)
                    sums[((size_t)blockIdx.x * a.rows + row0 + r) * width + tile[i].at + t.lane % 16] =
                        s_sum[r * (TILE_RANKS + 1) + t.lane];
        }
    }
}

// Four neighbouring outputs' columns of a row.
template <bool VEC>
__device__ __forceinline__ int4 load_columns(const int32_t* p, uint32_t step, uint32_t count) {
    int4 v{};
    if constexpr (VEC) {  // (fours are whole)
        if (count) v = load4(p);
        return v;
    }
    if (count > 0) v.x = load1(p);
    if (count > 1) v.y = load1(p + step);
    if (count > 2) v.z = load1(p + 2 * step);
    if (count > 3) v.w = load1(p + 3 * step);
    return v;
}

template <bool VEC>
__device__ __forceinline__ void store_columns(int32_t* p, uint32_t step, uint32_t count, int4 v) {
    if constexpr (VEC) {
        if (count) *(int4*)p = v;
        return;
    }
    if (count > 0) p[0] = v.x;
    if (count > 1) p[step] = v.y;
    if (count > 2) p[2 * (size_t)step] = v.z;
    if (count > 3) p[3 * (size_t)step] = v.w;
}

// u of output c of a lane's four from its accumulators; unit = 2^-bits. The
// vector units' part of a tile, so few operations: neighbouring accumulators
// share an int32 where they fit (NARROW: up to three steps, 2^29 a step), powers
// of two scale exactly, and an addend of 1.5 2^52 rounds to even.
enum class Sums { NARROW, LONG, WIDE };
template <Sums KIND, int SUMS>
__device__ __forceinline__ int32_t output_sum(const v4i (&acc)[SUMS], int c, uint32_t bits, double unit) {
    if constexpr (KIND != Sums::WIDE) {
        // Below 2^23 2^15 256 = 2^46: exact in double.
        double sum;
        if constexpr (KIND == Sums::NARROW) {
            const int32_t low = acc[0][c] + (acc[1][c] << 8), high = acc[2][c] + (acc[3][c] << 8);
            sum = fma((double)high, 65536.0 * unit, (double)low * unit);
        } else {
            sum = (double)acc[3][c];
#pragma unroll
            for (int d = 2; d >= 0; d--) sum = fma(sum, 256.0, (double)acc[d][c]);
            sum *= unit;
        }
        return (int32_t)(uint32_t)softmax_bits(fmin(fmax(sum, -2147483648.0), 2147483647.0) + SOFTMAX_ROUND);
    } else {
        int64_t sum = 0;
#pragma unroll
        for (int d = SUMS - 1; d >= 0; d--) sum = (sum << 8) + acc[d][c];
        return rounded(sum, bits);
    }
}

// The kind of an adapter's sums, its rank and whether its t is wide known.
__device__ __forceinline__ Sums kind_of(uint32_t rank, bool wide) {
    return wide ? Sums::WIDE : rank <= 192 ? Sums::NARROW : Sums::LONG;
}

// The digits of t of a tile's rows as operands of the matrix cores, in LDS:
// [64-rank step][16 rows][digit][lane].
struct Operand {
    v4i lane[64];
};
constexpr uint32_t DIGIT_PLANES = 5;
__device__ __forceinline__ uint32_t operand_at(uint32_t step, uint32_t g, uint32_t digit) { return (step * 2 + g) * DIGIT_PLANES + digit; }

// t of the rows of one adapter's part, from its sums by pieces, as operands in
// s_digits; by a workgroup of 256. What it returns tells whether a fourth digit
// was needed (above bit 23).
__device__ __forceinline__ uint32_t stage_digits(const IrisAdapterRows& a, const AdapterEntry& e, const int64_t* sums, uint32_t width,
                                                 uint32_t splits, uint32_t row0, uint32_t rows, Operand* s_digits) {
    const uint32_t steps = (e.rank + 63) / 64;
    uint32_t seen = 0;
    // Four values of a row a thread and turn (zeros past the rank and for
    // others' rows).
    for (uint32_t i = threadIdx.x; i < TILE_ROWS * steps * 16; i += 256) {
        const uint32_t r = i / (steps * 16), j = i % (steps * 16) * 4;
        int32_t v[4] = {};
        if (rows >> r & 1) {
            const int64_t* from = sums + (size_t)(row0 + r) * width + min(j, e.rank - 1);
            int64_t sum[4] = {};
            // Several pieces' loads at once; a value past the rank is the last again.
            const uint32_t last = e.rank - 1 - min(j, e.rank - 1);
            const size_t piece = (size_t)a.rows * width;
            auto add = [&](auto count, uint32_t q) {
                int64_t x[count][4];
#pragma unroll
                for (uint32_t k = 0; k < count; k++)
#pragma unroll
                    for (uint32_t c = 0; c < 4; c++) x[k][c] = from[min(q + k, splits - 1) * piece + min(c, last)];
#pragma unroll
                for (uint32_t k = 0; k < count; k++)
#pragma unroll
                    for (uint32_t c = 0; c < 4; c++) sum[c] += q + k < splits ? x[k][c] : 0;
            };
            if (splits <= 2) add(std::integral_constant<uint32_t, 2>{}, 0);
            else
                for (uint32_t q = 0; q < splits; q += 4) add(std::integral_constant<uint32_t, 4>{}, q);
#pragma unroll
            for (uint32_t c = 0; c < 4; c++) v[c] = j + c < e.rank ? rounded(sum[c], e.a_bits) : 0;
        }
        const int4 x = make_int4(v[0], v[1], v[2], v[3]);
        uint32_t plane[4];
        split4(x, plane, seen);
        const uint32_t lane = (j % 64 / 16) * 16 + r % 16, c = j % 16 / 4;
#pragma unroll
        for (uint32_t d = 0; d < DIGIT_PLANES; d++)
            ((uint32_t*)&s_digits[operand_at(j / 64, r / 16, d)].lane[lane])[c] = d < 4 ? plane[d] : fifth4(x);
    }
    return seen;
}

// Sixteen weights of a row of B from k on. The rank's padding may end at 8 of
// them: those behind it are another row's.
__device__ __forceinline__ void load_weights(const int16_t* w, uint32_t k, uint32_t stride, int4& b0, int4& b1) {
    b0 = k < stride ? load4((const int32_t*)(w + k)) : int4{};
    b1 = k + 8 < stride ? load4((const int32_t*)(w + k) + 4) : int4{};
}

// Tiles of 16 outputs for the rows of one adapter, into out. WIDE: values past
// three digits. One step's operands stay in registers where they are all (ONE).
template <bool VEC, Sums KIND, bool ONE>
__device__ __forceinline__ void expand_outputs(const IrisAdapterRows& a, const IrisAdapterPart& p, const AdapterEntry& e,
                                               const Operand* s_digits, const Tile& t, uint32_t row0, uint32_t rows, uint32_t i0,
                                               uint32_t i1) {
    constexpr int SUMS = KIND == Sums::WIDE ? 6 : 4, DIGITS = KIND == Sums::WIDE ? 5 : 3;
    const uint32_t n = t.lane & 15, group = t.lane >> 4, steps = ONE ? 1 : (e.rank + 63) / 64, b_stride = stride_of(e.rank);
    const double unit = ldexp(1.0, -(int)e.b_bits);
    v4i kept[2][DIGITS];
    if (ONE) {
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int d = 0; d < DIGITS; d++) kept[g][d] = s_digits[operand_at(0, g, d)].lane[t.lane];
    }
    // The next tile's y and first weights are under way while one is computed.
    int4 y[2], b0{}, b1{};
    auto load = [&](uint32_t i) {
        const int16_t* w = e.b + (size_t)min(i + n, p.rows - 1) * b_stride;
        const uint32_t first = i + 4 * group, count = first < i1 ? min(i1 - first, 4u) : 0;
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const uint32_t r = 16 * g + n;
            y[g] = load_columns<VEC>(a.y + (size_t)(row0 + r) * a.y_stride + p.first + (size_t)first * p.step, p.step,
                                     rows >> r & 1 ? count : 0);
        }
        load_weights(w, 16 * group, b_stride, b0, b1);
    };
    if (i0 + 16 * t.wave < i1) load(i0 + 16 * t.wave);
#pragma unroll 1
    for (uint32_t i = i0 + 16 * t.wave; i < i1; i += 64) {
        const uint32_t first = i + 4 * group, count = first < i1 ? min(i1 - first, 4u) : 0;
        const int4 was[2] = {y[0], y[1]};
        v4i acc[2][SUMS] = {};
        v4i low, high;
        split_weights(b0, b1, low, high);
        if (i + 64 < i1) load(i + 64);
#pragma unroll 1
        for (uint32_t step = 0;;) {
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int d = 0; d < DIGITS; d++) {
                    const v4i digit = ONE ? kept[g][d] : s_digits[operand_at(step, g, d)].lane[t.lane];
                    acc[g][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(low, digit, acc[g][d], 0, 0, 0);
                    acc[g][d + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(high, digit, acc[g][d + 1], 0, 0, 0);
                }
            if (ONE || ++step == steps) break;
            int4 c0{}, c1{};
            load_weights(e.b + (size_t)min(i + n, p.rows - 1) * b_stride, 64 * step + 16 * group, b_stride, c0, c1);
            split_weights(c0, c1, low, high);
        }
#pragma unroll
        for (int g = 0; g < 2; g++) {
            const uint32_t r = 16 * g + n;
            const int32_t old[4] = {was[g].x, was[g].y, was[g].z, was[g].w};
            int32_t out[4];
#pragma unroll
            for (int c = 0; c < 4; c++) out[c] = __builtin_elementwise_add_sat(old[c], output_sum<KIND>(acc[g], c, e.b_bits, unit));
            if (rows >> r & 1)
                store_columns<VEC>(a.out + (size_t)(row0 + r) * a.out_stride + p.first + (size_t)first * p.step, p.step, count,
                                   make_int4(out[0], out[1], out[2], out[3]));
        }
    }
}

// Workgroup: chunk blockIdx.x of the parts' outputs, row tile blockIdx.y, and
// blockIdx.z which of the tile's adapters. LDS: operands of the steps of max_rank.
//
// t is rounded and split once for a chunk, whose outputs then take a few steps of
// matrix products each and y's read and out's write in 16 bytes a lane: 4096 rows
// of 4096 outputs, rank 32, 43 us (134 MB at 3.1 TB/s; vector units issue in 40% of
// the cycles), 2309 rows of q|k|v at rank 64 39 us (113 MB, 2.9 TB/s). Chunks of 256
// outputs form t twice as often, of 1024 leave few workgroups: where 512 took 52 and
// 88 us, 256 took 68 and 96, 1024 51 and 93.
template <bool VEC>
__global__ __launch_bounds__(256) void expand_tile_kernel(const IrisAdapterRows a, const AdapterShape sh, const AdapterEntry* table,
                                                          const int64_t* sums, uint32_t splits, uint32_t slot_groups) {
    extern __shared__ Operand s_digits[];
    __shared__ uint32_t s_wide;
    const uint32_t row0 = blockIdx.y * TILE_ROWS, tid = threadIdx.x, turn = blockIdx.z;
    uint32_t chunk = blockIdx.x;
    const uint32_t part = part_of(sh, CHUNK_OUTPUTS, chunk);
    const IrisAdapterPart p = sh.parts[part];
    const uint32_t i0 = chunk * CHUNK_OUTPUTS, i1 = min(i0 + CHUNK_OUTPUTS, p.rows);
    const uint32_t width = sh.part_count * sh.max_rank;
    Tile t = tile_of(a, sh, row0, false);
    uint32_t copied = ~t.pending;  // rows that no adapter changes
    const bool copies = turn == 0 && a.out != a.y;
    for (uint32_t at = 0; t.pending; at++) {
        int32_t slot;
        const uint32_t rows = next_slot(t, slot);
        if (at % slot_groups != turn && !copies) continue;
        const AdapterEntry e = table[(size_t)slot * sh.part_count + part];
        if (!e.rank) copied |= rows;
        if (!e.rank || at % slot_groups != turn) continue;
        const uint32_t steps = (e.rank + 63) / 64;
        __syncthreads();  // the adapter before is done with the operands
        if (tid == 0) s_wide = 0;
        __syncthreads();
        const uint32_t seen = stage_digits(a, e, sums + part * sh.max_rank, width, splits, row0, rows, s_digits);
        if (seen >> 24) s_wide = 1;
        __syncthreads();
        const Sums kind = kind_of(e.rank, s_wide != 0);
        if (kind == Sums::WIDE) expand_outputs<VEC, Sums::WIDE, false>(a, p, e, s_digits, t, row0, rows, i0, i1);
        else if (kind == Sums::LONG) expand_outputs<VEC, Sums::LONG, false>(a, p, e, s_digits, t, row0, rows, i0, i1);
        else if (steps == 1) expand_outputs<VEC, Sums::NARROW, true>(a, p, e, s_digits, t, row0, rows, i0, i1);
        else expand_outputs<VEC, Sums::NARROW, false>(a, p, e, s_digits, t, row0, rows, i0, i1);
    }
    if (!copies) return;
    for (uint32_t r = t.wave; r < TILE_ROWS && row0 + r < a.rows; r += 4) {
        if (!(copied >> r & 1)) continue;
        for (uint32_t i = i0 + 4 * t.lane; i < i1; i += 256) {
            const size_t column = p.first + (size_t)i * p.step;
            const uint32_t count = min(i1 - i, 4u);
            store_columns<VEC>(a.out + (size_t)(row0 + r) * a.out_stride + column, p.step, count,
                               load_columns<VEC>(a.y + (size_t)(row0 + r) * a.y_stride + column, p.step, count));
        }
    }
}

// u of four outputs of both row groups, 16 outputs a wave from output i on.
template <Sums KIND>
__device__ __forceinline__ void tile_sums(const AdapterEntry& e, const IrisAdapterPart& p, const Operand* s_digits, const Tile& t,
                                          uint32_t i, int32_t (&u)[2][4]) {
    constexpr int SUMS = KIND == Sums::WIDE ? 6 : 4, DIGITS = KIND == Sums::WIDE ? 5 : 3;
    const uint32_t n = t.lane & 15, group = t.lane >> 4, steps = (e.rank + 63) / 64, b_stride = stride_of(e.rank);
    const int16_t* w = e.b + (size_t)min(i + n, p.rows - 1) * b_stride;
    const double unit = ldexp(1.0, -(int)e.b_bits);
    v4i acc[2][SUMS] = {};
#pragma unroll 1
    for (uint32_t step = 0; step < steps; step++) {
        int4 b0, b1;
        load_weights(w, 64 * step + 16 * group, b_stride, b0, b1);
        v4i low, high;
        split_weights(b0, b1, low, high);
#pragma unroll
        for (int g = 0; g < 2; g++)
#pragma unroll
            for (int d = 0; d < DIGITS; d++) {
                const v4i digit = s_digits[operand_at(step, g, d)].lane[t.lane];
                acc[g][d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(low, digit, acc[g][d], 0, 0, 0);
                acc[g][d + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(high, digit, acc[g][d + 1], 0, 0, 0);
            }
    }
#pragma unroll
    for (int g = 0; g < 2; g++)
#pragma unroll
        for (int c = 0; c < 4; c++) u[g][c] = output_sum<KIND>(acc[g], c, e.b_bits, unit);
}

// Two parts whose outputs take turns (gate and up): workgroup as
// expand_tile_kernel's, of both parts, so that a lane's four outputs of each are
// eight neighbours of a row. (Part by part every fourth byte of a line would be
// written at a time: 600 rows of 2 x 14336 at rank 16, 129 us against 75, which
// is 138 MB at 1.8 TB/s: y's loads wait for the sums before them.) LDS: operands of
// both.
__global__ __launch_bounds__(256) void expand_pair_kernel(const IrisAdapterRows a, const AdapterShape sh, const AdapterEntry* table,
                                                          const int64_t* sums, uint32_t splits, uint32_t slot_groups, uint32_t low) {
    extern __shared__ Operand s_digits[];
    __shared__ uint32_t s_wide;
    const uint32_t row0 = blockIdx.y * TILE_ROWS, tid = threadIdx.x, turn = blockIdx.z;
    const IrisAdapterPart p = sh.parts[low];  // the part of the even columns
    const uint32_t i0 = blockIdx.x * CHUNK_OUTPUTS, i1 = min(i0 + CHUNK_OUTPUTS, p.rows), width = sh.part_count * sh.max_rank;
    Operand* s_odd = s_digits + operand_at((sh.max_rank + 63) / 64, 0, 0);
    Tile t = tile_of(a, sh, row0, false);
    const uint32_t n = t.lane & 15, group = t.lane >> 4;
    uint32_t copied = ~t.pending;  // rows that no adapter changes
    const bool copies = turn == 0 && a.out != a.y;
    for (uint32_t at = 0; t.pending; at++) {
        int32_t slot;
        const uint32_t rows = next_slot(t, slot);
        if (at % slot_groups != turn && !copies) continue;
        const AdapterEntry even = table[(size_t)slot * 2 + low], odd = table[(size_t)slot * 2 + 1 - low];
        const bool none = !even.rank && !odd.rank;
        if (none) copied |= rows;
        if (none || at % slot_groups != turn) continue;
        __syncthreads();  // the adapter before is done with the operands
        if (tid == 0) s_wide = 0;
        __syncthreads();
        const uint32_t seen = stage_digits(a, even, sums + low * sh.max_rank, width, splits, row0, rows, s_digits) |
                              stage_digits(a, odd, sums + (1 - low) * sh.max_rank, width, splits, row0, rows, s_odd);
        if (seen >> 24) s_wide = 1;
        __syncthreads();
        const Sums kind = kind_of(max(even.rank, odd.rank), s_wide != 0);
#pragma unroll 1
        for (uint32_t i = i0 + 16 * t.wave; i < i1; i += 64) {
            const uint32_t first = i + 4 * group;  // (fours are whole)
            int4 y[2][2];
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (first < i1 && (rows >> (16 * g + n) & 1))
                        y[g][h] = load4(a.y + (size_t)(row0 + 16 * g + n) * a.y_stride + p.first + 2 * first + 4 * h);
            int32_t u[2][4], v[2][4];
            if (kind == Sums::NARROW) {
                tile_sums<Sums::NARROW>(even, p, s_digits, t, i, u), tile_sums<Sums::NARROW>(odd, p, s_odd, t, i, v);
            } else if (kind == Sums::LONG) {
                tile_sums<Sums::LONG>(even, p, s_digits, t, i, u), tile_sums<Sums::LONG>(odd, p, s_odd, t, i, v);
            } else {
                tile_sums<Sums::WIDE>(even, p, s_digits, t, i, u), tile_sums<Sums::WIDE>(odd, p, s_odd, t, i, v);
            }
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    if (first < i1 && (rows >> (16 * g + n) & 1))
                        *(int4*)(a.out + (size_t)(row0 + 16 * g + n) * a.out_stride + p.first + 2 * first + 4 * h) =
                            make_int4(__builtin_elementwise_add_sat(y[g][h].x, u[g][2 * h]), __builtin_elementwise_add_sat(y[g][h].y, v[g][2 * h]),
                                      __builtin_elementwise_add_sat(y[g][h].z, u[g][2 * h + 1]),
                                      __builtin_elementwise_add_sat(y[g][h].w, v[g][2 * h + 1]));
        }
    }
    if (!copies) return;
    for (uint32_t r = t.wave; r < TILE_ROWS && row0 + r < a.rows; r += 4) {
        if (!(copied >> r & 1)) continue;
        for (uint32_t i = 2 * i0 + 4 * t.lane; i < 2 * i1; i += 256)
            *(int4*)(a.out + (size_t)(row0 + r) * a.out_stride + p.first + i) = load4(a.y + (size_t)(row0 + r) * a.y_stride + p.first + i);
    }
}

// Workgroups that share the rank tiles of an adapter.
uint32_t rank_groups(const AdapterShape& s) { return (s.part_count * ((s.max_rank + 15) / 16) + 3) / 4; }

// Workgroups that share the adapters of a tile of rows: most tiles of prompts have
// one or two, those of short prompts or single tokens up to 32, and where tiles
// are few there is room for a workgroup each. (2309 rows of 19 prompts, sums of
// A x: 63 us with one, 42 with four.)
uint32_t slot_groups_of(uint32_t tiles) { return tiles <= 8 ? 32 : tiles <= 32 ? 16 : tiles <= 64 ? 8 : 4; }

// Pieces of the columns for a call of tiles: enough workgroups for the card (two
// a CU, which its registers hold), each with a step for every wave. More would only
// be more sums to write and add. (One piece holds any columns: a step adds at most
// 2 64 2^14 to an accumulator, and a wave has a quarter of at most 1024 steps.)
uint32_t splits_of(const AdapterShape& s, uint32_t rows) {
    const uint32_t tiles = (rows + TILE_ROWS - 1) / TILE_ROWS, steps = (s.cols + 63) / 64;
    return std::max(1u, std::min(std::min(512 / (tiles * rank_groups(s)), (steps + 3) / 4), MAX_SPLITS));
}

// Bytes of work space of a call: t itself for few rows, its sums by pieces for
// tiles. Where it goes by the ranks that the bank holds which of the two a call
// takes, this is the tiles', the larger.
uint64_t space_of(const AdapterShape& s, uint32_t rows) {
    const uint64_t values = (uint64_t)rows * s.part_count * s.max_rank;
    return few(rows, s.max_rank) ? values * 4 + 32 : values * splits_of(s, rows) * 8;
}

}  // namespace

struct IrisAdapterBank {
    AdapterShape shape{};
    int16_t* weights = nullptr;
    AdapterEntry* table = nullptr;  // [slots][parts]
    uint64_t slot_weights = 0;      // weights of a slot
    uint64_t part_at[IRIS_ADAPTER_PARTS] = {};
    uint32_t most_rows = 0, width = 0;
    std::vector<uint16_t> ranks;  // [slots][parts], as the table's
    uint32_t rank = 0;            // the largest of them
};

uint64_t iris_adapters_space(uint32_t cols, uint32_t part_count, uint32_t max_rank, uint32_t rows) {
    if (!rows || rows > 65535) return 0;
    AdapterShape s{};
    s.cols = cols, s.part_count = part_count, s.max_rank = max_rank;
    // What any number of rows up to these takes: whole tiles take the most.
    uint64_t bytes = space_of(s, rows);
    for (uint32_t n = rows / TILE_ROWS * TILE_ROWS; n; n -= TILE_ROWS) bytes = std::max(bytes, space_of(s, n));
    return std::max(bytes, space_of(s, std::min(std::min(rows, FEW_ROWS), std::max(FEW_RANKS / max_rank, 1u))));
}

extern "C" {

int iris_adapters_create(uint32_t cols, const IrisAdapterPart* parts, uint32_t part_count, uint32_t slots, uint32_t max_rank,
                         IrisAdapterBank** out) {
    if (!out) return IRIS_E_INVALID;
    *out = nullptr;
    if (!parts || !part_count || part_count > IRIS_ADAPTER_PARTS || !cols || cols % 32 || !slots || !max_rank) return IRIS_E_INVALID;
    if (cols > 65504 || slots > 65535 || max_rank > IRIS_ADAPTER_RANK) return IRIS_E_RANGE;
    for (uint32_t p = 0; p < part_count; p++) {
        if (!parts[p].rows || !parts[p].step) return IRIS_E_INVALID;
        if (parts[p].first + (uint64_t)(parts[p].rows - 1) * parts[p].step >= 1u << 24) return IRIS_E_RANGE;
    }
    // Two parts share an output where a column lies in both progressions.
    for (uint32_t p = 0; p < part_count; p++)
        for (uint32_t q = 0; q < p; q++)
            for (uint32_t i = 0; i < parts[p].rows; i++) {
                const int64_t off = (int64_t)parts[p].first + (int64_t)i * parts[p].step - parts[q].first;
                if (off >= 0 && off % parts[q].step == 0 && off / parts[q].step < parts[q].rows) return IRIS_E_INVALID;
            }
    IrisAdapterBank* b = new (std::nothrow) IrisAdapterBank();
    if (!b) return IRIS_E_NOMEM;
    AdapterShape& s = b->shape;
    s.cols = cols, s.part_count = part_count, s.slots = slots, s.max_rank = max_rank;
    for (uint32_t p = 0; p < part_count; p++) {
        s.parts[p] = parts[p];
        b->part_at[p] = b->slot_weights;
        b->slot_weights += (uint64_t)max_rank * cols + (uint64_t)parts[p].rows * stride_of(max_rank);
        b->slot_weights = (b->slot_weights + 127) & ~127ull;
        b->most_rows = std::max(b->most_rows, parts[p].rows);
        b->width = std::max(b->width, parts[p].first + (parts[p].rows - 1) * parts[p].step + 1);
    }
    try {
        b->ranks.assign((size_t)slots * part_count, 0);
    } catch (const std::bad_alloc&) {
        delete b;
        return IRIS_E_NOMEM;
    }
    const size_t entries = (size_t)slots * part_count * sizeof(AdapterEntry);
    hipError_t st = hipMalloc((void**)&b->weights, b->slot_weights * slots * 2);
    if (st == hipSuccess) st = hipMalloc((void**)&b->table, entries);
    if (st == hipSuccess) st = hipMemset(b->table, 0, entries);
    if (st == hipSuccess) st = hipDeviceSynchronize();
    if (st != hipSuccess) {
        iris_adapters_free(b);
        (void)hipGetLastError();  // returned here: not the next launch's to report
        return (int)st;
    }
    *out = b;
    return 0;
}

void iris_adapters_free(IrisAdapterBank* b) {
    if (!b) return;
    (void)hipFree(b->weights);
    (void)hipFree(b->table);
    delete b;
}

uint64_t iris_adapters_device_bytes(const IrisAdapterBank* b) {
    return b ? b->slot_weights * b->shape.slots * 2 + (uint64_t)b->shape.slots * b->shape.part_count * sizeof(AdapterEntry) : 0;
}

int iris_adapters_load(IrisAdapterBank* b, uint32_t slot, uint32_t part, const int16_t* a, uint32_t a_bits, const int16_t* w,
                       uint32_t b_bits, uint32_t rank) {
    if (!b || slot >= b->shape.slots || part >= b->shape.part_count || (rank && (!a || !w))) return IRIS_E_INVALID;
    const AdapterShape& s = b->shape;
    if (rank > s.max_rank || (rank && (a_bits > IRIS_ADAPTER_BITS || b_bits > IRIS_ADAPTER_BITS))) return IRIS_E_RANGE;
    const uint32_t rows = s.parts[part].rows, stride = stride_of(rank);
    // The two digits of each weight, A and then B with its rows padded by zeros.
    std::vector<uint16_t> digits;
    const size_t a_count = (size_t)rank * s.cols, count = a_count + (size_t)rows * stride;
    try {
        digits.assign(count, 0);
    } catch (const std::bad_alloc&) {
        return IRIS_E_NOMEM;
    }
    uint32_t past = 0;
    auto convert = [&past](const int16_t* from, uint16_t* to, size_t n) {
        uint32_t bad = 0;
        for (size_t i = 0; i < n; i++) {
            bad |= (uint32_t)(from[i] > IRIS_ADAPTER_WEIGHT) | (uint32_t)(from[i] < -IRIS_ADAPTER_WEIGHT);
            to[i] = digits_of(from[i]);
        }
        past |= bad;
    };
    convert(a, digits.data(), a_count);
    if (stride == rank) convert(w, digits.data() + a_count, (size_t)rows * rank);
    else
        for (uint32_t i = 0; i < rows; i++) convert(w + (size_t)i * rank, digits.data() + a_count + (size_t)i * stride, rank);
    if (past) return IRIS_E_RANGE;
    int16_t* to = b->weights + slot * b->slot_weights + b->part_at[part];
    AdapterEntry* entry = b->table + (size_t)slot * s.part_count + part;
    AdapterEntry e{};
    hipError_t st = hipDeviceSynchronize();
    if (st != hipSuccess) return (int)st;
    // (A copy that fails on the way leaves the part empty.)
    uint16_t& held = b->ranks[(size_t)slot * s.part_count + part];
    st = hipMemcpy(entry, &e, sizeof(e), hipMemcpyHostToDevice);
    if (st == hipSuccess) held = 0;
    if (st == hipSuccess && rank) {
        e.a = to, e.b = to + a_count;
        e.rank = rank, e.a_bits = a_bits, e.b_bits = b_bits;
        st = hipMemcpy(to, digits.data(), count * 2, hipMemcpyHostToDevice);
        if (st == hipSuccess) st = hipMemcpy(entry, &e, sizeof(e), hipMemcpyHostToDevice);
        if (st == hipSuccess) held = (uint16_t)rank;
    }
    b->rank = *std::max_element(b->ranks.begin(), b->ranks.end());
    return (int)st;
}

uint64_t iris_adapters_workspace_bytes(const IrisAdapterBank* b, uint32_t rows) {
    return b ? iris_adapters_space(b->shape.cols, b->shape.part_count, b->shape.max_rank, rows) : 0;
}

int iris_adapters_apply(const IrisAdapterBank* b, const IrisAdapterRows* a, void* space, uint64_t space_bytes, void* stream) {
    if (!b || !a) return IRIS_E_INVALID;
    if (!a->rows) return 0;
    if (!a->x || !a->y || !a->out || !a->slots || !space || misaligned(a->x) || misaligned(space) || a->x_stride % 4)
        return IRIS_E_INVALID;
    const AdapterShape& s = b->shape;
    if (a->x_stride < s.cols || a->y_stride < b->width || a->out_stride < b->width) return IRIS_E_INVALID;
    if (a->out == a->y && a->out_stride != a->y_stride) return IRIS_E_INVALID;
    if (a->rows > 65535) return IRIS_E_RANGE;
    if (space_bytes < space_of(s, a->rows)) return IRIS_E_RANGE;
    hipStream_t st = (hipStream_t)stream;
    if (!few(a->rows, b->rank)) {
        const uint32_t tiles = (a->rows + TILE_ROWS - 1) / TILE_ROWS, splits = splits_of(s, a->rows);
        const size_t lds = (s.max_rank + 63) / 64 * 2 * DIGIT_PLANES * sizeof(Operand);
        // Sixteen bytes of a row at a time where every part allows it.
        const bool aligned = !misaligned(a->y) && !misaligned(a->out) && a->y_stride % 4 == 0 && a->out_stride % 4 == 0;
        bool vec = aligned;
        for (uint32_t p = 0; p < s.part_count; p++) vec = vec && s.parts[p].step == 1 && s.parts[p].first % 4 == 0 && s.parts[p].rows % 4 == 0;
        // Two parts in turn whose fours of both are eight aligned neighbours.
        const uint32_t low = s.part_count == 2 && s.parts[1].first < s.parts[0].first;
        const bool pair = s.part_count == 2 && s.parts[0].step == 2 && s.parts[1].step == 2 && s.parts[0].rows == s.parts[1].rows &&
                          s.parts[1 - low].first == s.parts[low].first + 1 && s.parts[low].first % 4 == 0 && s.parts[0].rows % 4 == 0 &&
                          aligned;
        const uint32_t groups = slot_groups_of(tiles);
        const dim3 grid(pair ? (b->most_rows + CHUNK_OUTPUTS - 1) / CHUNK_OUTPUTS : chunks_of(s, CHUNK_OUTPUTS), tiles, groups);
        hipLaunchKernelGGL(shrink_tile_kernel, dim3(splits, tiles, rank_groups(s) * groups), dim3(256), 0, st, *a, s, b->table,
                           (int64_t*)space, groups);
        const int64_t* sums = (const int64_t*)space;
        if (pair) {
            const hipError_t limit = paged_lds_limit((const void*)expand_pair_kernel, 2 * lds);
            if (limit != hipSuccess) return (int)limit;
            hipLaunchKernelGGL(expand_pair_kernel, grid, dim3(256), 2 * lds, st, *a, s, b->table, sums, splits, groups, low);
        } else if (vec) {
            hipLaunchKernelGGL(expand_tile_kernel<true>, grid, dim3(256), lds, st, *a, s, b->table, sums, splits, groups);
        } else {
            hipLaunchKernelGGL(expand_tile_kernel<false>, grid, dim3(256), lds, st, *a, s, b->table, sums, splits, groups);
        }
        return (int)hipGetLastError();
    }
    const uint32_t ranks = std::max(b->rank, 1u);
    hipLaunchKernelGGL(shrink_row_kernel, dim3(s.part_count * ranks, a->rows), dim3(256), 0, st, *a, s, b->table, (int32_t*)space,
                       ranks);
    hipLaunchKernelGGL(expand_row_kernel, dim3(chunks_of(s, 256), a->rows), dim3(256), 0, st, *a,
                       s, b->table, (const int32_t*)space);
    return (int)hipGetLastError();
}

}  // extern "C"
