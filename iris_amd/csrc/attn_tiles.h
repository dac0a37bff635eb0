// Pieces of exact attention on the int8 matrix cores over rows of several
// sequences.
//
// An int32 value is five signed byte digits, v = sum_l 256^l d_l; one below
// 2^23 - 2^15 in magnitude three. A dot product modulo 2^64 is the sum over
// pairs of digit planes of exact int32 products, each pair shifted by
// 8 (l + m); pairs of one shift share an accumulator (at most five times
// 512 * 2^14 < 2^26 each). The usual values need nine products per 64
// dimensions, the widest 25.
//
// Tiles: scores are keys x queries (16 x 16): lane l holds query l % 16 and
// keys 4 (l / 16) + i of the tile. Within a 64-dimension step the operand
// byte 4 j + c of lane l is dimension 16 j + 4 (l / 16) + c, for queries and
// keys alike: 16-byte loads of a row's four consecutive values. Weights are
// the other product's left operand without leaving their lanes: byte 4 t + i
// of a 64-key step is key 16 t + 4 (l / 16) + i. Value tiles hold, as column
// l % 16 of tile t, dimension 4 (l % 16) + t of a 64-dimension block.
#pragma once

#include "detnum_dev.h"
#include "paged.h"
#include "softmax_double.h"

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr uint32_t TILE_BYTES = 1024;  // a 16 x 64 operand: 16 bytes per lane
constexpr int DIGITS = 5;              // of any int32
constexpr int NARROW = 3;              // of the usual values
constexpr int32_t BIG_WEIGHT = 32640;  // the first weight that needs a third digit

// The dimensions that a head's operand tiles hold.
constexpr uint32_t padded_head(uint32_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 256 ? 256 : 512; }

// The wave's index in its workgroup, known to be the same in every lane (what
// follows from it stays in scalar registers).
__device__ __forceinline__ uint32_t wave_index() { return (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)); }

// Loads from device memory by a pointer the compiler cannot place (flat loads
// would count as LDS accesses too, and every LDS wait as one for them).
__device__ __forceinline__ int4 load4(const int32_t* p) {
    const v4i v = *(const __attribute__((address_space(1))) v4i*)p;
    return make_int4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ int2 load2(const int32_t* p) {
    typedef int v2i __attribute__((ext_vector_type(2)));
    const v2i v = *(const __attribute__((address_space(1))) v2i*)p;
    return make_int2(v[0], v[1]);
}
__device__ __forceinline__ int32_t load1(const int32_t* p) { return *(const __attribute__((address_space(1))) int32_t*)p; }

// The four digit planes' dwords (byte c: value c's digit) of four values;
// `seen` collects what tells whether a fourth digit was needed.
__device__ __forceinline__ void split4(int4 v, uint32_t (&plane)[4], uint32_t& seen) {
    const uint32_t bias = 0x80808080u;
    const uint32_t x = ((uint32_t)v.x + bias) ^ bias, y = ((uint32_t)v.y + bias) ^ bias;
    const uint32_t z = ((uint32_t)v.z + bias) ^ bias, w = ((uint32_t)v.w + bias) ^ bias;
    seen |= x | y | z | w;
    const uint32_t xy = __builtin_amdgcn_perm(y, x, 0x05010400u), zw = __builtin_amdgcn_perm(w, z, 0x05010400u);
    const uint32_t xy2 = __builtin_amdgcn_perm(y, x, 0x07030602u), zw2 = __builtin_amdgcn_perm(w, z, 0x07030602u);
    plane[0] = __builtin_amdgcn_perm(zw, xy, 0x05040100u);
    plane[1] = __builtin_amdgcn_perm(zw, xy, 0x07060302u);
    plane[2] = __builtin_amdgcn_perm(zw2, xy2, 0x05040100u);
    plane[3] = __builtin_amdgcn_perm(zw2, xy2, 0x07060302u);
}

// The fifth digit's dword: one where the lower four cannot reach the value.
__device__ __forceinline__ uint32_t fifth4(int4 v) {
    const int32_t top = 0x7f7f7f7f;
    return (uint32_t)(v.x > top) | (uint32_t)(v.y > top) << 8 | (uint32_t)(v.z > top) << 16 | (uint32_t)(v.w > top) << 24;
}

// Whether a fourth digit was needed anywhere in the wave.
__device__ __forceinline__ bool is_wide(uint32_t seen) { return __any(seen >> 24) != 0; }

// The scores of a lane's four keys from the accumulators of LD digits each.
template <uint32_t HD, int LD>
__device__ __forceinline__ void scores_of(const v4i (&acc)[2 * LD - 1], int scaled, uint32_t scale_q32, int32_t (&sc)[4]) {
    constexpr int NS = 2 * LD - 1;
    if constexpr (LD == NARROW) {
        // The sum in double: exact below 2^53, else off by less than 2^-52 of
        // itself; a score near a rounding tie (one in 2^14) is redone exactly.
        const double scale = (double)scale_q32 * 0x1p-48;
        bool slow = false;
        double s[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (HD <= 128) {
                // Neighbouring accumulators fit an int32 (2 HD 2^14 2^8 <= 2^30).
                const int32_t low = acc[0][i] + (acc[1][i] << 8), mid = acc[2][i] + (acc[3][i] << 8);
                s[i] = fma(fma((double)acc[4][i], 65536.0, (double)mid), 65536.0, (double)low);
            } else {
                s[i] = (double)acc[NS - 1][i];
#pragma unroll
                for (int j = NS - 2; j >= 0; j--) s[i] = fma(s[i], 256.0, (double)acc[j][i]);
            }
        }
        // The integer nearest t = sum * scale / 2^48 by a rounding addend; the
        // reference's floor at 2^-32 moves t by under 2^-16. Unscaled, t =
        // sum / 2^16 of an exact sum rounds to even as the reference does.
        const double unit = scaled ? scale : 0x1p-16;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const double t = fma(s[i], unit, SOFTMAX_ROUND), n = t - SOFTMAX_ROUND;
            sc[i] = (int32_t)(uint32_t)softmax_bits(t);
            slow |= !(fabs(n) < 2147483647.0);
            if (scaled) slow |= !(fabs(fma(s[i], unit, -n)) <= 0.5 - 0x1p-15);
            else slow |= !(fabs(s[i]) < 0x1p53);
        }
        if (!__any(slow)) return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint64_t s = 0;  // the wrapping i64 dot product
#pragma unroll
        for (int j = 0; j < NS && j < 8; j++) s += (uint64_t)(int64_t)acc[j][i] << (8 * j);
        sc[i] = scaled ? dn::scaled_score_from_sum((int64_t)s, scale_q32) : dn::requantize((int64_t)s);
    }
}

// One 64-dimension step's products into the accumulators.
template <int LD>
__device__ __forceinline__ void dot_step(const v4i (&kf)[LD], const v4i (&qf)[LD], v4i (&acc)[2 * LD - 1]) {
#pragma unroll
    for (int l = 0; l < LD; l++)
#pragma unroll
        for (int m = 0; m < LD; m++)
            acc[l + m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf[l], qf[m], acc[l + m], 0, 0, 0);
}

// What turns a row's exp terms into weights: 2^16 over their sum (zero for a
// lane without a row: all its weights are zero), and whether a weight may need
// three digits. The sum itself is read again where a weight is formed exactly.
struct RowScale {
    double w;
    bool big;
    const double* sum;
    __device__ __forceinline__ RowScale(const double* total, bool valid) : sum(total) {
        w = valid ? 65536.0 / *total : 0.0;
        big = w * 4294967296.0 >= (double)BIG_WEIGHT - 1.0;
    }
};

__device__ __forceinline__ int32_t exact_weight(uint32_t kept, double total) {
    return dn::softmax_weight(kept == 0xffffffffu ? (uint64_t)dn::ONE_ACC : kept, (uint64_t)total, 4294967296.0 / total);
}

// The integer nearest a weight's quotient as double has it: off by under
// 2^-29 (and 2^-16 where the kept term stands for 2^32), while the quotient's
// own rounding in 32 fraction bits moves it by at most 2^-17. So unless it is
// near a rounding tie, within 2^-15 (one in 2^14), this is the weight.
__device__ __forceinline__ int32_t nearest_weight(uint32_t kept, double w_scale, bool& near) {
    const double k = (double)kept, t = fma(k, w_scale, SOFTMAX_ROUND);
    near = fabs(fma(k, w_scale, SOFTMAX_ROUND - t)) > 0.5 - 0x1p-15;
    return (int32_t)(uint32_t)softmax_bits(t);
}

// The weights of four kept terms, two digits each; those near a tie are formed
// again exactly, a third digit is left to on_big(i) and taken off the weight.
template <class OnBig>
__device__ __forceinline__ void weights_of(const uint32_t (&e)[4], const RowScale& s, double w_scale, int32_t (&w)[4],
                                           int32_t& wsum, OnBig&& on_big) {
    bool slow = s.big;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        bool near;
        w[i] = nearest_weight(e[i], w_scale, near);
        slow |= near;
    }
    if (__any(slow)) {
        // One piece of code for the four: four copies of it in every loop
        // would not stay in the instruction cache.
#pragma unroll 1
        for (int i = 0; i < 4; i++) {
            const uint32_t kept = i == 0 ? e[0] : i == 1 ? e[1] : i == 2 ? e[2] : e[3];
            int32_t x = i == 0 ? w[0] : i == 1 ? w[1] : i == 2 ? w[2] : w[3];
            bool near;
            nearest_weight(kept, w_scale, near);
            if (near) x = exact_weight(kept, *s.sum);
            if (x >= BIG_WEIGHT) {
                on_big(i);
                x -= 65536;
                wsum += 65536;
            }
            w[0] = i == 0 ? x : w[0], w[1] = i == 1 ? x : w[1], w[2] = i == 2 ? x : w[2], w[3] = i == 3 ? x : w[3];
        }
    }
    wsum += w[0] + w[1] + w[2] + w[3];
}

// What two digits hold of a weight: the weight, or 65536 less.
__device__ __forceinline__ int32_t two_digits(int32_t w) { return ((w + 0x8080) & 0xffff) - 0x8080; }

// The two digit planes' dwords of four weights, of each what two_digits() says.
__device__ __forceinline__ void weight_digits(const int32_t (&w)[4], uint32_t& low, uint32_t& high) {
    uint32_t d[4];
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = (uint32_t)(w[i] + 0x8080) ^ 0x8080u;
    const uint32_t a = __builtin_amdgcn_perm(d[1], d[0], 0x05010400u), b = __builtin_amdgcn_perm(d[3], d[2], 0x05010400u);
    low = __builtin_amdgcn_perm(b, a, 0x05040100u);
    high = __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Value products of one 64-key step: weights of two digits, values of LV.
template <int LV>
__device__ __forceinline__ void value_step(v4i w0, v4i w1, const v4i (&vf)[LV], v4i (&acc)[LV + 1]) {
#pragma unroll
    for (int b = 0; b < LV; b++) {
        acc[b] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w0, vf[b], acc[b], 0, 0, 0);
        acc[b + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w1, vf[b], acc[b + 1], 0, 0, 0);
    }
}

}  // namespace
