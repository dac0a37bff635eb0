// The softmax's exp term (softmax_exp_term, crates/det-num/src/ops.rs:508-556)
// of a score `diff` below its row's maximum, in double arithmetic for host and
// device alike.
//
// The reference's steps are integers: d = diff 2^16, k = floor(d / ln 2), r the
// remainder, r^2 .. r^5 each rounded to even at 32 fraction bits, their
// quotients by 2, 6, 24 and 120 rounded to even, their sum shifted right by k
// and rounded to even. A sum with 1.5 * 2^52 is a rounding to even of the other
// operand (below 2^51 in magnitude), and its low word that integer's. A
// fused multiply-add rounds the power's exact product once; the quotients by
// 6, 24 and 120 are rounded as products first, so that one that lies half way
// stays there. That no step turns on the products' own rounding is checked over
// all 2^20 differences with a non-zero term (tests/test_softmax_terms_host.py).
// About 29 double operations; the same steps with floor, rint and conversions
// take 30 and a dozen other instructions more.
#pragma once

#include <math.h>
#include <stdint.h>
#include <string.h>

#ifdef __HIPCC__
#define SOFTMAX_FN __host__ __device__ __forceinline__
#else
#define SOFTMAX_FN static inline
#endif

// The integer-rounding addend.
#define SOFTMAX_ROUND 6755399441055744.0

SOFTMAX_FN uint64_t softmax_bits(double x) {
    uint64_t b;
    memcpy(&b, &x, 8);
    return b;
}
SOFTMAX_FN double softmax_from_bits(uint64_t b) {
    double x;
    memcpy(&x, &b, 8);
    return x;
}

// The term (0 .. 2^32), and in *kept its 32 bits: 2^32, which only diff = 0
// gives, as 0xffffffff, which no other term is.
SOFTMAX_FN double softmax_term(uint32_t diff, uint32_t* kept) {
#ifdef __clang__
#pragma clang fp contract(off)
#endif
    const double M = SOFTMAX_ROUND;
    // From 2^20 on the term is zero: so it is at 2^22, by the shift.
    const double d = (double)(diff < (1u << 20) ? diff : 1u << 22);
    const double tk = fma(d, 65536.0 / 2977044472.0, -0.5) + M, k = tk - M;
    const double r = fma(k, -2977044472.0 / 65536.0, d);  // the remainder / 2^16
    const double rs = r * 0x1p-16;
    const double r2 = fma(r, r, M) - M, r3 = fma(r2, rs, M) - M, r4 = fma(r3, rs, M) - M, r5 = fma(r4, rs, M) - M;
    const double even = fma(r2, 0.5, M) - (r3 * (1.0 / 6) + M), odd = (r4 * (1.0 / 24) + M) - (r5 * (1.0 / 120) + M);
    const double approx = fma(r, -65536.0, 4294967296.0) + (even + odd);
    const double scale = softmax_from_bits((uint64_t)(1023u - (uint32_t)softmax_bits(tk)) << 52);  // 2^-k
    const double t = fma(approx, scale, M);
    *kept = diff ? (uint32_t)softmax_bits(t) : 0xffffffffu;
    return t - M;
}
