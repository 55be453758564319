// lbh_rows64.h — what the kernels share that compute rows in 64 bits between
// their loads and their roundings (lbh_norm.hip, lbh_block_norm.hip,
// lbh_experts_i8.hip): wave sums, reciprocals, the int8 rounding, words of row
// elements, the sigmoid.
#pragma once
#include "lbh_dev.h"
#include "lbh_rowtypes.h"

namespace lbh {

namespace {

// Sum and maximum over the 64 lanes: within rows of 16 through DPP, then across.
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, ((uint64_t)dpp_row<CTRL>((uint32_t)(b >> 32)) << 32) | dpp_row<CTRL>((uint32_t)b));
}
__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, o), hi = (uint32_t)__shfl_xor((int)(b >> 32), o);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ void wave_sum_max(double &sum, double &top) {
    sum += dpp_f64<0xB1>(sum), top = fmax(top, dpp_f64<0xB1>(top));     // quad_perm [1, 0, 3, 2]
    sum += dpp_f64<0x4E>(sum), top = fmax(top, dpp_f64<0x4E>(top));     // quad_perm [2, 3, 0, 1]
    sum += dpp_f64<0x141>(sum), top = fmax(top, dpp_f64<0x141>(top));   // row_half_mirror
    sum += dpp_f64<0x140>(sum), top = fmax(top, dpp_f64<0x140>(top));   // row_mirror
#pragma unroll
    for (int o = 16; o < 64; o *= 2) sum += shfl_xor_f64(sum, o), top = fmax(top, shfl_xor_f64(top, o));
}

// 1 / sqrt(x) and 1 / x to the last bits or so: the hardware's estimate and two
// Newton steps, a fraction of the library's latency, which a single row waits for.
// x >= 0; what the estimate does not take goes through the library.
__device__ __forceinline__ double rsqrt_f64(double x) {
    if (!(x > 0x1p-900 && x < 0x1p900)) return 1.0 / sqrt(x);
    double r = __builtin_amdgcn_rsq(x);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = __builtin_fma(0.5 * r, __builtin_fma(-x * r, r, 1.0), r);
    return r;
}
__device__ __forceinline__ double reciprocal_of(float x) {   // a normal value
    const double d = (double)x;
    double r = __builtin_amdgcn_rcp(d);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
    return r;
}

// The nearest integer of a * b (ties to even) for |a * b| < 2^31: the sum with
// 1.5 * 2^52 is rounded once and holds the integer in its low word.  (A row's
// largest value gives 127 (1 + 2^-24), which is 127.)
__device__ __forceinline__ int nearest_of_product(double a, double b) {
    return (int)(uint32_t)__builtin_bit_cast(uint64_t, __builtin_fma(a, b, 0x1.8p52));
}

// The nearest integer of x / s, ties to even, of 32-bit x and s with |x / s| <= 127
// (1 + 2^-24), from inv = 1 / s in 64 bits.  The product is off by 2^-45 at most, so a
// quotient that is a tie may land beside it; one that is none is at least 2^-26 away
// from a tie (2 x - (2 i + 1) s is a multiple of x's or s's last bit).  The first sum
// rounds to multiples of 2^-30, which puts the former on the tie and leaves the latter on
// their side; the second one is nearest_of_product's.
__device__ __forceinline__ int nearest_of_quotient(double x, double inv) {
    return (int)(uint32_t)__builtin_bit_cast(uint64_t, __builtin_fma(x, inv, 0x1.8p22) + (0x1.8p52 - 0x1.8p22));
}

// Eight consecutive elements in memory at any address of their type, as words of 16
// bytes (global memory takes a word at any address).
template <int TY>
__device__ __forceinline__ void load8(const row_t<TY> *p, float (&v)[8]) {
    constexpr int N = 16 / (int)sizeof(row_t<TY>);
#pragma unroll
    for (int i = 0; i < 8; i += N) {
        rvec<row_t<TY>, N> a;
        __builtin_memcpy(&a, p + i, sizeof a);
#pragma unroll
        for (int j = 0; j < N; ++j) v[i + j] = (float)a[j];
    }
}
template <int TY>
__device__ __forceinline__ void store8(row_t<TY> *p, const float (&v)[8]) {
    constexpr int N = 16 / (int)sizeof(row_t<TY>);
#pragma unroll
    for (int i = 0; i < 8; i += N) {
        rvec<row_t<TY>, N> a;
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = (row_t<TY>)v[i + j];
        __builtin_memcpy(p + i, &a, sizeof a);
    }
}

// 1 / (1 + exp(-g)) to some 2^-46 of itself: exp(x) = 2^n exp(f), |f| <= ln 2 / 2, by
// the series up to f^11 (what is cut off is below 0.3466^12 / 12! = 2^-47), n ln 2 in two
// parts.  The library's exp and division are exact to the last bit or so at more
// than twice the instructions, which a row of gates would wait for.  Below g = -708
// it is 0, as 1 / (1 + exp(-g)) is soon after.
__device__ __forceinline__ double sigmoid_f64(double g) {
    constexpr double LOG2E = 0x1.71547652b82fep+0, LN2_HI = 0x1.62e42fefa0000p-1, LN2_LO = 0x1.cf79abc9e3b3ap-40;
    const double x = fmin(fmax(-g, -708.0), 708.0);
    const double n = __builtin_rint(x * LOG2E);
    const double f = __builtin_fma(n, -LN2_LO, __builtin_fma(n, -LN2_HI, x));
    double e = 1.0 / 39916800.0;
    constexpr double C[] = {1.0 / 3628800.0, 1.0 / 362880.0, 1.0 / 40320.0, 1.0 / 5040.0, 1.0 / 720.0, 1.0 / 120.0,
                            1.0 / 24.0,      1.0 / 6.0,      0.5,           1.0,          1.0};
#pragma unroll
    for (int i = 0; i < 11; ++i) e = __builtin_fma(e, f, C[i]);
    const double d = 1.0 + __builtin_ldexp(e, (int)n);
    double r = __builtin_amdgcn_rcp(d);
#pragma unroll
    for (int i = 0; i < 2; ++i) r = __builtin_fma(r, __builtin_fma(-d, r, 1.0), r);
    return g < -708.0 ? 0.0 : g != g ? g : r;
}

}  // namespace

}  // namespace lbh
