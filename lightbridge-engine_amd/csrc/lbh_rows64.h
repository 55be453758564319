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

__device__ __forceinline__ double wave_sum(double v) {
    v += dpp_f64<0xB1>(v);    // quad_perm [1, 0, 3, 2]
    v += dpp_f64<0x4E>(v);    // quad_perm [2, 3, 0, 1]
    v += dpp_f64<0x141>(v);   // row_half_mirror
    v += dpp_f64<0x140>(v);   // row_mirror
#pragma unroll
    for (int o = 16; o < 64; o *= 2) v += shfl_xor_f64(v, o);
    return v;
}

// The exponential and the sigmoid to 2^-38.7 of themselves (measured against the
// library's: 2^-38.75 and 2^-38.77 at most).  exp(x) = 2^n 2^f with |f| <= 1/2 (n by a
// 32-bit rounding, which leaves f up to 2^-13 beyond; the product with log2(e) in 64
// bits), 2^f by a polynomial of degree eight through the Chebyshev nodes (off by 2^-38.77
// at most, 2^-38.75 with what f is beyond), the reciprocal by the hardware's estimate and
// one step of third order.  The library's exp and division cost more than twice the
// instructions, and a kernel of gated rows is bound by instructions.  Below g = -708 the sigmoid is 0, as its formula in
// 64 bits is from -745.
struct Exp64 {
    double c[8];
    // The coefficients in scalar registers, where an instruction takes them as they are
    // (as literals each costs two moves a use).
    __device__ __forceinline__ Exp64()
        : c{0x1.63b2d7971923fp-20, 0x1.00c0e4e15189cp-16, 0x1.4308c7183d6a2p-13, 0x1.5d877598350dep-10, 0x1.3b2ab70ad2565p-7, 0x1.c6b08da70cce3p-5, 0x1.ebfbdff82a734p-3, 0x1.62e42fef9cc69p-1} {
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("" : "+s"(c[i]));
    }
    __device__ __forceinline__ double sigmoid(float g) const {
        const float x = __builtin_amdgcn_fmed3f(-g, -708.0f, 708.0f);
        const double s = of((double)x, x);
        return g < -708.0f ? 0.0 : g != g ? (double)g : s;
    }
    __device__ __forceinline__ double sigmoid(double g) const {
        const double x = fmin(fmax(-g, -708.0), 708.0);
        const double s = of(x, (float)x);
        return g < -708.0 ? 0.0 : g != g ? g : s;
    }

    // exp(x), |x| <= 708; x32 is x to 32 bits.
    __device__ __forceinline__ double exp(double x, float x32) const {
        constexpr double LOG2E = 0x1.71547652b82fep+0;
        const float n = __builtin_rintf(x32 * (float)LOG2E);
        const double f = __builtin_fma(x, LOG2E, -(double)n);
        double e = c[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) e = __builtin_fma(e, f, c[i]);
        return __builtin_ldexp(__builtin_fma(e, f, 1.0), (int)n);
    }

private:
    // 1 / (1 + exp(x)), |x| <= 708.
    __device__ __forceinline__ double of(double x, float x32) const {
        const double d = 1.0 + exp(x, x32);
        const double r = __builtin_amdgcn_rcp(d), miss = __builtin_fma(-d, r, 1.0);
        return __builtin_fma(r, __builtin_fma(miss, miss, miss), r);
    }
};

// The larger of a and |b|: one instruction (fmax makes two, the first to quiet a NaN that
// cannot be there).  NaN in b leaves a.
__device__ __forceinline__ double max_abs(double a, double b) {
    asm("v_max_f64 %0, %0, |%1|" : "+v"(a) : "v"(b));
    return a;
}

}  // namespace

}  // namespace lbh
