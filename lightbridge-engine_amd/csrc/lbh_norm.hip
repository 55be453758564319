// lbh_norm.hip — root-mean-square norm of rows with the residual's addition,
// and the 8-bit outputs that the products read.
//
//   h  = hidden + delta           rounded to 32 bits, then to the rows' type (stored)
//   r  = 1 / sqrt(mean(h^2) + eps)
//   v  = h * weight * r
//   y  = v rounded to 32 bits, then to y's type
//   Q8_K of v rounded to 32 bits (quantize_row_q8_k, lbh_dev.h)
//   int8: s = max|v| / 127 rounded to 32 bits, q = v / s to the nearest integer, ties to even
//
// Everything between the loads and the roundings is in 64 bits: the product
// of two 32-bit values is exact there, and the sum's order moves r by some
// 1e-16 only (in 32 bits one 8-bit value in ten thousand falls on the other side
// of a rounding border when the order changes).  What order is left hangs on n
// alone.  The 64-bit rate of a CU equals its 32-bit rate, and the kernel stays
// bound by memory.
//
// max|v| = r * max|h * weight|, so the sum and the maximum come from one pass
// over the row, which stays in registers for the second one.
#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rows64.h"

namespace lbh {

namespace {

// One row by TPR threads, 8 * NV of its products h * weight in each thread's
// registers; longer rows are read a second time beyond those.  VEC: a thread's
// eight elements of a step are consecutive and moved as 16-byte words (n a multiple
// of 8); otherwise they lie TPR apart, one element a lane.  The choice hangs on n
// alone: the order of a row's sum moves r by 1e-16, and with it one float32 value in
// some 10^8 over a rounding border, so operands at other addresses and strides get
// the same form and the same bits.  (6007 x 4096 bf16 with the residual to int8 at odd
// addresses: 42 us in words, 129 in single elements.  Words with a scalar tail, in one form for both,
// put every load behind a branch of its own: 6007 x 4096 bf16 took 52 us instead of
// 38, and 333 x 7167 no less than this.)
template <int TY, int TPR, int NV, bool VEC, bool NORM>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm_rows(NormArgs p) {
    using T = row_t<TY>;
    using Product = std::conditional_t<NORM, double, float>;   // what waits in registers: h itself where there is no weight
    constexpr int RPW = TPR < 256 ? 256 / TPR : 1;   // rows per workgroup
    constexpr int NW = TPR / 64;                     // waves per row
    const int tid = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * RPW + threadIdx.x / TPR;
    const bool live = RPW == 1 || row < p.rows;
    const long long rr = live ? row : 0;
    const int n = p.n;
    const T *hid = static_cast<const T *>(p.hidden) + rr * p.hidden_stride;
    const T *del = p.delta ? static_cast<const T *>(p.delta) + rr * p.delta_stride : nullptr;
    T *ho = p.hidden_out && live ? static_cast<T *>(p.hidden_out) + rr * p.hidden_out_stride : nullptr;
    const float *w = NORM ? p.weight : nullptr;

    const int steps = (n + 8 * TPR - 1) / (8 * TPR);
    auto at = [&](int i, int j) { return VEC ? (i * TPR + tid) * 8 + j : (i * 8 + j) * TPR + tid; };
    // h of step i, what the row holds after the addition, from `src` (+ `add`).
    auto fetch = [&](int i, const T *src, const T *add, float (&h)[8], float (&wv)[8]) {
        if constexpr (VEC) {
            const int e = at(i, 0);
            if (e < n) {
                load8<TY>(src + e, h);
                if (add) {
                    float d[8];
                    load8<TY>(add + e, d);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = (float)(T)__fadd_rn(h[j], d[j]);
                }
                if (w) load8<T_F32>(w + e, wv);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) h[j] = wv[j] = 0.0f;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = at(i, j);
                h[j] = wv[j] = 0.0f;
                if (e < n) {
                    h[j] = (float)src[e];
                    if (add) h[j] = (float)(T)__fadd_rn(h[j], (float)add[e]);
                    if (w) wv[j] = w[e];
                }
            }
        }
        if (!w) {
#pragma unroll
            for (int j = 0; j < 8; ++j) wv[j] = 1.0f;
        }
    };
    // The addition's result is stored as soon as it is there (its own elements are
    // all a thread reads, so an update in place is safe).
    auto keep = [&](int i, const float (&h)[8]) {
        if (!ho) return;
        if constexpr (VEC) {
            if (at(i, 0) < n) store8<TY>(ho + at(i, 0), h);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at(i, j) < n) ho[at(i, j)] = (T)h[j];
        }
    };

    // A weight that is not finite shows in `odd`, an h that is not in the sum (without
    // a norm, in `odd`).
    double ssq = 0.0, top = 0.0;
    float odd = 0.0f;
    auto account = [&](const float (&h)[8], const float (&wv)[8], Product (&hw)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double x = (double)h[j];
            if constexpr (NORM) {
                hw[j] = x * (double)wv[j];
                ssq = __builtin_fma(x, x, ssq);
                odd = __builtin_fmaf(wv[j], 0.0f, odd);
            } else {
                hw[j] = h[j];
                odd = __builtin_fmaf(h[j], 0.0f, odd);
            }
            top = fmax(top, fabs((double)hw[j]));
        }
    };
    Product hw[NV][8];
    {
        float h[NV][8], wv[NV][8];
#pragma unroll
        for (int i = 0; i < NV; ++i) fetch(i, hid, del, h[i], wv[i]);
#pragma unroll
        for (int i = 0; i < NV; ++i) keep(i, h[i]), account(h[i], wv[i], hw[i]);
    }
    for (int i = NV; i < steps; ++i) {
        float h[8], wv[8];
        Product v[8];
        fetch(i, hid, del, h, wv);
        keep(i, h);
        account(h, wv, v);
    }

    // The row's sum and maximum; what is odd makes the sum NaN for the scale's sake.
    wave_sum_max(ssq, top);
    bool any_odd = __ballot(odd != odd) != 0;
    if constexpr (NW > 1) {
        __shared__ double s_sum[NW], s_top[NW];
        __shared__ int s_odd[NW];
        if ((tid & 63) == 0) s_sum[tid >> 6] = ssq, s_top[tid >> 6] = top, s_odd[tid >> 6] = any_odd;
        __syncthreads();
        ssq = 0.0, top = 0.0, any_odd = false;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            ssq += s_sum[i];
            top = fmax(top, s_top[i]);
            any_odd |= s_odd[i] != 0;
        }
    }
    // quantization of the rows as they are (no norm): r = 1
    const double r = NORM ? rsqrt_f64(__builtin_fma(ssq, p.inv_n, p.eps)) : 1.0;

    // The scale, and the factor that takes h * weight to int8: zero for a row
    // whose scale is zero (or below the least normal value, where it would
    // have lost bits) and for one that is not finite, whose scale is NaN.
    double to_q = 0.0;
    if (p.q) {
        const double s = top * r * (1.0 / 127.0);
        float scale = (float)s;
        if (any_odd || !(ssq < __builtin_inf()) || !(scale < __builtin_inff()))
            scale = __builtin_nanf("");
        else if (scale < 0x1p-126f)
            scale = 0.0f;
        else
            to_q = r * reciprocal_of(scale);
        if (tid == 0 && live) p.scale[rr] = scale;
    }
    const bool blank = to_q == 0.0;   // zeros, whatever the row holds
    auto int8_of = [&](Product x) { return NORM ? nearest_of_product(x, to_q) : nearest_of_quotient(x, to_q); };

    auto emit = [&](int i, const Product (&hw)[8]) {
        if constexpr (VEC) {
            const int e = at(i, 0);
            if (e >= n || !live) return;
            if (p.q) {
                uint32_t q[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    q[j >> 2] |= (uint32_t)(int8_of(hw[j]) & 0xff) << (8 * (j & 3));
                const uint2 word = blank ? make_uint2(0, 0) : make_uint2(q[0], q[1]);
                __builtin_memcpy(p.q + rr * p.q_stride + e, &word, sizeof word);
            }
            if (p.y || p.q8k) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (float)((double)hw[j] * r);
                if (p.y && p.y_type == T_F32)
                    store8<T_F32>(static_cast<float *>(p.y) + rr * p.y_stride + e, v);
                else if (p.y && p.y_type == T_F16)
                    store8<T_F16>(static_cast<_Float16 *>(p.y) + rr * p.y_stride + e, v);
                else if (p.y)
                    store8<T_BF16>(static_cast<__bf16 *>(p.y) + rr * p.y_stride + e, v);
                if constexpr (TPR > 64) {
                    extern __shared__ __align__(16) float s_v[];
                    if (p.q8k) {
                        *reinterpret_cast<float4 *>(s_v + e) = make_float4(v[0], v[1], v[2], v[3]);
                        *reinterpret_cast<float4 *>(s_v + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = at(i, j);
                if (e >= n || !live) continue;
                if (p.q) p.q[rr * p.q_stride + e] = (int8_t)(blank ? 0 : int8_of(hw[j]));
                if (p.y || p.q8k) {
                    const float v = (float)((double)hw[j] * r);
                    if (p.y && p.y_type == T_F32)
                        static_cast<float *>(p.y)[rr * p.y_stride + e] = v;
                    else if (p.y && p.y_type == T_F16)
                        static_cast<_Float16 *>(p.y)[rr * p.y_stride + e] = (_Float16)v;
                    else if (p.y)
                        static_cast<__bf16 *>(p.y)[rr * p.y_stride + e] = (__bf16)v;
                    if constexpr (TPR > 64) {
                        extern __shared__ __align__(16) float s_v[];
                        if (p.q8k) s_v[e] = v;
                    }
                }
            }
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) emit(i, hw[i]);
    // The rest of a long row again, from where the sum was stored if it was (hidden
    // may have been overwritten with it).
    for (int i = NV; i < steps; ++i) {
        float h[8], wv[8];
        Product v[8];
        fetch(i, ho ? ho : hid, ho ? nullptr : del, h, wv);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (Product)h[j] * (Product)wv[j];
        emit(i, v);
    }
    if constexpr (TPR > 64) {
        if (p.q8k) {
            extern __shared__ __align__(16) float s_v[];
            __syncthreads();
            const int nb = n / 256;
            for (int b0 = (tid >> 6) * 4; b0 < nb; b0 += NW * 4)
                quantize_blocks_wave(s_v, p.q8k + rr * (long long)nb * 292, b0, nb);
        }
    }
}

template <int TY, bool VEC, bool NORM>
hipError_t launch_norm_form(const NormArgs &a, hipStream_t s) {
    // The products of a row of 512 stay in the registers of 64 threads, of 2048 and
    // 4096 in 256 threads', of 8192 in 512 threads' (1024 threads leave room for one
    // workgroup on a CU: 333 rows of 7168 took two rounds), of 16384 in 1024
    // threads'.  Q8_K blocks go through LDS, which only the workgroup-per-row forms
    // have.  Measured as graph nodes, input and output bytes a second: 6007 x 4096 bf16
    // with the residual to int8 4.3 TB/s, int8 of 1024 x 13312 f32 5.0 TB/s; one row of
    // 4096 to int8 3.6 us and 64 rows to Q8_K 4.8 us, which is latency.
    const size_t lds = a.q8k ? (size_t)a.n * 4 : 0;
    if (a.n <= 512 && !a.q8k)
        hipLaunchKernelGGL((k_norm_rows<TY, 64, 1, VEC, NORM>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
    else if (a.n <= 2048)
        hipLaunchKernelGGL((k_norm_rows<TY, 256, 1, VEC, NORM>), dim3((unsigned)a.rows), dim3(256), lds, s, a);
    else if (a.n <= 4096)
        hipLaunchKernelGGL((k_norm_rows<TY, 256, 2, VEC, NORM>), dim3((unsigned)a.rows), dim3(256), lds, s, a);
    else if (a.n <= 8192)
        hipLaunchKernelGGL((k_norm_rows<TY, 512, 2, VEC, NORM>), dim3((unsigned)a.rows), dim3(512), lds, s, a);
    else
        hipLaunchKernelGGL((k_norm_rows<TY, 1024, 2, VEC, NORM>), dim3((unsigned)a.rows), dim3(1024), lds, s, a);
    return hipGetLastError();
}

template <int TY>
hipError_t launch_norm_typed(const NormArgs &a, bool vec, hipStream_t s) {
    if (a.norm) return vec ? launch_norm_form<TY, true, true>(a, s) : launch_norm_form<TY, false, true>(a, s);
    return vec ? launch_norm_form<TY, true, false>(a, s) : launch_norm_form<TY, false, false>(a, s);
}

}  // namespace

hipError_t launch_norm_rows(const NormArgs &a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    if (a.n < 1 || a.rows > 0x7fffffff) return hipErrorInvalidValue;
    const bool vec = a.n % 8 == 0;
    switch (a.type) {
    case T_F32: return launch_norm_typed<T_F32>(a, vec, s);
    case T_F16: return launch_norm_typed<T_F16>(a, vec, s);
    case T_BF16: return launch_norm_typed<T_BF16>(a, vec, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lbh
