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
// 1e-16 only, so an 8-bit value does not depend on how a row is split over
// lanes (in 32 bits one value in ten thousand falls on the other side of a
// rounding border when the order of the sum changes).  The 64-bit rate of a CU
// equals its 32-bit rate, and the kernel stays bound by memory.
//
// max|v| = r * max|h * weight|, so the sum and the maximum come from one pass
// over the row, which stays in registers for the second one.
#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rowtypes.h"

namespace lbh {

namespace {

// max that keeps a NaN once it has one.
__device__ __forceinline__ double max_nan(double m, double a) { return (a > m || a != a) ? a : m; }

__device__ __forceinline__ double shfl_xor_f64(double v, int o) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)b, o), hi = (uint32_t)__shfl_xor((int)(b >> 32), o);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// The nearest integer of a * b (ties to even) for |a * b| < 2^31: the sum with
// 1.5 * 2^52 is rounded once and holds the integer in its low word.
__device__ __forceinline__ int nearest_of_product(double a, double b) {
    return (int)(uint32_t)__builtin_bit_cast(uint64_t, __builtin_fma(a, b, 0x1.8p52));
}

template <int TY>
__device__ __forceinline__ void load8(const row_t<TY> *p, float (&v)[8]) {
    if constexpr (TY == T_F32) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const rvec<row_t<TY>, 8> a = *reinterpret_cast<const rvec<row_t<TY>, 8> *>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
    }
}
template <int TY>
__device__ __forceinline__ void store8(row_t<TY> *p, const float (&v)[8]) {
    if constexpr (TY == T_F32) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        rvec<row_t<TY>, 8> a;
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = (row_t<TY>)v[j];
        *reinterpret_cast<rvec<row_t<TY>, 8> *>(p) = a;
    }
}

// One row by TPR threads, 8 * NV of its elements in each thread's registers;
// longer rows are read a second time beyond those.  VEC: a thread's eight
// elements of a step are consecutive and moved as 16-byte words (every row of
// every operand aligned for it, n a multiple of 8); otherwise they lie TPR
// apart, one element a lane, at any alignment and length.
template <int TY, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_norm_rows(NormArgs p) {
    using T = row_t<TY>;
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
    const float *w = p.weight;

    const int steps = (n + 8 * TPR - 1) / (8 * TPR);
    auto at = [&](int i, int j) { return VEC ? (i * TPR + tid) * 8 + j : (i * 8 + j) * TPR + tid; };
    // h of step i: what the row holds after the addition
    auto fetch = [&](int i, float (&h)[8], float (&wv)[8]) {
        if constexpr (VEC) {
            const int e = at(i, 0);
            if (e < n) {
                load8<TY>(hid + e, h);
                if (del) {
                    float d[8];
                    load8<TY>(del + e, d);
#pragma unroll
                    for (int j = 0; j < 8; ++j) h[j] = (float)(T)__fadd_rn(h[j], d[j]);
                }
                if (w)
                    load8<T_F32>(w + e, wv);
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
                    h[j] = (float)hid[e];
                    if (del) h[j] = (float)(T)__fadd_rn(h[j], (float)del[e]);
                    if (w) wv[j] = w[e];
                }
            }
        }
        if (!w) {
#pragma unroll
            for (int j = 0; j < 8; ++j) wv[j] = 1.0f;
        }
    };

    float h[NV][8], wv[NV][8];
    double ssq = 0.0, top = 0.0;
    auto account = [&](const float (&a)[8], const float (&b)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double x = (double)a[j];
            ssq = __builtin_fma(x, x, ssq);
            top = max_nan(top, fabs(x * (double)b[j]));
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) fetch(i, h[i], wv[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) account(h[i], wv[i]);
    for (int i = NV; i < steps; ++i) {
        float a[8], b[8];
        fetch(i, a, b);
        account(a, b);
    }

    // The row's sum and maximum.
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        ssq += shfl_xor_f64(ssq, o);
        top = max_nan(top, shfl_xor_f64(top, o));
    }
    if constexpr (NW > 1) {
        __shared__ double s_sum[NW], s_top[NW];
        if ((tid & 63) == 0) s_sum[tid >> 6] = ssq, s_top[tid >> 6] = top;
        __syncthreads();
        ssq = 0.0, top = 0.0;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            ssq += s_sum[i];
            top = max_nan(top, s_top[i]);
        }
    }
    // quantization of the rows as they are (no norm): r = 1
    const double r = p.norm ? 1.0 / sqrt(ssq / (double)n + p.eps) : 1.0;

    // The scale, and the factor that takes h * weight to int8: zero for a row
    // whose scale is zero (or below the least normal value, where it would
    // have lost bits) and for one that is not finite, whose scale is NaN.
    float scale = 0.0f;
    double to_q = 0.0;
    if (p.q) {
        const double s = top * r / 127.0;
        scale = (float)s;
        if (!(ssq < __builtin_inf()) || !(s < 0x1.fffffep127))
            scale = __builtin_nanf("");
        else if (scale < 0x1p-126f)
            scale = 0.0f;
        else
            to_q = r / (double)scale;
        if (tid == 0 && live) p.scale[rr] = scale;
    }
    const bool bad = scale != scale;

    auto emit = [&](int i, const float (&a)[8], const float (&b)[8]) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)((double)a[j] * (double)b[j] * r);
        if constexpr (VEC) {
            const int e = at(i, 0);
            if (e >= n || !live) return;
            if (ho) store8<TY>(ho + e, a);
            if (p.q) {
                uint32_t q[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    q[j >> 2] |= (uint32_t)(uint8_t)(bad ? 0 : nearest_of_product((double)a[j] * (double)b[j], to_q))
                                 << (8 * (j & 3));
                *reinterpret_cast<uint2 *>(p.q + rr * p.q_stride + e) = make_uint2(q[0], q[1]);
            }
            if (p.y) {
                if (p.y_type == T_F32)
                    store8<T_F32>(static_cast<float *>(p.y) + rr * p.y_stride + e, v);
                else if (p.y_type == T_F16)
                    store8<T_F16>(static_cast<_Float16 *>(p.y) + rr * p.y_stride + e, v);
                else
                    store8<T_BF16>(static_cast<__bf16 *>(p.y) + rr * p.y_stride + e, v);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = at(i, j);
                if (e >= n || !live) continue;
                if (ho) ho[e] = (T)a[j];
                if (p.q)
                    p.q[rr * p.q_stride + e] =
                        (int8_t)(bad ? 0 : nearest_of_product((double)a[j] * (double)b[j], to_q));
                if (p.y) {
                    if (p.y_type == T_F32)
                        static_cast<float *>(p.y)[rr * p.y_stride + e] = v[j];
                    else if (p.y_type == T_F16)
                        static_cast<_Float16 *>(p.y)[rr * p.y_stride + e] = (_Float16)v[j];
                    else
                        static_cast<__bf16 *>(p.y)[rr * p.y_stride + e] = (__bf16)v[j];
                }
            }
        }
        if constexpr (TPR > 64) {
            if (p.q8k) {
                extern __shared__ float s_v[];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (at(i, j) < n) s_v[at(i, j)] = v[j];
            }
        }
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) emit(i, h[i], wv[i]);
    // the rest of a long row again, before this thread's own stores can change it
    for (int i = NV; i < steps; ++i) {
        float a[8], b[8];
        fetch(i, a, b);
        emit(i, a, b);
    }
    if constexpr (TPR > 64) {
        if (p.q8k) {
            extern __shared__ float s_v[];
            __syncthreads();
            const int nb = n / 256;
            for (int b0 = (tid >> 6) * 4; b0 < nb; b0 += NW * 4)
                quantize_blocks_wave(s_v, p.q8k + rr * (long long)nb * 292, b0, nb);
        }
    }
}

template <int TY, bool VEC>
hipError_t launch_norm_typed(const NormArgs &a, hipStream_t s) {
    // 64 threads hold a row of 512, 256 threads one of 4096 (4096 bf16 rows of
    // 4096: see k_norm_rows' figures), 1024 threads one of 16384.  Q8_K blocks
    // go through LDS, which only the workgroup-per-row forms have.
    if (a.n <= 512 && !a.q8k) {
        hipLaunchKernelGGL((k_norm_rows<TY, 64, 1, VEC>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
    } else {
        const size_t lds = a.q8k ? (size_t)a.n * 4 : 0;
        if (a.n <= 4096)
            hipLaunchKernelGGL((k_norm_rows<TY, 256, 2, VEC>), dim3((unsigned)a.rows), dim3(256), lds, s, a);
        else
            hipLaunchKernelGGL((k_norm_rows<TY, 1024, 2, VEC>), dim3((unsigned)a.rows), dim3(1024), lds, s, a);
    }
    return hipGetLastError();
}

bool aligned_rows(const void *p, long long stride, int elem, int bytes) {
    return !p || ((reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (stride * elem) % bytes == 0);
}

}  // namespace

hipError_t launch_norm_rows(const NormArgs &a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    if (a.n < 1 || a.rows > 0x7fffffff) return hipErrorInvalidValue;
    const int e = row_elem_bytes(a.type);
    const bool vec = a.n % 8 == 0 && aligned_rows(a.hidden, a.hidden_stride, e, 16) &&
                     aligned_rows(a.delta, a.delta_stride, e, 16) &&
                     aligned_rows(a.hidden_out, a.hidden_out_stride, e, 16) && aligned_rows(a.weight, 0, 4, 16) &&
                     aligned_rows(a.y, a.y_stride, row_elem_bytes(a.y_type), 16) && aligned_rows(a.q, a.q_stride, 1, 8);
    switch (a.type) {
    case T_F32: return vec ? launch_norm_typed<T_F32, true>(a, s) : launch_norm_typed<T_F32, false>(a, s);
    case T_F16: return vec ? launch_norm_typed<T_F16, true>(a, s) : launch_norm_typed<T_F16, false>(a, s);
    case T_BF16: return vec ? launch_norm_typed<T_BF16, true>(a, s) : launch_norm_typed<T_BF16, false>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lbh
