// lbh_block_norm.hip — a block's output back into the residual stream and the
// norm in front of the next block, in one pass over the rows.
//
//   p = block * post_weight / sqrt(mean(block^2) + post_eps)    (no post_weight: block)
//   p = p * a(gate)                                    a: as it is, sigmoid, silu
//   h = hidden + scale * p        rounded to 32 bits, then to the rows' type (stored)
//   v = h * weight / sqrt(mean(h^2) + eps)
//   y, Q8_K blocks, int8 rows of v as lbh_norm.hip makes them
//
// Bound by memory: each operand is read once and stays in registers across
// both reductions, and the row's two barriers are the latency of a single row.
// Two norm launches in its place read the sum again and store the normed block
// between them.  Everything between the loads and the roundings is in 64 bits,
// for the reasons lbh_norm.hip gives; the order of the sums hangs on n alone.
#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rows64.h"

namespace lbh {

namespace {

// The block-wide sum, and the second reduction's sum, maximum and oddness.
template <int NW>
struct RowScratch {
    double first[NW], sum[NW], top[NW];
    int odd[NW];
};

// One row by TPR threads, 8 * NV elements of each operand in a thread's registers
// (n <= 8 * NV * TPR).  VEC: a thread's eight elements of a step are consecutive (n a
// multiple of 8); otherwise they lie TPR apart.
template <int TY, int TPR, int NV, bool VEC>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_block_norm(BlockNormArgs p) {
    using T = row_t<TY>;
    constexpr int RPW = TPR < 256 ? 256 / TPR : 1;   // rows per workgroup
    constexpr int NW = TPR / 64;                     // waves per row
    const int tid = threadIdx.x % TPR;
    const long long row = (long long)blockIdx.x * RPW + threadIdx.x / TPR;
    const bool live = RPW == 1 || row < p.rows;
    const long long rr = live ? row : 0;
    const int n = p.n;
    const T *blk = static_cast<const T *>(p.block) + rr * p.block_stride;
    const T *hid = static_cast<const T *>(p.hidden) + rr * p.hidden_stride;
    const T *gat = p.gate ? static_cast<const T *>(p.gate) + rr * p.gate_stride : nullptr;
    T *ho = static_cast<T *>(p.hidden_out) + rr * p.hidden_out_stride;

    auto at = [&](int i, int j) { return VEC ? (i * TPR + tid) * 8 + j : (i * 8 + j) * TPR + tid; };
    // Elements of step i of a row, zeros (or `fill`) behind its end.
    auto take = [&](auto ty, const auto *src, int i, float (&v)[8], float fill) {
        if constexpr (VEC) {
            if (at(i, 0) < n) {
                load8<decltype(ty)::value>(src + at(i, 0), v);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = fill;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = at(i, j) < n ? (float)src[at(i, j)] : fill;
        }
    };
    using Row = std::integral_constant<int, TY>;
    using F32 = std::integral_constant<int, T_F32>;
    float o[NV][8], h[NV][8], g[NV][8], w1[NV][8], w2[NV][8];
#pragma unroll
    for (int i = 0; i < NV; ++i) take(Row{}, blk, i, o[i], 0.0f);
    if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i) take(F32{}, p.post_weight, i, w1[i], 0.0f);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) take(Row{}, hid, i, h[i], 0.0f);
    if (gat) {
#pragma unroll
        for (int i = 0; i < NV; ++i) take(Row{}, gat, i, g[i], 0.0f);
    }
    if (p.weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i) take(F32{}, p.weight, i, w2[i], 0.0f);
    }

    __shared__ RowScratch<NW> s_row[RPW];
    RowScratch<NW> &sc = s_row[RPW == 1 ? 0 : threadIdx.x / TPR];
    double r1 = 1.0;
    if (p.post_weight) {
        double ssq = 0.0, none = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) ssq = __builtin_fma((double)o[i][j], (double)o[i][j], ssq);
        wave_sum_max(ssq, none);
        if constexpr (NW > 1) {
            if ((tid & 63) == 0) sc.first[tid >> 6] = ssq;
            __syncthreads();
            ssq = 0.0;
#pragma unroll
            for (int i = 0; i < NW; ++i) ssq += sc.first[i];
        }
        r1 = rsqrt_f64(__builtin_fma(ssq, p.inv_n, p.post_eps));
    }

    // The stream after the block, and the products of the next norm.
    double hw[NV][8], ssq = 0.0, top = 0.0;
    float odd = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            double v = (double)o[i][j];
            if (p.post_weight) v = v * r1 * (double)w1[i][j];
            if (gat) {
                const double x = (double)g[i][j];
                double a = x;
                if (p.gate_act) {
                    a = sigmoid_f64(x);
                    if (p.gate_act == GATE_SILU) a *= x;
                }
                v *= a;
            }
            const float sum = (float)__builtin_fma(p.scale, v, (double)h[i][j]);
            h[i][j] = (float)(T)sum;
        }
        if (!live) continue;
        if constexpr (VEC) {
            if (at(i, 0) < n) store8<TY>(ho + at(i, 0), h[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (at(i, j) < n) ho[at(i, j)] = (T)h[i][j];
        }
    }
    if (!p.weight) return;   // the same for every thread
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double x = VEC ? (double)h[i][j] : at(i, j) < n ? (double)h[i][j] : 0.0;
            hw[i][j] = x * (double)w2[i][j];
            ssq = __builtin_fma(x, x, ssq);
            odd = __builtin_fmaf(w2[i][j], 0.0f, odd);
            top = fmax(top, fabs(hw[i][j]));
        }
    }
    wave_sum_max(ssq, top);
    bool any_odd = __ballot(odd != odd) != 0;
    if constexpr (NW > 1) {
        if ((tid & 63) == 0) sc.sum[tid >> 6] = ssq, sc.top[tid >> 6] = top, sc.odd[tid >> 6] = any_odd;
        __syncthreads();
        ssq = 0.0, top = 0.0, any_odd = false;
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            ssq += sc.sum[i];
            top = fmax(top, sc.top[i]);
            any_odd |= sc.odd[i] != 0;
        }
    }
    const double r = rsqrt_f64(__builtin_fma(ssq, p.inv_n, p.eps));
    double to_q = 0.0;   // zero: a row of zeros, or one that is not finite
    if (p.q) {
        const double s = top * r * (1.0 / 127.0);
        float scale = (float)s;
        if (any_odd || !(ssq < __builtin_inf()) || !(scale < __builtin_inff()))
            scale = __builtin_nanf("");
        else if (scale < 0x1p-126f)
            scale = 0.0f;
        else
            to_q = r * reciprocal_of(scale);
        if (tid == 0 && live) p.scales[rr] = scale;
    }
    const bool blank = to_q == 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        extern __shared__ __align__(16) float s_v[];
        if (!live) continue;
        if constexpr (VEC) {
            const int e = at(i, 0);
            if (e >= n) continue;
            if (p.q) {
                uint32_t q[2] = {0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j >> 2] |= (uint32_t)(nearest_of_product(hw[i][j], to_q) & 0xff) << (8 * (j & 3));
                const uint2 word = blank ? make_uint2(0, 0) : make_uint2(q[0], q[1]);
                __builtin_memcpy(p.q + rr * p.q_stride + e, &word, sizeof word);
            }
            if (p.y || p.q8k) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = (float)(hw[i][j] * r);
                if (p.y && p.y_type == T_F32)
                    store8<T_F32>(static_cast<float *>(p.y) + rr * p.y_stride + e, v);
                else if (p.y && p.y_type == T_F16)
                    store8<T_F16>(static_cast<_Float16 *>(p.y) + rr * p.y_stride + e, v);
                else if (p.y)
                    store8<T_BF16>(static_cast<__bf16 *>(p.y) + rr * p.y_stride + e, v);
                if (TPR > 64 && p.q8k) {
                    *reinterpret_cast<float4 *>(s_v + e) = make_float4(v[0], v[1], v[2], v[3]);
                    *reinterpret_cast<float4 *>(s_v + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int e = at(i, j);
                if (e >= n) continue;
                if (p.q) p.q[rr * p.q_stride + e] = (int8_t)(blank ? 0 : nearest_of_product(hw[i][j], to_q));
                if (p.y) {
                    const float v = (float)(hw[i][j] * r);
                    if (p.y_type == T_F32)
                        static_cast<float *>(p.y)[rr * p.y_stride + e] = v;
                    else if (p.y_type == T_F16)
                        static_cast<_Float16 *>(p.y)[rr * p.y_stride + e] = (_Float16)v;
                    else
                        static_cast<__bf16 *>(p.y)[rr * p.y_stride + e] = (__bf16)v;
                }
            }
        }
    }
    if constexpr (VEC && TPR > 64) {   // Q8_K rows are multiples of 256
        if (p.q8k) {
            extern __shared__ __align__(16) float s_v[];
            __syncthreads();
            const int nb = n / 256;
            for (int b0 = (tid >> 6) * 4; b0 < nb; b0 += NW * 4)
                quantize_blocks_wave(s_v, p.q8k + rr * (long long)nb * 292, b0, nb);
        }
    }
}

template <int TY, bool VEC>
hipError_t launch_form(const BlockNormArgs &a, hipStream_t s) {
    // Forms by the row's length, as the norm's.
    const size_t lds = a.q8k ? (size_t)a.n * 4 : 0;
    if (a.n <= 512 && !a.q8k)
        hipLaunchKernelGGL((k_block_norm<TY, 64, 1, VEC>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, s, a);
    else if (a.n <= 2048)
        hipLaunchKernelGGL((k_block_norm<TY, 256, 1, VEC>), dim3((unsigned)a.rows), dim3(256), lds, s, a);
    else if (a.n <= 4096)
        hipLaunchKernelGGL((k_block_norm<TY, 256, 2, VEC>), dim3((unsigned)a.rows), dim3(256), lds, s, a);
    else if (a.n <= 8192)
        hipLaunchKernelGGL((k_block_norm<TY, 512, 2, VEC>), dim3((unsigned)a.rows), dim3(512), lds, s, a);
    else
        hipLaunchKernelGGL((k_block_norm<TY, 1024, 2, VEC>), dim3((unsigned)a.rows), dim3(1024), lds, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs &a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    if (a.n < 1 || a.n > BLOCK_NORM_MAX || a.rows > 0x7fffffff) return hipErrorInvalidValue;
    const bool vec = a.n % 8 == 0;
    switch (a.type) {
    case T_F32: return vec ? launch_form<T_F32, true>(a, s) : launch_form<T_F32, false>(a, s);
    case T_F16: return vec ? launch_form<T_F16, true>(a, s) : launch_form<T_F16, false>(a, s);
    case T_BF16: return vec ? launch_form<T_BF16, true>(a, s) : launch_form<T_BF16, false>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lbh
