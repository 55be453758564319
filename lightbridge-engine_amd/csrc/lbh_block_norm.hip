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
// 4096 x 4096 bf16 to int8 rows: 28.6 us without a gate (4.1 TB/s), 46 through a sigmoid or
// silu, whose 64-bit exponentials bind it then (70 vector instructions for 64 elements); float32
// rows with the norm behind the block 44.7 us (4.9 TB/s); a single row 3.7 us.
#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rows64.h"

namespace lbh {

namespace {

enum : int { NO_GATE, AS_IS, ACTIVATED };

// Eight consecutive elements of a row as they are in memory.
template <int TY>
using raw8 = rvec<row_t<TY>, 8>;

// One row by TPR threads, 8 * NV elements of each operand in a thread's registers
// (n <= 8 * NV * TPR), 16-bit ones packed as they came until they are used.  A thread's
// eight elements of a step are consecutive and moved as words of 16 bytes at any
// address.  Where they reach past the row's end, the words are the row's last eight
// elements, shifted into place once everything is on its way: no load waits behind a
// branch (elements one by one, TPR apart, took twice as long: 333 x 4095 fp16 with
// gates 17.2 us).
// GATE: no gate, one as it is, one through an activation.
template <int TY, int TPR, int NV, int GATE>
__global__ void __launch_bounds__(TPR < 256 ? 256 : TPR) k_block_norm(BlockNormArgs p) {
    using T = row_t<TY>;
    constexpr int RPW = TPR < 256 ? 256 / TPR : 1;   // rows per workgroup
    constexpr int NW = TPR / 64;                     // waves per row
    const int tid = threadIdx.x % TPR;
    const int n = p.n;

    auto at = [&](int i) { return (i * TPR + tid) * 8; };
    auto take = [&](const auto *src, int i, auto &v) {
        if (n >= 8) {
            __builtin_memcpy(&v, src + min(at(i), n - 8), sizeof v);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = at(i) + j < n ? src[at(i) + j] : 0;
        }
    };
    // The words of a step that reaches past the end: shifted, zeros behind it.
    auto settle = [&](int i, auto &v) {
        const int over = at(i) + 8 - n;
        if (over <= 0 || n < 8) return;
#pragma unroll
        for (int s = 4; s; s /= 2)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (over & s) v[j] = v[j + s < 8 ? j + s : 7];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j + over >= 8) v[j] = 0;
    };
    const long long row = (long long)blockIdx.x * RPW + (RPW == 1 ? 0 : threadIdx.x / TPR);
    if (RPW > 1 && row >= p.rows) return;   // a wave with a row of its own, without a barrier
    const T *blk = static_cast<const T *>(p.block) + row * p.block_stride;
    const T *hid = static_cast<const T *>(p.hidden) + row * p.hidden_stride;
    T *ho = static_cast<T *>(p.hidden_out) + row * p.hidden_out_stride;
    raw8<TY> o[NV], x[NV], g[NV];
    raw8<T_F32> w1[NV], w2[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) take(blk, i, o[i]);
    if (p.post_weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i) take(p.post_weight, i, w1[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) w1[i] = 1.0f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) take(hid, i, x[i]);
    if constexpr (GATE != NO_GATE) {
        const T *gat = static_cast<const T *>(p.gate) + row * p.gate_stride;
#pragma unroll
        for (int i = 0; i < NV; ++i) take(gat, i, g[i]);
    }
    if (p.weight) {
#pragma unroll
        for (int i = 0; i < NV; ++i) take(p.weight, i, w2[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) w2[i] = 1.0f;
    }
    __shared__ double s_first[NW], s_sum[NW], s_top[NW];
    __shared__ int s_odd[NW];
    extern __shared__ __align__(16) float s_v[];

#pragma unroll
    for (int i = 0; i < NV; ++i) settle(i, o[i]);
    double r1 = p.scale;
    if (p.post_weight) {
        double ssq = 0.0;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) ssq = __builtin_fma((double)(float)o[i][j], (double)(float)o[i][j], ssq);
        ssq = wave_sum(ssq);
        if constexpr (NW > 1) {
            if ((tid & 63) == 0) s_first[tid >> 6] = ssq;
            __syncthreads();
            ssq = 0.0;
#pragma unroll
            for (int i = 0; i < NW; ++i) ssq += s_first[i];
        }
        r1 *= rsqrt_f64(__builtin_fma(ssq, p.inv_n, p.post_eps));
    }

    // The stream after the block, and the next norm's sums.
    double ssq = 0.0, top = 0.0;
    float odd = 0.0f;
    const Exp64 ex;
    const bool silu = p.gate_act == GATE_SILU;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        settle(i, x[i]);
        settle(i, w1[i]);
        settle(i, w2[i]);
        if constexpr (GATE != NO_GATE) settle(i, g[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            double v = (double)(float)o[i][j] * (double)w1[i][j];   // exact
            if constexpr (GATE == AS_IS) v *= (double)(float)g[i][j];
            if constexpr (GATE == ACTIVATED) {
                const float z = (float)g[i][j];
                v *= ex.sigmoid(z) * (double)(silu ? z : 1.0f);
            }
            x[i][j] = (T)(float)__builtin_fma(v, r1, (double)(float)x[i][j]);
            const double h = (double)(float)x[i][j];
            ssq = __builtin_fma(h, h, ssq);
            top = max_abs(top, h * (double)w2[i][j]);
            odd = __builtin_fmaf(w2[i][j], 0.0f, odd);
        }
        const int e = at(i), over = e + 8 - n;
        if (e >= n) continue;
        if (over <= 0) {
            __builtin_memcpy(ho + e, &x[i], sizeof x[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j + over < 8) ho[e + j] = x[i][j];
        }
    }
    if (!p.weight) return;   // the same for every thread
    wave_sum_max(ssq, top);
    bool any_odd = __ballot(odd != odd) != 0;
    if constexpr (NW > 1) {
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
        if (tid == 0) p.scales[row] = scale;
    }
    const bool blank = to_q == 0.0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int e = at(i), over = e + 8 - n;
        if (e >= n) continue;
        double hw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) hw[j] = (double)(float)x[i][j] * (double)w2[i][j];
        if (p.q) {
            uint32_t q[2] = {0, 0};
#pragma unroll
            for (int j = 0; j < 8; ++j) q[j >> 2] |= (uint32_t)(nearest_of_product(hw[j], to_q) & 0xff) << (8 * (j & 3));
            const uint2 word = blank ? make_uint2(0, 0) : make_uint2(q[0], q[1]);
            int8_t *to = p.q + row * p.q_stride + e;
            if (over <= 0) {
                __builtin_memcpy(to, &word, sizeof word);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j + over < 8) to[j] = (int8_t)((j < 4 ? word.x : word.y) >> (8 * (j & 3)));
            }
        }
        if (p.y || p.q8k) {
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = (float)(hw[j] * r);
            auto put = [&](auto ty) {
                using Y = row_t<decltype(ty)::value>;
                Y *to = static_cast<Y *>(p.y) + row * p.y_stride + e;
                if (over <= 0) {
                    store8<decltype(ty)::value>(to, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (j + over < 8) to[j] = (Y)v[j];
                }
            };
            if (p.y && p.y_type == T_F32)
                put(std::integral_constant<int, T_F32>());
            else if (p.y && p.y_type == T_F16)
                put(std::integral_constant<int, T_F16>());
            else if (p.y)
                put(std::integral_constant<int, T_BF16>());
            if (TPR > 64 && p.q8k) {   // n is a multiple of 256
                *reinterpret_cast<float4 *>(s_v + e) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(s_v + e + 4) = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }
    if constexpr (TPR > 64) {
        if (p.q8k) {
            __syncthreads();
            const int nb = n / 256;
            for (int b0 = (tid >> 6) * 4; b0 < nb; b0 += NW * 4)
                quantize_blocks_wave(s_v, p.q8k + row * (long long)nb * 292, b0, nb);
        }
    }
}

template <int TY, int GATE, int TPR, int NV>
hipError_t launch_rows(const BlockNormArgs &a, hipStream_t s) {
    constexpr int RPW = TPR < 256 ? 256 / TPR : 1;
    hipLaunchKernelGGL((k_block_norm<TY, TPR, NV, GATE>), dim3((unsigned)((a.rows + RPW - 1) / RPW)), dim3(TPR * RPW),
                       a.q8k ? (size_t)a.n * 4 : 0, s, a);
    return hipGetLastError();
}

// Two steps a thread keep more of a row's loads in flight than one step of twice as many
// threads (4096 x 4096 bf16: 27.6 against 32.4 us).  Workgroups that went through rows
// with the next row on its way and the weights kept had half the waves in the
// registers that took, and were slower (32.0; with gates 52 against 46).
template <int TY, int GATE>
hipError_t launch_form(const BlockNormArgs &a, hipStream_t s) {
    if (a.n <= 512 && !a.q8k) return launch_rows<TY, GATE, 64, 1>(a, s);
    if (a.n <= 2048) return launch_rows<TY, GATE, 256, 1>(a, s);
    if (a.n <= 4096) return launch_rows<TY, GATE, 256, 2>(a, s);
    if (a.n <= 8192) return launch_rows<TY, GATE, 512, 2>(a, s);
    return launch_rows<TY, GATE, 1024, 2>(a, s);
}

template <int TY>
hipError_t launch_gate(const BlockNormArgs &a, hipStream_t s) {
    if (!a.gate) return launch_form<TY, NO_GATE>(a, s);
    return a.gate_act == GATE_AS_IS ? launch_form<TY, AS_IS>(a, s) : launch_form<TY, ACTIVATED>(a, s);
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs &a, hipStream_t s) {
    if (a.rows <= 0) return hipSuccess;
    if (a.n < 1 || a.n > BLOCK_NORM_MAX || a.rows > 0x7fffffff) return hipErrorInvalidValue;
    switch (a.type) {
    case T_F32: return launch_gate<T_F32>(a, s);
    case T_F16: return launch_gate<T_F16>(a, s);
    case T_BF16: return launch_gate<T_BF16>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lbh
