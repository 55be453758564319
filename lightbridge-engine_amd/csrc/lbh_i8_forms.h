// lbh_i8_forms.h — the kernel forms of the 8-bit integer product (lbh_i8.hip
// has the mathematics and the weights' layout) and their launches, for the
// three translation units that differ in the epilogue alone: the product
// itself (lbh_i8.hip), with a bias and a sigmoid-like activation
// (lbh_i8_act.hip), with a bias and the normal distribution's (lbh_i8_gelu.hip).
#pragma once
#include <math.h>

#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rowtypes.h"

namespace lbh {

namespace {

// What a product's epilogue does beside the scales, the gated pair's SwiGLU and the
// residual: nothing, or bias, activation and the scale in front of the residual.
enum : int { EPI_NONE = 0, EPI_SIGMOID = 1, EPI_NORMAL = 2 };

typedef int i8_v4i __attribute__((ext_vector_type(4)));
typedef int i8_v16i __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void i8_lds;

// Token rows in LDS: 64 (128) bytes of a token are four (eight) pieces, piece c
// stored at c ^ swizzle, so that 16 lanes reading one piece of 16 tokens touch every
// bank.
__device__ __forceinline__ int token_swizzle(int t) { return (t >> 2) & 3; }
__device__ __forceinline__ int pair_swizzle(int t) { return (t >> 1) & 7; }

// ------------------------------------------------------------- the epilogue

// V consecutive elements as words of at most 16 bytes.
template <int OUT, int V>
__device__ __forceinline__ void load_row(const row_t<OUT> *p, float (&v)[V]) {
    constexpr int N = V * (int)sizeof(row_t<OUT>) > 16 ? 16 / (int)sizeof(row_t<OUT>) : V;
#pragma unroll
    for (int i = 0; i < V; i += N) {
        const rvec<row_t<OUT>, N> a = *reinterpret_cast<const rvec<row_t<OUT>, N> *>(p + i);
#pragma unroll
        for (int j = 0; j < N; ++j) v[i + j] = (float)a[j];
    }
}
template <int OUT, int V>
__device__ __forceinline__ void store_row(row_t<OUT> *p, const float (&v)[V]) {
    constexpr int N = V * (int)sizeof(row_t<OUT>) > 16 ? 16 / (int)sizeof(row_t<OUT>) : V;
#pragma unroll
    for (int i = 0; i < V; i += N) {
        rvec<row_t<OUT>, N> a;
#pragma unroll
        for (int j = 0; j < N; ++j) a[j] = (row_t<OUT>)v[i + j];
        *reinterpret_cast<rvec<row_t<OUT>, N> *>(p + i) = a;
    }
}

// The scales of channels c .. c + V - 1 (c % V == 0, V <= 16; channels past the last
// one have the zeros that fill its group, or those of the last group).
template <bool GATED, int V>
struct ChannelScales {
    float g[V], u[GATED ? V : 1];
    __device__ __forceinline__ ChannelScales(const I8Args &p, int c) {
        const int grp = min(c >> 4, (p.rows - 1) >> 4);
        const float *s = p.ws + (GATED ? 32 : 16) * grp + (c & 15);
        load_row<T_F32, V>(s, g);
        if constexpr (GATED) load_row<T_F32, V>(s + 16, u);
    }
};

// Their biases (the caller's, at any address: one at a time), where the epilogue has them.
template <bool GATED, int EPI, int V>
struct ChannelBiases {
    float g[EPI ? V : 1], u[EPI && GATED ? V : 1];
    __device__ __forceinline__ ChannelBiases(const I8Args &p, int c) {
        if constexpr (EPI != EPI_NONE) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                g[j] = p.bias ? p.bias[min(c + j, p.rows - 1)] : 0.0f;
                if constexpr (GATED) u[j] = p.up_bias ? p.up_bias[min(c + j, p.rows - 1)] : 0.0f;
            }
        }
    }
};

// The value as a 32-bit float: without this the compiler folds a product and its
// conversion to 16 bits into one rounding, in some of the forms and not in others.
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}

// 1 / (1 + exp(-g)).  exp(-g) = 2^z with z = -g log2(e) to some 40 bits (hi +
// lo), so the argument's rounding does not grow with |g|; from g = -126 ln 2 = -87.34
// down the reciprocal of 1 + e lies below the least normal float and is 0 (what is right
// is below 2^-119 |u|), so the exponent stays at g = -88, and above g = 104 (1 + e is 1),
// which also keeps infinities out of it; and 1 / d is the reciprocal with one
// Newton step.  The library's exp and division cost twice
// as many instructions, which is what bounds the epilogue.
__device__ __forceinline__ float exp_of(float x) {
    constexpr float LOG2E = 0x1.715476p+0f, LOG2E_LO = 0x1.4ae0cp-26f, LN2 = 0x1.62e43p-1f;
    const float hi = x * LOG2E;
    const float lo = __builtin_fmaf(x, LOG2E_LO, __builtin_fmaf(x, LOG2E, -hi));
    const float e = __builtin_amdgcn_exp2f(hi);
    return __builtin_fmaf(e, lo * LN2, e);
}
__device__ __forceinline__ float reciprocal_step(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
}
__device__ __forceinline__ float sigmoid_of(float g) {
    return reciprocal_step(1.0f + exp_of(__builtin_amdgcn_fmed3f(-g, -104.0f, 88.0f)));
}
__device__ __forceinline__ float swiglu(float g, float u) { return g * sigmoid_of(g) * u; }

// The same for outputs of 16 bits, without the steps that matter to 32: off by some 8 *
// 2^-24 and 2 * 2^-24 |g|, where the output's rounding is 2^-12 or 2^-9.  (With them the
// activations of 2048 x 13312 took 5 us more.)
__device__ __forceinline__ float sigmoid_of_16(float g) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(__builtin_amdgcn_fmed3f(-g, -104.0f, 88.0f) * 0x1.715476p+0f));
}

// x times the normal distribution's function of x.  Its lower tail is exp(-a^2 / 2)
// times a smooth function of a = |x|, here t P(t) with t = 1 / (1 + 0.35 a) and P of degree
// eight, fitted for the least relative error over 0 <= a <= 14 (as written here, in floats,
// 6.0e-8 or 2^-24); a^2 goes into the exponential in two parts (WIDE: an output of 32 bits).  Past a = 13.2 the tail is 0
// (what is right is below 2^-126 there, and up to 2^-122 |x| is given up).
template <bool WIDE>
__device__ __forceinline__ float normal_gate(float x) {
    const float a = fminf(fabsf(x), 14.0f);
    const float d = __builtin_fmaf(0.35f, a, 1.0f);
    const float t = WIDE ? reciprocal_step(d) : __builtin_amdgcn_rcpf(d);
    float p = -0x1.dd86ep-6f;
    constexpr float C[] = {0x1.26daap-3f, -0x1.05d9f4p-2f, 0x1.45fd1ap-3f, -0x1.7aa1a6p-6f, 0x1.b02928p-4f, 0x1.ead5dep-4f, 0x1.1e6fe6p-3f, 0x1.1df1d4p-3f};
#pragma unroll
    for (int i = 0; i < 8; ++i) p = __builtin_fmaf(p, t, C[i]);
    const float s = a * a;
    float e;
    if constexpr (WIDE) {
        e = exp_of(-0.5f * s);
        e = __builtin_fmaf(e, -0.5f * __builtin_fmaf(a, a, -s), e);
    } else {
        e = __builtin_amdgcn_exp2f(s * -0x1.715476p-1f);
    }
    const float tail = p * t * e;
    return x * (x > 0.0f ? 1.0f - tail : tail);
}

// The activation of a product's epilogue (I8Args::act) on V values.
template <int EPI, bool WIDE, int V>
__device__ __forceinline__ void activate(const I8Args &p, float (&v)[V]) {
    if constexpr (EPI == EPI_NORMAL) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = normal_gate<WIDE>(v[j]);
        return;
    }
    if (p.act == ACT_NONE) return;
    if (p.act <= ACT_RELU2) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float pos = v[j] < 0.0f ? 0.0f : v[j];   // a comparison, not fmaxf: NaN stays NaN
            v[j] = p.act == ACT_RELU ? pos : pos * pos;
        }
        return;
    }
    // v / (1 + exp(-z)): z = v, or sqrt(8 / pi) (v + 0.044715 v^3), whose v / 2 (1 + tanh(z / 2)) this is
    const bool tanh = p.act == ACT_GELU_TANH;
    constexpr float C1 = 0x1.988454p+0f, C3 = 0x1.2444f2p-4f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        float z = v[j];
        if (tanh) z *= __builtin_fmaf(v[j] * v[j], C3, C1);
        v[j] *= WIDE ? sigmoid_of(z) : sigmoid_of_16(z);
    }
}

// Channels c .. c + V - 1 of token t from their sums times the token's scale
// (`up`: of the second matrix of a gated pair).  INSIDE: all of them exist, rows
// are aligned to 16 bytes, and the residual's values (if any) are at hand.
template <int OUT, bool GATED, int EPI, bool INSIDE, int V>
__device__ __forceinline__ void finish(const I8Args &p, int t, int c, const float (&sum)[V], const float (&up)[V],
                                       const ChannelScales<GATED, V> &ws, const ChannelBiases<GATED, EPI, V> &bias,
                                       const rvec<row_t<OUT>, V> *residual = nullptr) {
    if (!INSIDE && c >= p.rows) return;
    float v[V];
    if constexpr (EPI != EPI_NONE) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = sum[j] * ws.g[j] + bias.g[j];
        activate<EPI, OUT == T_F32, V>(p, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (GATED) v[j] *= up[j] * ws.u[j] + bias.u[j];
            v[j] = rounded(v[j] * p.scale);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            v[j] = sum[j] * ws.g[j];
            if constexpr (GATED) v[j] = swiglu(v[j], up[j] * ws.u[j]);
            v[j] = rounded(v[j]);
        }
    }
    row_t<OUT> *y = static_cast<row_t<OUT> *>(p.y) + (long long)t * p.y_stride + c;
    if constexpr (INSIDE) {
        if (residual) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = rounded((float)(*residual)[j] + v[j]);
        }
        store_row<OUT, V>(y, v);
        return;
    }
    const row_t<OUT> *res = GATED || !p.residual
                                ? nullptr
                                : static_cast<const row_t<OUT> *>(p.residual) + (long long)t * p.residual_stride + c;
    if (p.vec_out && c + V <= p.rows) {
        if (res) {
            float r[V];
            load_row<OUT, V>(res, r);
#pragma unroll
            for (int j = 0; j < V; ++j) v[j] = rounded(r[j] + v[j]);
        }
        store_row<OUT, V>(y, v);
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (c + j < p.rows) y[j] = (row_t<OUT>)rounded(res ? (float)res[j] + v[j] : v[j]);
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_rsrc(const void *base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)(uint32_t)bytes, 0x00020000);
}

// 16 bytes at a byte offset, zero past the resource's end.  ONCE: non-temporal.
template <bool ONCE>
__device__ __forceinline__ i8_v4i i8_load(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_bit_cast(i8_v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, ONCE ? 2 : 0));
}

// 16 bytes a lane straight to LDS, lane l's at to + 16 l.
__device__ __forceinline__ void i8_copy(__amdgpu_buffer_rsrc_t r, uint8_t *to, uint32_t at, uint32_t uniform) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (i8_lds *)to, 16, at, uniform, 0, 0);
}

// The same with the wait left to the kernel, which counts its copies itself (the
// compiler waits for every copy before a read that might be of its target).
__device__ __forceinline__ i8_v4i i8_words(const void *base, long long bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return i8_v4i{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(a >> 32)),
                  __builtin_amdgcn_readfirstlane((int)(uint32_t)bytes), 0x00020000};
}
__device__ __forceinline__ void i8_copy_asm(const i8_v4i &r, uint32_t to, int plus, uint32_t at, uint32_t uniform) {
    asm volatile("s_add_u32 m0, %0, %1\n\ts_nop 0\n\tbuffer_load_dwordx4 %2, %3, %4 offen lds" ::"s"(to), "i"(plus),
                 "v"(at), "s"(r), "s"(uniform)
                 : "memory", "m0", "scc");
}

// ------------------------------------------------------- few tokens: streaming
//
// A workgroup takes R channel groups (gated: pairs of groups) and 16 * TT tokens
// over all of k; its eight waves take every eighth k tile and their integer sums
// are joined in LDS, so that a matrix of few channels still has every CU at work.
// Weights go straight to operand registers; tokens through LDS: 16 tokens x 64
// bytes read straight into operand registers touch 64 lines an instruction, which
// costs the L1 four times what the bytes do, and copied to LDS in the order of
// memory they touch 16 (64 tokens x 12288 channels x 4096: 25.9 -> 18.0 us).  With R =
// 2 the tokens of 32 channels are copied once: where the weights come from HBM, each
// workgroup's tokens beside them cost as much as a quarter of the weights (16 x 24000:
// 24.4 -> 20.0 us).  Each wave has two buffers of its own, so nobody waits for another
// wave before the join.  Bound: up to some 16 tokens the weights' bytes (one token
// x 12288 x 4096: 9.3 us, 5.4 TB/s), then the L1's (R + TT) KiB a k tile.
constexpr int ST_WAVES = 8;

template <int OUT, bool GATED, int EPI, int TT, int R, bool ONCE>
__global__ void __launch_bounds__(64 * ST_WAVES, 4) k_i8_stream(I8Args p) {
    constexpr int G = GATED ? 2 * R : R;
    __shared__ __align__(1024) uint8_t x0[ST_WAVES][TT * 1024], x1[ST_WAVES][TT * 1024];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int groups = (p.rows + 15) / 16 * (GATED ? 2 : 1), across = (groups + G - 1) / G;
    const int bx = blockIdx.x % across;
    const int t0 = (int)(blockIdx.x / across) * 16 * TT, nt = min(p.n_tokens - t0, 16 * TT);
    const int g0 = bx * G, last = min(groups - g0, G);
    const __amdgpu_buffer_rsrc_t rw = i8_rsrc(p.w + (long long)g0 * p.kt * 1024, (long long)last * p.kt * 1024);
    const __amdgpu_buffer_rsrc_t rx = i8_rsrc(p.x + (long long)t0 * p.x_stride, (long long)(nt - 1) * p.x_stride + p.k);
    uint32_t from[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i)
        from[i] = (uint32_t)min(16 * i + (lane >> 2), nt - 1) * (uint32_t)p.x_stride +
                  16 * ((lane & 3) ^ token_swizzle(lane >> 2));
    const int at = (lane & 15) * 64 + 16 * ((lane >> 4) ^ token_swizzle(lane & 15));
    i8_v4i acc[G][TT] = {}, a0[G], a1[G];
    auto ask = [&](uint8_t *x, i8_v4i (&a)[G], int kt) {
        // past the last tile (or group): out of the resource's range, zero
#pragma unroll
        for (int g = 0; g < G; ++g)
            a[g] = i8_load<ONCE>(rw, lane * 16 + (kt < p.kt ? g * p.kt + kt : G * p.kt) * 1024);
#pragma unroll
        for (int i = 0; i < TT; ++i)
            i8_copy(rx, x + i * 1024, from[i] + kt * 64, 0);
    };
    auto multiply = [&](const uint8_t *x, const i8_v4i (&a)[G]) {
        // everything but the other buffer's loads has arrived
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(G + TT) : "memory");
#pragma unroll
        for (int i = 0; i < TT; ++i) {
            const i8_v4i b = *reinterpret_cast<const i8_v4i *>(x + i * 1024 + at);
#pragma unroll
            for (int g = 0; g < G; ++g) acc[g][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[g], b, acc[g][i], 0, 0, 0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next copy into this buffer sets out
    };
    ask(x0[wid], a0, wid);
    for (int kt = wid; kt < p.kt; kt += 2 * ST_WAVES) {
        ask(x1[wid], a1, kt + ST_WAVES);
        multiply(x0[wid], a0);
        ask(x0[wid], a0, kt + 2 * ST_WAVES);
        multiply(x1[wid], a1);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // no copy is on its way into what follows
    __syncthreads();
    // The join: each wave's sums in its own half of the buffers, G * TT KiB from wave to wave.
    static_assert(G <= 2, "the sums of half the waves fit a buffer");
    auto sums = [&](int w) -> i8_v4i * {
        uint8_t *half = w < ST_WAVES / 2 ? x0[0] : x1[0];
        return reinterpret_cast<i8_v4i *>(half + w % (ST_WAVES / 2) * G * TT * 1024);
    };
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < TT; ++i) sums(wid)[(g * TT + i) * 64 + lane] = acc[g][i];
    __syncthreads();
    for (int j = wid; j < R * TT; j += ST_WAVES) {
        const int r = j / TT, i = j % TT;
        i8_v4i sum = {}, up = {};
#pragma unroll
        for (int w = 0; w < ST_WAVES; ++w) {
            sum += sums(w)[((GATED ? 2 * r : r) * TT + i) * 64 + lane];
            if constexpr (GATED) up += sums(w)[((2 * r + 1) * TT + i) * 64 + lane];
        }
        const int t = 16 * i + (lane & 15), c = (bx * R + r) * 16 + 4 * (lane >> 4);
        const ChannelScales<GATED, 4> ws(p, c);
        const ChannelBiases<GATED, EPI, 4> bias(p, c);
        const float xs = p.xs[t0 + min(t, nt - 1)];
        float u[4], v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)sum[e] * xs, u[e] = (float)up[e] * xs;
        if (t < nt) finish<OUT, GATED, EPI, false, 4>(p, t0 + t, c, v, u, ws, bias);
    }
}

// ------------------------------------------------------ many tokens: tiles
//
// A workgroup of four waves (2 x 2) computes 64 * CW channels x 64 * TW tokens,
// each wave CW x TW products of 32 x 32 with v_mfma_i32_32x32x32_i8.  k runs in
// stages of 64; operands are copied to LDS ahead of their use, with no registers in
// between: weights in their tile order, three stages ahead into a ring of four
// buffers; tokens likewise in rows of 64 bytes, or, in the small tiles, in rows of
// 128 bytes for a pair of stages, two pairs ahead into a ring of three.  (Rows of 64
// ask for every cache line twice, and the requests to L2 are what bounds the small
// tiles: 4096 x 12288 in T22 218 -> 199 us, 256 x 26624 53 -> 43.  The larger tiles
// have less LDS to spare, and start later with the longer rows: 512 x 12288 in T32
// 29.0 -> 30.2 us, T44 44.2 -> 47.1.)
template <int OUT, bool GATED, int EPI, int CW, int TW>
__global__ void __launch_bounds__(256, CW * TW > 8 ? 1 : 2) k_i8_tile(I8Args p) {
    constexpr int CH = 64 * CW, TK = 64 * TW;
    constexpr bool PAIRS = CW * TW <= 4;   // token rows of 128 bytes
    constexpr int W = CH * 64, X = TK * (PAIRS ? 128 : 64);   // a buffer of each ring
    __shared__ __align__(1024) uint8_t lds[4 * W + (PAIRS ? 3 : 4) * X];
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wc = wid & 1, wt = wid >> 1;
    // Tiles of the grid: workgroups go to the eight XCDs in turn, and each XCD
    // takes a contiguous run of tiles.  Within the run: panels of eight token
    // tiles, channel tiles one after the other inside, so that the tiles at work
    // at once share operands both ways.
    const int groups = (p.rows + 15) / 16 * (GATED ? 2 : 1);       // channel groups in memory
    const int n_tt = (p.n_tokens + TK - 1) / TK;
    const int total = gridDim.x, per = (total + 7) / 8;
    const int xcd = blockIdx.x & 7, ix = blockIdx.x >> 3;
    const int whole = total & 7 ? total & 7 : 8;                  // XCDs with `per` tiles, the others one less
    const int tile = xcd < whole ? xcd * per + ix : whole * per + (xcd - whole) * (per - 1) + ix;
    const int n_tc = total / n_tt, panel = tile / (8 * n_tc), width = min(8, n_tt - 8 * panel);
    const int in_panel = tile - panel * 8 * n_tc;
    const int tc = in_panel / width, tt = panel * 8 + in_panel % width;
    const int g0 = tc * (CH / 16), t0 = tt * TK;
    const int nt = min(p.n_tokens - t0, TK);
    const i8_v4i rw = i8_words(p.w + (long long)g0 * p.kt * 1024, (long long)min(groups - g0, CH / 16) * p.kt * 1024);
    const i8_v4i rx = i8_words(p.x + (long long)t0 * p.x_stride, (long long)(nt - 1) * p.x_stride + p.k);

    // The epilogue's layout and scales.
    constexpr int ROW = CW * 32;                                  // floats of a token, four by four at c ^ its mask
    constexpr int MASK = CW % 2 ? 7 : 15;
    constexpr int V = OUT == T_F32 ? 4 : 8;                       // channels of a lane
    constexpr int WIDE = GATED ? CW * 16 : CW * 32;               // channels of the wave
    constexpr int PER = WIDE / V, AT_ONCE = 64 / PER;             // lanes a token, tokens a pass
    const int lc = (lane % PER) * V;
    const int c = (GATED ? g0 / 2 : g0) * 16 + wc * WIDE + lc;
    const ChannelScales<GATED, V> ws(p, c);
    float xs[TW];
#pragma unroll
    for (int n = 0; n < TW; ++n) xs[n] = p.xs[t0 + min((wt * TW + n) * 32 + (lane & 31), nt - 1)];

    // What this wave copies in a stage: CW channel groups of 1 KiB (groups past the
    // last one repeat it), and TW pieces of 16 tokens x 64 bytes, or half of a pair's 2
    // * TW pieces of 8 tokens x 128 (tokens past the last one lie behind the resource's
    // end).
    const uint32_t stride = (uint32_t)p.x_stride;
    constexpr int TP = PAIRS ? 8 : 16;   // tokens of a piece
    uint32_t vb[2];   // even and odd pieces: the swizzles of tokens 8 apart differ
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = PAIRS ? 8 * i + (lane >> 3) : lane >> 2;
        vb[i] = (uint32_t)(wid * TW * 16 + (PAIRS ? lane >> 3 : lane >> 2)) * stride +
                16 * (PAIRS ? (lane & 7) ^ pair_swizzle(t) : (lane & 3) ^ token_swizzle(t));
    }
    const uint32_t w_lds = (uint32_t)(uintptr_t)(i8_lds *)lds + wid * CW * 1024;
    const uint32_t x_lds = (uint32_t)(uintptr_t)(i8_lds *)lds + 4 * W + wid * (16 / TP) * TW * 1024;
    uint32_t row[CW];   // this wave's channel groups
#pragma unroll
    for (int i = 0; i < CW; ++i) row[i] = (uint32_t)(min(wid * CW + i, groups - g0 - 1) * p.kt) * 1024u;
    auto copy_weights = [&](uint32_t buf, int i, uint32_t at) { i8_copy_asm(rw, w_lds + buf, i * 1024, lane * 16, row[i] + at); };
    auto copy_tokens = [&](uint32_t buf, int i, uint32_t at) {
        i8_copy_asm(rx, x_lds + buf, i * 1024, vb[i & 1] + ((uint32_t)(i * TP) * stride + at), 0);
    };

    // Operands of k piece j (32 of a stage's 64): lane l holds channel (token) l %
    // 32 and k 16 (l / 32) .. + 15 of the 32.
    const int l32 = lane & 31, hi = lane >> 5;
    const int a_at = wc * CW * 2048 + (l32 >> 4) * 1024 + hi * 256 + (l32 & 15) * 16;
    const int b_at = 4 * W + (wt * TW * 32 + l32) * (X / TK);
    const int b_piece = hi ^ (PAIRS ? pair_swizzle(l32) : token_swizzle(l32));
    i8_v4i a[2][CW], b[2][TW];
    // Operand i of a piece, in the order in which the products ask for them.
    auto read = [&](int i, int wbuf, int xbuf, int half, int j, i8_v4i (&fa)[CW], i8_v4i (&fb)[TW]) {
        if (i == 0 || i > TW)
            fa[i ? i - TW : 0] = *reinterpret_cast<const i8_v4i *>(lds + wbuf * W + a_at + (i ? i - TW : 0) * 2048 + j * 512);
        else
            fb[i - 1] = *reinterpret_cast<const i8_v4i *>(lds + xbuf * X + b_at + (i - 1) * (X / TK * 32) +
                                                          16 * (b_piece ^ (PAIRS ? 4 * half + 2 * j : 2 * j)));
    };
    i8_v16i acc[CW][TW] = {};
    // The products of one piece, with the reads of the next one and `copies` copies
    // set between them, one of each after a product.
    auto piece = [&](const i8_v4i (&fa)[CW], const i8_v4i (&fb)[TW], auto &&next, int copies, auto &&copy) __attribute__((always_inline)) {
        constexpr int N = CW * TW, READS = (CW + TW + N - 1) / N;
#pragma unroll
        for (int m = 0; m < N; ++m) {
#pragma unroll
            for (int i = m * READS; i < (m + 1) * READS; ++i)
                if (i < CW + TW) next(i);
            acc[m / TW][m % TW] =
                __builtin_amdgcn_mfma_i32_32x32x32_i8(fa[m / TW], fb[m % TW], acc[m / TW][m % TW], 0, 0, 0);
            if (m < copies) copy(m);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // Stage kt, the first or second `half` of its pair, in weight buffer wb and token
    // buffer xb; xn: the next stage's token buffer.  The weights of the third stage from
    // here go to the previous stage's buffer, and to buffer xf the tokens of that stage or
    // half of those of the second pair from here.  The last stages copy the last ones
    // again.
    auto stage = [&](int wb, int xb, int xn, int xf, int kt, int half) __attribute__((always_inline)) {
        const int ahead = min(kt + 3, p.kt - 1), at = PAIRS ? min(kt / 2 + 2, p.kt / 2 - 1) * 128 : ahead * 64;
        piece(a[0], b[0], [&](int i) { read(i, wb, xb, half, 1, a[1], b[1]); }, CW,
              [&](int i) { copy_weights(((wb + 3) & 3) * W, i, ahead * 1024); });
        // This wave's copies for the next stage are done (younger are at least two
        // stages' weights and one's tokens) and its reads of this one; then everybody's.
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * CW + TW) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        piece(a[1], b[1], [&](int i) { read(i, (wb + 1) & 3, xn, 1 - half, 0, a[0], b[0]); }, TW,
              [&](int i) { copy_tokens(xf * X, PAIRS ? half * TW + i : i, at); });
    };
    auto weights = [&](int kt) {
#pragma unroll
        for (int i = 0; i < CW; ++i) copy_weights(kt * W, i, kt * 1024);
    };
    auto tokens = [&](int n) {   // a stage's, or a pair's
#pragma unroll
        for (int i = 0; i < 16 / TP * TW; ++i) copy_tokens(n * X, i, n * (X / TK));
    };
    tokens(0), weights(0);
    if constexpr (PAIRS)
        weights(1), tokens(1), weights(2);
    else
        weights(1), tokens(1), weights(2), tokens(2);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * (CW + TW)) : "memory");   // the first stage's are done
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < CW + TW; ++i) read(i, 0, 0, 0, 0, a[0], b[0]);
    if constexpr (PAIRS) {
        for (int kt = 0, wb = 0, x = 0, xn = 1, xf = 2; kt < p.kt; kt += 2, wb ^= 2) {
            stage(wb, x, x, xf, kt, 0);
            stage(wb + 1, x, xn, xf, kt + 1, 1);
            const int done = x;
            x = xn, xn = xf, xf = done;
        }
    } else {
        for (int kt = 0; kt < p.kt; kt += 4) {   // k tiles are a multiple of four: k is padded to 256
            stage(0, 0, 1, 3, kt, 0);
            stage(1, 1, 2, 0, kt + 1, 1);
            stage(2, 2, 3, 1, kt + 2, 0);
            stage(3, 3, 0, 2, kt + 3, 1);
        }
    }

    // D of a 32 x 32 product: lane l holds token l % 32 and channels 8 q + 4 (l /
    // 32) + 0 .. 3, q < 4.  Each wave scales them by their token and turns 32
    // tokens at a time through its part of the LDS, so that a token's channels are
    // read, scaled and stored in words of 16 bytes, whole lines at a time (stored
    // straight from D, 16 bytes a token and line, the stores took a quarter of the
    // kernel).
    static_assert(32 * ROW * 4 == W, "a wave's part is a buffer of weights");
    const ChannelBiases<GATED, EPI, V> bias(p, c);   // (not before the products, whose registers they would take)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    float *turn = reinterpret_cast<float *>(lds + wid * W);
    const int from = GATED ? (lc >> 4) * 32 + (lc & 15) : lc;     // a gated pair's groups alternate
    auto put = [&](auto inside, auto with_residual) {
        constexpr bool INSIDE = decltype(inside)::value, RES = decltype(with_residual)::value;
        constexpr int PASSES = (32 + AT_ONCE - 1) / AT_ONCE;
#pragma unroll
        for (int n = 0; n < TW; ++n) {
            // The passes' residuals, on their way while the sums are turned.
            rvec<row_t<OUT>, V> res[RES ? PASSES : 1];
            if constexpr (RES) {
#pragma unroll
                for (int k = 0; k < PASSES; ++k) {
                    const int tl = min(k * AT_ONCE + lane / PER, 31);
                    res[k] = *reinterpret_cast<const rvec<row_t<OUT>, V> *>(
                        static_cast<const row_t<OUT> *>(p.residual) +
                        (long long)(t0 + (wt * TW + n) * 32 + tl) * p.residual_stride + c);
                }
            }
#pragma unroll
            for (int i = 0; i < CW; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4 *>(turn + l32 * ROW + 4 * ((8 * i + 2 * q + hi) ^ (l32 & MASK))) =
                        make_float4((float)acc[i][n][4 * q] * xs[n], (float)acc[i][n][4 * q + 1] * xs[n],
                                    (float)acc[i][n][4 * q + 2] * xs[n], (float)acc[i][n][4 * q + 3] * xs[n]);
            wave_sync();
            // With an activation the passes stay a loop: unrolled they outgrow the instruction cache, and
            // the largest tile's sums went to memory for it (2048 x 13312 x 4096: 2380 us).
            constexpr int UNROLL = EPI != EPI_NONE && !RES && CW == 4 ? 1 : PASSES;
#pragma unroll UNROLL
            for (int r = 0; r < 32; r += AT_ONCE) {
                const int tl = r + lane / PER, t = (wt * TW + n) * 32 + tl;
                const int tr = min(tl, 31);
                float g[V], u[V];
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    auto four = [&](int ch, float *to) {
                        const float4 f = *reinterpret_cast<const float4 *>(turn + tr * ROW + 4 * ((ch / 4) ^ (tr & MASK)));
                        to[0] = f.x, to[1] = f.y, to[2] = f.z, to[3] = f.w;
                    };
                    four(from + j, g + j);
                    if constexpr (GATED) four(from + 16 + j, u + j);
                }
                const bool mine = (64 % PER == 0 || lane < PER * AT_ONCE) && (32 % AT_ONCE == 0 || tl < 32);
                if (mine && (INSIDE || t < nt))
                    finish<OUT, GATED, EPI, INSIDE, V>(p, t0 + t, c, g, u, ws, bias, RES ? &res[r / AT_ONCE] : nullptr);
            }
            wave_sync();
            __builtin_amdgcn_sched_barrier(0);   // the next tokens' residuals do not need registers yet
        }
    };
    const bool inside = p.vec_out && nt == TK && (tc + 1) * (GATED ? CH / 2 : CH) <= p.rows;
    if constexpr (!GATED && CW < 4) {
        if (inside && p.residual) {
            put(std::true_type{}, std::true_type{});
            return;
        }
    }
    // (The largest tile has no registers to hold residuals in: it takes them as the ragged tiles do.)
    if (inside && (GATED || !p.residual))
        put(std::true_type{}, std::false_type{});
    else
        put(std::false_type{}, std::false_type{});
}

// The forms and what a call takes in each, in us.  Measured on k = 4096 (64 k tiles),
// time of the whole call as a graph node; estimate() and plan() use them.
struct Form {
    int cw, tw;           // tile: 64 * cw channels x 64 * tw tokens (stream, cw = 0: tw = TT, r = R)
    int r;
    float fixed, step;    // a round of one workgroup per CU: fixed + step * k tiles
};
constexpr Form FORMS[] = {
    {0, 1, 1, 0, 0},       {0, 2, 1, 0, 0},       {0, 2, 2, 0, 0},      {0, 4, 1, 0, 0},    {0, 4, 2, 0, 0},
    {1, 1, 0, 1.5f, 0.12f}, {2, 1, 0, 2.0f, 0.14f}, {2, 2, 0, 2.5f, 0.22f}, {3, 2, 0, 3.5f, 0.32f}, {4, 4, 0, 8.5f, 0.73f},
    {0, 1, 2, 0, 0}};
constexpr int N_FORMS = sizeof(FORMS) / sizeof(FORMS[0]);
static_assert(N_FORMS == I8_FORMS, "the forms a context can ask for");

long long groups_of(const I8Args &a) { return ((long long)a.rows + 15) / 16 * (a.gated ? 2 : 1); }

// Workgroups of a tile form.
long long tiles_of(const I8Args &a, const Form &f) {
    return (groups_of(a) + 4 * f.cw - 1) / (4 * f.cw) * ((a.n_tokens + 64 * f.tw - 1) / (64 * f.tw));
}

// Workgroups of a streaming form of 16 * tt tokens and r channel groups (or pairs).
long long streams_of(const I8Args &a, int tt, int r) {
    return ((long long)a.rows + 16 * r - 1) / (16 * r) * ((a.n_tokens + 16 * tt - 1) / (16 * tt));
}

// A launch counts its threads in 32 bits.
bool fits_a_launch(long long workgroups, int threads) { return workgroups * threads < 1ll << 32; }

template <int OUT, bool GATED, int EPI, int CW, int TW>
hipError_t launch_tile(const I8Args &a, hipStream_t s) {
    const long long grid = tiles_of(a, Form{CW, TW, 0, 0, 0});
    if (!fits_a_launch(grid, 256)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_i8_tile<OUT, GATED, EPI, CW, TW>), dim3((unsigned)grid), dim3(256), 0, s, a);
    return hipGetLastError();
}

// Weights of up to four tokens are read non-temporally from 64 MiB on: four such
// matrices fill the last cache (256 MB), so those of a model come from HBM at every
// step.  From HBM, one token: 2 * 13312 x 4096 21.8 -> 20.3 us, 24000 x 4096 18.8 ->
// 17.2, 8192 x 8192 15.0 -> 13.2; in a loop over one matrix, which stays in the cache,
// 18.9 -> 20.1, 15.7 -> 16.7, 11.8 -> 12.7.  With 16 tokens it gained 6% and lost 17%.
constexpr long long ONCE_BYTES = 64ll << 20;

template <int OUT, bool GATED, int EPI, int TT, int R>
hipError_t launch_stream(const I8Args &a, hipStream_t s) {
    const long long grid = streams_of(a, TT, R);
    if (!fits_a_launch(grid, 64 * ST_WAVES)) return hipErrorInvalidValue;
    if constexpr (TT == 1)
        if (a.n_tokens <= 4 && groups_of(a) * a.kt * 1024 >= ONCE_BYTES) {
            hipLaunchKernelGGL((k_i8_stream<OUT, GATED, EPI, TT, R, true>), dim3((unsigned)grid), dim3(64 * ST_WAVES), 0, s, a);
            return hipGetLastError();
        }
    hipLaunchKernelGGL((k_i8_stream<OUT, GATED, EPI, TT, R, false>), dim3((unsigned)grid), dim3(64 * ST_WAVES), 0, s, a);
    return hipGetLastError();
}

template <int OUT, bool GATED, int EPI>
hipError_t launch_form(const I8Args &a, int form, hipStream_t s) {
    if (form < 0 || form >= N_FORMS) return hipErrorInvalidValue;
    switch (form) {
    case 0: return launch_stream<OUT, GATED, EPI, 1, 1>(a, s);
    case 1: return launch_stream<OUT, GATED, EPI, 2, 1>(a, s);
    case 3: return launch_stream<OUT, GATED, EPI, 4, 1>(a, s);
    case 5: return launch_tile<OUT, GATED, EPI, 1, 1>(a, s);
    case 6: return launch_tile<OUT, GATED, EPI, 2, 1>(a, s);
    case 7: return launch_tile<OUT, GATED, EPI, 2, 2>(a, s);
    case 8: return launch_tile<OUT, GATED, EPI, 3, 2>(a, s);
    case 9: return launch_tile<OUT, GATED, EPI, 4, 4>(a, s);
    }
    if constexpr (!GATED) {
        if (form == 2) return launch_stream<OUT, GATED, EPI, 2, 2>(a, s);
        if (form == 4) return launch_stream<OUT, GATED, EPI, 4, 2>(a, s);
        if (form == 10) return launch_stream<OUT, GATED, EPI, 1, 2>(a, s);
    }
    if (form == 10) return launch_stream<OUT, GATED, EPI, 1, 1>(a, s);
    return launch_form<OUT, GATED, EPI>(a, form - 1, s);   // a forced form of two groups: a pair has them already
}


// A form of the product with the epilogue EPI.
template <int EPI>
hipError_t launch_epilogue(const I8Args &a, int form, hipStream_t s) {
    switch (a.out_type) {
    case T_F32: return a.gated ? launch_form<T_F32, true, EPI>(a, form, s) : launch_form<T_F32, false, EPI>(a, form, s);
    case T_F16: return a.gated ? launch_form<T_F16, true, EPI>(a, form, s) : launch_form<T_F16, false, EPI>(a, form, s);
    case T_BF16:
        return a.gated ? launch_form<T_BF16, true, EPI>(a, form, s) : launch_form<T_BF16, false, EPI>(a, form, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

}  // namespace lbh
