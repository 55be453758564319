// lbh_i8.hip — matrix product in 8-bit integers with a scale for each token
// and each channel, plain (with the residual's addition) and gated (SwiGLU of
// two products), and the layout of its weights.
//
//   y[t][c] = residual[t][c] + float(sum_i q[t][i] w[c][i]) * xs[t] * ws[c]
//   h[t][c] = g / (1 + exp(-g)) * u,   g, u: the gate's and the up's products
//
// The integer sums are exact (k * 128 * 128 < 2^31), so neither the split of k
// over waves nor the order of the joins changes a bit of the result.
//
// Weights are kept as tiles of 16 channels x 64 k, 1 KiB each in the order of
// v_mfma_i32_16x16x64_i8's operand (lane l: channel l % 16, k 16 (l / 16) ..
// + 15): a wave's 16 bytes a lane are one contiguous KiB.  Tiles of one
// channel group follow each other along k; a gated pair's gate and up groups
// alternate, so both products of a channel end in the same lane.  Channels and
// k are padded with zeros (k to 256), so what the rows hold behind k never
// counts.
#include <math.h>

#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rowtypes.h"

namespace lbh {

namespace {

typedef int i8_v4i __attribute__((ext_vector_type(4)));
typedef int i8_v16i __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) void i8_lds;

// Token rows in LDS: 64 (128) bytes of a token are four (eight) pieces, piece c
// stored at c ^ swizzle, so that 16 lanes reading one piece of 16 tokens touch every
// bank.
__device__ __forceinline__ int token_swizzle(int t) { return (t >> 2) & 3; }
__device__ __forceinline__ int pair_swizzle(int t) { return (t >> 1) & 7; }

// ------------------------------------------------------------- weight layout

struct I8LayoutArgs {
    int8_t *rowmajor;      // [rows][k]
    uint8_t *tiles;
    float *scales;         // row-major side: [rows]
    float *tile_scales;    // [groups * 16]
    long long rows, k;
    long long kt;          // k tiles of 64
    int step, part;        // channel group g of this matrix is group g * step + part of the tiles
};

// One thread per 16-byte piece of a tile.
__global__ void k_i8_to_tiles(I8LayoutArgs p) {
    const long long groups = (p.rows + 15) / 16, total = groups * p.kt * 64;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const int l = (int)(i & 63);
        const long long g = (i >> 6) / p.kt, t = (i >> 6) % p.kt;
        const long long row = g * 16 + (l & 15), k0 = t * 64 + 16 * (l >> 4);
        uint32_t q[4] = {0, 0, 0, 0};
        if (row < p.rows)
            for (int j = 0; j < 16; ++j)
                if (k0 + j < p.k) q[j >> 2] |= (uint32_t)(uint8_t)p.rowmajor[row * p.k + k0 + j] << (8 * (j & 3));
        const long long at = ((g * p.step + p.part) * p.kt + t) * 1024 + l * 16;
        *reinterpret_cast<uint4 *>(p.tiles + at) = make_uint4(q[0], q[1], q[2], q[3]);
        if (t == 0 && l < 16) p.tile_scales[(g * p.step + p.part) * 16 + l] = row < p.rows ? p.scales[row] : 0.0f;
    }
}

__global__ void k_i8_from_tiles(I8LayoutArgs p) {
    const long long groups = (p.rows + 15) / 16, total = groups * p.kt * 64;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const int l = (int)(i & 63);
        const long long g = (i >> 6) / p.kt, t = (i >> 6) % p.kt;
        const long long row = g * 16 + (l & 15), k0 = t * 64 + 16 * (l >> 4);
        if (row >= p.rows) continue;
        const uint8_t *src = p.tiles + ((g * p.step + p.part) * p.kt + t) * 1024 + l * 16;
        for (int j = 0; j < 16; ++j)
            if (k0 + j < p.k) p.rowmajor[row * p.k + k0 + j] = (int8_t)src[j];
        if (t == 0 && l < 16) p.scales[row] = p.tile_scales[(g * p.step + p.part) * 16 + l];
    }
}

// Rows of any alignment and length into rows of `pitch` (a multiple of 256)
// aligned bytes, zeros behind k.
__global__ void k_i8_align_rows(const int8_t *x, long long stride, int k, int pitch, long long n, uint8_t *out) {
    const int words = pitch / 16;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n * words;
         i += (long long)gridDim.x * blockDim.x) {
        const long long t = i / words;
        const int k0 = (int)(i % words) * 16;
        const int8_t *src = x + t * stride + k0;
        uint32_t q[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 16; ++j)
            if (k0 + j < k) q[j >> 2] |= (uint32_t)(uint8_t)src[j] << (8 * (j & 3));
        *reinterpret_cast<uint4 *>(out + t * pitch + k0) = make_uint4(q[0], q[1], q[2], q[3]);
    }
}

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

// The value as a 32-bit float: without this the compiler folds a product and its
// conversion to 16 bits into one rounding, in some of the forms and not in others.
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}

// g / (1 + exp(-g)) * u.  exp(-g) = 2^z with z = -g log2(e) to some 40 bits (hi +
// lo), so the argument's rounding does not grow with |g|; from g = -126 ln 2 = -87.34
// down the reciprocal of 1 + e lies below the least normal float and is 0 (what is right
// is below 2^-119 |u|), so the exponent stays at g = -88, and above g = 104 (1 + e is 1),
// which also keeps infinities out of it; and 1 / d is the reciprocal with one
// Newton step.  The library's exp and division cost twice
// as many instructions, which is what bounds the epilogue.
__device__ __forceinline__ float swiglu(float g, float u) {
    constexpr float LOG2E = 0x1.715476p+0f, LOG2E_LO = 0x1.4ae0cp-26f, LN2 = 0x1.62e43p-1f;
    const float x = __builtin_amdgcn_fmed3f(-g, -104.0f, 88.0f);
    const float hi = x * LOG2E;
    const float lo = __builtin_fmaf(x, LOG2E_LO, __builtin_fmaf(x, LOG2E, -hi));
    float e = __builtin_amdgcn_exp2f(hi);
    e = __builtin_fmaf(e, lo * LN2, e);
    const float d = 1.0f + e;
    float r = __builtin_amdgcn_rcpf(d);
    r = __builtin_fmaf(__builtin_fmaf(-d, r, 1.0f), r, r);
    return g * r * u;
}

// Channels c .. c + V - 1 of token t from their sums times the token's scale
// (`up`: of the second matrix of a gated pair).  INSIDE: all of them exist, rows
// are aligned to 16 bytes, and the residual's values (if any) are at hand.
template <int OUT, bool GATED, bool INSIDE, int V>
__device__ __forceinline__ void finish(const I8Args &p, int t, int c, const float (&sum)[V], const float (&up)[V],
                                       const ChannelScales<GATED, V> &ws,
                                       const rvec<row_t<OUT>, V> *residual = nullptr) {
    if (!INSIDE && c >= p.rows) return;
    float v[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        v[j] = sum[j] * ws.g[j];
        if constexpr (GATED) v[j] = swiglu(v[j], up[j] * ws.u[j]);
        v[j] = rounded(v[j]);
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

template <int OUT, bool GATED, int TT, int R, bool ONCE>
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
        const float xs = p.xs[t0 + min(t, nt - 1)];
        float u[4], v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (float)sum[e] * xs, u[e] = (float)up[e] * xs;
        if (t < nt) finish<OUT, GATED, false, 4>(p, t0 + t, c, v, u, ws);
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
template <int OUT, bool GATED, int CW, int TW>
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
#pragma unroll
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
                    finish<OUT, GATED, INSIDE, V>(p, t0 + t, c, g, u, ws, RES ? &res[r / AT_ONCE] : nullptr);
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

float estimate(const I8Args &a, const Form &f) {
    if (!(f.cw ? fits_a_launch(tiles_of(a, f), 256) : fits_a_launch(streams_of(a, f.tw, f.r), 64 * ST_WAVES)))
        return HUGE_VALF;   // 2 * 2^26 channels x 23 tokens in the streaming form of 16
    const float cu = (float)a.cu_count, bytes = (float)(groups_of(a) * a.kt) * 1024, k = (float)a.kt;
    if (f.cw) {
        const float tiles = (float)tiles_of(a, f), rounds = ceilf(tiles / cu);
        // the largest tile waits for its residuals (4096 x 12288: T44 227 us, T32 230)
        const float wait = a.residual && f.cw == 4 ? 18.0f * rounds : 0.0f;
        // Weights that only one tile of tokens reads come from memory at what a CU has
        // in flight: 17.5 KB/us with three stages of the smallest tile, 25.5 with more.
        float weights = bytes / 5.2e6f;
        if (a.n_tokens <= 64 * f.tw)
            weights = rounds * k * (float)f.cw * 4096 / (f.cw == 1 && rounds == 1 ? 17.5e3f : 25.5e3f);
        return 2.0f + wait + fmaxf(rounds * (f.fixed + f.step * k), weights);
    }
    // Two to four workgroups share a CU and its L1, which takes 19.5 ns for a KiB.
    // Tokens come from L2 beside the weights, each workgroup's its own: 17 TB/s
    // (10 to 17 where the weights come from HBM, 16 to 30 from the last cache).
    const int per = a.gated ? 2 * f.r : f.r;
    const float across = (float)((groups_of(a) + per - 1) / per);
    const float n = across * (float)((a.n_tokens + 16 * f.tw - 1) / (16 * f.tw));
    // too little in flight: 16 x 4096 (k = 13312) S12 20 us, S11 14
    if (f.tw == 1 && f.r == 2 && n < 0.75f * cu) return HUGE_VALF;
    const float tokens = across * (float)a.n_tokens * k * 64;
    const float memory = (f.r == 2 ? 1.75f : 1.0f) + bytes / 5.5e6f + tokens / 17e6f;
    return fmaxf(2.5f + ceilf(n / cu) * k * (float)(per + f.tw) * 0.0195f, memory);
}

// The form of the least estimate.  Measured in us, two matrices in turn (in the last
// cache) / ten of them (from HBM), for the choice and for the next one (tokens x
// channels, k = 4096, g: a gated pair; S: stream TT, R; T: tile cw, tw):
//   1 x 12288     S11 9.8 / 11.3    S12 10.1 / 12.2     16 x 12288    S12 10.5 / 13.1   S11 10.1 / 13.6
//   16 x 24000    S12 16.4 / 20.0   S11 16.8 / 24.4     32 x 12288    S22 11.8 / 15.9   T11 14.8 / 17.7
//   64 x 12288    T11 15.1 / 17.7   S22 16.8 / 20.0     128 x 12288   T21 15.8 / 19.9   T11 15.8 / 20.6
//   64 x 4096     S22 7.0 / 7.0     S12 8.0 / 8.1       96 x 4096     S42 8.3 / 8.4     S22 10.1 / 10.2
//   256 x 4096    T11 12.4 / 12.5   T21 13.5 / 13.6     300 x 8192    T22 19.6 / 21.6   T21 20.3 / 25.2
//   16 x 13312 g  T11 18.5 / 22.4   S11 19.0 / 23.0     32 x 8000 g   S21 12.6 / 16.2   T11 15.2 / 19.1
//   32 x 13312 g  T11 18.9 / 23.0   S21 20.7 / 28.6     128 x 13312 g T22 21.6 / 27.5   T21 23.0 / 33.3
// and with three matrices in turn:
//   512 x 12288   T32 29.2, T22 32.5                    1024 x 4096 (k = 13312)  T22 61, T32 64
//   1024 x 12288  T32 52.5, T44 54, T22 56              1024 x 26624  T44 120, T32 145
//   4096 x 12288  T44 180, T32 200, T22 202
// (Machines differ by some 5%.)
int plan(const I8Args &a) {
    int best = -1;
    float least = 0.0f;
    for (int i = 0; i < N_FORMS; ++i) {
        if (a.gated && !FORMS[i].cw && FORMS[i].r > 1) continue;   // a pair is two groups already
        const float t = estimate(a, FORMS[i]);
        if (best < 0 || t < least) best = i, least = t;
    }
    return best;
}

template <int OUT, bool GATED, int CW, int TW>
hipError_t launch_tile(const I8Args &a, hipStream_t s) {
    const long long grid = tiles_of(a, Form{CW, TW, 0, 0, 0});
    if (!fits_a_launch(grid, 256)) return hipErrorInvalidValue;
    hipLaunchKernelGGL((k_i8_tile<OUT, GATED, CW, TW>), dim3((unsigned)grid), dim3(256), 0, s, a);
    return hipGetLastError();
}

// Weights of up to four tokens are read non-temporally from 64 MiB on: four such
// matrices fill the last cache (256 MB), so those of a model come from HBM at every
// step.  From HBM, one token: 2 * 13312 x 4096 21.8 -> 20.3 us, 24000 x 4096 18.8 ->
// 17.2, 8192 x 8192 15.0 -> 13.2; in a loop over one matrix, which stays in the cache,
// 18.9 -> 20.1, 15.7 -> 16.7, 11.8 -> 12.7.  With 16 tokens it gained 6% and lost 17%.
constexpr long long ONCE_BYTES = 64ll << 20;

template <int OUT, bool GATED, int TT, int R>
hipError_t launch_stream(const I8Args &a, hipStream_t s) {
    const long long grid = streams_of(a, TT, R);
    if (!fits_a_launch(grid, 64 * ST_WAVES)) return hipErrorInvalidValue;
    if constexpr (TT == 1)
        if (a.n_tokens <= 4 && groups_of(a) * a.kt * 1024 >= ONCE_BYTES) {
            hipLaunchKernelGGL((k_i8_stream<OUT, GATED, TT, R, true>), dim3((unsigned)grid), dim3(64 * ST_WAVES), 0, s, a);
            return hipGetLastError();
        }
    hipLaunchKernelGGL((k_i8_stream<OUT, GATED, TT, R, false>), dim3((unsigned)grid), dim3(64 * ST_WAVES), 0, s, a);
    return hipGetLastError();
}

template <int OUT, bool GATED>
hipError_t launch_form(const I8Args &a, int form, hipStream_t s) {
    if (form < 0 || form >= N_FORMS) return hipErrorInvalidValue;
    switch (form) {
    case 0: return launch_stream<OUT, GATED, 1, 1>(a, s);
    case 1: return launch_stream<OUT, GATED, 2, 1>(a, s);
    case 3: return launch_stream<OUT, GATED, 4, 1>(a, s);
    case 5: return launch_tile<OUT, GATED, 1, 1>(a, s);
    case 6: return launch_tile<OUT, GATED, 2, 1>(a, s);
    case 7: return launch_tile<OUT, GATED, 2, 2>(a, s);
    case 8: return launch_tile<OUT, GATED, 3, 2>(a, s);
    case 9: return launch_tile<OUT, GATED, 4, 4>(a, s);
    }
    if constexpr (!GATED) {
        if (form == 2) return launch_stream<OUT, GATED, 2, 2>(a, s);
        if (form == 4) return launch_stream<OUT, GATED, 4, 2>(a, s);
        if (form == 10) return launch_stream<OUT, GATED, 1, 2>(a, s);
    }
    if (form == 10) return launch_stream<OUT, GATED, 1, 1>(a, s);
    return launch_form<OUT, GATED>(a, form - 1, s);   // a forced form of two groups: a pair has them already
}

template <int OUT>
hipError_t launch_out(const I8Args &a, hipStream_t s) {
    const int form = a.form ? a.form - 1 : plan(a);
    return a.gated ? launch_form<OUT, true>(a, form, s) : launch_form<OUT, false>(a, form, s);
}

int grid_of(long long threads) {
    const long long g = (threads + 255) / 256;
    return (int)(g < 1 ? 1 : g > 16384 ? 16384 : g);
}

}  // namespace

hipError_t launch_i8_layout(const int8_t *rowmajor, uint8_t *tiles, const float *scales, float *tile_scales,
                            long long rows, long long k, long long kt, int step, int part, int to_tiles, hipStream_t s) {
    const I8LayoutArgs a{const_cast<int8_t *>(rowmajor), tiles, const_cast<float *>(scales), tile_scales, rows, k, kt,
                         step, part};
    const int grid = grid_of((rows + 15) / 16 * kt * 64);
    if (to_tiles)
        hipLaunchKernelGGL(k_i8_to_tiles, dim3(grid), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL(k_i8_from_tiles, dim3(grid), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_i8_align_rows(const int8_t *x, long long stride, int k, int pitch, long long n, uint8_t *out,
                                hipStream_t s) {
    hipLaunchKernelGGL(k_i8_align_rows, dim3(grid_of(n * (pitch / 16))), dim3(256), 0, s, x, stride, k, pitch, n, out);
    return hipGetLastError();
}

hipError_t launch_i8_product(const I8Args &a, hipStream_t s) {
    if (a.n_tokens <= 0) return hipSuccess;
    switch (a.out_type) {
    case T_F32: return launch_out<T_F32>(a, s);
    case T_F16: return launch_out<T_F16>(a, s);
    case T_BF16: return launch_out<T_BF16>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace lbh
