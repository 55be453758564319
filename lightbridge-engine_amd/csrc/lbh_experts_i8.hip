// lbh_experts_i8.hip — the feed-forward half of a mixture-of-experts layer for
// few tokens, over int8 experts (lbh_i8.hip has the weights' layout).
//
//   h[p] = silu(g) * u          p = (token, slot): g, u the products of the slot's expert
//   y[t] = residual[t] + sum over slots coef[p] * down(int8 row of h[p]) + down_shared(int8 row of h_shared[t])
//
// Integer sums are exact in any order; everything behind them is in 64 bits
// (h is rounded to 32 bits once, y to 32 bits and its type), slots are added in their
// order and the shared expert last, so a token's result hangs on its own row,
// slots and weights alone, and the few roundings leave every int8 value of h where
// the formula puts it but for one in millions.
//
// Bound: each used expert's weights once from HBM, 3 n ffn bytes; the products
// themselves are a few percent of the matrix cores' rate.  So the launches go
// by the weights: k_experts_up takes (expert, 16 channels of gate and up) per
// workgroup with k split over its waves, k_experts_down takes 8 or 16 output channels
// over every used expert, so that the sum over a token's slots ends in one
// workgroup.  A matrix tile of 16 channels x 16 tokens costs the same for one
// token as for sixteen, and up to 64 tokens of an expert (in k_experts_down all of
// them) share one read of its weights.
// 192 experts of 4096 x 1536, top 8, a shared one of 4096: 1 token 39.6 us (5.1 TB/s of the used
// experts' bytes), 5 111 (6.1), 64 516 (6.6); on another machine 64 535 (6.4), 128 601 (6.1), 256 721
// (5.1: the shared expert's and the hot ones' gate and up are read up to four times).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rows64.h"

namespace lbh {

namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

// Waves of k_experts_up: four, so that a workgroup's start (ids, first weights) and end (the
// join, silu) are spread over four times as many bytes a wave as with sixteen; eight took
// 5 to 30% longer (8 tokens, 192 experts of 4096 x 1536: 182 against 160 us), two and one 5 to
// 20%.  Of k_experts_down, which has one workgroup a CU at n = 4096: sixteen (eight waves of
// units twice as long took 1 to 4% longer, twelve 1%).
constexpr int UP_WAVES = 4, WAVES = 16;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void *base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)(uint32_t)bytes, 0x00020000);
}
// 16 bytes at a byte offset, zero past the resource's end.  Weights are read non-temporally:
// a layer's used experts do not stay in the last cache until the model comes back to the
// layer, and pushing nothing out for them is faster in any case (5 tokens 112 against 139 us,
// 64 tokens 516 against 612).
template <bool ONCE>
__device__ __forceinline__ v4i load16(__amdgpu_buffer_rsrc_t r, uint32_t at) {
    return __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, ONCE ? 2 : 0));
}

__device__ __forceinline__ int lane_rank(uint64_t mask) {   // set bits below this lane
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
}

// The used experts, each with its (token, slot) pairs.  Up to 64 pairs each wave finds
// them by itself, a pair a lane; more are sorted by k_experts_plan.  Slots whose id
// is no expert are nobody's.
struct Used {
    int expert, count;   // wave-uniform
    int pairs;           // up to 64 pairs: lane i holds the i-th
    const int *list;     // more: the list
};

struct FewPairs {
    int id;            // lane p: pair p's expert, or -1
    __device__ __forceinline__ FewPairs(const ExpertsArgs &a) {
        const int lane = threadIdx.x & 63;
        const uint32_t raw = lane < a.pairs ? a.ids[lane] : ~0u;
        id = raw < (uint32_t)a.n_experts ? (int)raw : -1;
    }
    __device__ __forceinline__ Used of(int expert, uint64_t members) const {
        const int lane = threadIdx.x & 63;
        Used r;
        r.expert = expert;
        r.count = __builtin_popcountll(members);
        // member lanes to the front; the others to lanes behind them
        const int to = (members >> lane) & 1 ? lane_rank(members) : r.count + lane_rank(~members);
        r.pairs = __builtin_amdgcn_ds_permute(4 * to, lane);
        r.list = nullptr;
        return r;
    }
    // The expert whose first pair is pair p; count 0: pair p is no expert's first.
    __device__ __forceinline__ Used starting_at(int p) const {
        const int expert = __builtin_amdgcn_readlane(id, p);
        const uint64_t members = __ballot(id == expert);
        if (expert < 0 || (int)__builtin_ctzll(members) != p) return {};
        return of(expert, members);
    }
};

// Every used expert in turn, by the place of its first pair.
struct FewExperts : FewPairs {
    uint64_t first;
    __device__ __forceinline__ FewExperts(const ExpertsArgs &a) : FewPairs(a) {
        uint64_t left = __ballot(id >= 0);
        first = 0;
        while (left) {
            const int p = (int)__builtin_ctzll(left);
            first |= 1ull << p;
            left &= ~__ballot(id == __builtin_amdgcn_readlane(id, p));
        }
    }
    __device__ __forceinline__ int used() const { return __builtin_popcountll(first); }
    __device__ __forceinline__ Used at(int u) const {   // u < used()
        const int lane = threadIdx.x & 63;
        const uint64_t mine = __ballot(((first >> lane) & 1) && lane_rank(first) == u);
        const int expert = __builtin_amdgcn_readlane(id, (int)__builtin_ctzll(mine));
        return of(expert, __ballot(id == expert));
    }
};

struct ManyPairs {
    const ExpertsPlan *plan;
    __device__ __forceinline__ ManyPairs(const ExpertsArgs &a) : plan(a.plan) {}
    __device__ __forceinline__ int used() const { return __builtin_amdgcn_readfirstlane(plan->used); }
    __device__ __forceinline__ Used at(int u) const {
        const int from = __builtin_amdgcn_readfirstlane(plan->from[u]), to = __builtin_amdgcn_readfirstlane(plan->from[u + 1]);
        return {__builtin_amdgcn_readfirstlane(plan->expert[u]), to - from, 0, plan->pair + from};
    }
};

// The i-th pair of an expert (per lane; i < count).
template <bool FEW>
__device__ __forceinline__ int pair_at(const Used &u, int i) {
    if constexpr (FEW) return __builtin_amdgcn_ds_bpermute(4 * i, u.pairs);
    return u.list[i];
}

template <bool FEW>
using Experts = std::conditional_t<FEW, FewExperts, ManyPairs>;

// Sorts more than 64 pairs by expert.  The order of an expert's pairs among
// themselves hangs on the LDS atomics, and no result hangs on it: each pair has
// a column of its own in the products.
__global__ void __launch_bounds__(1024) k_experts_plan(ExpertsArgs a) {
    __shared__ int count[1024], at[1024], wave_used[16], wave_pairs[16];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    count[tid] = 0;
    __syncthreads();
    for (int p = tid; p < a.pairs; p += 1024)
        if (a.ids[p] < (uint32_t)a.n_experts) atomicAdd(&count[a.ids[p]], 1);
    __syncthreads();
    const int mine = count[tid];
    const uint64_t some = __ballot(mine != 0);
    int sum = mine;   // inclusive within the wave
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int below = __shfl_up(sum, o, 64);
        if (lane >= o) sum += below;
    }
    if (lane == 63) wave_pairs[wid] = sum, wave_used[wid] = __builtin_popcountll(some);
    __syncthreads();
    int u = lane_rank(some), from = sum - mine;
    for (int w = 0; w < wid; ++w) u += wave_used[w], from += wave_pairs[w];
    at[tid] = from;
    if (mine) a.plan->expert[u] = tid, a.plan->from[u] = from;
    if (tid == 1023) a.plan->used = u + (mine ? 1 : 0), a.plan->from[u + (mine ? 1 : 0)] = from + mine;
    __syncthreads();
    for (int p = tid; p < a.pairs; p += 1024)
        if (a.ids[p] < (uint32_t)a.n_experts) a.plan->pair[atomicAdd(&at[a.ids[p]], 1)] = p;
}

// ------------------------------------------------------------ gate and up
//
// A workgroup has 16 channels of an expert's gate and up; wave w takes the k tiles
// w, w + 4, ...  Tokens go straight to operand registers: 16 rows x 64 bytes an
// instruction touch more lines than copies through LDS would, but at most 16 tokens
// share a tile of weights that comes from HBM at a tenth of what the L1 moves.

// Pairs base .. base + 16 NT - 1 of the expert against this wave's k tiles; D tiles a step.
template <int NT, int D, bool FEW, bool SHARED>
__device__ __forceinline__ void up_tiles(const ExpertsArgs &a, const Used &u, int base, __amdgpu_buffer_rsrc_t rw,
                                         __amdgpu_buffer_rsrc_t rx, int wid, v4i (&g)[NT], v4i (&up)[NT]) {
    const int lane = threadIdx.x & 63;
    uint32_t row[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int n = min(base + 16 * i + (lane & 15), u.count - 1);
        const int t = SHARED ? n : pair_at<FEW>(u, n) / a.top_k;
        row[i] = (uint32_t)t * (uint32_t)a.x_stride + 16 * (lane >> 4);
    }
    const int kt = a.kt_n;
    v4i wg[2][D], wu[2][D], x[2][D][NT];
    auto ask = [&](int b, int k0) {
#pragma unroll
        for (int d = 0; d < D; ++d) {
            const int k = k0 + d * UP_WAVES;
            // past the last tile: out of the resource's range, zero
            wg[b][d] = load16<true>(rw, lane * 16 + (k < kt ? k : 2 * kt) * 1024);
            wu[b][d] = load16<true>(rw, lane * 16 + (k < kt ? kt + k : 2 * kt) * 1024);
        }
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < NT; ++i) x[b][d][i] = load16<false>(rx, row[i] + (k0 + d * UP_WAVES) * 64);
    };
    auto multiply = [&](int b) {
#pragma unroll
        for (int d = 0; d < D; ++d)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                g[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wg[b][d], x[b][d][i], g[i], 0, 0, 0);
                up[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wu[b][d], x[b][d][i], up[i], 0, 0, 0);
            }
    };
    ask(0, wid);
    for (int k = wid; k < kt; k += 2 * D * UP_WAVES) {
        ask(1, k + D * UP_WAVES);
        multiply(0);
        ask(0, k + 2 * D * UP_WAVES);
        multiply(1);
    }
}

template <int NT, int D, bool FEW, bool SHARED>
__device__ __forceinline__ void up_item(const ExpertsArgs &a, const Used &u, int base, int c0, __amdgpu_buffer_rsrc_t rw,
                                        const float *gs, const float *us, v4i (*s_sum)[UP_WAVES][64]) {
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const __amdgpu_buffer_rsrc_t rx = rsrc(a.x, (long long)(a.n_tokens - 1) * a.x_stride + a.x_bytes);
    v4i g[NT] = {}, up[NT] = {};
    up_tiles<NT, D, FEW, SHARED>(a, u, base, rw, rx, wid, g, up);
    const Exp64 ex;
    // One value a thread: token tid / 16, channel tid % 16.
    const int n0 = (tid >> 4) & 15, c = tid & 15, ffn = SHARED ? a.ffn_s : a.ffn;
    const int from = n0 + 16 * (c >> 2);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        __syncthreads();   // what was there has been read
        s_sum[0][wid][lane] = g[i], s_sum[1][wid][lane] = up[i];
        __syncthreads();
        const int n = base + 16 * i + n0;
        int pair_of_row = 0;   // every lane takes part in the exchange
        if constexpr (!SHARED) pair_of_row = pair_at<FEW>(u, min(n, u.count - 1));
        if (n < u.count && c0 + c < ffn && tid < 256) {
            int sg = 0, su = 0;
#pragma unroll
            for (int w = 0; w < UP_WAVES; ++w)
                sg += s_sum[0][w][from][c & 3], su += s_sum[1][w][from][c & 3];
            const int p = SHARED ? n : pair_of_row, t = SHARED ? n : p / a.top_k;
            const double xs = (double)a.x_scales[t];
            const double vg = (double)sg * xs * (double)gs[c], vu = (double)su * xs * (double)us[c];
            const float h = (float)(vg * ex.sigmoid(vg) * vu);
            if constexpr (SHARED)
                a.h_s[(long long)t * a.h_s_pitch + c0 + c] = h;
            else
                a.h[(long long)p * a.h_pitch + c0 + c] = h;
        }
    }
}

// Tiles of 16 tokens at once: as many as the call's tokens can fill.
template <int NT, bool FEW, bool SHARED>
__device__ __forceinline__ void up_expert(const ExpertsArgs &a, const Used &u, int c0, __amdgpu_buffer_rsrc_t rw,
                                          const float *gs, const float *us, v4i (*s_sum)[UP_WAVES][64]) {
    int base = 0;
    if constexpr (NT == 4)
        for (; u.count - base > 32; base += 64) up_item<4, 1, FEW, SHARED>(a, u, base, c0, rw, gs, us, s_sum);
    if constexpr (NT >= 2)
        for (; u.count - base > 16; base += 32) up_item<2, 2, FEW, SHARED>(a, u, base, c0, rw, gs, us, s_sum);
    for (; base < u.count; base += 16) up_item<1, 4, FEW, SHARED>(a, u, base, c0, rw, gs, us, s_sum);
}

// grid: (channel groups, the shared expert and one for each used expert or pair)
template <int NT, bool FEW>
__global__ void __launch_bounds__(64 * UP_WAVES, 4) k_experts_up(ExpertsArgs a) {
    __shared__ v4i s_sum[2][UP_WAVES][64];
    const int grp = blockIdx.x, c0 = grp * 16;
    const long long bytes = 2ll * a.kt_n * 1024;
    if (a.has_shared && blockIdx.y == 0) {
        if (c0 >= a.ffn_s) return;
        const float *s = a.shared.up_scales + grp * 32;
        const Used all{0, a.n_tokens, 0, nullptr};
        up_expert<NT, FEW, true>(a, all, c0, rsrc(a.shared.up + grp * bytes, bytes), s, s + 16, s_sum);
        return;
    }
    if (c0 >= a.ffn) return;
    const int i = blockIdx.y - a.has_shared;
    Used u;
    if constexpr (FEW) {   // a pair a row of the grid
        u = FewPairs(a).starting_at(i);
        if (!u.count) return;
    } else {
        const ManyPairs pairs(a);
        if (i >= pairs.used()) return;
        u = pairs.at(i);
    }
    const ExpertI8 e = a.experts[u.expert];
    const float *s = e.up_scales + grp * 32;
    up_expert<NT, FEW, false>(a, u, c0, rsrc(e.up + grp * bytes, bytes), s, s + 16, s_sum);
}

// ------------------------------------------------------ int8 rows of h
//
// The scale of a row and its values, as lbh_quantize_i8_rows makes them.
struct RowScale {
    float scale;
    double to_q;   // zero: a row of zeros, or one that is not finite
    // top: the row's largest |value|, or not finite if any value is not
    __device__ __forceinline__ explicit RowScale(float top) : to_q(0.0) {
        scale = (float)((double)top * (1.0 / 127.0));
        if (!(top < __builtin_inff()))
            scale = __builtin_nanf("");
        else if (scale < 0x1p-126f)
            scale = 0.0f;
        else
            to_q = reciprocal_of(scale);
    }
    __device__ __forceinline__ uint2 values(const float (&x)[8]) const {
        uint32_t w[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)(nearest_of_quotient((double)x[j], to_q) & 0xff) << (8 * (j & 3));
        return to_q == 0.0 ? make_uint2(0, 0) : make_uint2(w[0], w[1]);
    }
};
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = row16_max(v);
#pragma unroll
    for (int o = 16; o < 64; o *= 2) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
    return v;
}
// The bits of |v|, which are ordered as the values are, those that are not finite above the rest.
__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }
// Elements e .. e + 7 of a row of n, zeros behind its end (rows start at multiples of 16 bytes).
__device__ __forceinline__ void eight_of(const float *h, int e, int n, float (&v)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.0f;
    if (e + 8 <= n) {
        const float4 lo = *reinterpret_cast<const float4 *>(h + e), hi = *reinterpret_cast<const float4 *>(h + e + 4);
        v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
    } else if (e < n) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e + j < n) v[j] = h[e + j];
    }
}

// One row a workgroup.  Rows up to 4096 elements stay
// in registers, longer ones are read twice.
__global__ void __launch_bounds__(256) k_experts_quantize(ExpertsArgs a) {
    const int row = blockIdx.x, tid = threadIdx.x;
    const bool shared = row >= a.pairs;
    if (!shared && a.ids[row] >= (uint32_t)a.n_experts) return;
    const int n = shared ? a.ffn_s : a.ffn, kt = shared ? a.kt_fs : a.kt_f;
    const float *h = shared ? a.h_s + (long long)(row - a.pairs) * a.h_s_pitch : a.h + (long long)row * a.h_pitch;
    int8_t *q = shared ? a.hq_s + (long long)(row - a.pairs) * kt * 64 : a.hq + (long long)row * kt * 64;
    constexpr int NV = 2;
    auto take = [&](int i, float (&v)[8]) { eight_of(h, (i * 256 + tid) * 8, n, v); };
    const int steps = (n + 2047) / 2048;
    float v[NV][8];
    uint32_t top = 0;
    auto account = [&](const float (&x)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(x[j]));
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) take(i, v[i]);
#pragma unroll
    for (int i = 0; i < NV; ++i) account(v[i]);
    for (int i = NV; i < steps; ++i) {
        float x[8];
        take(i, x);
        account(x);
    }
    __shared__ uint32_t s_top[4];
    top = wave_max(top);
    if ((tid & 63) == 0) s_top[tid >> 6] = top;
    __syncthreads();
    const RowScale sc(__builtin_bit_cast(float, max(max(s_top[0], s_top[1]), max(s_top[2], s_top[3]))));
    if (tid == 0) a.h_scales[row] = sc.scale;
    auto put = [&](int i, const float (&x)[8]) {
        const int e = (i * 256 + tid) * 8;
        if (e < n) *reinterpret_cast<uint2 *>(q + e) = sc.values(x);
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) put(i, v[i]);
    for (int i = NV; i < steps; ++i) {
        float x[8];
        take(i, x);
        put(i, x);
    }
}

// ---------------------------------------------------------------- down
//
// A workgroup has CH output channels.  Its waves take units of (expert, DOWN_TILES k
// tiles) in turn, weights of the next unit on their way during the products of this
// one; the integer sums of a pair meet in LDS, where their order does not
// count, and the sum over a token's slots is made from there in the slots' order.
constexpr int DOWN_TILES = 4;
constexpr int FUSED_STEPS = 1;   // of 512 elements a wave

// FUSED (few pairs): the int8 rows are made here, by every workgroup for itself, in
// place of a launch of k_experts_quantize; the first weights are on their way meanwhile.
template <int OUT, bool FEW, bool FUSED, int CH>
__global__ void __launch_bounds__(64 * WAVES, 4) k_experts_down(ExpertsArgs a) {
    constexpr int PER_LOAD = 16 / CH, LOADS = DOWN_TILES / PER_LOAD;
    extern __shared__ __align__(16) int s_sum[];   // [rows][CH]; FUSED: int8 rows (shared, then routed), scales
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c0 = blockIdx.x * CH, grp = c0 / 16, rows = a.pairs + (a.has_shared ? a.n_tokens : 0);
    for (int i = tid; i < rows * CH / 4; i += 64 * WAVES) reinterpret_cast<v4i *>(s_sum)[i] = v4i{};
    uint8_t *s_hq = reinterpret_cast<uint8_t *>(s_sum + rows * CH), *s_hq_r = s_hq + (a.has_shared ? a.n_tokens * a.kt_fs * 64 : 0);
    float *s_scale = reinterpret_cast<float *>(s_hq_r + a.pairs * a.kt_f * 64);
    (void)s_scale;
    if constexpr (FUSED)
        for (int i = tid; i < rows; i += 64 * WAVES) s_scale[i] = 0.0f;   // the rows' maxima
    __syncthreads();   // the sums are zero

    struct Unit {
        Used u;
        bool shared;
        int kt, k0;
        __amdgpu_buffer_rsrc_t rw, rh;
    };
    auto shared_unit = [&](int j) {
        Unit r;
        r.u = Used{0, a.n_tokens, 0, nullptr};
        r.shared = true, r.kt = a.kt_fs, r.k0 = j * DOWN_TILES;
        r.rh = rsrc(a.hq_s, (long long)a.n_tokens * a.kt_fs * 64);
        r.rw = rsrc(a.shared.down + (long long)grp * r.kt * 1024, (long long)r.kt * 1024);
        return r;
    };
    auto row_of = [&](const Unit &r, int base) {
        const int n = min(base + (lane & 15), r.u.count - 1);
        return r.shared ? n : pair_at<FEW>(r.u, n);
    };
    // Of the 16 rows a load has for the matrix instruction, CH are channels of one k tile, the next CH those
    // channels of the next.
    const int lane_at = ((lane & 48) + c0 % 16 + lane % CH) * 16 + lane % 16 / CH * 1024;
    auto ask = [&](const Unit &r, v4i (&w)[LOADS]) {
#pragma unroll
        for (int d = 0; d < LOADS; ++d)   // past the last tile: zero
            w[d] = load16<true>(r.rw, lane_at + (r.k0 + d * PER_LOAD) * 1024);
    };
    auto tokens = [&](const Unit &r, int row, v4i (&x)[DOWN_TILES]) {
        if constexpr (FUSED) {   // rows end at k tiles: the tiles behind, whose weights are zero, repeat the last
            const uint8_t *from = (r.shared ? s_hq : s_hq_r) + row * (r.kt * 64) + 16 * (lane >> 4);
#pragma unroll
            for (int d = 0; d < DOWN_TILES; ++d) x[d] = *reinterpret_cast<const v4i *>(from + min(r.k0 + d, r.kt - 1) * 64);
            return;
        }
        const uint32_t at = (uint32_t)row * (uint32_t)(r.kt * 64) + 16 * (lane >> 4) + r.k0 * 64;
#pragma unroll
        for (int d = 0; d < DOWN_TILES; ++d) x[d] = load16<false>(r.rh, at + d * 64);
    };
    auto add = [&](const Unit &r, int base, int row, const v4i (&w)[LOADS], const v4i (&x)[DOWN_TILES]) {
        v4i sums[PER_LOAD] = {};   // the i-th: of every PER_LOAD-th k tile, in rows CH i .. CH i + CH - 1
#pragma unroll
        for (int d = 0; d < DOWN_TILES; ++d)
            sums[d % PER_LOAD] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[d / PER_LOAD], x[d], sums[d % PER_LOAD], 0, 0, 0);
        v4i acc = sums[0];
#pragma unroll
        for (int i = 1; i < PER_LOAD; ++i)
            if ((lane >> 4) * 4 / CH == i) acc = sums[i];
        if (base + (lane & 15) < r.u.count) {
            int *to = s_sum + ((r.shared ? a.pairs : 0) + row) * CH + 4 * (lane >> 4) % CH;
#pragma unroll
            for (int e = 0; e < 4; ++e) atomicAdd(to + e, acc[e]);
        }
    };
    v4i w0[LOADS], w1[LOADS], x0[DOWN_TILES], x1[DOWN_TILES];
    Unit r0, r1;
    // The shared expert's units come first: their weights can be asked for before the ids are there.
    const int per = (a.kt_f + DOWN_TILES - 1) / DOWN_TILES, first = a.has_shared ? (a.kt_fs + DOWN_TILES - 1) / DOWN_TILES : 0;
    if (wid < first) {
        r0 = shared_unit(wid);
        ask(r0, w0);
    }
    const Experts<FEW> pairs(a);
    const int units = first + pairs.used() * per;
    auto unit = [&](int j) {
        if (j < first) return shared_unit(j);
        Unit r;
        const int i = (j - first) / per;
        r.u = pairs.at(i);
        r.shared = false, r.kt = a.kt_f, r.k0 = ((j - first) - i * per) * DOWN_TILES;
        r.rh = rsrc(a.hq, (long long)a.pairs * a.kt_f * 64);
        r.rw = rsrc(a.experts[r.u.expert].down + (long long)grp * r.kt * 1024, (long long)r.kt * 1024);
        return r;
    };
    auto work = [&](const Unit &r, int row, const v4i (&w)[LOADS], const v4i (&x)[DOWN_TILES]) {
        add(r, 0, row, w, x);
        for (int base = 16; base < r.u.count; base += 16) {   // further tokens of the same weights
            v4i more[DOWN_TILES];
            const int other = row_of(r, base);
            tokens(r, other, more);
            add(r, base, other, w, more);
        }
    };
    int row0 = 0, row1 = 0;
    if (wid < units) {
        if (wid >= first) {
            r0 = unit(wid);
            ask(r0, w0);
        }
        row0 = row_of(r0, 0);
    }
    if constexpr (FUSED) {
        // 512 elements of a row a wave at once, all of them in registers between the maximum and the values.
        const int per_s = a.has_shared ? (a.ffn_s + 511) / 512 : 0, per_r = (a.ffn + 511) / 512;
        const int all_s = per_s * a.n_tokens, all = all_s + per_r * a.pairs;
        float v[FUSED_STEPS][8];
        auto place = [&](int i, int &row, int &e) {   // row: of the sums
            const int j = wid + i * WAVES;
            const bool sh = j < all_s;
            const int per = sh ? per_s : per_r, k = sh ? j : j - all_s;
            row = k / per + (sh ? a.pairs : 0), e = (k % per) * 512 + lane * 8;
            return j < all && (sh || a.ids[row] < (uint32_t)a.n_experts);
        };
#pragma unroll
        for (int i = 0; i < FUSED_STEPS; ++i) {
            int row, e;
            if (!place(i, row, e)) continue;
            if (row >= a.pairs)
                eight_of(a.h_s + (long long)(row - a.pairs) * a.h_s_pitch, e, a.ffn_s, v[i]);
            else
                eight_of(a.h + (long long)row * a.h_pitch, e, a.ffn, v[i]);
        }
#pragma unroll
        for (int i = 0; i < FUSED_STEPS; ++i) {
            int row, e;
            if (!place(i, row, e)) continue;
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, magnitude(v[i][j]));
            top = wave_max(top);
            if (lane == 0) atomicMax(reinterpret_cast<uint32_t *>(s_scale) + row, top);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < FUSED_STEPS; ++i) {
            int row, e;
            if (!place(i, row, e)) continue;
            const bool sh = row >= a.pairs;
            if (e < (sh ? a.ffn_s : a.ffn))
                *reinterpret_cast<uint2 *>((sh ? s_hq + (row - a.pairs) * (a.kt_fs * 64) : s_hq_r + row * (a.kt_f * 64)) + e) =
                    RowScale(s_scale[row]).values(v[i]);
        }
        __syncthreads();
    }
    if (wid < units) {
        tokens(r0, row0, x0);
        for (int j = wid; j < units; j += 2 * WAVES) {
            const bool next = j + WAVES < units;
            if (next) {
                r1 = unit(j + WAVES);
                row1 = row_of(r1, 0);
                ask(r1, w1), tokens(r1, row1, x1);
            }
            work(r0, row0, w0, x0);
            if (!next) break;
            if (j + 2 * WAVES < units) {
                r0 = unit(j + 2 * WAVES);
                row0 = row_of(r0, 0);
                ask(r0, w0), tokens(r0, row0, x0);
            }
            work(r1, row1, w1, x1);
        }
    }
    __syncthreads();
    using T = row_t<OUT>;
    auto scale_of = [&](int row) { return FUSED ? (double)RowScale(s_scale[row]).scale : (double)a.h_scales[row]; };
    for (int i = tid; i < a.n_tokens * CH; i += 64 * WAVES) {
        const int t = i / CH, c = c0 + i % CH;
        if (c >= a.n) continue;
        double sum = 0.0;
        for (int s = 0; s < a.top_k; ++s) {
            const int p = t * a.top_k + s;
            const uint32_t id = a.ids[p];
            if (id >= (uint32_t)a.n_experts) continue;
            const double scale = (double)a.coefs[p] * scale_of(p);
            sum += (double)s_sum[p * CH + i % CH] * (double)a.down_scales[(long long)id * a.down_pitch + c] * scale;
        }
        if (a.has_shared)
            sum += (double)s_sum[(a.pairs + t) * CH + i % CH] * (double)a.shared.down_scales[c] * scale_of(a.pairs + t);
        if (a.residual) sum += (double)static_cast<const T *>(a.residual)[(long long)t * a.residual_stride + c];
        static_cast<T *>(a.y)[(long long)t * a.y_stride + c] = (T)(float)sum;
    }
}

template <bool FEW>
hipError_t launch_up(const ExpertsArgs &a, hipStream_t s) {
    const int widest = a.has_shared && a.ffn_s > a.ffn ? a.ffn_s : a.ffn;
    const int used = FEW || a.pairs < a.n_experts ? a.pairs : a.n_experts;
    const dim3 grid((widest + 15) / 16, used + a.has_shared);
    if (a.n_tokens <= 16)
        hipLaunchKernelGGL((k_experts_up<1, FEW>), grid, dim3(64 * UP_WAVES), 0, s, a);
    else if (a.n_tokens <= 32)
        hipLaunchKernelGGL((k_experts_up<2, FEW>), grid, dim3(64 * UP_WAVES), 0, s, a);
    else
        hipLaunchKernelGGL((k_experts_up<4, FEW>), grid, dim3(64 * UP_WAVES), 0, s, a);
    return hipGetLastError();
}

template <int OUT, bool FEW, bool FUSED, int CH>
hipError_t launch_down(const ExpertsArgs &a, hipStream_t s) {
    auto kernel = k_experts_down<OUT, FEW, FUSED, CH>;
    const int rows = a.pairs + (a.has_shared ? a.n_tokens : 0);
    int lds = rows * CH * 4;
    if constexpr (FUSED) lds += 64 * (a.pairs * a.kt_f + (a.has_shared ? a.n_tokens * a.kt_fs : 0)) + rows * 4;
    if (lds > 64 * 1024) {
        const hipError_t e =
            hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(kernel, dim3((a.n + CH - 1) / CH), dim3(64 * WAVES), lds, s, a);
    return hipGetLastError();
}

// Up to 2048 channels sixteen a workgroup leave half the CUs without one, eight (whole 128-byte lines of the
// tiles) give each of them one: 64 experts of 2048 x 1024, 64 tokens 85.9 -> 80.2 us, 128 of 2048 x 1536 222.6 -> 204.8,
// 4 tokens 63.0 -> 57.6; one token of the former 11.6 -> 11.8.  Beyond, eight make more workgroups than there are CUs, which
// run them in turns (top 4 of 64 experts of n x 1024, 4 and 64 tokens, sixteen against eight: n = 2560 32.1 and 103.5
// against 35.8 and 118.2, 4096 37.6 and 130.4 against 42.0 and 142.8, 5120 50.7 and 187 against 54.3 and 192, 7168 63.7
// and 230 against 70.8 and 257; one token 13.6 to 23.9 against 16.5 to 29.8).  Four (half lines) for up to 1024 channels took
// as long or longer than eight (64 experts of 1024 x 512, 64 tokens 48.8 against 46.2).
template <int OUT, bool FEW, bool FUSED>
hipError_t launch_down(const ExpertsArgs &a, hipStream_t s) {
    return a.n <= 2048 ? launch_down<OUT, FEW, FUSED, 8>(a, s) : launch_down<OUT, FEW, FUSED, 16>(a, s);
}

template <bool FEW, bool FUSED>
hipError_t launch_layer(const ExpertsArgs &a, hipStream_t s) {
    hipError_t e;
    if constexpr (!FEW) {
        hipLaunchKernelGGL(k_experts_plan, dim3(1), dim3(1024), 0, s, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if ((e = launch_up<FEW>(a, s)) != hipSuccess) return e;
    if constexpr (!FUSED) {
        hipLaunchKernelGGL(k_experts_quantize, dim3(a.pairs + (a.has_shared ? a.n_tokens : 0)), dim3(256), 0, s, a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    switch (a.y_type) {
    case T_F32: return launch_down<T_F32, FEW, FUSED>(a, s);
    case T_F16: return launch_down<T_F16, FEW, FUSED>(a, s);
    case T_BF16: return launch_down<T_BF16, FEW, FUSED>(a, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_experts_i8(const ExpertsArgs &a, hipStream_t s) {
    if (a.n_tokens <= 0) return hipSuccess;
    if (a.n_tokens > EXPERTS_MAX_TOKENS || a.pairs != a.n_tokens * a.top_k || a.pairs < 1 || a.pairs > EXPERTS_MAX_PAIRS ||
        a.n_experts < 1 || a.n_experts > EXPERTS_MAX)
        return hipErrorInvalidValue;
    // Up to 64 pairs every wave finds its expert's pairs with a few ballots; a launch that sorts
    // them takes longer (64 pairs, 8 tokens of 4096 x 1536: 154 against 159 us).
    if (a.pairs > 64) return launch_layer<false, false>(a, s);
    // Rows that fit the waves' registers once are quantized inside k_experts_down: one token
    // of four experts of 2048 x 1024 11.9 us, with a launch for it 13.0; twice or four times as many
    // steps gain nothing (one token, eight of 4096 x 1536 and a shared one of 4096: 40.4 and 39.5).
    const long long steps = (long long)a.pairs * ((a.ffn + 511) / 512) + (long long)a.n_tokens * ((a.ffn_s + 511) / 512);
    if (steps <= FUSED_STEPS * WAVES) return launch_layer<true, true>(a, s);
    return launch_layer<true, false>(a, s);
}

}  // namespace lbh
