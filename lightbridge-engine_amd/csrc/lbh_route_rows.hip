// lbh_route_rows.hip — routing of a batch of rows: router logits, the best
// experts of each row and their coefficients.
//
//   l[t][e] = sum_i x[t][i] w[e][i]
//   mode 0: the top_k largest l, coefs = softmax over them * weight_scale
//   mode 1: the top_k largest sigmoid(l) + bias, coefs = sigmoid(l) / max(sum, 2^-14) * weight_scale
//
// Everything is in 64 bits (products of 32-bit values are exact there), ties go to the
// lower id, so a choice between two experts does not hang on the order of a
// sum unless their scores agree to some 1e-14; and that order is the same for any
// number of rows.  (The router of lbh_router.hip reproduces a sequential 32-bit
// sum instead, one token at a time, at 4096 dependent additions.)
//
// Products run on v_mfma_f64_16x16x4_f64, 16 experts x 16 rows.  The inner
// dimension is cut into 8 slices, each over a workgroup's four waves; few rows
// give every slice a workgroup of its own (its sums wait in the workspace), many
// rows let a workgroup go through all eight, with the sums added in the same
// order.  Bound: many rows by the matrix instruction (64 cycles for 1024 products), few by
// latency.
#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rows64.h"

namespace lbh {

namespace {

typedef double v4d __attribute__((ext_vector_type(4)));

template <int TY>
__device__ __forceinline__ void load4(const row_t<TY> *p, float (&v)[4]) {
    rvec<row_t<TY>, 4> a;
    __builtin_memcpy(&a, p, sizeof a);   // at any address of its type
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)a[j];
}

// grid: (16 experts, 16 rows, slices or 1)
template <int TY>
__global__ void __launch_bounds__(256) k_route_logits(RouteRowsArgs a) {
    __shared__ double s_part[4][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int e = min((int)blockIdx.x * 16 + (lane & 15), a.n_experts - 1);
    const int t = min((int)blockIdx.y * 16 + (lane & 15), a.n_tokens - 1);
    const float4 *w = reinterpret_cast<const float4 *>(a.w) + e;
    const row_t<TY> *x = static_cast<const row_t<TY> *>(a.x) + (long long)t * a.x_stride;
    const int steps = a.hidden / 16, q = lane >> 4;
    const int s0 = gridDim.z == 1 ? 0 : blockIdx.z, s1 = gridDim.z == 1 ? ROUTE_SLICES : s0 + 1;
    double total = 0.0;
    for (int s = s0; s < s1; ++s) {
        const int part = s * 4 + wid;
        int k = part * steps / (4 * ROUTE_SLICES);
        const int end = (part + 1) * steps / (4 * ROUTE_SLICES);
        v4d acc = {};
        // 16 of the inner dimension a step: the lane's four are those of 4 q .. 4 q + 3, product m takes the m-th of each
        auto ask = [&](int i, float4 &wv, float (&xv)[4]) {
            i = min(i, steps - 1);
            wv = w[(long long)(4 * i + q) * a.n_experts];
            load4<TY>(x + 16 * i + 4 * q, xv);
        };
        auto multiply = [&](const float4 &wv, const float (&xv)[4]) {
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)wv.x, (double)xv[0], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)wv.y, (double)xv[1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)wv.z, (double)xv[2], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)wv.w, (double)xv[3], acc, 0, 0, 0);
        };
        constexpr int AHEAD = 8;   // a slice of 4096 in flight at once
        float4 wv[AHEAD];
        float xv[AHEAD][4];
        for (; k < end; k += AHEAD) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) ask(k + i, wv[i], xv[i]);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (k + i < end) multiply(wv[i], xv[i]);
        }
        // D: lane l holds row l % 16 and experts 4 i + l / 16
        if (s > s0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) s_part[wid][lane & 15][4 * i + q] = acc[i];
        __syncthreads();
        const int r = tid >> 4, c = tid & 15;
        total += s_part[0][r][c] + s_part[1][r][c] + s_part[2][r][c] + s_part[3][r][c];
    }
    const int to = blockIdx.y * 16 + (tid >> 4), te = blockIdx.x * 16 + (tid & 15);
    if (to < a.n_tokens && te < a.n_experts)
        a.part[((long long)blockIdx.z * a.n_tokens + to) * a.n_experts + te] = total;
}

// Order of 64-bit floats as integers; 0 is below every finite one.
__device__ __forceinline__ unsigned long long key_of(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);   // -0 is 0
    return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ unsigned long long wave_max_key(unsigned long long v) {
    auto take = [&](unsigned long long o) { v = o > v ? o : v; };
    auto dpp = [&](auto ctrl) {
        constexpr int C = decltype(ctrl)::value;
        return (unsigned long long)dpp_row<C>((uint32_t)(v >> 32)) << 32 | dpp_row<C>((uint32_t)v);
    };
    take(dpp(std::integral_constant<int, 0xB1>()));    // quad_perm [1, 0, 3, 2]
    take(dpp(std::integral_constant<int, 0x4E>()));    // quad_perm [2, 3, 0, 1]
    take(dpp(std::integral_constant<int, 0x141>()));   // row_half_mirror
    take(dpp(std::integral_constant<int, 0x140>()));   // row_mirror
    // one value a row of 16 lanes: four scalars
    unsigned long long m = 0;
#pragma unroll
    for (int i = 0; i < 64; i += 16) {
        const unsigned long long o = (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), i) << 32 |
                                     (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, i);
        m = o > m ? o : m;
    }
    return m;
}

// A wave a row; lane l has experts l, l + 64, ...
__global__ void __launch_bounds__(256) k_route_select(RouteRowsArgs a, int parts) {
    constexpr int SLOTS = 4;   // up to 256 experts
    const int lane = threadIdx.x & 63;
    const long long t = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.n_tokens) return;
    double logit[SLOTS], weight[SLOTS];
    unsigned long long key[SLOTS];
    float bias[SLOTS];
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
        const int e = min(lane + 64 * k, a.n_experts - 1);
        bias[k] = a.mode ? a.bias[e] : 0.0f;
        logit[k] = 0.0;
        if (parts == 1) {
            logit[k] += a.part[t * a.n_experts + e];
        } else {
#pragma unroll
            for (int s = 0; s < ROUTE_SLICES; ++s) logit[k] += a.part[(s * (long long)a.n_tokens + t) * a.n_experts + e];
        }
    }
    bool bad = false;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
        const int e = lane + 64 * k;
        const bool some = e < a.n_experts;
        if (some && a.logits) a.logits[t * a.n_experts + e] = (float)logit[k];
        weight[k] = a.mode ? 1.0 / (1.0 + exp(-logit[k])) : logit[k];
        const double score = a.mode ? weight[k] + (double)bias[k] : logit[k];
        bad |= some && !(fabs(score) < __builtin_inf() && fabs(logit[k]) < __builtin_inf());
        key[k] = some ? key_of(score) : 0;
    }
    uint32_t *ids = a.ids + t * a.top_k;
    float *coefs = a.coefs + t * a.top_k;
    if (__ballot(bad)) {   // no order among such scores: every coefficient says so
        if (lane < a.top_k) ids[lane] = (uint32_t)lane, coefs[lane] = __builtin_nanf("");
        return;
    }
    bool taken[SLOTS] = {};
    double best = 0.0;   // the largest logit of a selection by logits
    for (int r = 0; r < a.top_k; ++r) {
        unsigned long long top = key[0];
#pragma unroll
        for (int k = 1; k < SLOTS; ++k) top = key[k] > top ? key[k] : top;
        const unsigned long long m = wave_max_key(top);
        if (r == 0) best = __builtin_bit_cast(double, m >> 63 ? m & ~(1ull << 63) : ~m);
        bool found = false;
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {   // the lowest id among equals
            const uint64_t equal = __ballot(key[k] == m);
            if (!found && equal) {
                found = true;
                if (lane == (int)__builtin_ctzll(equal)) taken[k] = true, key[k] = 0;
            }
        }
    }
    double sum = 0.0, none = 0.0;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
        if (!a.mode) weight[k] = taken[k] ? exp(logit[k] - best) : 0.0;
        if (taken[k]) sum += weight[k];
    }
    wave_sum_max(sum, none);
    if (a.mode) sum = fmax(sum, 0x1p-14);
    int at = 0;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
        const uint64_t mask = __ballot(taken[k]);
        const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
        if (taken[k]) {
            ids[at + rank] = (uint32_t)(lane + 64 * k);
            coefs[at + rank] = (float)(weight[k] / sum * a.weight_scale);
        }
        at += __builtin_popcountll(mask);
    }
}

template <int TY>
hipError_t launch_logits(const RouteRowsArgs &a, int parts, hipStream_t s) {
    hipLaunchKernelGGL((k_route_logits<TY>), dim3((a.n_experts + 15) / 16, (a.n_tokens + 15) / 16, parts), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_route_rows(const RouteRowsArgs &a, hipStream_t s) {
    if (a.n_tokens <= 0) return hipSuccess;
    if (a.n_experts < 1 || a.n_experts > 256 || a.hidden < 256 || a.hidden % 256 || a.top_k < 1 ||
        a.top_k > MOE_MAX_ROUTED || a.top_k > a.n_experts || (a.n_tokens + 15) / 16 > 65535)
        return hipErrorInvalidValue;
    const int parts = route_parts(a.n_tokens);
    hipError_t e;
    switch (a.x_type) {
    case T_F32: e = launch_logits<T_F32>(a, parts, s); break;
    case T_F16: e = launch_logits<T_F16>(a, parts, s); break;
    case T_BF16: e = launch_logits<T_BF16>(a, parts, s); break;
    default: return hipErrorInvalidValue;
    }
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_route_select, dim3((a.n_tokens + 3) / 4), dim3(256), 0, s, a, parts);
    return hipGetLastError();
}

}  // namespace lbh
