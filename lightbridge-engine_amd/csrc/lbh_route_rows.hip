// lbh_route_rows.hip — routing of a batch of rows: router logits, the best
// experts of each row and their coefficients.
//
//   l[t][e] = sum_i x[t][i] w[e][i]
//   mode 0: the top_k largest l, coefs = softmax over them * weight_scale
//   mode 1: the top_k largest sigmoid(l) + bias, coefs = sigmoid(l) / max(sum, 2^-14) * weight_scale
//
// Everything is in 64 bits (products of 32-bit values are exact there), ties go to the
// lower id, so a choice between two experts does not hang on the order of a
// sum unless their logits agree to some 1e-14 (nor, in mode 1, on the sigmoid's 2^-38.7
// unless their scores agree to some 1e-12); and that order is the same for any number of rows.  (The router of lbh_router.hip reproduces a sequential 32-bit
// sum instead, one token at a time, at 4096 dependent additions.)
//
// Products run on v_mfma_f64_16x16x4_f64, 16 experts x 16 rows.  The inner dimension
// is cut into 32 parts; the sums of eight parts are added in turn to one of four
// sums, and these in turn to the logit, whoever does it: few rows spread the parts
// over four workgroups of eight waves (their sums wait in the workspace), many rows
// over the four waves of one.  Bound: few rows by the latency of two launches (192 experts of
// 4096, both: 1 row 10.8 us, 64 13.5, 256 20.2), many by the matrix instruction, some 74
// cycles for 1024 products (1000 rows 42.9 us, 23 of them its own).
#include <type_traits>

#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_router.h"
#include "lbh_rows64.h"

namespace lbh {

namespace {

typedef double v4d __attribute__((ext_vector_type(4)));

// The inner dimension's units of 64 in 32 parts, eight for each of four sums.  MANY: a
// wave makes a sum, part after part; else a workgroup does, a part a wave.  grid: (16
// experts, 16 rows, 1 or the four sums)
template <int TY, bool MANY>
__global__ void __launch_bounds__(MANY ? 256 : 512) k_route_logits(RouteRowsArgs a) {
    constexpr int WAVES = MANY ? ROUTE_SUMS : ROUTE_PARTS;
    __shared__ double s_sum[WAVES][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int e = min((int)blockIdx.x * 16 + (lane & 15), a.n_experts - 1);
    const int t = min((int)blockIdx.y * 16 + (lane & 15), a.n_tokens - 1);
    const float4 *w = reinterpret_cast<const float4 *>(a.w) + e;
    const row_t<TY> *x = static_cast<const row_t<TY> *>(a.x) + (long long)t * a.x_stride;
    const int units = a.hidden / 64, q = lane >> 4;
    auto edge = [&](int part) { return part * units / (ROUTE_SUMS * ROUTE_PARTS); };
    int part = MANY ? wid * ROUTE_PARTS : blockIdx.z * ROUTE_PARTS + wid;
    const int first = edge(part), last = edge(part + (MANY ? ROUTE_PARTS : 1));
    v4d sum = {}, acc = {};
    // A unit is 64 of the inner dimension.  The lane's sixteen are those of 16 q .. 16 q + 15, so that a row's bytes are
    // read a whole line at a time; product i takes the i-th of each.  (Four of each 16, a quarter of the line, had the
    // lines come from L2 four times: 1000 rows 44 us.)
    struct Unit {
        float4 w[4];
        rvec<row_t<TY>, 16> x;
    };
    auto ask = [&](int k, Unit &v) {
        const int at = min(k, units - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[i] = w[(long long)(16 * at + 4 * q + i) * a.n_experts];
        __builtin_memcpy(&v.x, x + 64 * at + 16 * q, sizeof v.x);   // at any address of its type
    };
    // The end of the part that position `at` lies in (of narrow rows some parts are empty).
    auto end_of = [&](int at) {
        while (edge(part) <= at && edge(part) < last) ++part;
        return edge(part);
    };
    int next = end_of(first);
    auto multiply = [&](int k, const Unit &v) {
        if (k >= last) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = v.w[i];
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f.x, (double)(float)v.x[4 * i], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f.y, (double)(float)v.x[4 * i + 1], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f.z, (double)(float)v.x[4 * i + 2], acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)f.w, (double)(float)v.x[4 * i + 3], acc, 0, 0, 0);
        }
        if (MANY && k + 1 == next) {   // the part is done
            sum += acc;
            acc = v4d{};
            next = end_of(k + 1);
        }
    };
    Unit v0, v1;
    ask(first, v0);
    for (int k = first; k < last; k += 2) {
        ask(k + 1, v1);
        multiply(k, v0);
        ask(k + 2, v0);
        multiply(k + 1, v1);
    }
    if (!MANY) sum = acc;
    // D: lane l holds row l % 16 and experts 4 i + l / 16
#pragma unroll
    for (int i = 0; i < 4; ++i) s_sum[wid][lane & 15][4 * i + q] = sum[i];
    __syncthreads();
    if (tid >= 256) return;
    double total = 0.0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) total += s_sum[i][tid >> 4][tid & 15];
    const int to = blockIdx.y * 16 + (tid >> 4), te = blockIdx.x * 16 + (tid & 15);
    if (to < a.n_tokens && te < a.n_experts)
        a.part[((long long)blockIdx.z * a.n_tokens + to) * a.n_experts + te] = total;
}

// Order of 64-bit floats as integers; 0 is below every finite one.
__device__ __forceinline__ unsigned long long key_of(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v + 0.0);   // -0 is 0
    return b >> 63 ? ~b : b | 1ull << 63;
}
// A wave a row; lane l has experts l, l + 64, ...
__global__ void __launch_bounds__(256) k_route_select(RouteRowsArgs a, int parts) {
    constexpr int SLOTS = 4;   // up to 256 experts
    const int lane = threadIdx.x & 63;
    const long long t = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= a.n_tokens) return;
    const Exp64 ex;
    double logit[SLOTS];
    unsigned long long key[SLOTS];
    float bias[SLOTS];
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
        const int e = min(lane + 64 * k, a.n_experts - 1);
        bias[k] = a.mode ? a.bias[e] : 0.0f;
        const double *part = a.part + t * a.n_experts + e;
        double v[ROUTE_SUMS];   // one sum: the others are not added
#pragma unroll
        for (int s = 0; s < ROUTE_SUMS; ++s) v[s] = part[s < parts ? s * (long long)a.n_tokens * a.n_experts : 0];
        logit[k] = v[0];
#pragma unroll
        for (int s = 1; s < ROUTE_SUMS; ++s) logit[k] = s < parts ? logit[k] + v[s] : logit[k];
    }
    bool bad = false;
#pragma unroll
    for (int k = 0; k < SLOTS; ++k) {
        const int e = lane + 64 * k;
        const bool some = e < a.n_experts;
        if (some && a.logits) a.logits[t * a.n_experts + e] = (float)logit[k];
        const double score = a.mode ? ex.sigmoid(logit[k]) + (double)bias[k] : logit[k];
        bad |= some && !(fabs(score) < __builtin_inf() && fabs(logit[k]) < __builtin_inf());
        key[k] = some ? key_of(score) : 0;
    }
    uint32_t *ids = a.ids + t * a.top_k;
    float *coefs = a.coefs + t * a.top_k;
    if (__ballot(bad)) {   // no order among such scores: every coefficient says so
        if (lane < a.top_k) ids[lane] = (uint32_t)lane, coefs[lane] = __builtin_nanf("");
        return;
    }
    // Rounds of a maximum over the keys' upper words; where several have it, over their
    // lower words, and the lowest id among equals.  Lane r keeps what round r chose.
    int id = 0x7fffffff;
    double chosen = 0.0;
    for (int r = 0; r < a.top_k; ++r) {
        uint32_t high = 0, low = 0;
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) high = max(high, (uint32_t)(key[k] >> 32));
        high = wave_max_u32(high);
        int many = 0;
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) many += __builtin_popcountll(__ballot((uint32_t)(key[k] >> 32) == high));
        if (many > 1) {
#pragma unroll
            for (int k = 0; k < SLOTS; ++k)
                if ((uint32_t)(key[k] >> 32) == high) low = max(low, (uint32_t)key[k]);
            low = wave_max_u32(low);
        }
        bool found = false;
#pragma unroll
        for (int k = 0; k < SLOTS; ++k) {
            const uint64_t equal = __ballot((uint32_t)(key[k] >> 32) == high && (many == 1 || (uint32_t)key[k] == low));
            if (found || !equal) continue;   // the same for every lane
            found = true;
            const int from = (int)__builtin_ctzll(equal);
            const uint64_t bits = __builtin_bit_cast(uint64_t, logit[k]);
            const uint64_t l = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(bits >> 32), from) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, from);
            if (lane == r) id = from + 64 * k, chosen = __builtin_bit_cast(double, l);
            if (lane == from) key[k] = 0;
        }
    }
    const bool mine = lane < a.top_k;
    double weight;
    if (a.mode) {
        weight = ex.sigmoid(chosen);
    } else {
        double best = mine ? chosen : -__builtin_inf(), none = 0.0;
        wave_sum_max(none, best);
        const double x = fmax(chosen - best, -708.0);   // from there on its share of the sum is 0
        weight = ex.exp(x, (float)x);
    }
    double sum = wave_sum(mine ? weight : 0.0);
    if (a.mode) sum = fmax(sum, 0x1p-14);
    int at = 0;
    for (int r = 0; r < a.top_k; ++r) at += __builtin_amdgcn_readlane(id, r) < id;
    if (mine) ids[at] = (uint32_t)id, coefs[at] = (float)(weight / sum * a.weight_scale);
}

template <int TY>
hipError_t launch_logits(const RouteRowsArgs &a, int parts, hipStream_t s) {
    const dim3 grid((a.n_experts + 15) / 16, (a.n_tokens + 15) / 16, parts);
    if (parts == 1)
        hipLaunchKernelGGL((k_route_logits<TY, true>), grid, dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((k_route_logits<TY, false>), grid, dim3(512), 0, s, a);
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
