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
// k are padded with zeros (k to 128), so what the rows hold behind k never
// counts.
#include "lbh_dev.h"
#include "lbh_internal.h"
#include "lbh_rowtypes.h"

namespace lbh {

namespace {

typedef int i8_v4i __attribute__((ext_vector_type(4)));

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

// Rows of any alignment and length into rows of `pitch` (a multiple of 128)
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

template <int OUT>
__device__ __forceinline__ void load4(const row_t<OUT> *p, float (&v)[4]) {
    const rvec<row_t<OUT>, 4> a = *reinterpret_cast<const rvec<row_t<OUT>, 4> *>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (float)a[j];
}
template <int OUT>
__device__ __forceinline__ void store4(row_t<OUT> *p, const float (&v)[4]) {
    rvec<row_t<OUT>, 4> a;
#pragma unroll
    for (int j = 0; j < 4; ++j) a[j] = (row_t<OUT>)v[j];
    *reinterpret_cast<rvec<row_t<OUT>, 4> *>(p) = a;
}

// Four channels c .. c + 3 (c % 4 == 0) of token t from their integer sums
// (`up`: of the second matrix of a gated pair).  g: channel group of the tiles.
template <int OUT, bool GATED>
__device__ __forceinline__ void finish4(const I8Args &p, int t, int c, const i8_v4i &sum, const i8_v4i &up) {
    const float xs = p.xs[t];
    float v[4];
    const int gr = c >> 4;
    if constexpr (GATED) {
        const float4 sg = *reinterpret_cast<const float4 *>(p.ws + 32 * gr + (c & 15));
        const float4 su = *reinterpret_cast<const float4 *>(p.ws + 32 * gr + 16 + (c & 15));
        const float a[4] = {sg.x, sg.y, sg.z, sg.w}, b[4] = {su.x, su.y, su.z, su.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float g = (float)sum[j] * xs * a[j], u = (float)up[j] * xs * b[j];
            v[j] = g / (1.0f + expf(-g)) * u;
        }
    } else {
        const float4 s4 = *reinterpret_cast<const float4 *>(p.ws + 16 * gr + (c & 15));
        const float a[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (float)sum[j] * xs * a[j];
    }
    row_t<OUT> *y = static_cast<row_t<OUT> *>(p.y) + (long long)t * p.y_stride + c;
    const row_t<OUT> *res = GATED || !p.residual
                                ? nullptr
                                : static_cast<const row_t<OUT> *>(p.residual) + (long long)t * p.residual_stride + c;
    if (p.vec_out && c + 3 < p.rows) {
        if (res) {
            float r[4];
            load4<OUT>(res, r);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = r[j] + v[j];
        }
        store4<OUT>(y, v);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (c + j < p.rows) y[j] = (row_t<OUT>)(res ? (float)res[j] + v[j] : v[j]);
    }
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t i8_rsrc(const void *base, long long bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), (short)0, (int)(uint32_t)bytes, 0x00020000);
}

// ------------------------------------------------------- few tokens: streaming
//
// A workgroup takes one channel group (a gated pair's two) and up to 16 * TT
// tokens; its eight waves take every eighth k tile and their integer sums are
// joined in LDS.  Bound: the weights' bytes, each read once a token tile.
constexpr int ST_WAVES = 8;

template <int OUT, bool GATED, int TT>
__global__ void __launch_bounds__(64 * ST_WAVES) k_i8_stream(I8Args p) {
    constexpr int G = GATED ? 2 : 1;
    constexpr int U = TT == 1 ? 8 : 4;
    __shared__ __align__(16) i8_v4i s_sum[ST_WAVES][G * TT][64];
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
    const int t0 = blockIdx.y * 16 * TT, nt = min(p.n_tokens - t0, 16 * TT);
    const __amdgpu_buffer_rsrc_t rw =
        i8_rsrc(p.w + (long long)blockIdx.x * G * p.kt * 1024, (long long)G * p.kt * 1024);
    // Token rows end with their last byte: what a tile reads beyond is zero, and
    // what it reads of the next row meets the weights' zeros.  (All offsets are
    // vector offsets: the scalar one is left out of the range check.)
    const __amdgpu_buffer_rsrc_t rx = i8_rsrc(p.x + (long long)t0 * p.x_stride, (long long)(nt - 1) * p.x_stride + p.k);
    uint32_t xo[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i)
        xo[i] = (uint32_t)min(16 * i + (lane & 15), nt - 1) * (uint32_t)p.x_stride + 16 * (lane >> 4);
    i8_v4i acc[G][TT] = {};
    for (int k0 = wid; k0 < p.kt; k0 += ST_WAVES * U) {
        i8_v4i a[U][G], b[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int kt = k0 + ST_WAVES * u;
#pragma unroll
            for (int g = 0; g < G; ++g)   // past the last tile: out of the resource's range, zero
                a[u][g] = __builtin_bit_cast(
                    i8_v4i, __builtin_amdgcn_raw_buffer_load_b128(
                                rw, lane * 16 + (kt < p.kt ? (g * p.kt + kt) * 1024 : G * p.kt * 1024), 0, 0));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < TT; ++i)
                b[u][i] = __builtin_bit_cast(
                    i8_v4i, __builtin_amdgcn_raw_buffer_load_b128(rx, xo[i] + (k0 + ST_WAVES * u) * 64, 0, 0));
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < TT; ++i)
#pragma unroll
                for (int g = 0; g < G; ++g)
                    acc[g][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[u][g], b[u][i], acc[g][i], 0, 0, 0);
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
        for (int i = 0; i < TT; ++i) s_sum[wid][g * TT + i][lane] = acc[g][i];
    __syncthreads();
    for (int i = wid; i < TT; i += ST_WAVES) {
        i8_v4i sum = {}, up = {};
#pragma unroll
        for (int w = 0; w < ST_WAVES; ++w) {
            sum += s_sum[w][i][lane];
            if constexpr (GATED) up += s_sum[w][TT + i][lane];
        }
        const int t = 16 * i + (lane & 15);
        if (t < nt) finish4<OUT, GATED>(p, t0 + t, blockIdx.x * 16 + 4 * (lane >> 4), sum, up);
    }
}

template <int OUT, bool GATED>
hipError_t launch_typed(const I8Args &a, hipStream_t s) {
    const unsigned groups = (unsigned)((a.rows + 15) / 16);
    if (a.n_tokens <= 16)
        hipLaunchKernelGGL((k_i8_stream<OUT, GATED, 1>), dim3(groups, 1), dim3(64 * ST_WAVES), 0, s, a);
    else if (a.n_tokens <= 32)
        hipLaunchKernelGGL((k_i8_stream<OUT, GATED, 2>), dim3(groups, 1), dim3(64 * ST_WAVES), 0, s, a);
    else
        hipLaunchKernelGGL((k_i8_stream<OUT, GATED, 4>), dim3(groups, (unsigned)((a.n_tokens + 63) / 64)),
                           dim3(64 * ST_WAVES), 0, s, a);
    return hipGetLastError();
}

template <int OUT>
hipError_t launch_out(const I8Args &a, hipStream_t s) {
    return a.gated ? launch_typed<OUT, true>(a, s) : launch_typed<OUT, false>(a, s);
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
