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
#include "lbh_i8_forms.h"

namespace lbh {

namespace {

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
        // An activation's work behind the products, which the largest tile, alone on its CU,
        // shows twice as much of.  Measured over the product alone: 2048 x 13312 T44 111 us, none
        // 116, silu 130, gelu 135, T22 124, 128, 132, 133; gated 1024 x 13312 T44 117, silu 122, T22 128, 130.
        const float each = a.act == ACT_GELU ? 0.8e-4f : a.act >= ACT_SILU ? 0.6e-4f : 0.3e-4f;
        const float outputs = (float)(f.cw * f.tw) * 4096 / (a.gated ? 2 : 1);
        const float after = a.epilogue ? rounds * outputs * (f.cw == 4 ? 2 * each : each) : 0.0f;
        return 2.0f + wait + after + fmaxf(rounds * (f.fixed + f.step * k), weights);
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
    const int form = a.form ? a.form - 1 : plan(a);
    if (!a.epilogue) return launch_epilogue<EPI_NONE>(a, form, s);
    return a.act == ACT_GELU ? launch_i8_normal(a, form, s) : launch_i8_sigmoid(a, form, s);
}

}  // namespace lbh
