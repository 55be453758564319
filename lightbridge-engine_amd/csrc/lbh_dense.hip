// lbh_dense.hip — host side of the dense-block entry points of
// include/lightbridge_hip.h: RMS norm rows with 8-bit outputs, the 8-bit
// integer matrices and their products.
//
// Every argument is checked before the first launch; a refused call launches
// nothing and leaves its outputs as they were.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>
#include <new>

#include "../../include/lightbridge_hip.h"
#include "lbh_host.h"
#include "lbh_internal.h"
#include "lbh_rowtypes.h"

using namespace lbh;

// 8-bit integer channels in the product's tiles (lbh_i8.hip); gated: the gate's
// and the up's channel groups alternate.
struct lbh_i8_matrix {
    int device;
    size_t rows, k, kt, groups;   // groups: channel groups of one matrix
    int gated;
    uint8_t *tiles;
    float *scales;
    size_t bytes;
};

namespace {

constexpr size_t MAX_TOKENS = (size_t)1 << 20;
constexpr size_t MAX_STRIDE = (size_t)1 << 23;     // 256 rows stay below 2^31 bytes
constexpr size_t MAX_K = 131071;                   // k * 128 * 128 < 2^31: the sums are exact
constexpr size_t MAX_ROWS = (size_t)1 << 26;

bool float_rows_type(int ty) { return row_elem_bytes(ty) != 0; }

// Rows of an operand: `bytes` used bytes of every `pitch`.
struct Span {
    const void *p;
    size_t pitch, bytes, rows;
};
Span span_of(const void *p, size_t stride, size_t elem, size_t cols, size_t rows) {
    return {p, stride * elem, cols * elem, rows};
}

// Whether two operands share a byte.  Rows of one pitch may lie side by side
// in a wider buffer; different pitches are taken by their whole extent.
bool share(const Span &a, const Span &b) {
    if (!a.p || !b.p || !a.rows || !b.rows) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
    const uintptr_t xe = x + (a.rows - 1) * a.pitch + a.bytes, ye = y + (b.rows - 1) * b.pitch + b.bytes;
    if (xe <= y || ye <= x) return false;
    if (a.pitch != b.pitch || a.rows == 1 || b.rows == 1) return true;
    const size_t d = y >= x ? (y - x) % a.pitch : (a.pitch - (x - y) % a.pitch) % a.pitch;
    return d < a.bytes || a.pitch - d < b.bytes;
}
// The same operand twice (an update in place), or no byte in common.
bool same_or_apart(const Span &a, const Span &b) {
    return (a.p == b.p && (a.pitch == b.pitch || a.rows <= 1) && a.bytes == b.bytes) || !share(a, b);
}

bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

lbh_status check_norm(const NormArgs &a, lbh_error *err) {
    const size_t n = (size_t)a.n, rows = (size_t)a.rows;
    struct Op {
        const void *p;
        long long stride;
        int ty;
    } ops[] = {{a.hidden, a.hidden_stride, a.type}, {a.delta, a.delta_stride, a.type},
               {a.hidden_out, a.hidden_out_stride, a.type}, {a.y, a.y_stride, a.y_type}};
    for (int i = 0; i < 4; ++i) {
        if (!ops[i].p) continue;
        if ((size_t)ops[i].stride < n && rows > 1) return fail(err, LBH_DIMENSION_MISMATCH, ops[i].ty, i, n, ops[i].stride);
        if (!aligned_to(ops[i].p, row_elem_bytes(ops[i].ty))) return fail(err, LBH_INVALID_PARAMETER, ops[i].ty, i);
    }
    if (a.q && (size_t)a.q_stride < n && rows > 1) return fail(err, LBH_DIMENSION_MISMATCH, 0, 4, n, a.q_stride);
    if (!aligned_to(a.weight, 4) || !aligned_to(a.scale, 4) || !aligned_to(a.q8k, 4))
        return fail(err, LBH_INVALID_PARAMETER);
    // Outputs share no byte with each other or with an input, but for hidden
    // and delta updated in place.
    const size_t e = row_elem_bytes(a.type);
    const Span hid = span_of(a.hidden, a.hidden_stride, e, n, rows), del = span_of(a.delta, a.delta_stride, e, n, rows),
               ho = span_of(a.hidden_out, a.hidden_out_stride, e, n, rows),
               y = span_of(a.y, a.y_stride, a.y ? row_elem_bytes(a.y_type) : 0, n, rows),
               q = span_of(a.q, a.q_stride, 1, n, rows), q8 = {a.q8k, n / 256 * 292, n / 256 * 292, rows},
               sc = {a.scale, 4, 4, rows}, w = {a.weight, 4 * n, 4 * n, 1};
    const Span outs[] = {ho, y, q, q8, sc};
    for (int i = 0; i < 5; ++i) {
        for (int j = i + 1; j < 5; ++j)
            if (share(outs[i], outs[j])) return fail(err, LBH_INVALID_PARAMETER);
        if (share(outs[i], w)) return fail(err, LBH_INVALID_PARAMETER);
        if (i && (share(outs[i], hid) || share(outs[i], del))) return fail(err, LBH_INVALID_PARAMETER);
    }
    if (!same_or_apart(ho, hid) || !same_or_apart(ho, del)) return fail(err, LBH_INVALID_PARAMETER);
    return LBH_OK;
}

// What the four entry points have in common.
lbh_status norm_rows(lbh_ctx *ctx, NormArgs a, bool outputs_missing, size_t rows, size_t n, size_t hs, size_t ds,
                     size_t os, size_t ys, size_t qs, lbh_error *err) {
    if (!ctx) return fail(err, LBH_NULL_ARGUMENT);
    if (!float_rows_type(a.type)) return fail(err, LBH_UNSUPPORTED_TYPE, a.type);
    if (a.y && !float_rows_type(a.y_type)) return fail(err, LBH_UNSUPPORTED_TYPE, a.y_type);
    if (n == 0) return fail(err, LBH_ZERO_LOGICAL_ELEMENTS, a.type);
    if (a.norm && !(a.eps > 0.0 && a.eps < HUGE_VAL)) return fail(err, LBH_INVALID_PARAMETER, a.type);
    if (n > MAX_STRIDE || rows > MAX_TOKENS) return fail(err, LBH_UNSUPPORTED_SHAPE, a.type, 0, MAX_STRIDE, n);
    for (size_t s : {hs, ds, os, ys, qs})
        if (s > ((size_t)1 << 40)) return fail(err, LBH_UNSUPPORTED_SHAPE, a.type, 0, (size_t)1 << 40, s);
    if (rows == 0) return ok(err);   // no row, and no address asked for
    if (!a.hidden || (a.norm && !a.weight) || outputs_missing) return fail(err, LBH_NULL_ARGUMENT);
    a.rows = (long long)rows;
    a.n = (int32_t)n;
    a.inv_n = 1.0 / (double)n;
    a.hidden_stride = (long long)hs;
    a.delta_stride = (long long)ds;
    a.hidden_out_stride = (long long)os;
    a.y_stride = (long long)ys;
    a.q_stride = (long long)qs;
    const lbh_status st = check_norm(a, err);
    if (st) return st;
    DeviceGuard g(ctx->device);
    HIP_TRY(launch_norm_rows(a, ctx->stream));
    return ok(err);
}

void free_i8(lbh_i8_matrix *m) {
    if (!m) return;
    DeviceGuard g(m->device);
    if (m->tiles) (void)hipFree(m->tiles);
    if (m->scales) (void)hipFree(m->scales);
    delete m;
}

lbh_status check_i8_shape(size_t rows, size_t k, lbh_error *err) {
    if (k == 0) return fail(err, LBH_ZERO_LOGICAL_ELEMENTS);
    if (rows == 0) return fail(err, LBH_DIMENSION_MISMATCH, 0, 0, 1, 0);
    if (k > MAX_K) return fail(err, LBH_UNSUPPORTED_SHAPE, 0, 0, MAX_K, k);
    if (rows > MAX_ROWS) return fail(err, LBH_UNSUPPORTED_SHAPE, 0, 1, MAX_ROWS, rows);
    return LBH_OK;
}

// An empty matrix of the shape: tiles and scales allocated.
lbh_status alloc_i8(lbh_ctx *ctx, size_t rows, size_t k, int gated, lbh_i8_matrix **out, lbh_error *err) {
    lbh_i8_matrix *m = new (std::nothrow) lbh_i8_matrix();
    if (!m) return fail(err, LBH_HIP_ERROR);
    m->device = ctx->device;
    m->rows = rows;
    m->k = k;
    m->kt = (k + 255) / 256 * 4;
    m->groups = (rows + 15) / 16;
    m->gated = gated;
    const size_t all = m->groups * (gated ? 2 : 1), tb = all * m->kt * 1024, sb = all * 16 * sizeof(float);
    m->bytes = tb + sb;
    hipError_t e = hipMalloc(&m->tiles, tb);
    if (e == hipSuccess) e = hipMalloc(&m->scales, sb);
    if (e != hipSuccess) {
        free_i8(m);
        return hip_fail(err, e);
    }
    *out = m;
    return LBH_OK;
}

// Scales of one matrix, finite, on the device.
lbh_status check_i8_scales(lbh_ctx *ctx, const float *scales, size_t rows, uint32_t which, lbh_error *err) {
    HIP_TRY(launch_reset_status(ctx->status, ctx->stream));
    HIP_TRY(launch_find_nonfinite(scales, (long long)rows, &ctx->status->first_bad_scale, ctx->stream));
    HIP_TRY(hipMemcpyAsync(ctx->status_host, ctx->status, sizeof(DevStatus), hipMemcpyDeviceToHost, ctx->stream));
    HIP_TRY(hipStreamSynchronize(ctx->stream));
    const unsigned long long bad = ctx->status_host->first_bad_scale;
    if (bad == ~0ull) return LBH_OK;
    uint32_t bits = 0;
    HIP_TRY(hipMemcpy(&bits, scales + bad, 4, hipMemcpyDeviceToHost));
    return fail(err, LBH_NON_FINITE_SCALE, 0, 0, 0, 0, bits, which, bad);
}

// Device memory of one creation call, released on every way out.
struct Temp {
    void *p = nullptr;
    hipError_t get(size_t n) { return hipMalloc(&p, n); }
    ~Temp() {
        if (p) (void)hipFree(p);
    }
};

lbh_status create_i8(lbh_ctx *ctx, const int8_t *const *w, const float *const *scales, int parts, size_t rows, size_t k,
                     int on_device, lbh_i8_matrix **out, lbh_error *err) {
    if (!ctx || !out) return fail(err, LBH_NULL_ARGUMENT);
    *out = nullptr;
    for (int i = 0; i < parts; ++i)
        if (!w[i] || !scales[i]) return fail(err, LBH_NULL_ARGUMENT);
    for (int i = 0; i < parts; ++i)
        if (on_device && !aligned_to(scales[i], 4)) return fail(err, LBH_INVALID_PARAMETER);
    lbh_status st = check_i8_shape(rows, k, err);
    if (st) return st;
    DeviceGuard g(ctx->device);
    lbh_i8_matrix *m = nullptr;
    st = alloc_i8(ctx, rows, k, parts == 2, &m, err);
    if (st) return st;
    auto fill = [&]() -> lbh_status {
        for (int i = 0; i < parts; ++i) {
            Temp tw, ts;
            const int8_t *src = w[i];
            const float *sc = scales[i];
            if (!on_device) {
                HIP_TRY(tw.get(rows * k));
                HIP_TRY(ts.get(rows * sizeof(float)));
                HIP_TRY(hipMemcpyAsync(tw.p, w[i], rows * k, hipMemcpyHostToDevice, ctx->stream));
                HIP_TRY(hipMemcpyAsync(ts.p, scales[i], rows * sizeof(float), hipMemcpyHostToDevice, ctx->stream));
                src = static_cast<const int8_t *>(tw.p);
                sc = static_cast<const float *>(ts.p);
            }
            const lbh_status s2 = check_i8_scales(ctx, sc, rows, (uint32_t)i, err);
            if (s2) return s2;
            HIP_TRY(launch_i8_layout(src, m->tiles, sc, m->scales, (long long)rows, (long long)k, (long long)m->kt,
                                     parts, i, 1, ctx->stream));
            HIP_TRY(hipStreamSynchronize(ctx->stream));
        }
        return LBH_OK;
    };
    st = fill();
    if (st) {
        free_i8(m);
        return st;
    }
    *out = m;
    return ok(err);
}

lbh_status product(lbh_ctx *ctx, const lbh_i8_matrix *m, int gated, const int8_t *x, size_t x_stride, const float *xs,
                   size_t n_tokens, int32_t y_type, void *y, size_t y_stride, const void *residual,
                   size_t residual_stride, void *workspace, size_t workspace_len, lbh_error *err) {
    if (!ctx || !m) return fail(err, LBH_NULL_ARGUMENT);
    if (m->gated != gated || m->device != ctx->device) return fail(err, LBH_INVALID_PARAMETER, y_type);
    const size_t e = row_elem_bytes(y_type);
    if (!e) return fail(err, LBH_UNSUPPORTED_TYPE, y_type);
    if (n_tokens == 0) return ok(err);   // no token, and no address asked for
    if (!x || !xs || !y) return fail(err, LBH_NULL_ARGUMENT);
    if (n_tokens > MAX_TOKENS) return fail(err, LBH_UNSUPPORTED_SHAPE, y_type, 0, MAX_TOKENS, n_tokens);
    if (n_tokens == 1) x_stride = m->k, y_stride = m->rows, residual_stride = m->rows;
    if (x_stride < m->k) return fail(err, LBH_DIMENSION_MISMATCH, y_type, 0, m->k, x_stride);
    if (y_stride < m->rows) return fail(err, LBH_DIMENSION_MISMATCH, y_type, 1, m->rows, y_stride);
    if (residual && residual_stride < m->rows)
        return fail(err, LBH_DIMENSION_MISMATCH, y_type, 2, m->rows, residual_stride);
    if (x_stride > MAX_STRIDE || y_stride > ((size_t)1 << 40) || (residual && residual_stride > ((size_t)1 << 40)))
        return fail(err, LBH_UNSUPPORTED_SHAPE, y_type, 0, MAX_STRIDE, x_stride);
    if (!aligned_to(xs, 4) || !aligned_to(y, e) || (residual && !aligned_to(residual, e)))
        return fail(err, LBH_INVALID_PARAMETER, y_type);
    const Span sy = span_of(y, y_stride, e, m->rows, n_tokens), sx = span_of(x, x_stride, 1, m->k, n_tokens),
               ss = {xs, 4, 4, n_tokens}, sr = span_of(residual, residual_stride, e, m->rows, n_tokens);
    if (share(sy, sx) || share(sy, ss) || !same_or_apart(sy, sr)) return fail(err, LBH_INVALID_PARAMETER, y_type);
    DeviceGuard g(ctx->device);
    I8Args a{};
    a.w = m->tiles;
    a.ws = m->scales;
    a.x = x;
    a.xs = xs;
    a.y = y;
    a.residual = residual;
    a.x_stride = (long long)x_stride;
    a.y_stride = (long long)y_stride;
    a.residual_stride = (long long)residual_stride;
    a.n_tokens = (int32_t)n_tokens;
    a.rows = (int32_t)m->rows;
    a.k = (int32_t)m->k;
    a.kt = (int32_t)m->kt;
    a.out_type = y_type;
    a.gated = gated;
    a.cu_count = ctx->cu_count;
    a.form = ctx->i8_form;
    a.vec_out = aligned_to(y, 16) && y_stride * e % 16 == 0 &&
                (!residual || (aligned_to(residual, 16) && residual_stride * e % 16 == 0));
    if (!aligned_to(x, 16) || x_stride % 16 || m->k % 16) {
        // The kernels read rows as 16-byte words: such rows go to the workspace first.
        const size_t pitch = m->kt * 64, need = n_tokens * pitch;
        if (!workspace) return fail(err, LBH_NULL_ARGUMENT);
        if (!aligned_to(workspace, 16)) return fail(err, LBH_INVALID_PARAMETER);
        if (workspace_len < need) return fail(err, LBH_SCRATCH_TOO_SMALL, 0, n_tokens, need, workspace_len);
        const Span sw = {workspace, need, need, 1};
        if (share(sw, sx) || share(sw, ss) || share(sw, sy) || share(sw, sr)) return fail(err, LBH_INVALID_PARAMETER, y_type);
        HIP_TRY(launch_i8_align_rows(x, a.x_stride, a.k, (int)pitch, (long long)n_tokens,
                                     static_cast<uint8_t *>(workspace), ctx->stream));
        a.x = static_cast<const int8_t *>(workspace);
        a.x_stride = (long long)pitch;
        a.k = (int32_t)pitch;
    }
    HIP_TRY(launch_i8_product(a, ctx->stream));
    return ok(err);
}

}  // namespace

extern "C" {

lbh_status lbh_rms_norm_rows(lbh_ctx *ctx, int32_t type, const void *hidden, size_t hidden_stride, const void *delta,
                             size_t delta_stride, const float *weight, double eps, size_t rows, size_t n,
                             void *hidden_out, size_t hidden_out_stride, int32_t y_type, void *y, size_t y_stride,
                             lbh_error *err) {
    NormArgs a{};
    a.hidden = hidden, a.delta = delta, a.hidden_out = hidden_out, a.weight = weight, a.y = y;
    a.type = type, a.y_type = y_type, a.norm = 1, a.eps = eps;
    return norm_rows(ctx, a, !y, rows, n, hidden_stride, delta_stride, hidden_out_stride, y_stride, 0, err);
}

lbh_status lbh_rms_norm_q8_k_rows(lbh_ctx *ctx, int32_t type, const void *hidden, size_t hidden_stride,
                                  const void *delta, size_t delta_stride, const float *weight, double eps, size_t rows,
                                  size_t n, void *hidden_out, size_t hidden_out_stride, int32_t y_type, void *y,
                                  size_t y_stride, uint8_t *encoded, lbh_error *err) {
    if (!ctx) return fail(err, LBH_NULL_ARGUMENT);
    if (n % 256) return fail(err, LBH_LOGICAL_ELEMENTS_NOT_DIVISIBLE, LBH_Q8_K, 0, 256, n);
    if (n > (size_t)NORM_MAX_Q8K) return fail(err, LBH_UNSUPPORTED_SHAPE, LBH_Q8_K, 0, NORM_MAX_Q8K, n);
    NormArgs a{};
    a.hidden = hidden, a.delta = delta, a.hidden_out = hidden_out, a.weight = weight, a.y = y, a.q8k = encoded;
    a.type = type, a.y_type = y_type, a.norm = 1, a.eps = eps;
    return norm_rows(ctx, a, !encoded, rows, n, hidden_stride, delta_stride, hidden_out_stride, y_stride, 0, err);
}

lbh_status lbh_rms_norm_i8_rows(lbh_ctx *ctx, int32_t type, const void *hidden, size_t hidden_stride, const void *delta,
                                size_t delta_stride, const float *weight, double eps, size_t rows, size_t n,
                                void *hidden_out, size_t hidden_out_stride, int32_t y_type, void *y, size_t y_stride,
                                int8_t *q, size_t q_stride, float *scales, lbh_error *err) {
    NormArgs a{};
    a.hidden = hidden, a.delta = delta, a.hidden_out = hidden_out, a.weight = weight, a.y = y, a.q = q, a.scale = scales;
    a.type = type, a.y_type = y_type, a.norm = 1, a.eps = eps;
    return norm_rows(ctx, a, !q || !scales, rows, n, hidden_stride, delta_stride, hidden_out_stride, y_stride, q_stride,
                     err);
}

lbh_status lbh_quantize_i8_rows(lbh_ctx *ctx, int32_t type, const void *x, size_t x_stride, size_t rows, size_t n,
                                int8_t *q, size_t q_stride, float *scales, lbh_error *err) {
    NormArgs a{};
    a.hidden = x, a.q = q, a.scale = scales, a.type = type;
    return norm_rows(ctx, a, !q || !scales, rows, n, x_stride, 0, 0, 0, q_stride, err);
}

lbh_status lbh_i8_matrix_create(lbh_ctx *ctx, size_t rows, size_t k, const int8_t *weights, const float *scales,
                                int32_t on_device, lbh_i8_matrix **out, lbh_error *err) {
    return create_i8(ctx, &weights, &scales, 1, rows, k, on_device, out, err);
}

lbh_status lbh_i8_matrix_create_gated(lbh_ctx *ctx, size_t rows, size_t k, const int8_t *gate, const float *gate_scales,
                                      const int8_t *up, const float *up_scales, int32_t on_device, lbh_i8_matrix **out,
                                      lbh_error *err) {
    const int8_t *w[2] = {gate, up};
    const float *s[2] = {gate_scales, up_scales};
    return create_i8(ctx, w, s, 2, rows, k, on_device, out, err);
}

lbh_status lbh_i8_matrix_from_packed(lbh_ctx *ctx, const lbh_matrix *m, const lbh_matrix *up, lbh_i8_matrix **out,
                                     lbh_error *err) {
    if (!ctx || !out) return fail(err, LBH_NULL_ARGUMENT);
    *out = nullptr;
    if (!m) return fail(err, LBH_NULL_ARGUMENT);
    const lbh_matrix *src[2] = {m, up};
    const int parts = up ? 2 : 1;
    for (int i = 0; i < parts; ++i) {
        if (src[i]->device != ctx->device) return fail(err, LBH_INVALID_PARAMETER, src[i]->type);
        if (src[i]->type != LBH_F32 && !is_dot_type(src[i]->type)) return fail(err, LBH_UNSUPPORTED_TYPE, src[i]->type);
        if (src[i]->rows != m->rows) return fail(err, LBH_DIMENSION_MISMATCH, src[i]->type, 0, m->rows, src[i]->rows);
        if (src[i]->k != m->k) return fail(err, LBH_DIMENSION_MISMATCH, src[i]->type, 1, m->k, src[i]->k);
    }
    const size_t rows = m->rows, k = m->k;
    lbh_status st = check_i8_shape(rows, k, err);
    if (st) return st;
    DeviceGuard g(ctx->device);
    lbh_i8_matrix *q = nullptr;
    st = alloc_i8(ctx, rows, k, parts == 2, &q, err);
    if (st) return st;
    auto fill = [&]() -> lbh_status {
        // Rows decoded 64 MiB at a time (2^16 rows at most: k is 256 or more), quantized, then laid
        // out together.
        for (int i = 0; i < parts; ++i) {
            const lbh_matrix *s = src[i];
            size_t chunk = ((size_t)64 << 20) / (k * sizeof(float));
            chunk = chunk > rows ? rows : chunk;
            Temp values, codes, scales;
            HIP_TRY(values.get(chunk * k * sizeof(float)));
            HIP_TRY(codes.get(rows * k));
            HIP_TRY(scales.get(rows * sizeof(float)));
            MatView v{s->planes, s->type, (int32_t)s->nb, (int32_t)s->rows, MAT_ROW_MAJOR, (long long)(s->rows * s->nb),
                      (long long)s->bytes};
            for (size_t r0 = 0; r0 < rows; r0 += chunk) {
                const size_t n = rows - r0 < chunk ? rows - r0 : chunk;
                float *f = static_cast<float *>(values.p);
                if (s->type == LBH_F32)
                    HIP_TRY(launch_f32_rows(reinterpret_cast<const float *>(s->planes), (long long)rows, (long long)k,
                                            (long long)r0, (long long)n, f, ctx->stream));
                else
                    HIP_TRY(launch_dequant_rows(v, (long long)r0, (long long)n, f, ctx->stream));
                NormArgs a{};
                a.hidden = f, a.hidden_stride = (long long)k, a.type = T_F32;
                a.q = static_cast<int8_t *>(codes.p) + r0 * k, a.q_stride = (long long)k;
                a.scale = static_cast<float *>(scales.p) + r0, a.rows = (long long)n, a.n = (int32_t)k;
                HIP_TRY(launch_norm_rows(a, ctx->stream));
            }
            const float *sc = static_cast<const float *>(scales.p);
            const lbh_status s2 = check_i8_scales(ctx, sc, rows, (uint32_t)i, err);
            if (s2) return s2;
            HIP_TRY(launch_i8_layout(static_cast<const int8_t *>(codes.p), q->tiles, sc, q->scales, (long long)rows,
                                     (long long)k, (long long)q->kt, parts, i, 1, ctx->stream));
            HIP_TRY(hipStreamSynchronize(ctx->stream));
        }
        return LBH_OK;
    };
    st = fill();
    if (st) {
        free_i8(q);
        return st;
    }
    *out = q;
    return ok(err);
}

lbh_status lbh_i8_matrix_destroy(lbh_i8_matrix *m) {
    free_i8(m);
    return LBH_OK;
}

lbh_status lbh_i8_matrix_read(lbh_ctx *ctx, const lbh_i8_matrix *m, int32_t which, int8_t *weights_host,
                              size_t weights_len, float *scales_host, size_t scales_len, lbh_error *err) {
    if (!ctx || !m || !weights_host || !scales_host) return fail(err, LBH_NULL_ARGUMENT);
    if (which < 0 || which > m->gated || m->device != ctx->device) return fail(err, LBH_INVALID_PARAMETER);
    if (weights_len != m->rows * m->k) return fail(err, LBH_OUTPUT_LENGTH_MISMATCH, 0, 0, m->rows * m->k, weights_len);
    if (scales_len != m->rows) return fail(err, LBH_OUTPUT_LENGTH_MISMATCH, 0, 1, m->rows, scales_len);
    DeviceGuard g(ctx->device);
    Temp w, s;
    HIP_TRY(w.get(m->rows * m->k));
    HIP_TRY(s.get(m->rows * sizeof(float)));
    HIP_TRY(launch_i8_layout(static_cast<int8_t *>(w.p), m->tiles, static_cast<float *>(s.p), m->scales,
                             (long long)m->rows, (long long)m->k, (long long)m->kt, m->gated ? 2 : 1, which, 0,
                             ctx->stream));
    HIP_TRY(hipMemcpyAsync(weights_host, w.p, m->rows * m->k, hipMemcpyDeviceToHost, ctx->stream));
    HIP_TRY(hipMemcpyAsync(scales_host, s.p, m->rows * sizeof(float), hipMemcpyDeviceToHost, ctx->stream));
    HIP_TRY(hipStreamSynchronize(ctx->stream));
    return ok(err);
}

size_t lbh_i8_matrix_rows(const lbh_i8_matrix *m) { return m ? m->rows : 0; }
size_t lbh_i8_matrix_k(const lbh_i8_matrix *m) { return m ? m->k : 0; }
int32_t lbh_i8_matrix_gated(const lbh_i8_matrix *m) { return m ? m->gated : 0; }
size_t lbh_i8_matrix_device_bytes(const lbh_i8_matrix *m) { return m ? m->bytes : 0; }

size_t lbh_gemm_i8_workspace_bytes(const lbh_i8_matrix *m, size_t n_tokens) {
    return m && n_tokens <= MAX_TOKENS ? n_tokens * m->kt * 64 : 0;
}

lbh_status lbh_gemm_i8(lbh_ctx *ctx, const lbh_i8_matrix *m, const int8_t *x, size_t x_stride, const float *x_scales,
                       size_t n_tokens, int32_t y_type, void *y, size_t y_stride, const void *residual,
                       size_t residual_stride, void *workspace, size_t workspace_len, lbh_error *err) {
    return product(ctx, m, 0, x, x_stride, x_scales, n_tokens, y_type, y, y_stride, residual, residual_stride, workspace,
                   workspace_len, err);
}

lbh_status lbh_gemm_i8_swiglu(lbh_ctx *ctx, const lbh_i8_matrix *m, const int8_t *x, size_t x_stride,
                              const float *x_scales, size_t n_tokens, int32_t h_type, void *h, size_t h_stride,
                              void *workspace, size_t workspace_len, lbh_error *err) {
    return product(ctx, m, 1, x, x_stride, x_scales, n_tokens, h_type, h, h_stride, nullptr, 0, workspace, workspace_len,
                   err);
}

}  // extern "C"
