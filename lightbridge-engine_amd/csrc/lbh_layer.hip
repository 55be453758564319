// lbh_layer.hip — host side of the entry points around a layer's experts in
// 8-bit integers (include/lightbridge_hip.h): the norms around a block, the
// routing of rows, the int8 experts.
//
// Every argument is checked before the first launch; a refused call launches
// nothing and leaves its outputs as they were.
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstring>
#include <new>

#include "../../include/lightbridge_hip.h"
#include "lbh_host.h"
#include "lbh_internal.h"
#include "lbh_operands.h"
#include "lbh_rowtypes.h"

using namespace lbh;

// Experts of one layer: the tables of their matrices, which stay the caller's.
struct lbh_moe_i8 {
    int device;
    size_t n_experts, n, ffn, ffn_s;   // ffn_s == 0: no shared expert
    size_t kt_n, kt_f, kt_fs, down_pitch;
    ExpertI8 *experts;                 // device
    ExpertI8 shared;
    float *down_scales;                // device, [n_experts][down_pitch]
};

namespace {

constexpr size_t MAX_PITCH = (size_t)1 << 40;
constexpr size_t MAX_ROUTE_TOKENS = (size_t)1 << 19;

size_t up16(size_t n) { return (n + 15) / 16 * 16; }

// An operand's rows.
struct Rows {
    const void *p;
    size_t stride, elem, cols;
};

lbh_status check_rows(const Rows *r, int n, size_t rows, int ty, lbh_error *err) {
    for (int i = 0; i < n; ++i) {
        if (r[i].stride > MAX_PITCH) return fail(err, LBH_UNSUPPORTED_SHAPE, ty, i, MAX_PITCH, r[i].stride);
        if (!r[i].p) continue;
        if (r[i].stride < r[i].cols && rows > 1) return fail(err, LBH_DIMENSION_MISMATCH, ty, i, r[i].cols, r[i].stride);
        if (!aligned_to(r[i].p, r[i].elem)) return fail(err, LBH_INVALID_PARAMETER, ty, i);
    }
    return LBH_OK;
}
Span span_of(const Rows &r, size_t rows) { return span_of(r.p, r.stride, r.elem, r.cols, rows); }

void free_moe_i8(lbh_moe_i8 *m) {
    if (!m) return;
    DeviceGuard g(m->device);
    if (m->experts) (void)hipFree(m->experts);
    if (m->down_scales) (void)hipFree(m->down_scales);
    delete m;
}

// A gated pair [ffn][n] and its down matrix [n][ffn].
lbh_status check_expert(const lbh_ctx *ctx, const lbh_i8_matrix *up, const lbh_i8_matrix *down, size_t n, size_t ffn,
                        size_t which, lbh_error *err) {
    if (!up || !down) return fail(err, LBH_NULL_ARGUMENT, 0, which);
    if (up->device != ctx->device || down->device != ctx->device || !up->gated || down->gated)
        return fail(err, LBH_INVALID_PARAMETER, 0, which);
    if (up->k != n) return fail(err, LBH_DIMENSION_MISMATCH, 0, which, n, up->k);
    if (up->rows != ffn) return fail(err, LBH_DIMENSION_MISMATCH, 0, which, ffn, up->rows);
    if (down->rows != n) return fail(err, LBH_DIMENSION_MISMATCH, 0, which, n, down->rows);
    if (down->k != ffn) return fail(err, LBH_DIMENSION_MISMATCH, 0, which, ffn, down->k);
    if (n > 131071 || ffn > 131071) return fail(err, LBH_UNSUPPORTED_SHAPE, 0, which, 131071, n > ffn ? n : ffn);
    return LBH_OK;
}

// The workspace's parts, each on 256 bytes.
struct ExpertsSpace {
    size_t plan, x, h, h_s, hq, hq_s, scales, bytes;
    ExpertsSpace(const lbh_moe_i8 &m, size_t tokens, size_t top_k) {
        const size_t pairs = tokens * top_k;
        bytes = 0;
        auto part = [&](size_t n) {
            const size_t at = bytes;
            bytes += (n + 255) / 256 * 256;
            return at;
        };
        plan = part(sizeof(ExpertsPlan));
        x = part(tokens * m.kt_n * 64);
        h = part(pairs * up16(m.ffn) * 4);
        h_s = part(m.ffn_s ? tokens * up16(m.ffn_s) * 4 : 0);
        hq = part(pairs * m.kt_f * 64);
        hq_s = part(m.ffn_s ? tokens * m.kt_fs * 64 : 0);
        scales = part((pairs + tokens) * 4);
    }
};
bool experts_shape(size_t tokens, size_t top_k) {
    return tokens <= (size_t)EXPERTS_MAX_TOKENS && top_k >= 1 && top_k <= (size_t)MOE_MAX_ROUTED &&
           tokens * top_k <= (size_t)EXPERTS_MAX_PAIRS;
}

}  // namespace

extern "C" {

lbh_status lbh_block_norm_rows(lbh_ctx *ctx, int32_t type, const void *block, size_t block_stride,
                               const float *post_weight, double post_eps, const void *gate, size_t gate_stride,
                               int32_t gate_act, double scale, const void *hidden, size_t hidden_stride,
                               void *hidden_out, size_t hidden_out_stride, const float *weight, double eps, size_t rows,
                               size_t n, int32_t y_type, void *y, size_t y_stride, int8_t *q, size_t q_stride,
                               float *scales, uint8_t *encoded, lbh_error *err) {
    if (!ctx) return fail(err, LBH_NULL_ARGUMENT);
    const size_t e = row_elem_bytes(type);
    if (!e) return fail(err, LBH_UNSUPPORTED_TYPE, type);
    if (y && !row_elem_bytes(y_type)) return fail(err, LBH_UNSUPPORTED_TYPE, y_type);
    if (n == 0) return fail(err, LBH_ZERO_LOGICAL_ELEMENTS, type);
    if (n > (size_t)BLOCK_NORM_MAX) return fail(err, LBH_UNSUPPORTED_SHAPE, type, 0, BLOCK_NORM_MAX, n);
    if (rows > MAX_TOKENS) return fail(err, LBH_UNSUPPORTED_SHAPE, type, 0, MAX_TOKENS, rows);
    if (encoded && n % 256) return fail(err, LBH_LOGICAL_ELEMENTS_NOT_DIVISIBLE, LBH_Q8_K, 0, 256, n);
    // (a scale beyond the float range times 1 / sqrt(post_eps) could be infinite, and zeros NaN)
    if (!(std::fabs(scale) <= FLT_MAX) || gate_act < GATE_AS_IS || gate_act > GATE_SILU || (!gate && gate_act) ||
        (post_weight && !(post_eps > 0.0 && post_eps < HUGE_VAL)) || (weight && !(eps > 0.0 && eps < HUGE_VAL)))
        return fail(err, LBH_INVALID_PARAMETER, type);
    const bool outputs = y || q || scales || encoded;
    if (rows == 0) return ok(err);   // no row, and no address asked for
    if (!block || !hidden || !hidden_out || !q != !scales || (weight != nullptr) != outputs)
        return fail(err, LBH_NULL_ARGUMENT, type);
    const bool one_gate = gate && gate_stride == 0;   // one row of gates for every row
    const Rows ops[] = {{block, block_stride, e, n}, {hidden, hidden_stride, e, n},
                        {gate, one_gate ? n : gate_stride, e, n}, {hidden_out, hidden_out_stride, e, n},
                        {y, y_stride, y ? (size_t)row_elem_bytes(y_type) : 1, n}, {q, q_stride, 1, n}};
    const lbh_status st = check_rows(ops, 6, rows, type, err);
    if (st) return st;
    if (!aligned_to(post_weight, 4) || !aligned_to(weight, 4) || !aligned_to(scales, 4) || !aligned_to(encoded, 4))
        return fail(err, LBH_INVALID_PARAMETER, type);
    // Outputs share no byte with each other or with an input, but for the stream
    // over hidden or the block's output.
    const size_t blocks = encoded ? n / 256 * 292 : 0;
    const Span ins[] = {span_of(ops[0], rows), span_of(ops[1], rows), span_of(ops[2], one_gate ? 1 : rows),
                        {post_weight, 4 * n, 4 * n, 1}, {weight, 4 * n, 4 * n, 1}};
    const Span outs[] = {span_of(ops[3], rows), span_of(ops[4], rows), span_of(ops[5], rows), {encoded, blocks, blocks, rows},
                         {scales, 4, 4, rows}};
    for (int i = 0; i < 5; ++i) {
        for (int j = i + 1; j < 5; ++j)
            if (share(outs[i], outs[j])) return fail(err, LBH_INVALID_PARAMETER, type);
        for (int j = 0; j < 5; ++j)
            if (i == 0 && j < 2 ? !same_or_apart(outs[i], ins[j]) : share(outs[i], ins[j]))
                return fail(err, LBH_INVALID_PARAMETER, type);
    }
    BlockNormArgs a{};
    a.block = block, a.hidden = hidden, a.gate = gate, a.hidden_out = hidden_out, a.post_weight = post_weight;
    a.weight = weight, a.y = y, a.q8k = encoded, a.q = q, a.scales = scales;
    a.block_stride = (long long)block_stride, a.hidden_stride = (long long)hidden_stride;
    a.gate_stride = (long long)gate_stride, a.hidden_out_stride = (long long)hidden_out_stride;
    a.y_stride = (long long)y_stride, a.q_stride = (long long)q_stride;
    a.rows = (long long)rows, a.n = (int32_t)n, a.type = type, a.y_type = y_type, a.gate_act = gate_act;
    a.post_eps = post_eps, a.eps = eps, a.inv_n = 1.0 / (double)n, a.scale = scale;
    DeviceGuard g(ctx->device);
    HIP_TRY(launch_block_norm(a, ctx->stream));
    return ok(err);
}

size_t lbh_router_route_rows_workspace_bytes(const lbh_router *r, size_t n_tokens) {
    if (!r || n_tokens > MAX_ROUTE_TOKENS) return 0;
    return (size_t)route_parts((long long)n_tokens) * n_tokens * r->n_experts * sizeof(double);
}

size_t lbh_router_route_rows_workspace_bytes_up_to(const lbh_router *r, size_t n_tokens) {
    if (!r || n_tokens > MAX_ROUTE_TOKENS) return 0;
    // Rows have as many parts up to ROUTE_FEW as they ever have, and fewer behind it: the most is at one of the two ends.
    const size_t few = n_tokens < (size_t)ROUTE_FEW ? n_tokens : (size_t)ROUTE_FEW;
    const size_t all = lbh_router_route_rows_workspace_bytes(r, n_tokens), most = lbh_router_route_rows_workspace_bytes(r, few);
    return all > most ? all : most;
}

lbh_status lbh_router_route_rows(lbh_ctx *ctx, const lbh_router *r, int32_t type, const void *x, size_t x_stride,
                                 size_t n_tokens, size_t top_k, int32_t mode, double weight_scale, uint32_t *ids,
                                 float *coefs, float *logits, void *workspace, size_t workspace_len, lbh_error *err) {
    if (!ctx || !r) return fail(err, LBH_NULL_ARGUMENT);
    const size_t e = row_elem_bytes(type);
    if (!e) return fail(err, LBH_UNSUPPORTED_TYPE, type);
    if (r->device != ctx->device || (mode != 0 && mode != 1) || !std::isfinite(weight_scale))
        return fail(err, LBH_INVALID_PARAMETER, type);
    if (mode == 1 && !r->bias) return fail(err, LBH_NULL_ARGUMENT, type);
    if (top_k == 0 || top_k > r->n_experts || top_k > (size_t)MOE_MAX_ROUTED)
        return fail(err, LBH_UNSUPPORTED_SHAPE, type, 0, r->n_experts < (size_t)MOE_MAX_ROUTED ? r->n_experts : MOE_MAX_ROUTED, top_k);
    if (n_tokens > MAX_ROUTE_TOKENS) return fail(err, LBH_UNSUPPORTED_SHAPE, type, 1, MAX_ROUTE_TOKENS, n_tokens);
    if (n_tokens == 0) return ok(err);
    if (!x || !ids || !coefs || !workspace) return fail(err, LBH_NULL_ARGUMENT, type);
    const Rows rows = {x, x_stride, e, r->hidden};
    const lbh_status st = check_rows(&rows, 1, n_tokens, type, err);
    if (st) return st;
    if (!aligned_to(ids, 4) || !aligned_to(coefs, 4) || !aligned_to(logits, 4) || !aligned_to(workspace, 8))
        return fail(err, LBH_INVALID_PARAMETER, type);
    const size_t need = lbh_router_route_rows_workspace_bytes(r, n_tokens);
    if (workspace_len < need) return fail(err, LBH_SCRATCH_TOO_SMALL, type, n_tokens, need, workspace_len);
    const size_t routes = n_tokens * top_k * 4, all = n_tokens * r->n_experts * 4;
    const Span in = span_of(rows, n_tokens);
    const Span outs[] = {{ids, routes, routes, 1}, {coefs, routes, routes, 1}, {logits, all, all, 1}, {workspace, need, need, 1}};
    for (int i = 0; i < 4; ++i) {
        if (share(outs[i], in)) return fail(err, LBH_INVALID_PARAMETER, type);
        for (int j = i + 1; j < 4; ++j)
            if (share(outs[i], outs[j])) return fail(err, LBH_INVALID_PARAMETER, type);
    }
    RouteRowsArgs a{};
    a.w = r->w, a.bias = r->bias, a.x = x, a.x_stride = (long long)x_stride, a.part = static_cast<double *>(workspace);
    a.ids = ids, a.coefs = coefs, a.logits = logits, a.weight_scale = weight_scale;
    a.n_tokens = (int32_t)n_tokens, a.n_experts = (int32_t)r->n_experts, a.hidden = (int32_t)r->hidden;
    a.top_k = (int32_t)top_k, a.mode = mode, a.x_type = type;
    DeviceGuard g(ctx->device);
    HIP_TRY(launch_route_rows(a, ctx->stream));
    return ok(err);
}

lbh_status lbh_moe_i8_create(lbh_ctx *ctx, const lbh_i8_matrix *const *gate_up, const lbh_i8_matrix *const *down,
                             size_t n_experts, const lbh_i8_matrix *shared_gate_up, const lbh_i8_matrix *shared_down,
                             lbh_moe_i8 **out, lbh_error *err) {
    if (!ctx || !out) return fail(err, LBH_NULL_ARGUMENT);
    *out = nullptr;
    if (n_experts == 0) return fail(err, LBH_DIMENSION_MISMATCH, 0, 0, 1, 0);
    if (n_experts > (size_t)EXPERTS_MAX) return fail(err, LBH_UNSUPPORTED_SHAPE, 0, 0, EXPERTS_MAX, n_experts);
    if (!gate_up || !down || !gate_up[0] || !shared_gate_up != !shared_down) return fail(err, LBH_NULL_ARGUMENT);
    const size_t n = gate_up[0]->k, ffn = gate_up[0]->rows;
    lbh_status st;
    for (size_t i = 0; i < n_experts; ++i)
        if ((st = check_expert(ctx, gate_up[i], down[i], n, ffn, i, err))) return st;
    if (shared_gate_up && (st = check_expert(ctx, shared_gate_up, shared_down, n, shared_gate_up->rows, n_experts, err)))
        return st;
    DeviceGuard g(ctx->device);
    lbh_moe_i8 *m = new (std::nothrow) lbh_moe_i8();
    ExpertI8 *table = new (std::nothrow) ExpertI8[n_experts];
    if (!m || !table) {
        delete m;
        delete[] table;
        return fail(err, LBH_HIP_ERROR);
    }
    auto view = [](const lbh_i8_matrix *up, const lbh_i8_matrix *dn) {
        return ExpertI8{up->tiles, dn->tiles, up->scales, dn->scales};
    };
    for (size_t i = 0; i < n_experts; ++i) table[i] = view(gate_up[i], down[i]);
    m->device = ctx->device, m->n_experts = n_experts, m->n = n, m->ffn = ffn;
    m->kt_n = gate_up[0]->kt, m->kt_f = down[0]->kt, m->down_pitch = up16(n);
    if (shared_gate_up) {
        m->ffn_s = shared_gate_up->rows, m->kt_fs = shared_down->kt;
        m->shared = view(shared_gate_up, shared_down);
    }
    auto fill = [&]() -> lbh_status {
        HIP_TRY(hipMalloc(&m->experts, n_experts * sizeof(ExpertI8)));
        HIP_TRY(hipMalloc(&m->down_scales, n_experts * m->down_pitch * sizeof(float)));
        HIP_TRY(hipMemcpyAsync(m->experts, table, n_experts * sizeof(ExpertI8), hipMemcpyHostToDevice, ctx->stream));
        for (size_t i = 0; i < n_experts; ++i)
            HIP_TRY(hipMemcpyAsync(m->down_scales + i * m->down_pitch, down[i]->scales, m->down_pitch * sizeof(float),
                                   hipMemcpyDeviceToDevice, ctx->stream));
        HIP_TRY(hipStreamSynchronize(ctx->stream));
        return LBH_OK;
    };
    st = fill();
    delete[] table;
    if (st) {
        free_moe_i8(m);
        return st;
    }
    *out = m;
    return ok(err);
}

lbh_status lbh_moe_i8_destroy(lbh_moe_i8 *m) {
    free_moe_i8(m);
    return LBH_OK;
}

size_t lbh_moe_i8_workspace_bytes(const lbh_moe_i8 *m, size_t n_tokens, size_t top_k) {
    return m && n_tokens && experts_shape(n_tokens, top_k) ? ExpertsSpace(*m, n_tokens, top_k).bytes : 0;
}

lbh_status lbh_moe_i8_forward(lbh_ctx *ctx, const lbh_moe_i8 *m, const int8_t *x, size_t x_stride, const float *x_scales,
                              const uint32_t *ids, const float *coefs, size_t n_tokens, size_t top_k, int32_t y_type,
                              void *y, size_t y_stride, const void *residual, size_t residual_stride, void *workspace,
                              size_t workspace_len, lbh_error *err) {
    if (!ctx || !m) return fail(err, LBH_NULL_ARGUMENT);
    if (m->device != ctx->device) return fail(err, LBH_INVALID_PARAMETER, y_type);
    const size_t e = row_elem_bytes(y_type);
    if (!e) return fail(err, LBH_UNSUPPORTED_TYPE, y_type);
    if (n_tokens == 0) return ok(err);   // no token, and no address asked for
    if (!experts_shape(n_tokens, top_k)) return fail(err, LBH_UNSUPPORTED_SHAPE, y_type, n_tokens, EXPERTS_MAX_PAIRS, top_k);
    if (!x || !x_scales || !ids || !coefs || !y || !workspace) return fail(err, LBH_NULL_ARGUMENT, y_type);
    if (n_tokens == 1) x_stride = m->n, y_stride = m->n, residual_stride = m->n;
    if (x_stride > MAX_STRIDE) return fail(err, LBH_UNSUPPORTED_SHAPE, y_type, 0, MAX_STRIDE, x_stride);
    const Rows ops[] = {{x, x_stride, 1, m->n}, {y, y_stride, e, m->n}, {residual, residual ? residual_stride : 0, e, m->n}};
    const lbh_status st = check_rows(ops, 3, n_tokens, y_type, err);
    if (st) return st;
    if (!aligned_to(x_scales, 4) || !aligned_to(ids, 4) || !aligned_to(coefs, 4) || !aligned_to(workspace, 16))
        return fail(err, LBH_INVALID_PARAMETER, y_type);
    const size_t pairs = n_tokens * top_k;
    const ExpertsSpace at(*m, n_tokens, top_k);
    if (workspace_len < at.bytes) return fail(err, LBH_SCRATCH_TOO_SMALL, 0, n_tokens, at.bytes, workspace_len);
    const Span sx = span_of(ops[0], n_tokens), sy = span_of(ops[1], n_tokens), sr = span_of(ops[2], n_tokens),
               ss = {x_scales, 4, 4, n_tokens}, si = {ids, 4 * pairs, 4 * pairs, 1}, sc = {coefs, 4 * pairs, 4 * pairs, 1},
               sw = {workspace, at.bytes, at.bytes, 1};
    for (const Span *in : {&sx, &ss, &si, &sc})
        if (share(sy, *in) || share(sw, *in)) return fail(err, LBH_INVALID_PARAMETER, y_type);
    if (!same_or_apart(sy, sr) || share(sw, sy) || share(sw, sr)) return fail(err, LBH_INVALID_PARAMETER, y_type);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    ExpertsArgs a{};
    a.experts = m->experts, a.down_scales = m->down_scales, a.shared = m->shared, a.has_shared = m->ffn_s != 0;
    a.n_experts = (int32_t)m->n_experts, a.n = (int32_t)m->n, a.ffn = (int32_t)m->ffn, a.ffn_s = (int32_t)m->ffn_s;
    a.kt_n = (int32_t)m->kt_n, a.kt_f = (int32_t)m->kt_f, a.kt_fs = (int32_t)m->kt_fs, a.down_pitch = (int32_t)m->down_pitch;
    a.x = x, a.x_scales = x_scales, a.x_stride = (long long)x_stride, a.x_bytes = (int32_t)m->n;
    a.n_tokens = (int32_t)n_tokens, a.top_k = (int32_t)top_k, a.pairs = (int32_t)pairs, a.ids = ids, a.coefs = coefs;
    a.y = y, a.residual = residual, a.y_stride = (long long)y_stride, a.residual_stride = (long long)residual_stride;
    a.y_type = y_type, a.plan = reinterpret_cast<ExpertsPlan *>(ws + at.plan);
    a.h = reinterpret_cast<float *>(ws + at.h), a.h_s = reinterpret_cast<float *>(ws + at.h_s);
    a.h_pitch = (long long)up16(m->ffn), a.h_s_pitch = (long long)up16(m->ffn_s);
    a.hq = reinterpret_cast<int8_t *>(ws + at.hq), a.hq_s = reinterpret_cast<int8_t *>(ws + at.hq_s);
    a.h_scales = reinterpret_cast<float *>(ws + at.scales);
    DeviceGuard g(ctx->device);
    if (!aligned_to(x, 16) || x_stride % 16 || m->n % 16) {   // read as 16-byte words: such rows are copied first
        const size_t pitch = m->kt_n * 64;
        HIP_TRY(launch_i8_align_rows(x, a.x_stride, a.n, (int)pitch, (long long)n_tokens, ws + at.x, ctx->stream));
        a.x = reinterpret_cast<const int8_t *>(ws + at.x);
        a.x_stride = (long long)pitch, a.x_bytes = (int32_t)pitch;
    }
    HIP_TRY(launch_experts_i8(a, ctx->stream));
    return ok(err);
}

}  // extern "C"
