// lbh_operands.h — checks of operands that the host sides of the dense block and
// of the layer around the experts share (lbh_dense.hip, lbh_layer.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "lbh_rowtypes.h"

namespace {

constexpr size_t MAX_TOKENS = (size_t)1 << 20;
constexpr size_t MAX_STRIDE = (size_t)1 << 23;     // 256 rows stay below 2^31 bytes
constexpr size_t MAX_K = 131071;                   // k * 128 * 128 < 2^31: the sums are exact
constexpr size_t MAX_ROWS = (size_t)1 << 26;

bool float_rows_type(int ty) { return lbh::row_elem_bytes(ty) != 0; }

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

// Device memory of one creation call, released on every way out.
struct Temp {
    void *p = nullptr;
    hipError_t get(size_t n) { return hipMalloc(&p, n); }
    ~Temp() {
        if (p) (void)hipFree(p);
    }
};

}  // namespace
