// lbh_rowtypes.h — the element types of row operands (32-bit and 16-bit
// floats) and their conversions, shared by the norm and 8-bit product kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace lbh {

// GGML type ids of row elements (T_F32 is in lbh_layout.h).
enum : int { T_F16 = 1, T_BF16 = 30 };

constexpr int row_elem_bytes(int ty) { return ty == 0 ? 4 : ty == T_F16 || ty == T_BF16 ? 2 : 0; }

template <int TY>
struct RowElem;
template <>
struct RowElem<0> {
    using T = float;
};
template <>
struct RowElem<T_F16> {
    using T = _Float16;
};
template <>
struct RowElem<T_BF16> {
    using T = __bf16;
};
template <int TY>
using row_t = typename RowElem<TY>::T;

// N consecutive elements as one vector (N * size 8 or 16 bytes a load).
template <typename T, int N>
using rvec __attribute__((ext_vector_type(N))) = T;

}  // namespace lbh
