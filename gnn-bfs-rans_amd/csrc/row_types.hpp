// Row element types of the operators on activation rows (rms_norm.hip,
// rotary.hip, cross_attn*.hip): fp32, bf16 and fp16 in memory, fp32 in
// registers; one rounding, to nearest even, at the store.
#pragma once

#include "common.hpp"

namespace mignn {

using bf16_t = __bf16;
using f16_t = _Float16;

// N consecutive elements at any element alignment: the hardware's unaligned
// vector access (one dwordx4 for 16 bytes, whatever the row pitch's parity).
template <typename T, int N>
struct RowVec {
    T v[N];
};

template <typename T, int N>
__device__ __forceinline__ void load_row(const T* p, float (&o)[N]) {
    RowVec<T, N> t;
    __builtin_memcpy(&t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = static_cast<float>(t.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* p, const float (&o)[N]) {
    RowVec<T, N> t;
#pragma unroll
    for (int i = 0; i < N; ++i) t.v[i] = static_cast<T>(o[i]);
    __builtin_memcpy(p, &t, sizeof(t));
}

inline int row_type_size(int dtype) { return dtype == MIGNN_ROW_F32 ? 4 : 2; }
inline bool row_type_ok(int dtype) { return dtype >= MIGNN_ROW_F32 && dtype <= MIGNN_ROW_F16; }

}  // namespace mignn
