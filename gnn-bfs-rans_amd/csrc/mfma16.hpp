// 16-bit matrix instructions on LDS tiles, shared by cross_attn16.hip (16-bit
// rows) and cross_attn32.hip (fp32 rows as three bf16 terms).
#pragma once

#include "cross_attn.hpp"

namespace mignn {

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));
using s16x4 = __attribute__((ext_vector_type(4))) short;
using lds_s16x4 = __attribute__((address_space(3))) s16x4;

__device__ __forceinline__ f32x16 mfma16(vec8<bf16_t> a, vec8<bf16_t> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma16(vec8<f16_t> a, vec8<f16_t> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Row pitch of a tile in bytes: its width plus 32, so that neither 8 rows'
// 16-byte reads nor 4 rows' transposed reads meet in a bank
template <int DP>
constexpr int pitch() { return DP * 2 + 32; }

// the transposed read's share of a lane: row 4 half + (l % 16) / 4, columns
// 16 ((l / 16) % 2) + 4 (l % 4) ..+3
template <int DP>
__device__ __forceinline__ int tr_lane(int lane) {
    return (4 * (lane >> 5) + ((lane & 15) >> 2)) * pitch<DP>() + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;
}

// A operand of a product over rows row + (the accumulator's order of 16) of a
// tile: columns 32 b + l % 32
template <typename T, int DP>
__device__ __forceinline__ vec8<T> tr_frag(const char* tile, int trl, int row, int b) {
    const char* p = tile + trl + row * pitch<DP>() + 64 * b;
    union {
        s16x4 h[2];
        vec8<T> v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * pitch<DP>()));
    return u.v;
}

// A operand of a product over columns: row r + l % 32, columns 16 i + 8 half ..+7
template <typename T, int DP>
__device__ __forceinline__ vec8<T> row_frag(const char* tile, int r, int i, int col, int half) {
    return *reinterpret_cast<const vec8<T>*>(tile + (r + col) * pitch<DP>() + 32 * i + 16 * half);
}

// Which of a tile's keys take part (bit = key), for every lane: the mask's
// byte is loaded ahead of the rows it goes with and looked at when they are (a
// comparison at the load would wait for every load before it)
struct KeyBits {
    uint32_t byte;
    int left;
    __device__ __forceinline__ void load(const CrossArgs& a, int64_t key0, int n, int lane) {
        left = n;
        byte = 1u;
        if (a.mask && n > 0) byte = a.mask[key0 + (lane < n ? lane : n - 1)];
    }
    __device__ __forceinline__ uint64_t bits(int lane) const {
        return __builtin_amdgcn_ballot_w64(lane < left && byte != 0u);
    }
};

// maximum and sum of a wave's two halves, in both
__device__ __forceinline__ float swap_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_add(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// an accumulator (columns of the result in its rows) times f to a row in memory
template <typename T, int DP>
__device__ __forceinline__ void store_acc(T* p, const f32x16 (&acc)[DP / 32], float f, int d, int half) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int c = 32 * b + 8 * g + 4 * half;
            if (c < d) {
                const float o[4] = {acc[b][4 * g] * f, acc[b][4 * g + 1] * f, acc[b][4 * g + 2] * f,
                                    acc[b][4 * g + 3] * f};
                store_row(p + c, o);
            }
        }
}

// the running maximum is raised when a score passes it by this power of two
constexpr float MAX_SLACK = 6.f;

}  // namespace mignn
