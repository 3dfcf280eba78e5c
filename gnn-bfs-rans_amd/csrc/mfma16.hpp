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

// LDS tile of rows of DP 16-bit columns: row r at r ROWB, its 16-byte chunk c
// in place c ^ h(r).  h is chosen so that in any 16 rows (aligned) one chunk of
// each, and in any 4 rows (aligned) four neighbouring chunks, lie in different
// banks, whether 128 or 256 bytes go by a cycle: the reads of a product over
// columns (16 bytes a lane, a lane a row) and the transposed reads (4 rows x 16
// columns a 16-lane group).  (A pitch of the width plus 32 bytes, without h,
// spent 40 % of its LDS cycles on conflicts of the former.)
template <int DP>
struct TileRow {
    static constexpr int BYTES = DP == 96 ? 256 : DP * 2;
    __device__ __forceinline__ static int h(int r) {
        if constexpr (DP == 32) return (((r >> 1) ^ (r >> 3)) & 1) << 1 | ((r >> 2) & 1);
        if constexpr (DP == 64) return ((r & 3) << 1 | ((r >> 2) & 1)) ^ ((r >> 3) & 1) << 1;
        return (r & 3) << 1 | ((r >> 2) & 1) | (((r >> 3) ^ r) & 1) << 3;
    }
    // byte of column c (a multiple of 4) in row r
    __device__ __forceinline__ static int at(int r, int c) {
        return r * BYTES + (((c >> 3) ^ h(r)) << 4) + 2 * (c & 7);
    }
};

// A lane's byte offsets in a tile
template <int DP>
struct TileLane {
    int row[DP / 16];        // row l % 32, columns 16 i + 8 (l / 32) ..+7
    int tr[DP / 32][2];      // rows 4 (l / 32) + (l % 16) / 4 (+ 8), columns 32 b + 16 ((l / 16) % 2) + 4 (l % 4) ..+3
    __device__ __forceinline__ explicit TileLane(int lane) {
        const int half = lane >> 5, r = lane & 31, q = 4 * half + ((lane & 15) >> 2);
        const int c = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) row[i] = TileRow<DP>::at(r, 16 * i + 8 * half);
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
            tr[b][0] = TileRow<DP>::at(q, 32 * b + c);
            tr[b][1] = TileRow<DP>::at(q + 8, 32 * b + c);
        }
    }
};

// A operand of a product over rows r (a multiple of 16) + (the accumulator's
// order of 16) of a tile: columns 32 b + l % 32
template <typename T, int DP>
__device__ __forceinline__ vec8<T> tr_frag(const char* tile, const TileLane<DP>& tl, int r, int b) {
    const char* p = tile + r * TileRow<DP>::BYTES;
    union {
        s16x4 h[2];
        vec8<T> v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + tl.tr[b][0]));
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + tl.tr[b][1]));
    return u.v;
}

// A operand of a product over columns 16 i ..+15: rows r (a multiple of 32) + l % 32
template <typename T, int DP>
__device__ __forceinline__ vec8<T> row_frag(const char* tile, const TileLane<DP>& tl, int r, int i) {
    return *reinterpret_cast<const vec8<T>*>(tile + r * TileRow<DP>::BYTES + tl.row[i]);
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
