// Root-mean-square norm of rows with the residual's addition, and its
// gradients (mignn_rms_norm, mignn_rms_norm_backward).
//
//   s = x + r,   rstd = (sum_h s_h^2 / H + eps)^-1/2,   y = s rstd w
//   g = dy w:    ds = rstd (g - s rstd^2 / H sum_h g_h s_h) + ds_out
//                dx = dr = ds,   dw = sum_rows dy s rstd
//
// Bound by memory: every tensor is read or written once.  A row lives in the
// registers of `lpr` lanes (a power of two, so that narrow rows share a wave)
// as NPT vectors of 16 bytes; its sums are butterflies over those lanes.  A
// width that is no multiple of the vector takes its last vector from the
// row's end: the elements that two lanes then hold are counted once and
// stored twice with the same bits.  The sums and s itself stay in fp32: y is
// rounded once, from the unrounded s, so a 16-bit backward reads x and r
// again instead of the stored s.
//
// Measured: 1M x 128 bf16 with residual 183 us (1.02 GB at 5.6 TB/s; a plain
// copy reaches 5.1).  49181 x 256 fp32: forward 34 us, gradients 35, the
// weight's partial sums 4.3 (7 more when they are read one after another).
#include "row_types.hpp"

namespace mignn {
namespace {

constexpr int NORM_WAVES = 4;
constexpr int NORM_MAX_GRID = 1024;

struct NormArgs {
    const void *x, *r, *w, *dy, *ds;
    void *y, *s;
    float* dw_part;   // the blocks' partial weight gradients, or
    void* dw;         // the only block's
    int64_t ldx, ldr, lddy, ldds, ldy, lds, n;
    int h, lpr;
    float eps;
    bool w_f32;
};

template <typename T, int VEC>
__device__ __forceinline__ void load_weight(const NormArgs& a, int c, float (&w)[VEC]) {
    if (a.w_f32) load_row(static_cast<const float*>(a.w) + c, w);
    else load_row(static_cast<const T*>(a.w) + c, w);
}

// Column chunk j of lane `sub`: its first column, and the first of its
// elements that no earlier chunk holds (VEC: the chunk does not exist).
template <int VEC>
__device__ __forceinline__ int chunk_begin(int chunk, int h, int& own) {
    const int c = chunk * VEC;
    own = 0;
    if (c + VEC <= h) return c;
    own = c < h ? c - (h - VEC) : VEC;
    return h - VEC;
}

template <typename T, int VEC, int NPT>
__global__ __launch_bounds__(NORM_WAVES * 64) void rms_norm_kernel(NormArgs a) {
    const int lane = threadIdx.x & 63, sub = lane & (a.lpr - 1);
    const int64_t rpw = 64 / a.lpr;
    const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * NORM_WAVES + (threadIdx.x >> 6)) * rpw +
                         lane / a.lpr;
    const int64_t step = static_cast<int64_t>(gridDim.x) * NORM_WAVES * rpw;
    float w[NPT][VEC];
    int col[NPT], own[NPT];
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
        col[j] = chunk_begin<VEC>(sub + j * a.lpr, a.h, own[j]);
        load_weight<T, VEC>(a, col[j], w[j]);
    }
    // every lane of a wave runs the same number of rounds (the butterflies
    // need all of a row's lanes)
    const int64_t first = row0 - lane / a.lpr;
    for (int64_t base = first; base < a.n; base += step) {
        const int64_t row = base + lane / a.lpr;
        const bool live = row < a.n;
        float s[NPT][VEC];
        float sum = 0.f;
        if (live) {
#pragma unroll
            for (int j = 0; j < NPT; ++j) {
                if (own[j] == VEC) continue;
                load_row(static_cast<const T*>(a.x) + row * a.ldx + col[j], s[j]);
                if (a.r) {
                    float r[VEC];
                    load_row(static_cast<const T*>(a.r) + row * a.ldr + col[j], r);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) s[j][i] += r[i];
                }
            }
#pragma unroll
            for (int j = 0; j < NPT; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (i >= own[j]) sum = fmaf(s[j][i], s[j][i], sum);
        }
        for (int m = 1; m < a.lpr; m <<= 1) sum += __shfl_xor(sum, m);
        const float rstd = 1.f / sqrtf(sum / static_cast<float>(a.h) + a.eps);
        if (live) {
#pragma unroll
            for (int j = 0; j < NPT; ++j) {
                if (own[j] == VEC) continue;
                float y[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) y[i] = s[j][i] * rstd * w[j][i];
                store_row(static_cast<T*>(a.y) + row * a.ldy + col[j], y);
                if (a.s) store_row(static_cast<T*>(a.s) + row * a.lds + col[j], s[j]);
            }
        }
    }
}

template <typename T, int VEC, int NPT>
__global__ __launch_bounds__(NORM_WAVES * 64) void rms_norm_backward_kernel(NormArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (a.lpr - 1);
    const int64_t rpw = 64 / a.lpr;
    const int64_t first = (static_cast<int64_t>(blockIdx.x) * NORM_WAVES + wave) * rpw;
    const int64_t step = static_cast<int64_t>(gridDim.x) * NORM_WAVES * rpw;
    float w[NPT][VEC], dw[NPT][VEC];
    int col[NPT], own[NPT];
#pragma unroll
    for (int j = 0; j < NPT; ++j) {
        col[j] = chunk_begin<VEC>(sub + j * a.lpr, a.h, own[j]);
        load_weight<T, VEC>(a, col[j], w[j]);
#pragma unroll
        for (int i = 0; i < VEC; ++i) dw[j][i] = 0.f;
    }
    for (int64_t base = first; base < a.n; base += step) {
        const int64_t row = base + lane / a.lpr;
        const bool live = row < a.n;
        float s[NPT][VEC], dy[NPT][VEC];
        float ss = 0.f, gs = 0.f;
        if (live) {
#pragma unroll
            for (int j = 0; j < NPT; ++j) {
                if (own[j] == VEC) continue;
                load_row(static_cast<const T*>(a.x) + row * a.ldx + col[j], s[j]);
                load_row(static_cast<const T*>(a.dy) + row * a.lddy + col[j], dy[j]);
                if (a.r) {
                    float r[VEC];
                    load_row(static_cast<const T*>(a.r) + row * a.ldr + col[j], r);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) s[j][i] += r[i];
                }
            }
#pragma unroll
            for (int j = 0; j < NPT; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (i >= own[j]) {
                        ss = fmaf(s[j][i], s[j][i], ss);
                        gs = fmaf(dy[j][i] * w[j][i], s[j][i], gs);
                    }
        }
        for (int m = 1; m < a.lpr; m <<= 1) {
            ss += __shfl_xor(ss, m);
            gs += __shfl_xor(gs, m);
        }
        const float inv_h = 1.f / static_cast<float>(a.h);
        const float rstd = 1.f / sqrtf(ss * inv_h + a.eps);
        const float c = gs * inv_h * rstd * rstd;
        if (live) {
#pragma unroll
            for (int j = 0; j < NPT; ++j) {
                if (own[j] == VEC) continue;
                float o[VEC];
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    o[i] = rstd * (dy[j][i] * w[j][i] - s[j][i] * c);
                    dw[j][i] = fmaf(dy[j][i], s[j][i] * rstd, dw[j][i]);
                }
                if (a.ds) {
                    float d[VEC];
                    load_row(static_cast<const T*>(a.ds) + row * a.ldds + col[j], d);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) o[i] += d[i];
                }
                store_row(static_cast<T*>(a.y) + row * a.ldy + col[j], o);
            }
        }
    }
    if (!a.dw_part && !a.dw) return;
    // this block's row of the [grid, H] partial weight gradients: rows of one
    // wave by butterflies over its row groups, the waves through LDS
    extern __shared__ float part[];   // [NORM_WAVES][h]
#pragma unroll
    for (int j = 0; j < NPT; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float v = dw[j][i];
            for (int m = a.lpr; m < 64; m <<= 1) v += __shfl_xor(v, m);
            if (lane < a.lpr && own[j] != VEC && i >= own[j]) part[wave * a.h + col[j] + i] = v;
        }
    __syncthreads();
    for (int c = threadIdx.x; c < a.h; c += NORM_WAVES * 64) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < NORM_WAVES; ++k) v += part[k * a.h + c];
        if (a.dw_part) a.dw_part[static_cast<int64_t>(blockIdx.x) * a.h + c] = v;
        else if (a.w_f32) static_cast<float*>(a.dw)[c] = v;
        else static_cast<T*>(a.dw)[c] = static_cast<T>(v);
    }
}

// dw[c] = sum of the blocks' partials: 8 columns a block, 128 threads a column
// that take every 128th partial (all in flight), their sums by a fixed tree
template <typename W>
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float* part, int blocks, int h, W* dw) {
    __shared__ float acc[1024];
    const int c = blockIdx.x * 8 + (threadIdx.x & 7), k0 = threadIdx.x >> 3;
    float v = 0.f;
    if (c < h) {
#pragma unroll
        for (int i = 0; i < NORM_MAX_GRID / 128; ++i) {
            const int k = k0 + 128 * i;
            if (k < blocks) v += part[static_cast<int64_t>(k) * h + c];
        }
    }
    acc[threadIdx.x] = v;
    __syncthreads();
    for (int m = 512; m >= 8; m >>= 1) {
        if (threadIdx.x < m) acc[threadIdx.x] += acc[threadIdx.x + m];
        __syncthreads();
    }
    if (threadIdx.x < 8 && c < h) dw[c] = static_cast<W>(acc[threadIdx.x]);
}

struct NormShape {
    int vec, npt, lpr;
    unsigned grid;
};

// 16-byte vectors unless the row is shorter than one; lanes a row: the power
// of two that holds it, at most a wave
NormShape norm_shape(int64_t n, int h, int dtype) {
    NormShape s;
    s.vec = 16 / row_type_size(dtype);
    if (h < s.vec) s.vec = 1;
    const int chunks = (h + s.vec - 1) / s.vec;
    s.lpr = 1;
    while (s.lpr < 64 && s.lpr < chunks) s.lpr <<= 1;
    s.npt = 1;
    while (s.npt * s.lpr < chunks) s.npt <<= 1;
    const int64_t rows = NORM_WAVES * (64 / s.lpr);
    s.grid = grid_for(n, static_cast<int>(rows), NORM_MAX_GRID);
    return s;
}

// Few rows' weight gradient: one block takes all of them, in up to four
// rounds, and writes it; a second kernel and its partial sums would cost more
// (a training step of 16 x 128 rows from PyTorch: 74 us with them, 59 without)
NormShape norm_backward_shape(int64_t n, int h, int dtype, bool dw) {
    NormShape s = norm_shape(n, h, dtype);
    if (dw && n <= 4 * NORM_WAVES * (64 / s.lpr)) s.grid = 1;
    return s;
}

template <typename T, int VEC, int NPT>
int launch_norm(const NormArgs& a, const NormShape& s, bool backward, hipStream_t st) {
    if (backward) {
        hipLaunchKernelGGL((rms_norm_backward_kernel<T, VEC, NPT>), dim3(s.grid),
                           dim3(NORM_WAVES * 64),
                           a.dw_part || a.dw ? NORM_WAVES * a.h * sizeof(float) : 0, st, a);
        return launch_status("rms_norm_backward_kernel");
    }
    hipLaunchKernelGGL((rms_norm_kernel<T, VEC, NPT>), dim3(s.grid), dim3(NORM_WAVES * 64), 0, st, a);
    return launch_status("rms_norm_kernel");
}

template <typename T>
int launch_norm_type(const NormArgs& a, const NormShape& s, bool backward, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    if (s.vec == 1) return launch_norm<T, 1, 1>(a, s, backward, st);
    switch (s.npt) {
        case 1: return launch_norm<T, V, 1>(a, s, backward, st);
        case 2: return launch_norm<T, V, 2>(a, s, backward, st);
        case 4: return launch_norm<T, V, 4>(a, s, backward, st);
        case 8:   // 2048 columns of fp32; 16-bit rows of that width take 4 vectors
            if constexpr (V == 4) return launch_norm<T, V, 8>(a, s, backward, st);
            break;
        default: break;
    }
    set_error("rms_norm: no kernel for h = %d", a.h);
    return MIGNN_ERR_UNSUPPORTED;
}

int norm_dispatch(const NormArgs& a, const NormShape& s, int dtype, bool backward, hipStream_t st) {
    switch (dtype) {
        case MIGNN_ROW_F32: return launch_norm_type<float>(a, s, backward, st);
        case MIGNN_ROW_BF16: return launch_norm_type<bf16_t>(a, s, backward, st);
        default: return launch_norm_type<f16_t>(a, s, backward, st);
    }
}

int norm_check(const char* who, const void* x, int64_t ldx, const void* r, int64_t ldr,
               const void* w, int64_t n, int h, float eps, int dtype) {
    MIGNN_REQUIRE(row_type_ok(dtype), "%s: unknown row type %d", who, dtype);
    MIGNN_REQUIRE(n >= 0 && h > 0 && h <= MIGNN_RMS_NORM_MAX_H, "%s: n = %lld, h = %d (1..%d)", who,
                  static_cast<long long>(n), h, MIGNN_RMS_NORM_MAX_H);
    MIGNN_REQUIRE(eps >= 0.f, "%s: eps must not be negative", who);
    MIGNN_REQUIRE(n == 0 || (x && w), "%s: null pointer", who);
    MIGNN_REQUIRE(ldx >= h || n <= 1, "%s: row stride %lld below h = %d", who,
                  static_cast<long long>(ldx), h);
    MIGNN_REQUIRE(!r || ldr >= h || n <= 1, "%s: residual row stride %lld below h = %d", who,
                  static_cast<long long>(ldr), h);
    return MIGNN_OK;
}

}  // namespace
}  // namespace mignn

using namespace mignn;

extern "C" int mignn_rms_norm(const void* x, int64_t ldx, const void* residual, int64_t ldr,
                              const void* weight, int weight_f32, int64_t n, int h, float eps,
                              int dtype, void* y, int64_t ldy, void* s, int64_t lds, void* stream) {
    if (int rc = norm_check("rms_norm", x, ldx, residual, ldr, weight, n, h, eps, dtype)) return rc;
    if (n == 0) return MIGNN_OK;
    MIGNN_REQUIRE(y && (ldy >= h || n == 1) && (!s || lds >= h || n == 1),
                  "rms_norm: bad output pointer or row stride");
    NormArgs a{};
    a.x = x, a.r = residual, a.w = weight, a.y = y, a.s = s;
    a.ldx = ldx, a.ldr = ldr, a.ldy = ldy, a.lds = lds, a.n = n;
    a.h = h, a.eps = eps, a.w_f32 = weight_f32 != 0;
    const NormShape sh = norm_shape(n, h, dtype);
    a.lpr = sh.lpr;
    return norm_dispatch(a, sh, dtype, false, as_stream(stream));
}

extern "C" size_t mignn_rms_norm_backward_scratch_bytes(int64_t n, int h, int dtype) {
    if (n < 0 || h <= 0 || h > MIGNN_RMS_NORM_MAX_H || !row_type_ok(dtype)) {
        set_error("rms_norm_backward_scratch_bytes: bad arguments");
        return 0;
    }
    const unsigned grid = norm_backward_shape(n, h, dtype, true).grid;
    return grid == 1 ? 0 : static_cast<size_t>(grid) * h * sizeof(float);
}

extern "C" int mignn_rms_norm_backward(const void* x, int64_t ldx, const void* residual,
                                       int64_t ldr, const void* weight, int weight_f32, int64_t n,
                                       int h, float eps, int dtype, const void* dy, int64_t lddy,
                                       const void* ds, int64_t ldds, void* dx, int64_t lddx,
                                       void* dw, void* scratch, size_t scratch_bytes,
                                       void* stream) {
    if (int rc = norm_check("rms_norm_backward", x, ldx, residual, ldr, weight, n, h, eps, dtype))
        return rc;
    MIGNN_REQUIRE((n == 0 || (dy && dx)) && (!dw || weight), "rms_norm_backward: null pointer");
    MIGNN_REQUIRE(n <= 1 || (lddy >= h && lddx >= h && (!ds || ldds >= h)),
                  "rms_norm_backward: row stride below h");
    const NormShape sh = norm_backward_shape(n, h, dtype, dw != nullptr);
    const bool parts = dw && sh.grid > 1;
    const size_t need = parts ? static_cast<size_t>(sh.grid) * h * sizeof(float) : 0;
    if (scratch_bytes < need) {
        set_error("rms_norm_backward: scratch %zu bytes, need %zu", scratch_bytes, need);
        return MIGNN_ERR_SCRATCH;
    }
    MIGNN_REQUIRE(!parts || (scratch && aligned16(scratch)), "rms_norm_backward: scratch pointer");
    NormArgs a{};
    a.x = x, a.r = residual, a.w = weight, a.dy = dy, a.ds = ds, a.y = dx;
    a.dw_part = parts ? static_cast<float*>(scratch) : nullptr;
    a.dw = parts ? nullptr : dw;
    a.ldx = ldx, a.ldr = ldr, a.lddy = lddy, a.ldds = ldds, a.ldy = lddx, a.n = n;
    a.h = h, a.lpr = sh.lpr, a.eps = eps, a.w_f32 = weight_f32 != 0;
    hipStream_t st = as_stream(stream);
    // n == 0 runs no row: the block's partial is then the empty sum, 0
    if (n > 0 || dw)
        if (int rc = norm_dispatch(a, sh, dtype, true, st)) return rc;
    if (!parts) return MIGNN_OK;
    const dim3 grid((h + 7) / 8);
    const int blocks = static_cast<int>(sh.grid);
    if (weight_f32 || dtype == MIGNN_ROW_F32)
        hipLaunchKernelGGL(rms_norm_dw_kernel<float>, grid, dim3(1024), 0, st, a.dw_part, blocks, h,
                           static_cast<float*>(dw));
    else if (dtype == MIGNN_ROW_BF16)
        hipLaunchKernelGGL(rms_norm_dw_kernel<bf16_t>, grid, dim3(1024), 0, st, a.dw_part, blocks, h,
                           static_cast<bf16_t*>(dw));
    else
        hipLaunchKernelGGL(rms_norm_dw_kernel<f16_t>, grid, dim3(1024), 0, st, a.dw_part, blocks, h,
                           static_cast<f16_t*>(dw));
    return launch_status("rms_norm_dw_kernel");
}
