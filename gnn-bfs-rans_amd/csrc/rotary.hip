// Rotary positions over several axes (mignn_rotary): the pairs of a head's
// columns turned by the row's coordinates.
//
//   pair j of axis a(j):  t = pos[a] f_j,   (u, v) -> (u cos t - v sin t, v cos t + u sin t)
//
// A pair is columns (j, j + pairs), or (2j, 2j + 1) when interleaved; columns
// from 2 pairs on pass through.  The gradient is the rotation by -t.
//
// Bound by memory: x read once and y written once.  The angle is formed in
// fp64 as a number of turns (the table holds f_j / 2 pi), of which the
// fraction goes to fp32: a far position costs no accuracy, and one thread's
// sine and cosine serve all heads of a row.
#include "row_types.hpp"

namespace mignn {
namespace {

struct RotArgs {
    const void *x, *pos;
    void* y;
    const double* freq;
    const int32_t* axis;
    int64_t ldt, ldh, ldp, ldyt, ldyh, n;
    int heads, d, pairs, pos_type, chunks, pass;
    bool inverse;
};

__device__ __forceinline__ double load_pos(const RotArgs& a, int64_t row, int axis) {
    const int64_t i = row * a.ldp + axis;
    switch (a.pos_type) {
        case MIGNN_POS_F32: return static_cast<const float*>(a.pos)[i];
        case MIGNN_POS_F64: return static_cast<const double*>(a.pos)[i];
        case MIGNN_POS_I32: return static_cast<const int32_t*>(a.pos)[i];
        default: return static_cast<double>(static_cast<const int64_t*>(a.pos)[i]);
    }
}

// V pairs a thread; chunk c < chunks: pairs, the last chunk ending at the last
// pair (pairs >= V, or V = 1); the chunks after them: columns passed through.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
    const int per_row = a.chunks + a.pass;
    const int64_t total = a.n * per_row;
    for (int64_t t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; t < total;
         t += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t row = t / per_row;
        const int c = static_cast<int>(t - row * per_row);
        const T* x = static_cast<const T*>(a.x) + row * a.ldt;
        T* y = static_cast<T*>(a.y) + row * a.ldyt;
        if (c >= a.chunks) {
            const int c0 = 2 * a.pairs + (c - a.chunks) * V;
            for (int h = 0; h < a.heads; ++h)
                for (int i = c0; i < a.d && i < c0 + V; ++i) y[h * a.ldyh + i] = x[h * a.ldh + i];
            continue;
        }
        int j0 = c * V;
        if (j0 > a.pairs - V) j0 = a.pairs - V;
        float cs[V], sn[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double turns = load_pos(a, row, a.axis[j0 + i]) * a.freq[j0 + i];
            const float f = static_cast<float>(turns - rint(turns));
            sincospif(2.f * f, &sn[i], &cs[i]);
            if (a.inverse) sn[i] = -sn[i];
        }
        for (int h = 0; h < a.heads; ++h) {
            const T* xh = x + h * a.ldh;
            T* yh = y + h * a.ldyh;
            if constexpr (INTERLEAVED) {
                float u[2 * V], o[2 * V];
                load_row(xh + 2 * j0, u);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    o[2 * i] = u[2 * i] * cs[i] - u[2 * i + 1] * sn[i];
                    o[2 * i + 1] = u[2 * i + 1] * cs[i] + u[2 * i] * sn[i];
                }
                store_row(yh + 2 * j0, o);
            } else {
                float u[V], v[V], o[V], q[V];
                load_row(xh + j0, u);
                load_row(xh + a.pairs + j0, v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    o[i] = u[i] * cs[i] - v[i] * sn[i];
                    q[i] = v[i] * cs[i] + u[i] * sn[i];
                }
                store_row(yh + j0, o);
                store_row(yh + a.pairs + j0, q);
            }
        }
    }
}

template <typename T>
int launch_rotary(RotArgs a, bool interleaved, hipStream_t st) {
    // 16 bytes an access: V pairs of two rows' halves, or V / 2 interleaved
    constexpr int V = 16 / sizeof(T);
    const int v = a.pairs < V ? 1 : (interleaved ? V / 2 : V);
    a.chunks = (a.pairs + v - 1) / v;
    a.pass = (a.d - 2 * a.pairs + v - 1) / v;
    const unsigned grid = grid_for(a.n * (a.chunks + a.pass), 256);
#define MIGNN_ROT(VV, I) \
    hipLaunchKernelGGL((rotary_kernel<T, VV, I>), dim3(grid), dim3(256), 0, st, a)
    if (v == 1) {
        if (interleaved) MIGNN_ROT(1, true);
        else MIGNN_ROT(1, false);
    } else if (interleaved) {
        MIGNN_ROT(V / 2, true);
    } else {
        MIGNN_ROT(V, false);
    }
#undef MIGNN_ROT
    return launch_status("rotary_kernel");
}

}  // namespace
}  // namespace mignn

using namespace mignn;

extern "C" int mignn_rotary(const void* x, int64_t ldt, int64_t ldh, int64_t n, int heads, int d,
                            const void* pos, int pos_type, int64_t ldp, const double* freq,
                            const int32_t* axis, int pairs, int interleaved, int inverse,
                            int dtype, void* y, int64_t ldyt, int64_t ldyh, void* stream) {
    MIGNN_REQUIRE(row_type_ok(dtype), "rotary: unknown row type %d", dtype);
    MIGNN_REQUIRE(pos_type >= MIGNN_POS_F32 && pos_type <= MIGNN_POS_I64,
                  "rotary: unknown position type %d", pos_type);
    MIGNN_REQUIRE(n >= 0 && heads >= 0 && d > 0 && pairs > 0 && 2 * static_cast<int64_t>(pairs) <= d,
                  "rotary: n = %lld, heads = %d, d = %d, pairs = %d", static_cast<long long>(n),
                  heads, d, pairs);
    if (n == 0 || heads == 0) return MIGNN_OK;
    MIGNN_REQUIRE(x && pos && freq && axis && y, "rotary: null pointer");
    RotArgs a{};
    a.x = x, a.pos = pos, a.y = y, a.freq = freq, a.axis = axis;
    a.ldt = ldt, a.ldh = ldh, a.ldp = ldp, a.ldyt = ldyt, a.ldyh = ldyh, a.n = n;
    a.heads = heads, a.d = d, a.pairs = pairs, a.pos_type = pos_type, a.inverse = inverse != 0;
    hipStream_t st = as_stream(stream);
    switch (dtype) {
        case MIGNN_ROW_F32: return launch_rotary<float>(a, interleaved != 0, st);
        case MIGNN_ROW_BF16: return launch_rotary<bf16_t>(a, interleaved != 0, st);
        default: return launch_rotary<f16_t>(a, interleaved != 0, st);
    }
}
