// Rotary positions over several axes (mignn_rotary): the pairs of a head's
// columns turned by the row's coordinates.
//
//   pair j of axis a(j):  t = pos[a] f_j,   (u, v) -> (u cos t - v sin t, v cos t + u sin t)
//
// A pair is columns (j, j + pairs), or (2j, 2j + 1) when interleaved; columns
// from 2 pairs on pass through.  The gradient is the rotation by -t.
//
// Bound by memory: x read once and y written once.  A workgroup takes a run of
// rows: first the sine and cosine of its rows' angles, once for all heads, into
// LDS, then the rows in the order of memory, 16 bytes an access.  The angle is
// formed in fp64 as a number of turns (the table holds f_j / 2 pi), of which
// the fraction goes to fp32: a far position costs no accuracy.
//
// Measured: 1M x 4 x 32 fp32, three axes, 188 us (1.04 GB at 5.5 TB/s);
// 49181 x 8 x 64 bf16 18 us (5.6).
#include "row_types.hpp"

namespace mignn {
namespace {

struct RotArgs {
    const void *x, *pos;
    void* y;
    const double* freq;
    const int32_t* axis;
    int64_t ldt, ldh, ldp, ldyt, ldyh, n;
    int heads, d, pairs, pos_type, chunks, pass, rows;   // rows of a workgroup
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

// Sine and cosine of f turns, |f| <= 1/2: the nearest quarter turn taken off
// (exactly), Taylor's polynomials to the 9th and 10th power of what is left
// (|2 pi r| <= pi / 4: cut off below 2e-9), and the quarter's exchange and signs.
__device__ __forceinline__ void sincos_turns(float f, float& sn, float& cs) {
    const float q = rintf(4.f * f), r = fmaf(q, -0.25f, f), z = r * r;
    const float s = r * fmaf(z, fmaf(z, fmaf(z, fmaf(z, 42.0586939f, -76.7058597f), 81.6052493f),
                                     -41.3417022f), 6.28318531f);
    const float c = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -26.4262568f, 60.2446414f), -85.4568172f),
                                              64.9393940f), -19.7392088f), 1.f);
    const int n = static_cast<int>(q);
    sn = n & 1 ? c : s;
    cs = n & 1 ? s : c;
    if (n & 2) sn = -sn;
    if ((n + 1) & 2) cs = -cs;
}

// V pairs an access; chunk c < chunks of a head: pairs, the last chunk ending
// at the last pair (pairs >= V, or V = 1); the chunks after them: columns
// passed through.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(256) void rotary_kernel(RotArgs a) {
    extern __shared__ __attribute__((aligned(16))) float trig[];   // [rows][cos: pairs | sin: pairs]
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * a.rows;
    const int rows = a.n - row0 < a.rows ? static_cast<int>(a.n - row0) : a.rows;
    // a thread keeps its pair and goes through the rows
    const int lanes = a.pairs < 256 ? a.pairs : 256, step = 256 / lanes;
    const int first = threadIdx.x / lanes;
    if (first < step)
        for (int j = threadIdx.x - first * lanes; j < a.pairs; j += 256) {
            const int axis = a.axis[j];
            const double freq = a.freq[j];
#pragma unroll 4
            for (int r = first; r < rows; r += step) {
                const double turns = load_pos(a, row0 + r, axis) * freq;
                float sn, cs;
                sincos_turns(static_cast<float>(turns - rint(turns)), sn, cs);
                trig[2 * r * a.pairs + j] = cs;
                trig[(2 * r + 1) * a.pairs + j] = a.inverse ? -sn : sn;
            }
        }
    __syncthreads();
    // (indices carried along: divisions would cost as much as the rest)
    const int per_head = a.chunks + a.pass, per_row = a.heads * per_head;
    const int dr = 256 / per_row, du = 256 - dr * per_row, dh = du / per_head, dc = du - dh * per_head;
    int r = threadIdx.x / per_row, h = (threadIdx.x - r * per_row) / per_head;
    int c = threadIdx.x - r * per_row - h * per_head;
    for (; r < rows; r += dr, h += dh, c += dc) {
        if (c >= per_head) c -= per_head, ++h;
        if (h >= a.heads) {
            h -= a.heads;
            if (++r >= rows) break;
        }
        const T* x = static_cast<const T*>(a.x) + (row0 + r) * a.ldt + h * a.ldh;
        T* y = static_cast<T*>(a.y) + (row0 + r) * a.ldyt + h * a.ldyh;
        if (c >= a.chunks) {
            const int c0 = 2 * a.pairs + (c - a.chunks) * V;
            for (int k = c0; k < a.d && k < c0 + V; ++k) y[k] = x[k];
            continue;
        }
        int j0 = c * V;
        if (j0 > a.pairs - V) j0 = a.pairs - V;
        float cs[V], sn[V];
        load_row(trig + 2 * r * a.pairs + j0, cs);
        load_row(trig + (2 * r + 1) * a.pairs + j0, sn);
        if constexpr (INTERLEAVED) {
            float v[2 * V], o[2 * V];
            load_row(x + 2 * j0, v);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                o[2 * k] = v[2 * k] * cs[k] - v[2 * k + 1] * sn[k];
                o[2 * k + 1] = v[2 * k + 1] * cs[k] + v[2 * k] * sn[k];
            }
            store_row(y + 2 * j0, o);
        } else {
            float v[V], w[V], o[V], q[V];
            load_row(x + j0, v);
            load_row(x + a.pairs + j0, w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                o[k] = v[k] * cs[k] - w[k] * sn[k];
                q[k] = w[k] * cs[k] + v[k] * sn[k];
            }
            store_row(y + j0, o);
            store_row(y + a.pairs + j0, q);
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
    // rows of a workgroup: about four accesses a thread, and at most 16 KB of angles
    const int64_t per_row = static_cast<int64_t>(a.heads) * (a.chunks + a.pass);
    int64_t rows = (1024 + per_row - 1) / per_row;
    if (rows > 2048 / a.pairs) rows = 2048 / a.pairs;
    a.rows = rows < 1 ? 1 : static_cast<int>(rows);
    const int64_t blocks = (a.n + a.rows - 1) / a.rows;
    // (a launch's threads are counted in 32 bits)
    MIGNN_REQUIRE(blocks <= UINT32_MAX / 256 && per_row <= INT32_MAX / 4096, "rotary: too many rows or heads");
    const unsigned grid = static_cast<unsigned>(blocks);
    const size_t lds = static_cast<size_t>(a.rows) * a.pairs * 2 * sizeof(float);
#define MIGNN_ROT(VV, I) \
    hipLaunchKernelGGL((rotary_kernel<T, VV, I>), dim3(grid), dim3(256), lds, st, a)
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
    MIGNN_REQUIRE(pairs <= MIGNN_ROTARY_MAX_PAIRS, "rotary: %d pairs (at most %d)", pairs,
                  MIGNN_ROTARY_MAX_PAIRS);
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
