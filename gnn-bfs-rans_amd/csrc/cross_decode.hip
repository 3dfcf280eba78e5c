// Cross attention of few rows (probe points): up to CROSS_FEW rows of one
// sequence and kv head -- queries times heads of the group -- against all its
// keys (formulas: cross_attn.hip).
//
// Bound by memory: K and V are read once, for all rows, and nothing is
// computed twice.  A key's row is spread over LPK lanes, 16 bytes each, so a
// wave reads 64 / LPK keys at a time, UNROLL of them in flight; the scores
// are butterflies over the LPK lanes, and every group of lanes keeps a running
// maximum, sum and output of its own keys in registers.  No LDS until the end,
// where the groups and then the block's waves are joined.  The matrix
// instructions would spend 32 columns on these rows, and the staging of tiles
// costs more than the arithmetic: fp32 here for every type.
//
// Measured: 64 bf16 probes, 8 heads over 2 of 64 columns, 416 MB of keys and
// values (12,700 keys a sequence): 91 us (4.5 TB/s) + 5 for the join; one fp32 probe of 4
// heads of 32 over 12225 keys 5 us + 3.3 (two launches of nearly empty time).
// The vector unit is the next bound: bf16 scores by two-element dot products
// took 106 to 95 us, a second key in flight a lane from four rows on 117 to
// 110; a third wave a SIMD spills and takes 320.
#include "cross_attn.hpp"

namespace mignn {
namespace {

constexpr int WAVES = 4;

// sum over the LPK (4..32) lanes of a key, for each of them: butterflies whose
// exchanges are lane permutations of the adder itself (a mirror of 8 or 16
// lanes serves as an exchange of their halves once the halves are uniform)
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int LPK>
__device__ __forceinline__ float key_sum(float v) {
    v = dpp_add<0xb1>(v);                            // quad_perm 1 0 3 2
    v = dpp_add<0x4e>(v);                            // quad_perm 2 3 0 1
    if constexpr (LPK >= 8) v = dpp_add<0x141>(v);   // row_half_mirror
    if constexpr (LPK >= 16) v = dpp_add<0x140>(v);  // row_mirror
    if constexpr (LPK >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
}

// <a, b> of a lane's 16 bytes: bf16 two at a time, products and sum in fp32
template <typename T, int V>
__device__ __forceinline__ float dot(const RowVec<T, V>& a, const RowVec<T, V>& b) {
    float x = 0.f;
    if constexpr (__is_same(T, bf16_t)) {
        typedef T pair __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < V; i += 2)
            x = __builtin_amdgcn_fdot2_f32_bf16(pair{a.v[i], a.v[i + 1]}, pair{b.v[i], b.v[i + 1]}, x, false);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x = fmaf(static_cast<float>(a.v[i]), static_cast<float>(b.v[i]), x);
    }
    return x;
}

// One thread's share of UNROLL keys, in flight
template <typename T, int UNROLL>
struct KeyLoad {
    static constexpr int V = 16 / sizeof(T);
    RowVec<T, V> k[UNROLL], v[UNROLL];
    uint32_t ok[UNROLL];   // as loaded: a comparison here would wait for all loads before it
};

// R rows (a power of two that holds the sequence's); LPK lanes a key, V elements each
template <typename T, int R, int LPK>
__global__ __launch_bounds__(WAVES * 64) void cross_few_kernel(CrossArgs a) {
    constexpr int V = 16 / sizeof(T), KPW = 64 / LPK, UNROLL = R >= 4 ? 2 : 4;
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = a.items[item];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPK, grp = lane / LPK;
    const int c0 = sub * V;
    const bool in = c0 < a.d;
    const int rows = it.r1 - it.r0;
    RowVec<T, V> q[R];
    float o[R][V], m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY, l[r] = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) o[r][i] = 0.f;
        q[r] = RowVec<T, V>{};
        if (r < rows && in) {
            const int row = it.r0 + r, t = row / a.group;
            __builtin_memcpy(&q[r], static_cast<const T*>(a.q) + (it.q_begin + static_cast<int64_t>(t)) * a.ldq +
                                        (kvh * a.group + row - t * a.group) * a.ldqh + c0, 16);
        }
    }
    const T* kb = static_cast<const T*>(a.k) + kvh * a.ldkh + c0;
    const T* vb = static_cast<const T*>(a.v) + kvh * a.ldvh + c0;
    KeyLoad<T, UNROLL> now, next;
    auto load = [&](KeyLoad<T, UNROLL>& n, int k0) {
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int k = k0 + u * KPW + grp;
            const int64_t key = it.k_begin + static_cast<int64_t>(k < it.c1 ? k : it.c1 - 1);
            n.ok[u] = a.mask ? a.mask[key] : 1u;
            n.k[u] = n.v[u] = RowVec<T, V>{};
            if (in) {
                __builtin_memcpy(&n.k[u], kb + key * a.ldk, 16);
                __builtin_memcpy(&n.v[u], vb + key * a.ldv, 16);
            }
        }
    };
    constexpr int STEP = WAVES * KPW * UNROLL;
    int k0 = it.c0 + wave * KPW * UNROLL;
    if (k0 < it.c1) load(now, k0);
    for (; k0 < it.c1; k0 += STEP, now = next) {
        if (k0 + STEP < it.c1) load(next, k0 + STEP);
        bool ok[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) ok[u] = now.ok[u] != 0u && k0 + u * KPW + grp < it.c1;
        float s[R][UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float x = key_sum<LPK>(dot(q[r], now.k[u]));
                s[r][u] = ok[u] ? x * a.c : -INFINITY;
            }
        // what the mask leaves out may hold anything, and 0 inf is no 0
        float vf[UNROLL][V];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) vf[u][i] = ok[u] ? static_cast<float>(now.v[u].v[i]) : 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mn = m[r];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) mn = fmaxf(mn, s[r][u]);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float f = __builtin_amdgcn_exp2f(m[r] - base);
            m[r] = mn;
            l[r] *= f;
#pragma unroll
            for (int i = 0; i < V; ++i) o[r][i] *= f;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const float p = __builtin_amdgcn_exp2f(s[r][u] - base);
                l[r] += p;
#pragma unroll
                for (int i = 0; i < V; ++i) o[r][i] = fmaf(p, vf[u][i], o[r][i]);
            }
        }
    }
    // the wave's groups, then the block's waves: each joined onto the largest maximum
    __shared__ float st[WAVES][R][2];
    __shared__ float os[WAVES][R][LPK * V];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float mx = m[r];
#pragma unroll
        for (int b = LPK; b < 64; b <<= 1) mx = fmaxf(mx, __shfl_xor(mx, b));
        const float f = __builtin_amdgcn_exp2f(m[r] - (mx == -INFINITY ? 0.f : mx));
        l[r] *= f;
#pragma unroll
        for (int b = LPK; b < 64; b <<= 1) l[r] += __shfl_xor(l[r], b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            o[r][i] *= f;
#pragma unroll
            for (int b = LPK; b < 64; b <<= 1) o[r][i] += __shfl_xor(o[r][i], b);
            if (grp == 0) os[wave][r][c0 + i] = o[r][i];
        }
        if (lane == 0) st[wave][r][0] = mx, st[wave][r][1] = l[r];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * a.d; i += WAVES * 64) {
        const int r = i / a.d, c = i - r * a.d;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) mx = fmaxf(mx, st[w][r][0]);
        const float base = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = __builtin_amdgcn_exp2f(st[w][r][0] - base);
            sum = fmaf(st[w][r][1], f, sum);
            v = fmaf(os[w][r][c], f, v);
        }
        if (it.slot >= 0) {
            float* p = a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * CROSS_FEW + r) * (a.d + 2);
            p[c] = v;
            if (c == 0) p[a.d] = mx, p[a.d + 1] = sum;
            continue;
        }
        const int row = it.r0 + r, t = row / a.group;
        const int64_t at = (it.q_begin + static_cast<int64_t>(t)) * a.heads + kvh * a.group + row - t * a.group;
        const float out = sum == 0.f ? 0.f : v / sum;
        static_cast<T*>(a.out)[at * a.d + c] = static_cast<T>(out);
        if (a.o32) a.o32[at * a.d + c] = out;
        if (a.lse && c == 0) a.lse[at] = sum == 0.f ? INFINITY : base + log2f(sum);
    }
}

template <typename T, int R>
void launch_few(const CrossArgs& a, hipStream_t st) {
    const dim3 grid(cross_grid(a)), block(WAVES * 64);
    const int lanes = a.d / (16 / static_cast<int>(sizeof(T)));
#define MIGNN_FEW(L) hipLaunchKernelGGL((cross_few_kernel<T, R, L>), grid, block, 0, st, a)
    if (lanes <= 4) MIGNN_FEW(4);
    else if (lanes <= 8) MIGNN_FEW(8);
    else if (lanes <= 16) MIGNN_FEW(16);
    else if constexpr (sizeof(T) == 4) MIGNN_FEW(32);
#undef MIGNN_FEW
}

template <typename T>
void launch_few_t(const CrossArgs& a, hipStream_t st) {
    const int rows = a.rows;
    if (rows <= 1) launch_few<T, 1>(a, st);
    else if (rows <= 2) launch_few<T, 2>(a, st);
    else if (rows <= 4) launch_few<T, 4>(a, st);
    else launch_few<T, CROSS_FEW>(a, st);
}

}  // namespace

int cross_few(const CrossArgs& a, int dtype, hipStream_t st) {
    if (dtype == MIGNN_ROW_F32) launch_few_t<float>(a, st);
    else if (dtype == MIGNN_ROW_BF16) launch_few_t<bf16_t>(a, st);
    else launch_few_t<f16_t>(a, st);
    return launch_status("cross_few_kernel");
}

}  // namespace mignn
