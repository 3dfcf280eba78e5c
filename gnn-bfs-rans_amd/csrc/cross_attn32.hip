// The forward of cross attention for fp32 rows on the bf16 matrix instructions
// (formulas: cross_attn.hip; structure: cross_attn16.hip).
//
// An fp32 number is the sum of three bf16 numbers, x = h + m + l: each the
// rounding of what is left, each remainder exact, 8 bits apiece.  A product of
// two such sums keeps the six terms down to 2^-16 of it (h h, h m, m h, m m,
// h l, l h); what is left out is below 2^-24 of |x y|, fp32's own rounding.
// bf16 has fp32's range, so no scales are needed and magnitudes may differ as
// they like; only an infinite key or value (or one that rounds to a bf16
// infinity, from 2^127.99 on) makes NaN of every row that reads it.
//
// Six bf16 products take 192 cycles for 32 x 32 x 16 where the fp32 matrix
// instruction takes 512.  K and V are split once a workgroup, on their way
// into LDS; q at the start; P in registers, in place.
#include "mfma16.hpp"

namespace mignn {
namespace {

using B = bf16_t;

// (two numbers at a time: one conversion instruction makes a pair)
__device__ __forceinline__ void split2(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
    typedef B pair __attribute__((ext_vector_type(2)));
    auto bits = [](pair p) { return __builtin_bit_cast(uint32_t, p); };
    h = bits(pair{static_cast<B>(a), static_cast<B>(b)});
    a -= __uint_as_float(h << 16), b -= __uint_as_float(h & 0xffff0000u);
    m = bits(pair{static_cast<B>(a), static_cast<B>(b)});
    a -= __uint_as_float(m << 16), b -= __uint_as_float(m & 0xffff0000u);
    l = bits(pair{static_cast<B>(a), static_cast<B>(b)});
}

struct Frag3 {
    vec8<B> h, m, l;
};
__device__ __forceinline__ Frag3 split8(const float (&x)[8]) {
    union {
        uint32_t u[4];
        vec8<B> v;
    } h, m, l;
#pragma unroll
    for (int i = 0; i < 4; ++i) split2(x[2 * i], x[2 * i + 1], h.u[i], m.u[i], l.u[i]);
    return {h.v, m.v, l.v};
}

// c + a b, the small terms first
__device__ __forceinline__ f32x16 mfma3(const Frag3& a, const Frag3& b, f32x16 c) {
    c = mfma16(a.l, b.h, c);
    c = mfma16(a.h, b.l, c);
    c = mfma16(a.m, b.m, c);
    c = mfma16(a.m, b.h, c);
    c = mfma16(a.h, b.m, c);
    return mfma16(a.h, b.h, c);
}

// One thread's share of KT rows of fp32, split at the store into three tiles
template <int DP, int KT, int NT>
struct Stage3 {
    static constexpr int C4 = DP / 4, N = KT * C4 / NT, TILE = KT * pitch<DP>();
    static_assert(KT * C4 % NT == 0, "tile share");
    f32x4 v[N];
    int off[N];
    uint32_t bytes;
    __device__ __forceinline__ static int row(int j) { return (threadIdx.x + j * NT) / C4; }
    __device__ __forceinline__ static int chunk(int j) { return (threadIdx.x + j * NT) % C4; }
    __device__ __forceinline__ void init(int64_t ld, int d) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            off[j] = chunk(j) * 4 < d ? static_cast<int>((row(j) * ld + chunk(j) * 4) * 4) : NO_LOAD;
        bytes = uniform(static_cast<int>((KT * ld + d) * 4));
    }
    __device__ __forceinline__ void load(const float* base, int left) {
        const i32x4 rsrc = buffer_rsrc(uniform(base), bytes);
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = raw_buffer_load_f32x4(rsrc, left >= KT || row(j) < left ? off[j] : NO_LOAD, 0, 0);
    }
    // rows whose bit is clear as zeros
    __device__ __forceinline__ void write(char* tile, uint64_t keep) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!((keep >> row(j)) & 1u)) v[j] = f32x4{};
            uint2 h, m, l;
            split2(v[j][0], v[j][1], h.x, m.x, l.x);
            split2(v[j][2], v[j][3], h.y, m.y, l.y);
            char* p = tile + row(j) * pitch<DP>() + chunk(j) * 8;
            *reinterpret_cast<uint2*>(p) = h;
            *reinterpret_cast<uint2*>(p + TILE) = m;
            *reinterpret_cast<uint2*>(p + 2 * TILE) = l;
        }
    }
};

template <int DP, int KT>
__device__ __forceinline__ Frag3 row3(const char* tile, int r, int i, int col, int half) {
    constexpr int TILE = KT * pitch<DP>();
    return {row_frag<B, DP>(tile, r, i, col, half), row_frag<B, DP>(tile + TILE, r, i, col, half),
            row_frag<B, DP>(tile + 2 * TILE, r, i, col, half)};
}
template <int DP, int KT>
__device__ __forceinline__ Frag3 tr3(const char* tile, int trl, int row, int b) {
    constexpr int TILE = KT * pitch<DP>();
    return {tr_frag<B, DP>(tile, trl, row, b), tr_frag<B, DP>(tile + TILE, trl, row, b),
            tr_frag<B, DP>(tile + 2 * TILE, trl, row, b)};
}

// KT keys a tile: 64 at the narrowest heads, else 32 (three tiles each of K
// and V, twice: 74 to 111 KB of LDS)
template <int DP, int KT, int NW>
__global__ __launch_bounds__(NW * 64, DP <= 64 ? 2 : 1) void cross_fwd32_kernel(CrossArgs a) {
    constexpr int TILE3 = 3 * KT * pitch<DP>(), NT = NW * 64, KB = KT / 32;
    constexpr f32x16 zero = {};
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE3];   // K, V; twice
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const int trl = tr_lane<DP>(lane);
    const int row = it.r0 + wave * 32 + col;
    const int qt = row / a.group, qh = kvh * a.group + row - qt * a.group;
    const int64_t token = it.q_begin + static_cast<int64_t>(qt);
    const int64_t at = token * a.heads + qh;
    Frag3 qf[DP / 16];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        float x[8] = {};
        const int c = 16 * i + 8 * half;
        if (row < it.r1 && c < a.d) load_row(static_cast<const float*>(a.q) + token * a.ldq + qh * a.ldqh + c, x);
        qf[i] = split8(x);
    }
    f32x16 o[DP / 32] = {};
    float m = -INFINITY, l = 0.f;   // m: the maximum in use, raw scores
    const float* kbase = static_cast<const float*>(a.k) + kvh * a.ldkh;
    const float* vbase = static_cast<const float*>(a.v) + kvh * a.ldvh;
    Stage3<DP, KT, NT> sk, sv;
    sk.init(a.ldk, a.d);
    sv.init(a.ldv, a.d);
    KeyBits kb;
    constexpr uint64_t ALL = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
    uint64_t bits;
    auto load = [&](int k0) {
        const int64_t key0 = it.k_begin + static_cast<int64_t>(k0);
        const int left = it.c1 - k0 < KT ? it.c1 - k0 : KT;
        kb.load(a, key0, left, lane);
        sk.load(kbase + key0 * a.ldk, left);
        sv.load(vbase + key0 * a.ldv, left);
    };
    auto write = [&](int buf) {
        bits = kb.bits(lane);
        sk.write(lds + buf * 2 * TILE3, bits);
        sv.write(lds + buf * 2 * TILE3 + TILE3, bits);
    };
    int k0 = it.c0, buf = 0;
    load(k0);   // (an item without keys goes through one tile in which none takes part)
    write(0);
    __syncthreads();
    do {
        const char* kt = lds + buf * 2 * TILE3;
        const char* vt = kt + TILE3;
        const bool more = k0 + KT < it.c1;
        if (more) load(k0 + KT);
        f32x16 s[KB];
#pragma unroll
        for (int hb = 0; hb < KB; ++hb)
#pragma unroll
            for (int i = 0; i < DP / 16; ++i)
                s[hb] = mfma3(row3<DP, KT>(kt, 32 * hb, i, col, half), qf[i], i == 0 ? zero : s[hb]);
        if (bits != ALL) {
            const uint64_t mine = bits >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16 * KB; ++r)
                if (!((mine >> (32 * (r >> 4) + acc_row(r & 15))) & 1u)) s[r >> 4][r & 15] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int r = 1; r < 16 * KB; ++r) mx = fmaxf(mx, s[r >> 4][r & 15]);
        mx = swap_max(mx);
        if (__any((mx - m) * a.c > MAX_SLACK)) {
            const float mn = fmaxf(m, mx);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) o[b] *= alpha;
        }
        const float shift = -(m == -INFINITY ? 0.f : m) * a.c;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16 * KB; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[r >> 4][r & 15], a.c, shift));
            s[r >> 4][r & 15] = p;
            sum += p;
        }
        l += sum;
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = s[t >> 1][8 * (t & 1) + i];
            const Frag3 p = split8(x);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) o[b] = mfma3(tr3<DP, KT>(vt, trl, 16 * t, b), p, o[b]);
        }
        if (more) write(buf ^ 1);
        __syncthreads();
        buf ^= 1;
        k0 += KT;
    } while (k0 < it.c1);
    l = swap_add(l);
    if (row >= it.r1) return;
    const float m2 = (m == -INFINITY ? 0.f : m) * a.c;
    if (it.slot >= 0) {
        float* p = a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * a.tile + row - it.r0) * (a.d + 2);
        store_acc<float, DP>(p, o, 1.f, a.d, half);
        if (half == 0) p[a.d] = m == -INFINITY ? -INFINITY : m2;
        else p[a.d + 1] = l;
        return;
    }
    store_acc<float, DP>(static_cast<float*>(a.out) + at * a.d, o, l == 0.f ? 0.f : 1.f / l, a.d, half);
    if (a.lse && half == 0) a.lse[at] = l == 0.f ? INFINITY : m2 + log2f(l);
}

template <int DP>
void launch32(const CrossArgs& a, hipStream_t st) {
    constexpr int KT = DP == 32 ? 64 : 32;
    hipLaunchKernelGGL((cross_fwd32_kernel<DP, KT, 4>), dim3(cross_grid(a)), dim3(256), 0, st,
                       a);
}

}  // namespace

int cross_forward32(const CrossArgs& a, hipStream_t st) {
    if (a.d <= 32) launch32<32>(a, st);
    else if (a.d <= 64) launch32<64>(a, st);
    else if (a.d <= 96) launch32<96>(a, st);
    else launch32<128>(a, st);
    return launch_status("cross_fwd32_kernel");
}

}  // namespace mignn
