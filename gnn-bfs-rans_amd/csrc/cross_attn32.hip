// Cross attention of fp32 rows on the bf16 matrix instructions (formulas:
// cross_attn.hip; structure: cross_attn16.hip).
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
// instruction takes 512 (which measured, at 12225 x 12225 x 4 x 32: 840 us
// against 468, 163 TFLOP/s; a plain fp32 product of 8192^3 reaches 153).  The
// tiles are split once a workgroup, on their way into LDS; what a wave owns at
// the start; P and dS in registers, in place.  Bound by the vector unit (80 %
// busy, most of it the splits; the matrix unit 47 %).  Trained, 19488 rows
// against 379 keys in three sequences, 4 heads of 64: forward 27 us, dq 44, dk
// / dv 62.
#include "mfma16.hpp"

namespace mignn {
namespace {

using B = bf16_t;

constexpr int KT = 32;   // rows of an LDS tile

// x = h + m + l, two numbers at a time: one instruction converts a pair
__device__ __forceinline__ uint32_t pair_bits(float a, float b) {
    typedef float f32pair __attribute__((ext_vector_type(2)));
    typedef B pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32pair{a, b}), pair));
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& h, uint32_t& m, uint32_t& l) {
    h = pair_bits(a, b);
    a -= __uint_as_float(h << 16), b -= __uint_as_float(h & 0xffff0000u);
    m = pair_bits(a, b);
    a -= __uint_as_float(m << 16), b -= __uint_as_float(m & 0xffff0000u);
    l = pair_bits(a, b);
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

// N fragments of a row
template <int DP>
__device__ __forceinline__ void load_frag3(Frag3 (&f)[DP / 16], const float* p, int d, int half) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        float x[8] = {};
        const int c = 16 * i + 8 * half;
        if (p && c < d) load_row(p + c, x);
        f[i] = split8(x);
    }
}

__device__ __forceinline__ Frag3 split_acc(const f32x16& w, int t) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = w[8 * t + i];
    return split8(x);
}

// One thread's share of KT rows of fp32, split at the store into three tiles
template <int DP, int NT>
struct Stage3 {
    static constexpr int C4 = DP / 4, N = KT * C4 / NT, TILE = KT * TileRow<DP>::BYTES;
    static_assert(KT * C4 % NT == 0, "tile share");
    f32x4 v[N];
    int off[N], lds[N];
    uint32_t bytes;
    __device__ __forceinline__ static int row(int j) { return (threadIdx.x + j * NT) / C4; }
    __device__ __forceinline__ static int chunk(int j) { return (threadIdx.x + j * NT) % C4; }
    // tile row r is row r / group, head r % group of a matrix of strides ldt, ldh
    __device__ __forceinline__ void init(int64_t ldt, int64_t ldh, int group, int d) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int t = row(j) / group, h = row(j) - t * group;
            off[j] = chunk(j) * 4 < d ? static_cast<int>((t * ldt + h * ldh + chunk(j) * 4) * 4) : NO_LOAD;
            lds[j] = TileRow<DP>::at(row(j), chunk(j) * 4);
        }
        bytes = uniform(static_cast<int>((KT / group * ldt + group * ldh + d) * 4));
    }
    __device__ __forceinline__ void load(const float* base, int left) {
        const i32x4 rsrc = buffer_rsrc(uniform(base), bytes);
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = raw_buffer_load_f32x4(rsrc, left >= KT || row(j) < left ? off[j] : NO_LOAD, 0, 0);
    }
    // rows whose bit is clear as zeros
    __device__ __forceinline__ void write(char* tile, uint32_t keep) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (!((keep >> row(j)) & 1u)) v[j] = f32x4{};
            uint2 h, m, l;
            split2(v[j][0], v[j][1], h.x, m.x, l.x);
            split2(v[j][2], v[j][3], h.y, m.y, l.y);
            char* p = tile + lds[j];
            *reinterpret_cast<uint2*>(p) = h;
            *reinterpret_cast<uint2*>(p + TILE) = m;
            *reinterpret_cast<uint2*>(p + 2 * TILE) = l;
        }
    }
};

template <int DP>
__device__ __forceinline__ Frag3 row3(const char* tile, const TileLane<DP>& tl, int i) {
    constexpr int TILE = KT * TileRow<DP>::BYTES;
    return {row_frag<B, DP>(tile, tl, 0, i), row_frag<B, DP>(tile + TILE, tl, 0, i),
            row_frag<B, DP>(tile + 2 * TILE, tl, 0, i)};
}
template <int DP>
__device__ __forceinline__ Frag3 tr3(const char* tile, const TileLane<DP>& tl, int row, int b) {
    constexpr int TILE = KT * TileRow<DP>::BYTES;
    return {tr_frag<B, DP>(tile, tl, row, b), tr_frag<B, DP>(tile + TILE, tl, row, b),
            tr_frag<B, DP>(tile + 2 * TILE, tl, row, b)};
}

// (three tiles each of K and V, twice: 25 KB of LDS for heads of 32, 98 KB for
// 128; 64 keys a tile measured 5 % slower)
template <int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW == 1 ? 1 : DP <= 64 ? 3 : 1) void cross_fwd32_kernel(
    CrossArgs a) {
    constexpr int TILE3 = 3 * KT * TileRow<DP>::BYTES, NT = NW * 64;
    constexpr f32x16 zero = {};
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE3];   // K, V; twice
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const TileLane<DP> tl(lane);
    const int row = it.r0 + wave * 32 + col;
    const int qt = row / a.group, qh = kvh * a.group + row - qt * a.group;
    const int64_t token = it.q_begin + static_cast<int64_t>(qt);
    const int64_t at = token * a.heads + qh;
    Frag3 qf[DP / 16];
    load_frag3<DP>(qf, row < it.r1 ? static_cast<const float*>(a.q) + token * a.ldq + qh * a.ldqh : nullptr,
                   a.d, half);
    f32x16 o[DP / 32] = {};
    float m = -INFINITY, l = 0.f;   // m: the maximum in use, raw scores
    const float* kbase = static_cast<const float*>(a.k) + kvh * a.ldkh;
    const float* vbase = static_cast<const float*>(a.v) + kvh * a.ldvh;
    Stage3<DP, NT> sk, sv;
    sk.init(a.ldk, 0, 1, a.d);
    sv.init(a.ldv, 0, 1, a.d);
    KeyBits kb;
    uint32_t bits;
    auto load = [&](int k0) {
        const int64_t key0 = it.k_begin + static_cast<int64_t>(k0);
        const int left = it.c1 - k0 < KT ? it.c1 - k0 : KT;
        kb.load(a, key0, left, lane);
        sk.load(kbase + key0 * a.ldk, left);
        sv.load(vbase + key0 * a.ldv, left);
    };
    auto write = [&](int buf) {
        bits = static_cast<uint32_t>(kb.bits(lane));
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
        f32x16 s;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i)
            s = mfma3(row3<DP>(kt, tl, i), qf[i], i == 0 ? zero : s);
        if (bits != ~0u) {
            const uint32_t mine = bits >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!((mine >> acc_row(r)) & 1u)) s[r] = -INFINITY;
        }
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
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
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, shift));
            sum += s[r];
        }
        l += sum;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Frag3 p = split_acc(s, t);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) o[b] = mfma3(tr3<DP>(vt, tl, 16 * t, b), p, o[b]);
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

template <int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW > 1 && DP <= 64 ? 2 : 1) void cross_dq32_kernel(CrossArgs a) {
    constexpr int TILE3 = 3 * KT * TileRow<DP>::BYTES, NT = NW * 64;
    constexpr f32x16 zero = {};
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE3];   // K, V; twice
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const TileLane<DP> tl(lane);
    const int row = it.r0 + wave * 32 + col;
    const bool live = row < it.r1;
    const int qt = row / a.group, qh = kvh * a.group + row - qt * a.group;
    const int64_t token = it.q_begin + static_cast<int64_t>(qt);
    const int64_t at = token * a.heads + qh;
    Frag3 qf[DP / 16], gf[DP / 16];
    load_frag3<DP>(qf, live ? static_cast<const float*>(a.q) + token * a.ldq + qh * a.ldqh : nullptr, a.d, half);
    const float* dout = live ? static_cast<const float*>(a.dout) + token * a.lddo + qh * a.lddoh : nullptr;
    load_frag3<DP>(gf, dout, a.d, half);
    float delta = 0.f;
    if (live) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int c = 16 * i + 8 * half;
            if (c >= a.d) continue;
            float x[8], y[8];
            load_row(a.out32 + at * a.d + c, x);
            load_row(dout + c, y);
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf(x[e], y[e], delta);
        }
    }
    delta = swap_add(delta);
    // the dk / dv kernel's: written by the item of the row's first keys
    if (live && half == 0 && it.c0 == 0) a.delta[at] = delta;
    const float lse = live ? a.lse[at] : INFINITY;
    f32x16 acc[DP / 32] = {};
    const float* kbase = static_cast<const float*>(a.k) + kvh * a.ldkh;
    const float* vbase = static_cast<const float*>(a.v) + kvh * a.ldvh;
    Stage3<DP, NT> sk, sv;
    sk.init(a.ldk, 0, 1, a.d);
    sv.init(a.ldv, 0, 1, a.d);
    KeyBits kb;
    uint32_t bits;
    auto load = [&](int k0) {
        const int64_t key0 = it.k_begin + static_cast<int64_t>(k0);
        const int left = it.c1 - k0 < KT ? it.c1 - k0 : KT;
        kb.load(a, key0, left, lane);
        sk.load(kbase + key0 * a.ldk, left);
        sv.load(vbase + key0 * a.ldv, left);
    };
    auto write = [&](int buf) {
        bits = static_cast<uint32_t>(kb.bits(lane));
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
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            s = mfma3(row3<DP>(kt, tl, i), qf[i], i == 0 ? zero : s);
            dp = mfma3(row3<DP>(vt, tl, i), gf[i], i == 0 ? zero : dp);
        }
        const uint32_t mine = bits >> (4 * half);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lse)) * (dp[r] - delta);
            s[r] = (mine >> acc_row(r)) & 1u ? p : 0.f;
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Frag3 p = split_acc(s, t);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) acc[b] = mfma3(tr3<DP>(kt, tl, 16 * t, b), p, acc[b]);
        }
        if (more) write(buf ^ 1);
        __syncthreads();
        buf ^= 1;
        k0 += KT;
    } while (k0 < it.c1);
    if (!live) return;
    if (it.slot >= 0)
        store_acc<float, DP>(a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * a.tile + row - it.r0) * a.d,
                             acc, a.scale, a.d, half);
    else
        store_acc<float, DP>(static_cast<float*>(a.out) + at * a.d, acc, a.scale, a.d, half);
}

template <int DP, int NW>
__global__ __launch_bounds__(NW * 64, NW > 1 && DP <= 32 ? 2 : 1) void cross_dkv32_kernel(CrossArgs a) {
    constexpr int TILE3 = 3 * KT * TileRow<DP>::BYTES, NT = NW * 64;
    constexpr f32x16 zero = {};
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE3];   // q, do; twice
    __shared__ __attribute__((aligned(16))) float st[2][2][KT];    // lse, delta
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const TileLane<DP> tl(lane);
    const int key = it.r0 + wave * 32 + col;
    const int64_t kt = it.k_begin + static_cast<int64_t>(key);
    const bool live = key < it.r1, keep = live && (!a.mask || a.mask[kt]);
    Frag3 kf[DP / 16], vf[DP / 16];
    load_frag3<DP>(kf, keep ? static_cast<const float*>(a.k) + kt * a.ldk + kvh * a.ldkh : nullptr, a.d, half);
    load_frag3<DP>(vf, keep ? static_cast<const float*>(a.v) + kt * a.ldv + kvh * a.ldvh : nullptr, a.d, half);
    f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    const float* qbase = static_cast<const float*>(a.q) + it.q_begin * a.ldq + kvh * a.group * a.ldqh;
    const float* gbase = static_cast<const float*>(a.dout) + it.q_begin * a.lddo + kvh * a.group * a.lddoh;
    Stage3<DP, NT> sq, sg;
    sq.init(a.ldq, a.ldqh, a.group, a.d);
    sg.init(a.lddo, a.lddoh, a.group, a.d);
    // whole queries a tile: the offsets are the same in every tile
    const int tokens = KT / a.group, step = tokens * a.group;
    const int my_t = threadIdx.x / a.group, my_h = threadIdx.x - my_t * a.group;
    float lse = INFINITY, delta = 0.f;
    int left = 0;
    auto load = [&](int r0, int t0) {
        left = it.c1 - r0 < step ? it.c1 - r0 : step;
        sq.load(qbase + t0 * a.ldq, left);
        sg.load(gbase + t0 * a.lddo, left);
        if (threadIdx.x < KT) {   // rows past the end: lse = inf, P = 0
            lse = INFINITY, delta = 0.f;
            if (static_cast<int>(threadIdx.x) < left) {
                const int64_t at = (it.q_begin + static_cast<int64_t>(t0 + my_t)) * a.heads + kvh * a.group + my_h;
                lse = a.lse[at];
                delta = a.delta[at];
            }
        }
    };
    auto write = [&](int buf) {
        sq.write(lds + buf * 2 * TILE3, ~0u);
        sg.write(lds + buf * 2 * TILE3 + TILE3, ~0u);
        if (threadIdx.x < KT) st[buf][0][threadIdx.x] = lse, st[buf][1][threadIdx.x] = delta;
    };
    int r0 = it.c0, t0 = it.c0 / a.group, buf = 0;
    load(r0, t0);   // (an item without rows goes through one tile of P = 0)
    write(0);
    __syncthreads();
    do {
        const char* qt = lds + buf * 2 * TILE3;
        const char* gt = qt + TILE3;
        const bool more = r0 + step < it.c1;
        if (more) load(r0 + step, t0 + tokens);
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            s = mfma3(row3<DP>(qt, tl, i), kf[i], i == 0 ? zero : s);
            dp = mfma3(row3<DP>(gt, tl, i), vf[i], i == 0 ? zero : dp);
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 x = ld4(&st[buf][0][8 * g + 4 * half]), y = ld4(&st[buf][1][8 * g + 4 * half]);
            const float lv[4] = {x.x, x.y, x.z, x.w}, ev[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = 4 * g + e;
                s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lv[e]));
                dp[r] = s[r] * (dp[r] - ev[e]);
            }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const Frag3 p = split_acc(s, t), ds = split_acc(dp, t);
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                dv[b] = mfma3(tr3<DP>(gt, tl, 16 * t, b), p, dv[b]);
                dk[b] = mfma3(tr3<DP>(qt, tl, 16 * t, b), ds, dk[b]);
            }
        }
        if (more) write(buf ^ 1);
        __syncthreads();
        buf ^= 1;
        r0 += step;
        t0 += tokens;
    } while (r0 < it.c1);
    if (!live) return;
    // a key that the mask leaves out has no gradient, whatever its rows hold
    if (!keep) {
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) dk[b] = dv[b] = f32x16{};
    }
    if (it.slot >= 0) {
        float* p = a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * a.tile + key - it.r0) * (2 * a.d);
        store_acc<float, DP>(p, dk, a.scale, a.d, half);
        store_acc<float, DP>(p + a.d, dv, 1.f, a.d, half);
    } else {
        const int64_t at = (kt * a.kv_heads + kvh) * a.d;
        store_acc<float, DP>(static_cast<float*>(a.dk) + at, dk, a.scale, a.d, half);
        store_acc<float, DP>(static_cast<float*>(a.dv) + at, dv, 1.f, a.d, half);
    }
}

template <int DP, int NW>
void launch32(const CrossArgs& a, int pass, hipStream_t st) {
    const dim3 grid(cross_grid(a)), block(NW * 64);
    if (pass == MIGNN_CROSS_FORWARD)
        hipLaunchKernelGGL((cross_fwd32_kernel<DP, NW>), grid, block, 0, st, a);
    else if (pass == MIGNN_CROSS_DQ)
        hipLaunchKernelGGL((cross_dq32_kernel<DP, NW>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((cross_dkv32_kernel<DP, NW>), grid, block, 0, st, a);
}

template <int DP>
void launch32_d(const CrossArgs& a, int pass, hipStream_t st) {
    if (a.tile == CROSS_ROWS) launch32<DP, 1>(a, pass, st);
    else launch32<DP, 4>(a, pass, st);
}

}  // namespace

int cross_pass32(const CrossArgs& a, int pass, hipStream_t st) {
    if (a.d <= 32) launch32_d<32>(a, pass, st);
    else if (a.d <= 64) launch32_d<64>(a, pass, st);
    else if (a.d <= 96) launch32_d<96>(a, pass, st);
    else launch32_d<128>(a, pass, st);
    return launch_status("cross attention kernel (fp32)");
}

}  // namespace mignn
