// Cross attention of bf16 and fp16 rows on the 16-bit matrix instructions
// (formulas and pass structure: cross_attn.hip).
//
// A wave owns 32 rows (forward, dq) or keys (dk / dv) as MFMA columns.  The
// other side comes in LDS tiles of 64, double buffered through registers:
// while a tile is worked on, the next one's rows are in flight.
//   S^T (keys x rows)   A = key rows, 16 bytes a lane;  B = q, in registers
//   O^T (d x rows)      A = V^T, read transposed from the row-major tile
//                       (ds_read_b64_tr_b16: 4 rows x 16 columns a 16-lane
//                       group);  B = P^T, the accumulator of S^T rounded in
//                       place: the product over keys takes them in the order
//                       in which its registers hold them
// dq and dk / dv are made of the same two forms.
//
// P and dS are rounded to the rows' type ahead of their second product (the
// matrix instruction takes both operands in one type), which adds to a result
// about what its own rounding does; statistics, sums and accumulators are fp32.
// Where rows or results are few (the plan's rule) the roundings' remainders go
// through a second product (REST), and only the output's rounding is left.
// bf16 has fp32's range.  fp16 has not: a weight of 1 / 5000 is already
// subnormal there, so P is carried up by a constant power of two and dS by one
// that each row (dq) or key (dk) lowers when its values would not fit
// (DsScale); the results are brought back in fp32.
//
// Bound by issue: the vector unit (exponentials, maxima, roundings) and the
// matrix unit take turns within a wave, so it is other waves that fill the gaps
// (busy, of 128 columns: 45 % each; of 64: 62 / 36 % in the forward, 58 / 46 in dq,
// 47 / 43 in dk / dv).  Measured (a plain product of
// 8192^3 reaches 1203 TFLOP/s in bf16, 1150 in fp16): 49181 rows x 4096 keys x 4
// heads over 2 of 64, bf16: forward 270 us (763 TFLOP/s), dq 340 (909), dk / dv
// 460 (897); 2 x 16384^2 x 8 x 128, fp16: forward 2370 (928; 2105 us with the
// softmax left out).  Heads to 64 run forward and dq at three waves a SIMD (dk
// / dv, and all of 128 columns, spill there: 2790 us).  Tiles of 32 keys cost
// 270 -> 296 us, reads of LDS ahead of time by fences of the scheduler 350 -> 404.
#include "mfma16.hpp"

namespace mignn {
namespace {

constexpr int KT = CROSS_STAGE;

// B operand rows held in registers
template <typename T, int DP>
__device__ __forceinline__ void load_frag16(vec8<T> (&f)[DP / 16], const T* p, int d, int half) {
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) {
        const int c = 16 * i + 8 * half;
        f[i] = vec8<T>{};
        if (p && c < d) f[i] = *reinterpret_cast<const vec8<T>*>(p + c);
    }
}

// registers 8 t ..+7 of a 32 x 32 accumulator as the B operand of 16 rows
template <typename T>
__device__ __forceinline__ vec8<T> pack8(const f32x16& w, int t) {
    vec8<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(w[8 * t + i]);
    return v;
}

// what pack8's rounding left, rounded
template <typename T>
__device__ __forceinline__ vec8<T> rest8(const f32x16& w, const vec8<T>& v, int t) {
    vec8<T> x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<T>(w[8 * t + i] - static_cast<float>(v[i]));
    return x;
}

// One thread's share of a 64-row tile on its way from memory to LDS: buffer
// loads at constant offsets from a scalar base that moves on with the tiles
template <typename T, int DP, int NT>
struct Stage {
    static constexpr int C8 = DP / 8, N = KT * C8 / NT;
    static_assert(KT * C8 % NT == 0, "tile share");
    f32x4 v[N];
    int off[N], lds[N];
    uint32_t bytes;
    __device__ __forceinline__ static int row(int j) { return (threadIdx.x + j * NT) / C8; }
    __device__ __forceinline__ static int chunk(int j) { return (threadIdx.x + j * NT) % C8; }
    // tile row r is row r / group, head r % group of a matrix of strides ldt, ldh
    __device__ __forceinline__ void init(int64_t ldt, int64_t ldh, int group, int d) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int t = row(j) / group, h = row(j) - t * group;
            off[j] = chunk(j) * 8 < d ? static_cast<int>((t * ldt + h * ldh + chunk(j) * 8) * sizeof(T))
                                      : NO_LOAD;
            lds[j] = TileRow<DP>::at(row(j), chunk(j) * 8);
        }
        // (63 rows' and all heads' strides fit: checked by the host)
        bytes = uniform(static_cast<int>((KT / group * ldt + group * ldh + d) * sizeof(T)));
    }
    // the `left` rows from `base` on; zeros after them
    __device__ __forceinline__ void load(const T* base, int left) {
        const i32x4 rsrc = buffer_rsrc(uniform(base), bytes);
#pragma unroll
        for (int j = 0; j < N; ++j)
            v[j] = raw_buffer_load_f32x4(rsrc, left >= KT || row(j) < left ? off[j] : NO_LOAD, 0, 0);
    }
    __device__ __forceinline__ void write(char* tile) const {
#pragma unroll
        for (int j = 0; j < N; ++j)
            *reinterpret_cast<f32x4*>(tile + lds[j]) = v[j];
    }
    // rows whose bit is clear as zeros
    __device__ __forceinline__ void write(char* tile, uint64_t keep) const {
        if (keep == ~0ull) return write(tile);
#pragma unroll
        for (int j = 0; j < N; ++j)
            *reinterpret_cast<f32x4*>(tile + lds[j]) =
                (keep >> row(j)) & 1u ? v[j] : f32x4{};
    }
};

// fp16's P is kept 2^8 up: a weight down to 2^-22 of the largest keeps its
// full precision, and 2^(8 + 6) stays below fp16's largest.  bf16 has fp32's
// range.
template <typename T>
constexpr float P_UP = 0.f;
template <>
constexpr float P_UP<f16_t> = 8.f;
template <typename T>
constexpr bool NARROW = sizeof(T) == 2 && !__is_same(T, bf16_t);
// P's power of two in the dk / dv kernel, where it is at most 1
template <typename T>
constexpr float PB_UP = NARROW<T> ? 14.f : 0.f;

// dS of one row (or key) as fp16: 2^up dS.  When a value passes 2^15, `up` is
// lowered so that the largest comes to 2^8 and what is summed so far is
// brought along, in the same way as a softmax's maximum.
template <typename T>
struct DsScale {
    float up = NARROW<T> ? 12.f : 0.f;
    template <int NB>
    __device__ __forceinline__ bool fit(f32x16& ds, f32x16 (&acc)[NB]) {
        if constexpr (!NARROW<T>) return false;
        float mx = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, fabsf(ds[r]));
        if (!__any(mx > 32768.f)) return false;
        mx = swap_max(mx);
        const int e = static_cast<int>((__float_as_uint(mx) >> 23) & 255u) - 127 - 7;
        const float down = mx > 32768.f ? static_cast<float>(e) : 0.f;
        const float f = __builtin_amdgcn_exp2f(-down);
        up -= down;
        ds *= f;
#pragma unroll
        for (int b = 0; b < NB; ++b) acc[b] *= f;
        return true;
    }
    __device__ __forceinline__ float back() const { return NARROW<T> ? __builtin_amdgcn_exp2f(-up) : 1.f; }
};

template <typename T, int DP, int NW, bool REST>
__global__ __launch_bounds__(NW * 64, NW > 1 ? (DP <= 64 ? 3 : 2) : DP == 32 ? 2 : 1) void cross_fwd16_kernel(CrossArgs a) {
    constexpr int TILE = KT * TileRow<DP>::BYTES, NT = NW * 64;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE];   // K, V; twice
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const TileLane<DP> tl(lane);
    constexpr f32x16 zero = {};
    vec8<T> qf[DP / 16];
    const int row = it.r0 + wave * 32 + col;
    const int t = row / a.group, h = kvh * a.group + row - t * a.group;
    const int64_t token = it.q_begin + static_cast<int64_t>(t);
    const int64_t at = token * a.heads + h;
    load_frag16<T, DP>(qf, row < it.r1 ? static_cast<const T*>(a.q) + token * a.ldq + h * a.ldqh
                                               : nullptr, a.d, half);
    f32x16 o[DP / 32] = {};
    float m = -INFINITY, l = 0.f;   // m: the maximum in use, raw scores
    const T* kbase = static_cast<const T*>(a.k) + kvh * a.ldkh;
    const T* vbase = static_cast<const T*>(a.v) + kvh * a.ldvh;
    Stage<T, DP, NT> sk, sv;
    sk.init(a.ldk, 0, 1, a.d);
    sv.init(a.ldv, 0, 1, a.d);
    KeyBits kb;
    uint64_t bits = 0;
    if (it.c0 < it.c1) {
        const int64_t key0 = it.k_begin + static_cast<int64_t>(it.c0);
        const int left = it.c1 - it.c0;
        kb.load(a, key0, left, lane);
        sk.load(kbase + key0 * a.ldk, left);
        sv.load(vbase + key0 * a.ldv, left);
        bits = kb.bits(lane);
        sk.write(lds);
        sv.write(lds + TILE, bits);
    }
    __syncthreads();
    int buf = 0;
    for (int k0 = it.c0; k0 < it.c1; k0 += KT) {
        const char* kt = lds + buf * 2 * TILE;
        const char* vt = kt + TILE;
        const bool more = k0 + KT < it.c1;
        if (more) {
            const int64_t key0 = it.k_begin + static_cast<int64_t>(k0 + KT);
            const int left = it.c1 - k0 - KT;
            kb.load(a, key0, left, lane);
            sk.load(kbase + key0 * a.ldk, left);
            sv.load(vbase + key0 * a.ldv, left);
        }
        f32x16 s[2];
#pragma unroll
        for (int hb = 0; hb < 2; ++hb)
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const vec8<T> f = row_frag<T, DP>(kt, tl, 32 * hb, i);
                s[hb] = mfma16(f, qf[i], i == 0 ? zero : s[hb]);
            }
        if (bits != ~0ull) {
            const uint64_t mine = bits >> (4 * half);
#pragma unroll
            for (int hb = 0; hb < 2; ++hb)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> (32 * hb + acc_row(r))) & 1u)) s[hb][r] = -INFINITY;
        }
        float mx = s[0][0];
#pragma unroll
        for (int r = 1; r < 32; ++r) mx = fmaxf(mx, s[r >> 4][r & 15]);
        mx = swap_max(mx);
        // (m = -inf: any score raises it)
        if (__any((mx - m) * a.c > MAX_SLACK)) {
            const float mn = fmaxf(m, mx);
            const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.c);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) o[b] *= alpha;
        }
        const float shift = P_UP<T> - (m == -INFINITY ? 0.f : m) * a.c;
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[r >> 4][r & 15], a.c, shift));
            s[r >> 4][r & 15] = p;
            sum += p;
        }
        l += sum;
#pragma unroll
        for (int t = 0; t < KT / 16; ++t) {
            const vec8<T> p = pack8<T>(s[t >> 1], t & 1);
            const vec8<T> rest = REST ? rest8<T>(s[t >> 1], p, t & 1) : p;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) {
                const vec8<T> f = tr_frag<T, DP>(vt, tl, 16 * t, b);
                if constexpr (REST) o[b] = mfma16(f, rest, o[b]);
                o[b] = mfma16(f, p, o[b]);
            }
        }
        if (more) {
            char* dst = lds + (buf ^ 1) * 2 * TILE;
            bits = kb.bits(lane);
            sk.write(dst);
            sv.write(dst + TILE, bits);
        }
        __syncthreads();
        buf ^= 1;
    }
    const float sum = swap_add(l);
    if (row >= it.r1) return;
    const float m2 = (m == -INFINITY ? 0.f : m) * a.c - P_UP<T>;
    if (it.slot >= 0) {
        float* p = a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * (NW * 32) +
                             row - it.r0) * (a.d + 2);
        store_acc<float, DP>(p, o, 1.f, a.d, half);
        if (half == 0) p[a.d] = m == -INFINITY ? -INFINITY : m2;
        else p[a.d + 1] = sum;
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    store_acc<T, DP>(static_cast<T*>(a.out) + at * a.d, o, inv, a.d, half);
    if (a.o32) store_acc<float, DP>(a.o32 + at * a.d, o, inv, a.d, half);
    if (a.lse && half == 0) a.lse[at] = sum == 0.f ? INFINITY : m2 + log2f(sum);
}

template <typename T, int DP, int NW, bool REST>
__global__ __launch_bounds__(NW * 64, NW > 1 ? (DP <= 64 ? 3 : 2) : DP == 32 ? 2 : 1) void cross_dq16_kernel(CrossArgs a) {
    constexpr int TILE = KT * TileRow<DP>::BYTES, NT = NW * 64;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE];
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const TileLane<DP> tl(lane);
    constexpr f32x16 zero = {};
    vec8<T> qf[DP / 16], gf[DP / 16];
    const int row = it.r0 + wave * 32 + col;
    const bool live = row < it.r1;
    const int t = row / a.group, h = kvh * a.group + row - t * a.group;
    const int64_t token = it.q_begin + static_cast<int64_t>(t);
    const int64_t at = token * a.heads + h;
    load_frag16<T, DP>(qf, live ? static_cast<const T*>(a.q) + token * a.ldq + h * a.ldqh : nullptr,
                       a.d, half);
    load_frag16<T, DP>(gf, live ? static_cast<const T*>(a.dout) + token * a.lddo + h * a.lddoh
                                    : nullptr, a.d, half);
    float del = 0.f;
    if (live) {
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
            const int c = 16 * i + 8 * half;
            if (c >= a.d) continue;
            const float4 x = ld4(a.out32 + at * a.d + c), y = ld4(a.out32 + at * a.d + c + 4);
            const float ov[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) del = fmaf(ov[e], static_cast<float>(gf[i][e]), del);
        }
    }
    const float delta = swap_add(del);
    // the dk / dv kernel's: written by the item of the row's first keys
    if (live && half == 0 && it.c0 == 0) a.delta[at] = delta;
    const float lse = live ? a.lse[at] : INFINITY;
    f32x16 acc[DP / 32] = {};
    DsScale<T> sc;
    const T* kbase = static_cast<const T*>(a.k) + kvh * a.ldkh;
    const T* vbase = static_cast<const T*>(a.v) + kvh * a.ldvh;
    Stage<T, DP, NT> sk, sv;
    sk.init(a.ldk, 0, 1, a.d);
    sv.init(a.ldv, 0, 1, a.d);
    KeyBits kb;
    uint64_t bits = 0;
    if (it.c0 < it.c1) {
        const int64_t key0 = it.k_begin + static_cast<int64_t>(it.c0);
        const int left = it.c1 - it.c0;
        kb.load(a, key0, left, lane);
        sk.load(kbase + key0 * a.ldk, left);
        sv.load(vbase + key0 * a.ldv, left);
        bits = kb.bits(lane);
        sk.write(lds, bits);
        sv.write(lds + TILE, bits);
    }
    __syncthreads();
    int buf = 0;
    for (int k0 = it.c0; k0 < it.c1; k0 += KT) {
        const char* kt = lds + buf * 2 * TILE;
        const char* vt = kt + TILE;
        const bool more = k0 + KT < it.c1;
        if (more) {
            const int64_t key0 = it.k_begin + static_cast<int64_t>(k0 + KT);
            const int left = it.c1 - k0 - KT;
            kb.load(a, key0, left, lane);
            sk.load(kbase + key0 * a.ldk, left);
            sv.load(vbase + key0 * a.ldv, left);
        }
#pragma unroll
        for (int hb = 0; hb < 2; ++hb) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const vec8<T> fk = row_frag<T, DP>(kt, tl, 32 * hb, i);
                const vec8<T> fv = row_frag<T, DP>(vt, tl, 32 * hb, i);
                s = mfma16(fk, qf[i], i == 0 ? zero : s);
                dp = mfma16(fv, gf[i], i == 0 ? zero : dp);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, sc.up - lse)) * (dp[r] - delta);
            if (bits != ~0ull) {
                const uint32_t mine = static_cast<uint32_t>(bits >> (32 * hb + 4 * half));
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((mine >> acc_row(r)) & 1u)) s[r] = 0.f;
            }
            sc.fit(s, acc);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const vec8<T> p = pack8<T>(s, t);
                const vec8<T> rest = REST ? rest8<T>(s, p, t) : p;
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) {
                    const vec8<T> f = tr_frag<T, DP>(kt, tl, 32 * hb + 16 * t, b);
                    if constexpr (REST) acc[b] = mfma16(f, rest, acc[b]);
                    acc[b] = mfma16(f, p, acc[b]);
                }
            }
        }
        if (more) {
            char* dst = lds + (buf ^ 1) * 2 * TILE;
            bits = kb.bits(lane);
            sk.write(dst, bits);
            sv.write(dst + TILE, bits);
        }
        __syncthreads();
        buf ^= 1;
    }
    if (row >= it.r1) return;
    const float f = a.scale * sc.back();
    if (it.slot >= 0)
        store_acc<float, DP>(a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * (NW * 32) +
                                         row - it.r0) * a.d, acc, f, a.d, half);
    else
        store_acc<T, DP>(static_cast<T*>(a.out) + at * a.d, acc, f, a.d, half);
}

template <typename T, int DP, int NW, bool REST>
__global__ __launch_bounds__(NW * 64, DP <= (NW > 1 ? 96 : 32) ? 2 : 1) void cross_dkv16_kernel(CrossArgs a) {
    constexpr int TILE = KT * TileRow<DP>::BYTES, NT = NW * 64;
    __shared__ __attribute__((aligned(16))) char lds[4 * TILE];
    __shared__ __attribute__((aligned(16))) float st[2][2][KT];   // lse, delta
    int item, kvh;
    if (!cross_work(a, item, kvh)) return;
    const CrossItem it = load_item(a, item);
    const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5, wave = threadIdx.x >> 6;
    const TileLane<DP> tl(lane);
    constexpr f32x16 zero = {};
    vec8<T> kf[DP / 16], vf[DP / 16];
    const int key = it.r0 + wave * 32 + col;
    const int64_t kt = it.k_begin + static_cast<int64_t>(key);
    const bool keep = key < it.r1 && (!a.mask || a.mask[kt]);
    load_frag16<T, DP>(kf, keep ? static_cast<const T*>(a.k) + kt * a.ldk + kvh * a.ldkh : nullptr,
                       a.d, half);
    load_frag16<T, DP>(vf, keep ? static_cast<const T*>(a.v) + kt * a.ldv + kvh * a.ldvh : nullptr,
                       a.d, half);
    f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};
    DsScale<T> sc;
    float gain = __builtin_amdgcn_exp2f(sc.up - PB_UP<T>);   // dS's power of two over P's
    const T* qbase = static_cast<const T*>(a.q) + it.q_begin * a.ldq + kvh * a.group * a.ldqh;
    const T* gbase = static_cast<const T*>(a.dout) + it.q_begin * a.lddo + kvh * a.group * a.lddoh;
    Stage<T, DP, NT> sq, sg;
    sq.init(a.ldq, a.ldqh, a.group, a.d);
    sg.init(a.lddo, a.lddoh, a.group, a.d);
    // whole queries a tile: the offsets are the same in every tile
    const int tokens = KT / a.group, step = tokens * a.group;
    const int my_t = threadIdx.x / a.group, my_h = threadIdx.x - my_t * a.group;
    float lse = INFINITY, delta = 0.f;
    auto load = [&](int r0, int t0) {
        const int left = it.c1 - r0 < step ? it.c1 - r0 : step;
        sq.load(qbase + t0 * a.ldq, left);
        sg.load(gbase + t0 * a.lddo, left);
        if (threadIdx.x < KT) {   // rows past the end: lse = inf, P = 0
            lse = INFINITY, delta = 0.f;
            if (static_cast<int>(threadIdx.x) < left) {
                const int64_t at = (it.q_begin + static_cast<int64_t>(t0 + my_t)) * a.heads + kvh * a.group + my_h;
                lse = a.lse[at] - PB_UP<T>;
                delta = a.delta[at];
            }
        }
    };
    auto write = [&](int buf) {
        sq.write(lds + buf * 2 * TILE);
        sg.write(lds + buf * 2 * TILE + TILE);
        if (threadIdx.x < KT) st[buf][0][threadIdx.x] = lse, st[buf][1][threadIdx.x] = delta;
    };
    if (it.c0 < it.c1) {
        load(it.c0, it.c0 / a.group);
        write(0);
    }
    __syncthreads();
    int buf = 0;
    for (int r0 = it.c0, t0 = it.c0 / a.group; r0 < it.c1; r0 += step, t0 += tokens) {
        const char* qt = lds + buf * 2 * TILE;
        const char* gt = qt + TILE;
        const bool more = r0 + step < it.c1;
        if (more) load(r0 + step, t0 + tokens);
#pragma unroll
        for (int rb = 0; rb < 2; ++rb) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < DP / 16; ++i) {
                const vec8<T> fq = row_frag<T, DP>(qt, tl, 32 * rb, i);
                const vec8<T> fg = row_frag<T, DP>(gt, tl, 32 * rb, i);
                s = mfma16(fq, kf[i], i == 0 ? zero : s);
                dp = mfma16(fg, vf[i], i == 0 ? zero : dp);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 x = ld4(&st[buf][0][32 * rb + 8 * g + 4 * half]);
                const float4 y = ld4(&st[buf][1][32 * rb + 8 * g + 4 * half]);
                const float lv[4] = {x.x, x.y, x.z, x.w}, ev[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * g + e;
                    s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.c, -lv[e]));
                    dp[r] = s[r] * (dp[r] - ev[e]);
                    if constexpr (NARROW<T>) dp[r] *= gain;
                }
            }
            if (sc.fit(dp, dk)) gain = __builtin_amdgcn_exp2f(sc.up - PB_UP<T>);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const vec8<T> p = pack8<T>(s, t), ds = pack8<T>(dp, t);
                const vec8<T> p_rest = REST ? rest8<T>(s, p, t) : p;
                const vec8<T> ds_rest = REST ? rest8<T>(dp, ds, t) : ds;
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) {
                    const vec8<T> fg = tr_frag<T, DP>(gt, tl, 32 * rb + 16 * t, b);
                    const vec8<T> fq = tr_frag<T, DP>(qt, tl, 32 * rb + 16 * t, b);
                    if constexpr (REST) {
                        dv[b] = mfma16(fg, p_rest, dv[b]);
                        dk[b] = mfma16(fq, ds_rest, dk[b]);
                    }
                    dv[b] = mfma16(fg, p, dv[b]);
                    dk[b] = mfma16(fq, ds, dk[b]);
                }
            }
        }
        if (more) write(buf ^ 1);
        __syncthreads();
        buf ^= 1;
    }
    if (key >= it.r1) return;
    // a key that the mask leaves out has no gradient, whatever its rows hold
    if (!keep) {
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) dk[b] = dv[b] = f32x16{};
    }
    const float fk = a.scale * sc.back(), fv = __builtin_amdgcn_exp2f(-PB_UP<T>);
    if (it.slot >= 0) {
        float* p = a.part + ((static_cast<int64_t>(it.slot) * a.kv_heads + kvh) * (NW * 32) +
                             key - it.r0) * (2 * a.d);
        store_acc<float, DP>(p, dk, fk, a.d, half);
        store_acc<float, DP>(p + a.d, dv, fv, a.d, half);
    } else {
        const int64_t at = ((it.k_begin + static_cast<int64_t>(key)) * a.kv_heads + kvh) * a.d;
        store_acc<T, DP>(static_cast<T*>(a.dk) + at, dk, fk, a.d, half);
        store_acc<T, DP>(static_cast<T*>(a.dv) + at, dv, fv, a.d, half);
    }
}

template <typename T, int DP, int NW, bool REST>
void launch16_tile(const CrossArgs& a, int pass, hipStream_t st) {
    const dim3 grid(cross_grid(a)), block(NW * 64);
    if (pass == MIGNN_CROSS_FORWARD)
        hipLaunchKernelGGL((cross_fwd16_kernel<T, DP, NW, REST>), grid, block, 0, st, a);
    else if (pass == MIGNN_CROSS_DQ)
        hipLaunchKernelGGL((cross_dq16_kernel<T, DP, NW, REST>), grid, block, 0, st, a);
    else
        hipLaunchKernelGGL((cross_dkv16_kernel<T, DP, NW, REST>), grid, block, 0, st, a);
}

template <typename T, int DP>
void launch16(const CrossArgs& a, int pass, hipStream_t st) {
    if (a.tile == CROSS_ROWS) launch16_tile<T, DP, 1, true>(a, pass, st);
    else if (a.exact) launch16_tile<T, DP, 4, true>(a, pass, st);
    else launch16_tile<T, DP, 4, false>(a, pass, st);
}

template <typename T>
void launch16_d(const CrossArgs& a, int pass, hipStream_t st) {
    if (a.d <= 32) launch16<T, 32>(a, pass, st);
    else if (a.d <= 64) launch16<T, 64>(a, pass, st);
    else if (a.d <= 96) launch16<T, 96>(a, pass, st);
    else launch16<T, 128>(a, pass, st);
}

}  // namespace

int cross_pass16(const CrossArgs& a, int pass, int dtype, hipStream_t st) {
    if (dtype == MIGNN_ROW_BF16) launch16_d<bf16_t>(a, pass, st);
    else launch16_d<f16_t>(a, pass, st);
    return launch_status("cross attention kernel (16 bit)");
}

}  // namespace mignn
