// Cross attention of query rows to the states of another mesh
// (mignn_cross_attn_forward, mignn_cross_attn_backward): the work plan and
// the joins of split work.
//
//   s_ij = scale <q_i, k_j> over the keys j of the row's sequence that the mask keeps
//   P_ij = 2^(c <q_i, k_j> - lse_i),  c = scale log2 e,  lse_i = log2 sum_j 2^(c <q_i, k_j>)
//   o_i  = sum_j P_ij v_j
//   delta_i = <do_i, o_i>;  dS_ij = P_ij (<do_i, v_j> - delta_i)
//   dq_i = scale sum_j dS_ij k_j;  dk_j = scale sum_i dS_ij q_i;  dv_j = sum_i P_ij do_i
//
// (scores and P are made again in each of the two gradient kernels, seven
// products where four are new: dq's own kernel needs no atomics)
//
// One pass over the keys with the running maximum and sum of the softmax;
// scores and P stay in registers: S^T = K Q^T puts a query in a lane's column,
// so the maximum and the sum are in-lane but for one exchange between the
// wave's halves, and the result registers of S^T are, as they stand, the B
// operand of O^T = V^T P^T (the product over keys takes them in the order in
// which the accumulator holds them).  dq runs like the forward; dk and dv
// swap the roles (a wave owns 32 keys, rows go by), so nothing is added
// atomically and results do not depend on the order of workgroups.  The query
// heads that share a kv head are rows of one tile: their keys are read once,
// and dk, dv sum over them in place.
#include "cross_attn.hpp"

#include <algorithm>
#include <cstdlib>

namespace mignn {
namespace {

// partial results: [slot][kv head][rows of the tile][d + 2] (forward: o
// unnormalised, maximum, sum; dq: dq; dk / dv: dk and dv, 2 d)
__device__ __forceinline__ float* part_row(const CrossArgs& a, int slot, int kvh, int r, int rows,
                                           int width) {
    return a.part + ((static_cast<int64_t>(slot) * a.kv_heads + kvh) * rows + r) * width;
}

// Joins the parts of split rows onto their largest maximum.  Few parts: 4
// columns of a row a thread.
template <typename T>
__global__ __launch_bounds__(256) void cross_join_fwd_kernel(CrossArgs a) {
    const CrossJoin jn = a.joins[blockIdx.x];
    const int kvh = blockIdx.y, i = blockIdx.z * 256 + threadIdx.x, d4 = a.d / 4;
    const int r = i / d4, c = (i - r * d4) * 4;
    if (r >= jn.r1 - jn.r0) return;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * a.tile * (a.d + 2);   // part to part
    const float* src = part_row(a, jn.slot, kvh, r, a.tile, a.d + 2);
    float m = -INFINITY;
    for (int p = 0; p < jn.parts; ++p) m = fmaxf(m, src[p * step + a.d]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < jn.parts; ++p) {
        float x[4];
        load_row(src + p * step + c, x);
        const float f = __builtin_amdgcn_exp2f(src[p * step + a.d] - base);
        l = fmaf(src[p * step + a.d + 1], f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    const int row = jn.r0 + r, t = row / a.group;
    const int64_t at = (jn.begin + static_cast<int64_t>(t)) * a.heads + kvh * a.group + (row - t * a.group);
    store_row(static_cast<T*>(a.out) + at * a.d + c, o);
    if (a.o32) store_row(a.o32 + at * a.d + c, o);
    if (a.lse && c == 0) a.lse[at] = l == 0.f ? INFINITY : base + log2f(l);
}

// Many parts of few rows: a row a workgroup, 4 columns of a part a thread, so
// that most parts are in flight at once.
template <typename T>
__global__ __launch_bounds__(256) void cross_join_few_kernel(CrossArgs a) {
    __shared__ float ms[4], ls[4], os[4][128];
    const CrossJoin jn = a.joins[blockIdx.x];
    const int kvh = blockIdx.y, r = blockIdx.z, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (r >= jn.r1 - jn.r0) return;
    const int d4 = a.d / 4;
    int lp = 2;   // lanes of a part
    while (lp < d4) lp <<= 1;
    const int groups = 256 / lp, g = threadIdx.x / lp, c = (threadIdx.x & (lp - 1)) * 4;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * a.tile * (a.d + 2);
    const float* src = part_row(a, jn.slot, kvh, r, a.tile, a.d + 2);
    float m = -INFINITY;
#pragma unroll 4
    for (int p = g; p < jn.parts; p += groups) m = fmaxf(m, src[p * step + a.d]);
    for (int b = lp; b < 64; b <<= 1) m = fmaxf(m, __shfl_xor(m, b));
    if (lane == 0) ms[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(ms[0], ms[1]), fmaxf(ms[2], ms[3]));
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = g; p < jn.parts; p += groups) {
        const float* part = src + p * step;
        float x[4] = {0.f, 0.f, 0.f, 0.f};
        if (c < a.d) load_row(part + c, x);
        const float f = __builtin_amdgcn_exp2f(part[a.d] - base);
        l = fmaf(part[a.d + 1], f, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
    }
    for (int b = lp; b < 64; b <<= 1) {
        l += __shfl_xor(l, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], b);
    }
    if (lane < lp) {
#pragma unroll
        for (int e = 0; e < 4; ++e) os[wave][c + e] = o[e];
        if (lane == 0) ls[wave] = l;
    }
    __syncthreads();
    if (threadIdx.x >= lp || c >= a.d) return;
    l = ls[0] + ls[1] + ls[2] + ls[3];
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (os[0][c + e] + os[1][c + e] + os[2][c + e] + os[3][c + e]) * inv;
    const int row = jn.r0 + r, t = row / a.group;
    const int64_t at = (jn.begin + static_cast<int64_t>(t)) * a.heads + kvh * a.group + (row - t * a.group);
    store_row(static_cast<T*>(a.out) + at * a.d + c, o);
    if (a.o32) store_row(a.o32 + at * a.d + c, o);
    if (a.lse && c == 0) a.lse[at] = l == 0.f ? INFINITY : base + log2f(l);
}

// Sums the parts of split gradients in slot order, 4 columns of a row a thread:
// dq, or dk and dv side by side.
template <typename T>
__global__ __launch_bounds__(256) void cross_join_grad_kernel(CrossArgs a, bool dkv) {
    const CrossJoin jn = a.joins[blockIdx.x];
    const int width = dkv ? 2 * a.d : a.d, w4 = width / 4;
    const int kvh = blockIdx.y, i = blockIdx.z * 256 + threadIdx.x;
    const int r = i / w4, c = (i - r * w4) * 4;
    if (r >= jn.r1 - jn.r0) return;
    const int64_t step = static_cast<int64_t>(a.kv_heads) * a.tile * width;
    const float* src = part_row(a, jn.slot, kvh, r, a.tile, width) + c;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int p = 0; p < jn.parts; ++p) {
        float x[4];
        load_row(src + p * step, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
    const int row = jn.r0 + r;
    if (dkv) {
        const int64_t at = ((jn.begin + static_cast<int64_t>(row)) * a.kv_heads + kvh) * a.d;
        store_row(c < a.d ? static_cast<T*>(a.dk) + at + c : static_cast<T*>(a.dv) + at + c - a.d, v);
    } else {
        const int t = row / a.group;
        const int64_t at = (jn.begin + static_cast<int64_t>(t)) * a.heads + kvh * a.group + (row - t * a.group);
        store_row(static_cast<T*>(a.out) + at * a.d + c, v);
    }
}

// ---------------------------------------------------------------------------
// Plan

// Tiles of the "r" side (rows or keys) times chunks of the "c" side.
struct PassShape {
    int64_t tile;     // rows of a tile
    bool exact;       // carries the remainders of P's and dS's rounding (16-bit rows; in tiles of 32 always)
    int64_t longest;  // of the r side
    int64_t slots;    // workgroups that chunks are made for
    int64_t least;    // shortest chunk
    int64_t rest;     // the same for what whole tiles leave over
    double start, join, part;   // a workgroup's start, a join and each of its parts, in rows of the c side
    int64_t unit;     // chunks are a multiple of it
};
struct PassPlan {
    int64_t items = 0, whole = 0, joins = 0, slots = 0;
};
struct Sequence {
    int64_t rn, cn, qb, kb;   // r and c side, first query and key
};

int64_t up(int64_t n, int64_t unit) { return (n + unit - 1) / unit * unit; }

// Tile: 8 rows where no sequence has more (forward: cross_few), 32 (one wave)
// where none has more than 32, else 128, four waves that share the staging of
// the other side.  (32 for longer sequences saves padding but not time: LDS
// holds few such workgroups; keys of three sequences of 78, 134 and 167: dk /
// dv 108 us in tiles of 32, 61 in tiles of 128.)
//
// The remainders of P's and dS's rounding to 16 bits are carried where that
// costs little or where their loss shows most.  Errors against 64 bits, in units
// of what the output's own rounding leaves (bf16 1.7e-3, fp16 2.1e-4): 1.0 with
// the remainders, 1.4 without.  They are half the matrix work again: 49181 x
// 4096 x 4 heads over 2 of 64, trained, would take 1425 for 1013 us, 2 x 16384^2 x 8
// x 128 3197 for 2313.  They are carried
//   for few results (a kv head's output is below 32 KB): such a launch seldom is
//     bound by the matrix unit (127 rows of 128, 262144 keys, 4 heads: forward 162
//     -> 187 us, dq 202 -> 197, dk / dv 243 -> 283);
//   in gradients that go through one LDS tile: bound by memory, and a few large
//     weights' errors are most of a result's (dv of 35 sequences of one row, 2606
//     keys, 2 heads of 24, fp16: 1.54 without), while a row's dS sum to 0, which
//     takes the keys' common part out of dq but not out of the roundings (2 x 5742
//     x up to 5 keys, 8 heads over 2 of 24, bf16: 1.65).  36675 rows or keys x 64 x 4
//     heads over 2 of 64: dq 25.0 -> 25.3 us, dk / dv 21.3 -> 24.6; 4 of 128: 58 -> 54,
//     63 -> 67.  (The forward stays below 1.42 without.);
//   in dq of heads to 16 columns, where the common part is much of a key at any
//     length (16 columns 1.50 -> 1.03; without them 24 columns 1.48, 32 1.46, 64
//     1.43).  Up to 8 of 12077 x 13392 x 2 heads of 16, trained, 916 -> 1025 us.
//
// Few results take tiles of 32 as long as that is the faster: those spread over
// more CUs, but each stages its own copy of the other side.  bf16, 4 heads,
// rows x other side x columns, us in tiles of 32 / 128:
//   forward  128 x 4096 x 64  14 / 18   40 x 32768 x 32  22 / 40    250 x 32768 x 64  51 / 51
//            40 x 262144 x 64 97 / 135  127 x 4096 x 128 20 / 24    128 x 262144 x 64 171 / 134
//            40 x 32768 x 128 60 / 52   127 x 32768 x 128 83 / 56   250 x 262144 x 64 288 / 176
//   dq       128 x 4096 x 64  13 / 15   40 x 32768 x 32  30 / 25    8 of 40 x 32768 x 32 52 / 60
//            250 x 4096 x 64  18 / 19   128 x 262144 x 32 147 / 74  127 x 32768 x 128 93 / 44
//   dk / dv  128 x 4096 x 64  18 / 19   40 x 32768 x 32  34 / 28    8 of 40 x 32768 x 32 57 / 86
//            250 x 4096 x 64  27 / 16   128 x 262144 x 32 161 / 101 127 x 32768 x 128 133 / 50
PassShape pass_shape(const Sequence* seq, int64_t batch, int pass, int d, int dtype, int group) {
    const bool dkv = pass == MIGNN_CROSS_DKV;
    PassShape s{128, false, 0, 512, 128, 128, 64.0, 0.0, 0.0, dkv ? CROSS_STAGE / group * group : CROSS_STAGE};
    int64_t results = 0;   // of one kv head
    double work = 0.0;     // products of one kv head and form
    int64_t other = 0;     // longest of the c side
    for (int64_t b = 0; b < batch; ++b) {
        s.longest = seq[b].rn > s.longest ? seq[b].rn : s.longest;
        other = seq[b].cn > other ? seq[b].cn : other;
        results += seq[b].rn * d;
        work += static_cast<double>(seq[b].rn) * static_cast<double>(seq[b].cn) * d;
    }
    const double limit = pass == MIGNN_CROSS_FORWARD ? (d <= 64 ? 0x1p30 : 0x1p27) : d <= 32 ? 0x1p29 : 0x1p25;
    const bool few = dtype != MIGNN_ROW_F32 && results < 16384;
    if (pass == MIGNN_CROSS_FORWARD && s.longest <= CROSS_FEW) s.tile = CROSS_FEW;
    else if (s.longest <= CROSS_ROWS || (few && work <= limit)) s.tile = CROSS_ROWS;
    const bool lossy = pass != MIGNN_CROSS_FORWARD && (other <= CROSS_STAGE || (!dkv && d <= 16));
    s.exact = s.tile == 128 && dtype != MIGNN_ROW_F32 && (few || lossy);
    // Workgroups that chunks are made for.  Four waves: two a CU (a forward or
    // dq of narrow heads holds three; made for 768, 12225^2 fp32 took 475 -> 489
    // us), one where the heads are wide and much is held in fp32.  One wave:
    // eight a CU, more than LDS holds of wide heads (16 bits: five of 64
    // columns, two of 128; fp32 one of 128), and joins are not priced there.
    // (4096: the same; 1024: the same, or less: 16 of 20 rows x 4096 keys of 64,
    // bf16, forward 27 -> 23 us.)
    const bool wide = dtype == MIGNN_ROW_F32 ? d > 64 || (dkv && d > 32) : dkv && d > 96;
    if (s.tile != 128) {
        s.slots = 2048;
        return s;
    }
    if (wide) s.slots = 256;
    // 4 us to start a workgroup (its rows and first tile), 5 for a join's
    // launch, 0.15 for each part it goes through, against the time of a row of
    // the c side.  (A least chunk of 256 and no price on parts: 20
    // sequences of up to 419 rows, 529 keys, 2 heads of 128, fp32 57 us, now 36; a least
    // of 64 without the prices, 2 of 27 rows, 17025 keys, fp32: 45 -> 56.)
    const double ns = (d + 31) / 32 * 32 * (dtype == MIGNN_ROW_F32 ? 0.55 : 0.12) *
                      (pass == MIGNN_CROSS_FORWARD ? 1.0 : pass == MIGNN_CROSS_DQ ? 1.5 : 2.0);
    s.start = 4000.0 / ns, s.join = 5000.0 / ns, s.part = 150.0 / ns;
    if (dtype == MIGNN_ROW_F32) s.least = 64;
    s.rest = 256;   // (128: 49181 rows x 4096 keys bf16, trained, 1038 -> 1046 us)
    return s;
}

// The chunk length that ends first when the tiles are fewer than the slots:
// rounds of `slots` workgroups, each a chunk and the cost of starting one
int64_t pick_chunk(const PassShape& s, const Sequence* seq, int64_t batch, int kv_heads) {
    int64_t longest = 0;
    for (int64_t b = 0; b < batch; ++b) longest = seq[b].cn > longest ? seq[b].cn : longest;
    int64_t best = up(longest > 0 ? longest : 1, s.unit);
    double best_cost = -1.0;
    int64_t last = 0;
    for (int64_t parts = 1; parts <= 256; ++parts) {
        const int64_t len = up((longest + parts - 1) / parts, s.unit);
        if (parts > 1 && len < s.least) break;
        if (len == last) continue;
        last = len;
        double items = 0.0;
        for (int64_t b = 0; b < batch; ++b)
            if (seq[b].cn > 0)
                items += static_cast<double>((seq[b].rn + s.tile - 1) / s.tile) *
                         static_cast<double>((seq[b].cn + len - 1) / len);
        const int64_t rounds = (static_cast<int64_t>(items) * kv_heads + s.slots - 1) / s.slots;
        const double cost = static_cast<double>(rounds) * (static_cast<double>(len) + s.start) +
                            (parts > 1 ? s.join + s.part * static_cast<double>(parts) : 0.0);
        if (best_cost < 0.0 || cost < best_cost) best = len, best_cost = cost;
    }
    return best;
}

// Whole tiles as long as they fill the slots round by round; what is left over
// (all of it, when the tiles are fewer than the slots) is split along the c
// side so that it fills the last round.
PassPlan plan_pass(const PassShape& s, const Sequence* seq, int64_t batch, int kv_heads, bool dkv,
                   CrossItem* items, CrossJoin* joins) {
    int64_t tiles = 0;
    for (int64_t b = 0; b < batch; ++b) tiles += (seq[b].rn + s.tile - 1) / s.tile;
    const int64_t whole = tiles * kv_heads / s.slots * s.slots / kv_heads;
    const int64_t rest = (tiles - whole) * kv_heads;
    const int64_t chunk = whole == 0 ? pick_chunk(s, seq, batch, kv_heads) : 0;
    const int64_t split = rest > 0 ? s.slots / rest : 1;
    PassPlan p;
    int64_t t = 0;
    for (int64_t b = 0; b < batch; ++b) {
        const int64_t rn = seq[b].rn, cn = seq[b].cn;
        for (int64_t r0 = 0; r0 < rn; r0 += s.tile, ++t) {
            const int64_t r1 = r0 + s.tile < rn ? r0 + s.tile : rn;
            int64_t parts = 1;
            if (t >= whole && cn > 0) {
                parts = whole == 0 ? (cn + chunk - 1) / chunk : split;
                const int64_t least = whole == 0 ? s.least : s.rest;
                if (parts > cn / least) parts = cn / least;
                if (parts < 1) parts = 1;
            }
            // equal parts, each a multiple of the unit but the last
            const int64_t len = cn == 0 ? 0 : up((cn + parts - 1) / parts, s.unit);
            if (len > 0) parts = (cn + len - 1) / len;
            if (joins && parts > 1)
                joins[p.joins] = {static_cast<int32_t>(dkv ? seq[b].kb : seq[b].qb), static_cast<int32_t>(r0),
                                  static_cast<int32_t>(r1), static_cast<int32_t>(p.slots),
                                  static_cast<int32_t>(parts), {0, 0, 0}};
            for (int64_t k = 0; k < parts; ++k) {
                if (items) {
                    const int64_t c0 = k * len, c1 = c0 + len < cn ? c0 + len : cn;
                    items[p.items] = {static_cast<int32_t>(seq[b].qb), static_cast<int32_t>(seq[b].kb),
                                      static_cast<int32_t>(r0), static_cast<int32_t>(r1),
                                      static_cast<int32_t>(c0), static_cast<int32_t>(c1),
                                      parts > 1 ? static_cast<int32_t>(p.slots + k) : -1, 0};
                }
                ++p.items;
            }
            if (t < whole) ++p.whole;
            if (parts > 1) {
                ++p.joins;
                p.slots += parts;
            }
        }
    }
    return p;
}

int64_t part_width(int pass, int d) {
    return pass == MIGNN_CROSS_FORWARD ? d + 2 : pass == MIGNN_CROSS_DQ ? d : 2 * d;
}

template <typename T>
void launch_join(const CrossArgs& a, int pass, hipStream_t st) {
    const unsigned rows = a.rows < a.tile ? a.rows : a.tile;
    auto grid = [&](unsigned width) { return dim3(a.n_joins, a.kv_heads, (rows * (width / 4) + 255) / 256); };
    const bool dkv = pass == MIGNN_CROSS_DKV;
    if (pass != MIGNN_CROSS_FORWARD)
        hipLaunchKernelGGL(cross_join_grad_kernel<T>, grid(dkv ? 2 * a.d : a.d), dim3(256), 0, st, a, dkv);
    else if (a.tile == 128)
        hipLaunchKernelGGL(cross_join_fwd_kernel<T>, grid(a.d), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL(cross_join_few_kernel<T>, dim3(a.n_joins, a.kv_heads, rows), dim3(256), 0, st, a);
}

int run_pass(CrossArgs a, const mignn_cross_pass& ps, int pass, int dtype, hipStream_t st) {
    a.items = static_cast<const CrossItem*>(ps.items);
    a.joins = static_cast<const CrossJoin*>(ps.joins);
    a.n_items = ps.n_items, a.n_joins = ps.n_joins, a.n_whole = ps.n_whole, a.rows = ps.rows;
    a.tile = ps.tile & ~MIGNN_CROSS_EXACT, a.exact = (ps.tile & MIGNN_CROSS_EXACT) != 0;
    if (a.n_items > 0) {
        int rc;
        if (a.tile == CROSS_FEW) rc = cross_few(a, dtype, st);
        else if (dtype == MIGNN_ROW_F32) rc = cross_pass32(a, pass, st);
        else rc = cross_pass16(a, pass, dtype, st);
        if (rc) return rc;
    }
    if (a.n_joins == 0) return MIGNN_OK;
    switch (dtype) {
        case MIGNN_ROW_F32: launch_join<float>(a, pass, st); break;
        case MIGNN_ROW_BF16: launch_join<bf16_t>(a, pass, st); break;
        default: launch_join<f16_t>(a, pass, st); break;
    }
    return launch_status("cross attention join");
}

// dims of a plan's pass (mignn_cross_plan): items, joins, slots, scratch bytes
int check_dims(const char* who, int heads, int kv_heads, int d, int dtype) {
    MIGNN_REQUIRE(row_type_ok(dtype), "%s: unknown row type %d", who, dtype);
    MIGNN_REQUIRE(kv_heads > 0 && heads > 0 && heads % kv_heads == 0 && heads <= 65535,
                  "%s: %d query heads over %d key heads", who, heads, kv_heads);
    MIGNN_REQUIRE(heads / kv_heads <= MIGNN_CROSS_MAX_GROUP, "%s: more than %d query heads a key head", who,
                  MIGNN_CROSS_MAX_GROUP);
    MIGNN_REQUIRE(d > 0 && d % 8 == 0 && d <= MIGNN_CROSS_MAX_D, "%s: head width %d (a multiple of 8, <= %d)",
                  who, d, MIGNN_CROSS_MAX_D);
    return MIGNN_OK;
}

int check_rows(const char* who, const char* what, const void* p, int64_t ldt, int64_t ldh,
               int dtype) {
    const int64_t es = row_type_size(dtype);
    MIGNN_REQUIRE(p && aligned16(p) && ldt >= 0 && ldh >= 0 && ldt * es % 16 == 0 &&
                      ldh * es % 16 == 0,
                  "%s: %s needs a 16-byte aligned pointer and strides", who, what);
    // the staging of 64 rows addresses them by 32-bit offsets
    MIGNN_REQUIRE(ldt <= MIGNN_CROSS_MAX_STRIDE && ldh <= MIGNN_CROSS_MAX_STRIDE,
                  "%s: %s has strides above %d elements", who, what, MIGNN_CROSS_MAX_STRIDE);
    return MIGNN_OK;
}

}  // namespace
}  // namespace mignn

using namespace mignn;

extern "C" int mignn_cross_plan(const int64_t* q_lens, const int64_t* k_lens, int64_t batch,
                                int heads, int kv_heads, int d, int dtype, int pass, void* items,
                                void* joins, int64_t* info) {
    if (int rc = check_dims("cross_plan", heads, kv_heads, d, dtype)) return rc;
    MIGNN_REQUIRE(pass >= MIGNN_CROSS_FORWARD && pass <= MIGNN_CROSS_DKV, "cross_plan: unknown pass %d",
                  pass);
    MIGNN_REQUIRE(batch >= 0 && (batch == 0 || (q_lens && k_lens)) && info,
                  "cross_plan: null pointer or negative batch");
    const int64_t group = heads / kv_heads;
    int64_t queries = 0, keys = 0;
    for (int64_t b = 0; b < batch; ++b) {
        MIGNN_REQUIRE(q_lens[b] >= 0 && k_lens[b] >= 0, "cross_plan: negative length in sequence %lld",
                      static_cast<long long>(b));
        MIGNN_REQUIRE(q_lens[b] <= INT32_MAX / group - 1024 && k_lens[b] <= INT32_MAX - 1024,
                      "cross_plan: sequence %lld too long", static_cast<long long>(b));
        queries += q_lens[b];
        keys += k_lens[b];
        MIGNN_REQUIRE(queries <= INT32_MAX && keys <= INT32_MAX, "cross_plan: more than 2^31 - 1 rows");
    }
    Sequence* seq = static_cast<Sequence*>(malloc(sizeof(Sequence) * (batch > 0 ? batch : 1)));
    MIGNN_REQUIRE(seq, "cross_plan: out of host memory");
    const bool dkv = pass == MIGNN_CROSS_DKV;
    queries = keys = 0;
    for (int64_t b = 0; b < batch; ++b) {
        const int64_t rows = q_lens[b] * group;
        seq[b] = {dkv ? k_lens[b] : rows, dkv ? rows : k_lens[b], queries, keys};
        queries += q_lens[b];
        keys += k_lens[b];
    }
    // the longest first: what starts last should be short
    std::stable_sort(seq, seq + batch, [](const Sequence& x, const Sequence& y) { return x.cn > y.cn; });
    const PassShape sh = pass_shape(seq, batch, pass, d, dtype, static_cast<int>(group));
    const PassPlan p = plan_pass(sh, seq, batch, kv_heads, dkv, static_cast<CrossItem*>(items),
                                 static_cast<CrossJoin*>(joins));
    free(seq);
    // (a launch's threads are counted in 32 bits)
    MIGNN_REQUIRE(p.items * kv_heads <= UINT32_MAX / 256 - 16, "cross_plan: too many tiles (%lld of %d key heads)",
                  static_cast<long long>(p.items), kv_heads);
    info[0] = p.items;
    info[1] = p.joins;
    info[2] = p.slots * kv_heads * sh.tile * part_width(pass, d) * static_cast<int64_t>(sizeof(float));
    info[3] = queries;
    info[4] = keys;
    info[5] = sh.tile | (sh.exact ? MIGNN_CROSS_EXACT : 0);
    info[6] = sh.longest;
    info[7] = p.whole;
    return MIGNN_OK;
}

extern "C" int mignn_cross_attn_forward(const mignn_cross_call* c, void* out, float* out32, float* lse,
                                        void* stream) {
    MIGNN_REQUIRE(c, "cross_attn_forward: null call");
    const char* who = "cross_attn_forward";
    if (int rc = check_dims(who, c->heads, c->kv_heads, c->d, c->dtype)) return rc;
    const mignn_cross_pass& ps = c->pass[MIGNN_CROSS_FORWARD];
    if (ps.n_items == 0) return MIGNN_OK;
    MIGNN_REQUIRE(c->scale > 0.f && c->scale <= 3.0e38f, "%s: scale must be positive", who);
    if (int rc = check_rows(who, "q", c->q, c->ldq, c->ldqh, c->dtype)) return rc;
    if (c->n_keys > 0) {
        if (int rc = check_rows(who, "k", c->k, c->ldk, c->ldkh, c->dtype)) return rc;
        if (int rc = check_rows(who, "v", c->v, c->ldv, c->ldvh, c->dtype)) return rc;
    }
    MIGNN_REQUIRE(out && aligned16(out) && (!out32 || aligned16(out32)), "%s: output pointer", who);
    MIGNN_REQUIRE(ps.items && (ps.n_joins == 0 || ps.joins), "%s: no plan", who);
    if (ps.part_bytes > 0 && (!c->scratch || c->scratch_bytes < static_cast<size_t>(ps.part_bytes))) {
        set_error("%s: scratch %zu bytes, need %lld", who, c->scratch_bytes,
                  static_cast<long long>(ps.part_bytes));
        return MIGNN_ERR_SCRATCH;
    }
    CrossArgs a{};
    a.q = c->q, a.k = c->k, a.v = c->v, a.mask = c->key_mask;
    a.out = out, a.o32 = out32, a.lse = lse, a.part = static_cast<float*>(c->scratch);
    a.ldq = c->ldq, a.ldqh = c->ldqh, a.ldk = c->ldk, a.ldkh = c->ldkh, a.ldv = c->ldv, a.ldvh = c->ldvh;
    a.heads = c->heads, a.kv_heads = c->kv_heads, a.group = c->heads / c->kv_heads, a.d = c->d;
    a.scale = c->scale, a.c = c->scale * LOG2E;
    return run_pass(a, ps, MIGNN_CROSS_FORWARD, c->dtype, as_stream(stream));
}

extern "C" int mignn_cross_attn_backward(const mignn_cross_call* c, const void* dout, int64_t lddo,
                                         int64_t lddoh, const float* out32, const float* lse,
                                         float* delta, void* dq, void* dk, void* dv, void* stream) {
    MIGNN_REQUIRE(c, "cross_attn_backward: null call");
    const char* who = "cross_attn_backward";
    if (int rc = check_dims(who, c->heads, c->kv_heads, c->d, c->dtype)) return rc;
    const mignn_cross_pass &pq = c->pass[MIGNN_CROSS_DQ], &pk = c->pass[MIGNN_CROSS_DKV];
    MIGNN_REQUIRE(c->scale > 0.f && c->scale <= 3.0e38f, "%s: scale must be positive", who);
    if (pq.n_items > 0) {
        if (int rc = check_rows(who, "q", c->q, c->ldq, c->ldqh, c->dtype)) return rc;
        if (int rc = check_rows(who, "dout", dout, lddo, lddoh, c->dtype)) return rc;
        MIGNN_REQUIRE(out32 && aligned16(out32) && lse && delta && dq && aligned16(dq) && pq.items,
                      "%s: null or unaligned pointer", who);
    }
    const bool keys = dk || dv;
    if (c->n_keys > 0) {
        if (int rc = check_rows(who, "k", c->k, c->ldk, c->ldkh, c->dtype)) return rc;
        if (int rc = check_rows(who, "v", c->v, c->ldv, c->ldvh, c->dtype)) return rc;
        MIGNN_REQUIRE(!keys || (dk && dv && aligned16(dk) && aligned16(dv) && pk.items),
                      "%s: null or unaligned pointer", who);
    }
    const int64_t need = pq.part_bytes > pk.part_bytes ? pq.part_bytes : pk.part_bytes;
    if (need > 0 && (!c->scratch || c->scratch_bytes < static_cast<size_t>(need))) {
        set_error("%s: scratch %zu bytes, need %lld", who, c->scratch_bytes, static_cast<long long>(need));
        return MIGNN_ERR_SCRATCH;
    }
    CrossArgs a{};
    a.q = c->q, a.k = c->k, a.v = c->v, a.mask = c->key_mask;
    a.dout = dout, a.out32 = out32, a.lse = const_cast<float*>(lse), a.delta = delta;
    a.out = dq, a.dk = dk, a.dv = dv, a.part = static_cast<float*>(c->scratch);
    a.ldq = c->ldq, a.ldqh = c->ldqh, a.ldk = c->ldk, a.ldkh = c->ldkh, a.ldv = c->ldv, a.ldvh = c->ldvh;
    a.lddo = lddo, a.lddoh = lddoh;
    a.heads = c->heads, a.kv_heads = c->kv_heads, a.group = c->heads / c->kv_heads, a.d = c->d;
    a.scale = c->scale, a.c = c->scale * LOG2E;
    for (int pass : {MIGNN_CROSS_DQ, MIGNN_CROSS_DKV}) {   // dq first: it writes delta
        if (pass == MIGNN_CROSS_DKV && !keys) break;
        if (int rc = run_pass(a, c->pass[pass], pass, c->dtype, as_stream(stream))) return rc;
    }
    return MIGNN_OK;
}
