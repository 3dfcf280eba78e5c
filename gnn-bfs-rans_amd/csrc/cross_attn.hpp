// Shared by the cross-attention sources (cross_attn.hip: plan, joins, entry
// points; cross_attn16.hip: 16-bit rows; cross_attn32.hip: fp32 rows;
// cross_decode.hip: few rows).
#pragma once

#include "row_types.hpp"

namespace mignn {

using f32x16 = __attribute__((ext_vector_type(16))) float;

constexpr int CROSS_ROWS = 32;    // rows (or keys) a wave owns: one MFMA tile edge
constexpr int CROSS_FEW = 8;      // rows that cross_few takes
constexpr int CROSS_STAGE = 64;   // rows of an LDS tile of the 16-bit kernels
constexpr float LOG2E = 1.44269504088896340736f;

// One workgroup's share of a pass, per kv head.  "Rows" are the (query, head
// of the group) pairs of one sequence: row r is query r / G, head kvh G + r % G.
// Forward and dq: r0..r1 rows of the tile, c0..c1 keys to go through;
// dk / dv:        r0..r1 keys of the tile, c0..c1 rows to go through.
struct CrossItem {
    int32_t q_begin, k_begin;   // first query / key of the sequence
    int32_t r0, r1, c0, c1;
    int32_t slot;               // partial results' slot, -1: the item is its tile's only one
    int32_t reserved;
};
static_assert(sizeof(CrossItem) == MIGNN_CROSS_ITEM_BYTES, "plan item layout");

// The items of one tile that several workgroups share: slots slot .. slot + parts - 1.
struct CrossJoin {
    int32_t begin;              // first query (forward, dq) or key (dk / dv) of the sequence
    int32_t r0, r1;
    int32_t slot, parts;
    int32_t reserved[3];
};
static_assert(sizeof(CrossJoin) == MIGNN_CROSS_ITEM_BYTES, "plan join layout");

struct CrossArgs {
    const void *q, *k, *v;
    const uint8_t* mask;
    const void* dout;
    const float* out32;          // fp32 outputs of the forward (training)
    void *out, *dk, *dv;         // out: the forward's output or dq
    float *o32, *lse, *delta;
    float* part;                 // partial results
    const CrossItem* items;
    const CrossJoin* joins;
    int64_t ldq, ldqh, ldk, ldkh, ldv, ldvh, lddo, lddoh;
    int32_t n_items, n_whole, n_joins, heads, kv_heads, group, d;
    int32_t tile, rows;          // of the pass: rows (keys) of a tile, of the longest sequence
    int32_t exact;               // 16-bit rows: the roundings' remainders are carried
    float scale, c;              // c = scale log2(e)
};

// A uniform value that the compiler cannot see to be one
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint64_t uniform(const void* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    return static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(v)))) |
           static_cast<uint64_t>(static_cast<uint32_t>(uniform(static_cast<int>(v >> 32)))) << 32;
}
__device__ __forceinline__ CrossItem load_item(const CrossArgs& a, int item) {
    CrossItem it = a.items[item];
    it.q_begin = uniform(it.q_begin), it.k_begin = uniform(it.k_begin);
    it.r0 = uniform(it.r0), it.r1 = uniform(it.r1);
    it.c0 = uniform(it.c0), it.c1 = uniform(it.c1);
    it.slot = uniform(it.slot);
    return it;
}

// 16 bytes at base + voffset; a lane whose bytes do not end by num_records
// reads zeros and asks for nothing
__device__ f32x4 raw_buffer_load_f32x4(i32x4 rsrc, int voffset, int soffset, int aux) __asm(
    "llvm.amdgcn.raw.buffer.load.v4f32");
constexpr int NO_LOAD = INT32_MIN;   // a voffset past every num_records

// Block -> (item, kv head): the whole tiles' items first, then the split ones'.
// Consecutive blocks go to the 8 XCDs in turn; each XCD gets one run of the
// (head-major) work, so that the tiles that read one head's keys and values
// share an L2.
__device__ __forceinline__ bool cross_work(const CrossArgs& a, int& item, int& kvh) {
    int n = a.n_whole, first = 0;
    uint32_t b = blockIdx.x;
    const uint32_t whole = (static_cast<uint32_t>(n) * a.kv_heads + 7u) / 8u * 8u;
    if (b >= whole) b -= whole, first = n, n = a.n_items - n;
    const uint32_t total = static_cast<uint32_t>(n) * a.kv_heads, per = (total + 7u) / 8u;
    const uint32_t w = (b & 7u) * per + (b >> 3);
    if ((b >> 3) >= per || w >= total) return false;
    kvh = w / n;
    item = first + w - static_cast<uint32_t>(kvh) * n;
    return true;
}
inline unsigned cross_grid(const CrossArgs& a) {
    auto up8 = [](int64_t n) { return (n + 7) / 8 * 8; };
    return static_cast<unsigned>(up8(static_cast<int64_t>(a.n_whole) * a.kv_heads) +
                                 up8(static_cast<int64_t>(a.n_items - a.n_whole) * a.kv_heads));
}

// Position in the sequence of an accumulator's element: MFMA 32x32 results
// hold D[8 (r / 4) + 4 (lane / 32) + r % 4][lane % 32] in register r.
__device__ __forceinline__ constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

// the 16-bit rows' kernels of a pass (cross_attn16.hip)
int cross_pass16(const CrossArgs& a, int pass, int dtype, hipStream_t st);
// the fp32 rows' (cross_attn32.hip)
int cross_pass32(const CrossArgs& a, int pass, hipStream_t st);
// the forward of up to CROSS_FEW rows a sequence (cross_decode.hip)
int cross_few(const CrossArgs& a, int dtype, hipStream_t st);

}  // namespace mignn
