// Parts of the tensor-core kernel of the attention of drafted tokens: masks, products, TMA, the order of the ring, queries and values.
#pragma once

#include <cuda.h>

#include "common.h"
#include "sm100_host.cuh"
#include "sm100_ptx.cuh"
#include "tree.cuh"
#include "turns.cuh"

namespace flat {
namespace tree_tc {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.0f;  // log2 domain: the running maximum is followed only when it grows by more

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Which of the 64 tokens from t0 on drafted token `node` sees, pages aside; own: its first 64 mask bits.
__device__ __forceinline__ uint64_t visible(const TreeParams &p, const TreeSequence &s, int node, int t0, uint64_t own) {
    auto ones = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
    const uint64_t live = ones(s.len - t0);
    uint64_t drafts = 0;
    if (t0 + 64 > s.len) {
        const int j = t0 - s.len;  // drafted token of the first column, if not negative
        if (!p.mask) {
            drafts = p.causal ? ones(node - j + 1) : ~0ull;
        } else if (j <= 0) {
            drafts = own << -j;  // -j < 64
        } else if (p.mask_words <= 2) {
            drafts = j < 64 ? own >> j : 0ull;
        } else {
            const uint32_t *row = p.mask + (int64_t)(s.first + node) * p.mask_words;
            auto word = [&](int i) { return i < p.mask_words ? (uint64_t)row[i] : 0ull; };
            const int w = j >> 5, shift = j & 31;
            drafts = (word(w) | word(w + 1) << 32) >> shift;
            if (shift) drafts |= word(w + 2) << (64 - shift);
        }
    }
    return (live | (drafts & ~live)) & ones(s.tokens - t0);
}

// D[tmem] (+)= A B^T with both operands in shared memory, 128-byte swizzle, rows in groups of 8: A's groups 1024 bytes apart, B's B_SBO.
template <int B_SBO>
__device__ __forceinline__ void mma_scores(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        ".reg .b64 da, db;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "mov.b64 da, {%1, %5};\n"
        "mov.b64 db, {%2, %6};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n"
        "}\n" ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"((1024 >> 4) | (1 << 14) | (2 << 29)),
        "n"((B_SBO >> 4) | (1 << 14) | (2 << 29))
        : "memory");
}
template <int B_SBO>
__device__ __forceinline__ void mma_values(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        ".reg .b64 db;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "mov.b64 db, {%2, %5};\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n"
        "}\n" ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(idesc), "r"(accumulate), "n"((B_SBO >> 4) | (1 << 14) | (2 << 29))
        : "memory");
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap *map, int group, int head, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3, %4}], [%5];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(group), "r"(head), "r"(bar)
        : "memory");
}

// Order of the tiles of a segment of n tiles in the ring: the first `ahead` K tiles, then V tile v and K tile v + ahead for each v.
__device__ __forceinline__ int k_entry(int i, int ahead) { return i < ahead ? i : 2 * i - ahead + 1; }
__device__ __forceinline__ int v_entry(int v, int n, int ahead) { return min(n, ahead) + v + min(v, max(0, n - ahead)); }

// The pool rows of a sequence's boxes, 32 at a time, a box per lane, the next 32 on their way.
struct BoxRows {
    const int32_t *table;
    int page_size, box_rows, tokens, base, lane;
    int page, in_page, page_next, in_page_next;
    __device__ __forceinline__ void fetch(int box, int &to, int &in) {
        const int t = box * box_rows;
        to = -2;  // nothing to read: zeros
        in = 0;
        if (t < tokens) {
            const int logical = t / page_size;
            to = max(table[logical], -1);
            in = t - logical * page_size;
        }
    }
    __device__ __forceinline__ void start(const TreeParams &p, int seq, int seq_tokens, int token0, int rows) {
        lane = threadIdx.x & 31;
        table = p.page_tables + (int64_t)seq * p.max_pages;
        page_size = p.page_size;
        box_rows = rows;
        tokens = seq_tokens;
        base = token0 / rows;
        fetch(base + lane, page, in_page);
        fetch(base + 32 + lane, page_next, in_page_next);
    }
    __device__ __forceinline__ void seek(int box) {  // boxes are asked for in order, a tile's at a time
        if (box - base < 32) return;
        base += 32;
        page = page_next;
        in_page = in_page_next;
        fetch(base + 32 + lane, page_next, in_page_next);
    }
};


// Values of a V tile (64 dims of 8 tokens a KB, GROUP bytes for 8 tokens) from token `from` on: rows from `live` on become zero, and so
// do values that are not finite.  A whole warp; returns whether this lane met such a value.
template <int BOXES, int TOKENS> __device__ __forceinline__ bool clear_values(uint8_t *tile, int from, int live) {
    bool met = false;
#pragma unroll 2
    for (int i = threadIdx.x & 31; i < (TOKENS - from) * BOXES * 8; i += 32) {
        const int row = from + i / (BOXES * 8), e8 = i % (BOXES * 8);
        uint4 *x = reinterpret_cast<uint4 *>(tile + (row >> 3) * (1024 * BOXES) + (e8 >> 3) * 1024 + (row & 7) * 128 + ((e8 & 7) << 4));
        if (row >= live) {
            *x = make_uint4(0, 0, 0, 0);
            continue;
        }
        const uint4 y = *x;
        const uint32_t in[4] = {y.x, y.y, y.z, y.w};
        uint32_t out[4];
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            out[e] = in[e];
            if ((in[e] & 0x7f80u) == 0x7f80u) out[e] &= 0xffff0000u, bad = true;
            if ((in[e] & 0x7f800000u) == 0x7f800000u) out[e] &= 0x0000ffffu, bad = true;
        }
        if (bad) {
            *x = make_uint4(out[0], out[1], out[2], out[3]);
            met = true;
        }
    }
    return met;
}

// 8 dims of a query: turned, and written as the sum of two bf16 numbers at `to` and `to` + LO.  The first one is cut off, not rounded, and
// 2^-30 of the value goes to the second: both then have the value's sign (down to 2^-96), so that their products with a K that is infinite
// are the same infinity and not its difference.  What is left over is below 2^(e - 7) for a value of 2^e to 2^(e + 1), and bf16 numbers
// there are 2^(e - 15) apart: the sum is off by 2^-16 of the value at most.
template <int LO> __device__ __forceinline__ void write_query(uint4 raw, const float2 (&cs)[4], uint8_t *to) {
    const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float a = __uint_as_float(x[e] << 16), b = __uint_as_float(x[e] & 0xffff0000u);
        const float u = a * cs[e].x - b * cs[e].y, v = a * cs[e].y + b * cs[e].x;
        const uint32_t ub = __float_as_uint(u), vb = __float_as_uint(v);
        hi[e] = __byte_perm(ub, vb, 0x7632);  // the upper halves
        lo[e] = pack_bf16(fmaf(u, 0x1p-30f, u - __uint_as_float(ub & 0xffff0000u)), fmaf(v, 0x1p-30f, v - __uint_as_float(vb & 0xffff0000u)));
    }
    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(to + LO) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

// 16 dims from c on of drafted tokens [t0, t1) of a sequence whose V is not finite, added to a row that sees them.
__device__ __forceinline__ void add_not_finite(const TreeParams &p, const TreeSequence &s, int seq, int kv_head, int node, int t0, int t1, int c, float *o) {
    for (int t = max(s.len, t0); t < min(s.tokens, t1); ++t) {
        if (!tree_sees(p, s, node, t - s.len)) continue;
        const int page = p.page_tables[(int64_t)seq * p.max_pages + t / p.page_size];
        if ((unsigned)page >= (unsigned)p.physical_pages) continue;
        const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(p.v) + (((int64_t)page * p.page_size + t % p.page_size) * p.kv_heads + kv_head) * p.head_dim + c;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float y = __bfloat162float(v[e]);
            if (!isfinite(y)) o[e] += y;
        }
    }
}

// 5-D map over (64 dims, token of 8, 64-dim block, group of 8 tokens, head) of a pool, with a box of one head's `box_rows` tokens.
inline int make_pool_map(flat_ctx *ctx, CUtensorMap *map, const void *base, int head_dim, uint64_t rows, int kv_heads, int box_rows) {
    EncodeFn fn = encode_fn();
    if (!fn) return fail(ctx, FLAT_ERR_UNAVAILABLE, "cuTensorMapEncodeTiled is not available from this driver");
    const cuuint64_t row_bytes = (cuuint64_t)kv_heads * head_dim * 2;
    cuuint64_t dims[5] = {64, 8, (cuuint64_t)head_dim / 64, rows / 8, (cuuint64_t)kv_heads};
    cuuint64_t strides[4] = {row_bytes, 128, row_bytes * 8, (cuuint64_t)head_dim * 2};
    cuuint32_t box[5] = {64, 8, (cuuint32_t)head_dim / 64, (cuuint32_t)box_rows / 8, 1};
    cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(ctx, FLAT_ERR_EXECUTION, "cuTensorMapEncodeTiled failed with %d", (int)r);
    return FLAT_OK;
}

}  // namespace tree_tc
}  // namespace flat
