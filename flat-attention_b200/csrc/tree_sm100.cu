// Attention of drafted tokens over a paged cache on the tensor cores: bf16, head_dim 64 or 128, pages of a multiple of 16 tokens.
//
//   rows of one (sequence, KV head): (drafted token, head of the group), n * G of them, all against the same keys and values
//   S = Q K^T (SS MMA, 128 rows x 64 tokens)  ->  P = exp2(S - m)  ->  O += P V (A operand from TMEM)
//
// The bytes are those of K and V, read once; with many drafted tokens the products cost as much, so both are kept going at once: two
// warps stream tiles of 128 tokens by TMA, a box per page or tile, into a ring whatever item is at hand; one thread issues all
// products; two groups of four warps ("slots") each own a 128-row accumulator and work a softmax row per thread, without shuffles.
//   more than 128 rows: slot w has rows 128 w .. and both slots take every tile, which crosses into the SM once for 256 rows;
//   otherwise:          both slots have the same rows and take the tiles in turn, and their states are joined at the end.  A slot is
//                       a chain (scores, softmax, values), and one alone does not keep up with the memory.
// P lies over the scores it comes from; the products of one thread execute in order, so the next scores of a slot cannot overtake
// the product that reads its P, and a slot that sees its scores knows that its last value product is complete.  Tiles of 64 tokens
// with two score tiles a slot were slower: the queries cross from shared memory for every tile, which at 64 tokens takes the tensor
// core longer than the product (a product of 128 x 64 x 16 every 46 clk, of 128 x 128 x 16 every 64).
//
// Work: the tiles of all (sequence, KV head, 256 rows) items stand in one line, which is cut into equal spans, one per CTA, whatever
// the lengths are.  Every CTA adds the lengths up itself, so nothing is planned on the host.  An item that a span's end cuts is
// joined by a small second kernel from the parts, in order; everything else is written directly.
//
// Roundings: q enters as the sum of two bf16 numbers (the tensor core takes one type, and K is bf16; q alone would cost 2^-9 of the
// scores: 1.7 times the error of the bf16 result, where this way is 1.4 times it), P as bf16, sums and statistics are f32.
// The running maximum is followed only when it grows by more than 2^8, which keeps the accumulator out of the loop; P then
// reaches 2^8, sums stay far inside f32.
//
// Tokens that a row does not see: its score is replaced by -inf.  P = 0 alone would not do for V that is not finite, so another
// warp goes over the V tiles that hold drafted tokens or the end of a sequence before they are used: rows behind the end (whatever
// an earlier owner of the page left) become zero, and so do values of drafted tokens that are not finite; these are then added to
// the rows that see them at the end, where they were met at all.
#include <cuda.h>

#include "common.h"
#include "sm100_host.cuh"
#include "sm100_ptx.cuh"
#include "tree.cuh"
#include "turns.cuh"

namespace flat {
namespace {

using namespace sm100;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kRescaleThreshold = 8.0f;  // log2 domain
constexpr int kTok = 128, kSlotRows = 128, kItemRows = 2 * kSlotRows;
constexpr int kSoftmaxWarps = 8, kKWarp = 8, kVWarp = 9, kMmaWarp = 10;  // ... and one that goes over V tiles
constexpr int kThreads = 384;
constexpr int kValidRing = 16;   // tiles between the producer and the slowest softmax warp: the ring's and four more
constexpr int kPoisonRing = 16;  // segments between the fixing warp and the slowest softmax warp
constexpr int kMergeChunks = 8;  // blocks per item, 32 rows each

// NARROW: no item has more than 128 rows; the ring takes the second slot's queries' place.
// A K or V tile lies in shared memory as [8 tokens][64 dims of D][token of the 8][64 dims]: one TMA box of any number of tokens
// then writes all D dims.
template <int D, bool NARROW> struct Cfg {
    static constexpr int kBoxes = D / 64;
    static constexpr int kQBox = kSlotRows * 128, kQTile = kQBox * kBoxes;  // one of the two summands of a slot's queries
    static constexpr int kGroup = 1024 * kBoxes;                            // 8 tokens
    static constexpr int kKvTile = kTok / 8 * kGroup;
    static constexpr int kQBytes = (NARROW ? 2 : 4) * kQTile;
    static constexpr int kStages = (224 * 1024 - kQBytes) / kKvTile;  // D = 128: 5 and 3, D = 64: 12 and 10
    static constexpr int kSmem = kQBytes + kStages * kKvTile + 1024;
};

struct Record {  // an item that begins in this CTA and ends in a later one
    int seq, kv_head, pair, parts;
};
struct KernelParams {
    TreeParams t;
    CUtensorMap map_k, map_v;
    uint32_t idesc_qk, idesc_pv;
    int box_rows;      // tokens of a TMA box: 16, 32, 64 or 128, a divisor of the page size
    float *part_o;     // [2 per CTA][256 rows][D], not normalised
    float2 *part_ml;   // [2 per CTA][256 rows] maximum (log2 domain) and sum
    Record *records;   // [CTA]
};

// A part of an item that one CTA works on.
struct Segment {
    TreeSequence s;
    int seq, kv_head, pair;  // pair: which 256 rows
    int rows;                // of the pair
    int j0, j1, tiles;       // its tiles, and the item's
    int64_t item_end;        // on the line
};

__device__ __forceinline__ int64_t units_of(const TreeParams &p, const TreeSequence &s) {
    if (s.nodes == 0) return 0;
    const int64_t pairs = ((int64_t)s.nodes * p.group + kItemRows - 1) / kItemRows;
    return pairs * p.kv_heads * max(1, (s.tokens + kTok - 1) / kTok);
}

// A CTA's walk over its span; every role makes it for itself.
struct Walk {
    int64_t at, end, seq_start;
    int seq;
    __device__ __forceinline__ bool next(const TreeParams &p, Segment &g) {
        while (at < end) {
            const TreeSequence s = tree_sequence(p, seq);
            const int64_t units = units_of(p, s);
            if (at >= seq_start + units) {
                seq_start += units;
                ++seq;
                continue;
            }
            const int tiles = max(1, (s.tokens + kTok - 1) / kTok);
            const int64_t x = at - seq_start, item = x / tiles;
            const int pairs = (int)(((int64_t)s.nodes * p.group + kItemRows - 1) / kItemRows);
            g.s = s;
            g.seq = seq;
            g.kv_head = (int)(item / pairs);
            g.pair = (int)(item % pairs);
            g.rows = min(kItemRows, s.nodes * p.group - g.pair * kItemRows);
            g.tiles = tiles;
            g.j0 = (int)(x - item * tiles);
            g.j1 = (int)min((int64_t)tiles, g.j0 + (end - at));
            g.item_end = seq_start + (item + 1) * tiles;
            at += g.j1 - g.j0;
            return true;
        }
        return false;
    }
};

__device__ __forceinline__ void record_timeout(const KernelParams &p, int where) {
    p.t.status->code = FLAT_ERR_DEVICE_WAIT_TIMEOUT;
    p.t.status->where = where;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Whether tile j of the segment's item holds drafted tokens or is its last: its V tile is gone over before it is used.  (Every
// item has such a tile, so the warp that does it is never more than the ring ahead.)
__device__ __forceinline__ bool is_tail(const Segment &g, int j) { return (j + 1) * kTok > g.s.len || j + 1 == g.tiles; }

// Which of the 64 tokens from t0 on drafted token `node` sees; valid: 16-token groups whose page is in the pool (4 bits).
__device__ __forceinline__ uint64_t visible(const TreeParams &p, const TreeSequence &s, int node, int t0, uint32_t valid) {
    auto ones = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
    const uint64_t live = ones(s.len - t0);
    uint64_t drafts = 0;
    if (t0 + 64 > s.len) {
        const int j = t0 - s.len;  // drafted token of the first column, if not negative
        if (!p.mask) {
            drafts = p.causal ? ones(node - j + 1) : ~0ull;
        } else {
            const uint32_t *row = p.mask + (int64_t)(s.first + node) * p.mask_words;
            auto word = [&](int i) { return i < p.mask_words ? (uint64_t)row[i] : 0ull; };
            if (j <= 0) {
                drafts = (word(0) | word(1) << 32) << -j;  // -j < 64
            } else {
                const int w = j >> 5, shift = j & 31;
                drafts = (word(w) | word(w + 1) << 32) >> shift;
                if (shift) drafts |= word(w + 2) << (64 - shift);
            }
        }
    }
    uint64_t on = (live | (drafts & ~live)) & ones(s.tokens - t0);
    if (valid != 0xf)
        for (int i = 0; i < 4; ++i)
            if (!((valid >> i) & 1)) on &= ~(0xffffull << (16 * i));
    return on;
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
    __device__ __forceinline__ void start(const TreeParams &p, const Segment &g, int rows) {
        lane = threadIdx.x & 31;
        table = p.page_tables + (int64_t)g.seq * p.max_pages;
        page_size = p.page_size;
        box_rows = rows;
        tokens = g.s.tokens;
        base = g.j0 * (kTok / rows);
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

template <int D, bool NARROW> __global__ void __launch_bounds__(kThreads, 1) tree_sm100_kernel(const __grid_constant__ KernelParams p) {
    using C = Cfg<D, NARROW>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *q_s = smem;                // [slot][summand]; at the end of a segment, results on their way out
    uint8_t *kv_s = smem + C::kQBytes;  // ring
    __shared__ uint64_t bars[4 * C::kStages + 9];
    __shared__ uint64_t turns_s[D / 2];
    __shared__ uint32_t tmem_slot[1];
    __shared__ int abort_word;
    __shared__ uint32_t valid_s[kValidRing];
    __shared__ int poison_s[kPoisonRing];
    __shared__ int64_t sums_s[kThreads / 32];
    __shared__ int64_t start_s[2];
    volatile int *abort_flag = &abort_word;

    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };                        // tile landed
    auto empty = [&](int s) { return bar0 + 8u * (C::kStages + s); };        // tile used
    auto fixed = [&](int s) { return bar0 + 8u * (2 * C::kStages + s); };    // V tile with drafted tokens gone over
    auto to_fix = [&](int s) { return bar0 + 8u * (3 * C::kStages + s); };   // such a tile has been requested
    auto s_full = [&](int w) { return bar0 + 8u * (4 * C::kStages + w); };       // scores of the slot's tile, and its last value product
    auto p_full = [&](int w) { return bar0 + 8u * (4 * C::kStages + 2 + w); };   // P written
    auto o_final = [&](int w) { return bar0 + 8u * (4 * C::kStages + 4 + w); };  // the slot's last value product of the segment
    const uint32_t q_ready = bar0 + 8u * (4 * C::kStages + 6);    // queries of the segment written
    const uint32_t q_free = bar0 + 8u * (4 * C::kStages + 7);     // a segment's queries and results are not needed any more
    const uint32_t join_full = bar0 + 8u * (4 * C::kStages + 8);  // slot 1's statistics written

    const int warp = warp_index_uniform(), lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_dependency_launch();
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(fixed(s), 1);
            mbar_init(to_fix(s), 1);
        }
        for (int w = 0; w < 2; ++w) {
            mbar_init(s_full(w), 1);
            mbar_init(p_full(w), 4);
            mbar_init(o_final(w), 1);
        }
        mbar_init(q_ready, kSoftmaxWarps);
        mbar_init(q_free, kSoftmaxWarps);
        mbar_init(join_full, 4);
        mbar_fence_init();
        fence_proxy_async();
        tma_prefetch_desc(&p.map_k);
        tma_prefetch_desc(&p.map_v);
    }
    if (threadIdx.x < kPoisonRing) poison_s[threadIdx.x] = 0;
    if (threadIdx.x < D / 2) turns_s[threadIdx.x] = p.t.freq.turns[threadIdx.x];
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(tmem_slot), 512);
        tmem_relinquish();
    }

    // The line's length, and the sequence that this CTA's span starts in.
    int64_t total = 0;
    for (int base = 0; base < p.t.num_seqs; base += kThreads) {
        const int seq = base + threadIdx.x;
        if (seq < p.t.num_seqs) {
            const TreeSequence s = tree_sequence(p.t, seq);
            total += units_of(p.t, s);
            if (s.code && blockIdx.x == 0) tree_report(p.t, s.code, seq);
        }
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    if (lane == 0) sums_s[warp] = total;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    total = 0;
    for (int i = 0; i < kThreads / 32; ++i) total += sums_s[i];
    const int64_t span = max((int64_t)1, (total + gridDim.x - 1) / gridDim.x);
    const int64_t begin = min(total, span * blockIdx.x), end = min(total, begin + span);
    if (begin < end) {
        int64_t before = 0;  // units of the sequences of earlier passes
        for (int base = 0;; base += kThreads) {
            const int seq = base + threadIdx.x;
            const int64_t units = seq < p.t.num_seqs ? units_of(p.t, tree_sequence(p.t, seq)) : 0;
            int64_t upto = units;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t y = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += y;
            }
            __syncthreads();
            if (lane == 31) sums_s[warp] = upto;
            __syncthreads();
            int64_t pass = 0;
            for (int i = 0; i < kThreads / 32; ++i) {
                if (i < warp) upto += sums_s[i];
                pass += sums_s[i];
            }
            upto += before;
            if (begin < upto && begin >= upto - units) {
                start_s[0] = seq;
                start_s[1] = upto - units;
            }
            before += pass;
            if (before > begin) break;
        }
    }
    if (threadIdx.x == 0) p.records[blockIdx.x].parts = 0;
    __syncthreads();
    const uint32_t tmem_base = *tmem_slot;
    auto col_o = [](int w) { return (uint32_t)(w * D); };
    auto col_s = [](int w) { return (uint32_t)(2 * D + w * kTok); };
    Walk walk{begin, end, start_s[1], (int)start_s[0]};
    Segment g;

    if (warp < kSoftmaxWarps) {
        // ================= queries, softmax, results =================
        const int w = warp >> 2, row = threadIdx.x & (kSlotRows - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's quarter of the TMEM lanes
        int count = 0;      // tiles of this slot so far
        int tile_base = 0;  // tiles of this CTA before the segment
        int finals = 0;     // segments in which this slot had tiles
        int joins = 0;
        bool ok = true;
        for (int k = 0; ok && walk.next(p.t, g); ++k) {
            const bool shared = NARROW || g.rows <= kSlotRows;
            const int n = g.j1 - g.j0, r_begin = g.pair * kItemRows;
            {
                // A thread takes 8 dims of up to four heads of a drafted token, whose angles are the same.  The loads of a step are
                // all in flight during the step before; the first ones while other warps finish the segment before.
                const int node_lo = r_begin / p.t.group, node_hi = (r_begin + g.rows - 1) / p.t.group;
                const int quads = (p.t.group + 3) / 4, tasks = (node_hi - node_lo + 1) * quads * (D / 8);
                struct Raw {
                    uint4 q[4];
                    int position;
                } now, next;
                auto request = [&](int i, Raw &x) {
                    const int c = i % (D / 8), nq = i / (D / 8), node = node_lo + nq / quads, h = nq % quads * 4;
                    x.position = p.t.positions[g.s.first + node];
                    const char *from = static_cast<const char *>(p.t.q) +
                                       (((int64_t)(g.s.first + node) * p.t.q_heads + g.kv_head * p.t.group + h) * D + c * 8) * 2;
                    const int r = node * p.t.group - r_begin + h;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (h + e < p.t.group && r + e >= 0 && r + e < g.rows) x.q[e] = *reinterpret_cast<const uint4 *>(from + e * D * 2);
                };
                if ((int)threadIdx.x < tasks) request(threadIdx.x, now);
                if (k > 0 && !mbar_wait_warp(q_free, (k - 1) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 330 + w);
                    ok = false;
                    break;
                }
                for (int i = threadIdx.x; i < tasks; i += kSoftmaxWarps * 32) {
                    if (i + kSoftmaxWarps * 32 < tasks) request(i + kSoftmaxWarps * 32, next);
                    const int c = i % (D / 8), nq = i / (D / 8), node = node_lo + nq / quads, h = nq % quads * 4;
                    float2 cs[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        cs[e] = turn_of_fast(now.position, turns_s[c * 4 + e]);
                        cs[e].x *= p.t.scale * kLog2e;
                        cs[e].y *= p.t.scale * kLog2e;
                    }
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int r = node * p.t.group - r_begin + h + q;
                        if (h + q >= p.t.group || r < 0 || r >= g.rows) continue;
                        const uint32_t x[4] = {now.q[q].x, now.q[q].y, now.q[q].z, now.q[q].w};
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float a = __uint_as_float(x[e] << 16), b = __uint_as_float(x[e] & 0xffff0000u);
                            const float u = a * cs[e].x - b * cs[e].y, v = a * cs[e].y + b * cs[e].x;
                            const __nv_bfloat162 h2 = __floats2bfloat162_rn(u, v);
                            const float2 f = __bfloat1622float2(h2);
                            hi[e] = *reinterpret_cast<const uint32_t *>(&h2);
                            lo[e] = pack_bf16(u - f.x, v - f.y);
                        }
                        const int rr = r & (kSlotRows - 1);
                        uint8_t *to = q_s + (r >> 7) * 2 * C::kQTile + (c >> 3) * C::kQBox + rr * 128 + (((c & 7) ^ (rr & 7)) << 4);
                        *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                        *reinterpret_cast<uint4 *>(to + C::kQTile) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                    }
                    now = next;
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);

            const int r = r_begin + (shared ? 0 : w * kSlotRows) + row;  // of the (sequence, KV head)
            const bool live = r < r_begin + g.rows;
            const int node = live ? r / p.t.group : 0;
            const int warp_rows = g.rows - (shared ? 0 : w * kSlotRows) - (warp & 3) * 32;  // of this warp's 32
            float m = -INFINITY, l = 0.f;
            int mine = 0;  // tiles of this slot in this segment
            for (int i = shared ? w : 0; i < n; i += shared ? 2 : 1, ++mine, ++count) {
                if (!mbar_wait_warp(s_full(w), count & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 300 + w);
                    ok = false;
                    break;
                }
                if (warp_rows > 0) {
                    tc_fence_after();
                    const int t0 = (g.j0 + i) * kTok;
                    const uint32_t valid = valid_s[(tile_base + i) % kValidRing];
                    const bool masked = t0 + kTok > g.s.len || valid != 0xff;
                    uint64_t on0 = ~0ull, on1 = ~0ull;
                    if (masked) {
                        on0 = visible(p.t, g.s, node, t0, valid & 0xf);
                        on1 = visible(p.t, g.s, node, t0 + 64, valid >> 4);
                    }
                    // Scores 0..63 stay in registers from the maximum on, 64..127 are read again: P lies over the first half.
                    uint32_t a[32], b[32];
                    auto request = [&](int c, uint32_t (&x)[32]) { tmem_ld32(tmem_base + lanes + col_s(w) + 32 * c, x); };
                    auto mask = [&](int c, uint32_t (&x)[32]) {
                        if (!masked) return;
                        const uint32_t bits = (uint32_t)((c & 2 ? on1 : on0) >> (32 * (c & 1)));
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((bits >> e) & 1)) x[e] = 0xff800000u;  // -inf
                    };
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    auto maximum = [&](const uint32_t (&x)[32]) {
#pragma unroll
                        for (int e = 0; e < 32; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(x[e]));
                    };
                    request(2, a);
                    request(3, b);
                    tc_wait_ld();
                    mask(2, a);
                    mask(3, b);
                    maximum(a);
                    maximum(b);
                    request(0, a);
                    request(1, b);
                    tc_wait_ld();
                    mask(0, a);
                    mask(1, b);
                    maximum(a);
                    maximum(b);
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    const bool grows = live && top > m + (mine ? kRescaleThreshold : 0.f);
                    if (__any_sync(0xffffffffu, grows)) {
                        const float now = grows ? top : m, f = grows ? ex2(m - now) : 1.f;  // m = -inf gives 0
                        m = now;
                        l *= f;
                        if (mine > 0) {
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                tmem_ld16(tmem_base + lanes + col_o(w) + c, o);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st16(tmem_base + lanes + col_o(w) + c, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.f : m;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};
                    auto weights = [&](int c, uint32_t (&x)[32]) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float pa = ex2(__uint_as_float(x[e]) - base), pb = ex2(__uint_as_float(x[e + 1]) - base);
                            sum[(e >> 1) & 3] += pa + pb;
                            x[e / 2] = pack_bf16(pa, pb);
                        }
                        tmem_st16(tmem_base + lanes + col_s(w) + 16 * c, x);
                    };
                    weights(0, a);
                    request(2, a);
                    weights(1, b);
                    tc_wait_ld();
                    request(3, b);
                    mask(2, a);
                    weights(2, a);
                    tc_wait_ld();
                    mask(3, b);
                    weights(3, b);
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tc_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(w));
            }
            tile_base += n;
            if (!ok) break;
            if (mine > 0) {
                if (!mbar_wait_warp(o_final(w), finals++ & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 320 + w);
                    ok = false;
                    break;
                }
                tc_fence_after();
            }
            // where this warp's rows pass on their way out: over the queries, which no product reads any more (of the shared ones, once
            // both slots are through)
            uint8_t *stage = q_s + (shared ? 0 : w * 2 * C::kQTile) + (warp & 3) * (32 * D * 4);
            // ---- the slots' states, where they share rows, are joined by slot 0, which reads both accumulators
            float keep = 1.f, other = 0.f;  // factors of this slot's accumulator and of slot 1's
            if (shared) {
                float2 *join_ml = reinterpret_cast<float2 *>(stage);
                if (w == 1) {
                    if (mine > 0) join_ml[lane] = make_float2(m, l);
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(join_full);
                } else {
                    if (!mbar_wait_warp(join_full, joins++ & 1, abort_flag)) {
                        if (lane == 0) record_timeout(p, 340);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    if (n > 1) {
                        const float2 ml = join_ml[lane];
                        const float mx = fmaxf(m, ml.x);
                        keep = l == 0.f ? 0.f : ex2(m - mx);  // a slot that has seen nothing counts for nothing; a NaN counts
                        other = ml.y == 0.f ? 0.f : ex2(ml.x - mx);
                        l = (l == 0.f ? 0.f : keep * l) + (ml.y == 0.f ? 0.f : other * ml.y);
                        m = mx;
                        __syncwarp();
                    }
                }
            }
            const bool whole = g.j0 == 0 && g.j1 == g.tiles;
            if (warp_rows > 0 && !(shared && w == 1)) {
                const int64_t part = ((int64_t)blockIdx.x * 2 + (g.j0 == 0 ? 1 : 0)) * kItemRows + (r - r_begin);
                const int64_t out = (int64_t)(g.s.first + node) * p.t.q_heads + g.kv_head * p.t.group + (live ? r % p.t.group : 0);
                const bool nothing = l == 0.f;
                const float inv = whole ? (nothing ? 0.f : 1.0f / l) : 1.f;
                keep *= inv;
                other *= inv;
                const int poison = *reinterpret_cast<volatile int *>(&poison_s[k % kPoisonRing]);
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t raw[16], raw1[16];
                    float o[16];
                    tmem_ld16(tmem_base + lanes + col_o(w) + c, raw);
                    if (shared && n > 1) tmem_ld16(tmem_base + lanes + col_o(1) + c, raw1);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        o[e] = keep == 0.f ? 0.f : __uint_as_float(raw[e]) * keep;
                        if (shared && n > 1 && other != 0.f) o[e] = fmaf(__uint_as_float(raw1[e]), other, o[e]);
                    }
                    if (poison && live) {  // drafted tokens of this segment whose V is not finite, for the rows that see them
                        for (int t = max(g.s.len, g.j0 * kTok); t < min(g.s.tokens, g.j1 * kTok); ++t) {
                            if (!tree_sees(p.t, g.s, node, t - g.s.len)) continue;
                            const int page = p.t.page_tables[(int64_t)g.seq * p.t.max_pages + t / p.t.page_size];
                            if ((unsigned)page >= (unsigned)p.t.physical_pages) continue;
                            const __nv_bfloat16 *v = static_cast<const __nv_bfloat16 *>(p.t.v) +
                                                     (((int64_t)page * p.t.page_size + t % p.t.page_size) * p.t.kv_heads + g.kv_head) * D + c;
#pragma unroll
                            for (int e = 0; e < 16; ++e) {
                                const float y = __bfloat162float(v[e]);
                                if (!isfinite(y)) o[e] += y;
                            }
                        }
                    }
                    // 16-byte chunks of a row, exchanged within groups of eight so that neither side meets a bank twice
                    if (whole) {
                        uint8_t *to = stage + lane * (D * 2);
                        *reinterpret_cast<uint4 *>(to + (((c / 8) ^ (lane & 7)) << 4)) =
                            make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
                        *reinterpret_cast<uint4 *>(to + (((c / 8 + 1) ^ (lane & 7)) << 4)) =
                            make_uint4(pack_bf16(o[8], o[9]), pack_bf16(o[10], o[11]), pack_bf16(o[12], o[13]), pack_bf16(o[14], o[15]));
                    } else {
                        uint8_t *to = stage + lane * (D * 4);
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            *reinterpret_cast<float4 *>(to + (((c / 4 + e) ^ (lane & 7)) << 4)) = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
                if (live) {
                    if (whole) p.t.lse[out] = nothing ? -INFINITY : (m + log2f(l)) * kLn2;
                    else p.part_ml[part] = make_float2(m, l);
                }
                __syncwarp();
                const int rows = min(32, warp_rows);
                if (whole) {
                    constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;  // lanes of a row
                    const int c = lane % kLanes;
#pragma unroll 4
                    for (int i = 0; i < 32; i += kAtOnce) {
                        const int rr = i + lane / kLanes;
                        const int64_t to = __shfl_sync(0xffffffffu, out, rr);
                        if (rr < rows)
                            reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.t.o) + to * D)[c] =
                                *reinterpret_cast<const uint4 *>(stage + rr * (D * 2) + ((c ^ (rr & 7)) << 4));
                    }
                } else {
                    constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;
                    const int c = lane % kLanes;
                    const int64_t first = __shfl_sync(0xffffffffu, part, 0);
#pragma unroll 4
                    for (int i = 0; i < 32; i += kAtOnce) {
                        const int rr = i + lane / kLanes;
                        if (rr < rows)
                            reinterpret_cast<uint4 *>(p.part_o + (first + rr) * D)[c] =
                                *reinterpret_cast<const uint4 *>(stage + rr * (D * 4) + ((c ^ (rr & 7)) << 4));
                    }
                }
            }
            tc_fence_before();  // the next segment's first value product starts the accumulator anew
            if (threadIdx.x == 0 && g.j0 == 0 && !whole) {
                Record &to = p.records[blockIdx.x];
                to.seq = g.seq;
                to.kv_head = g.kv_head;
                to.pair = g.pair;
                to.parts = (int)((g.item_end - 1) / span) - (int)blockIdx.x + 1;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(q_free);
        }
    } else if (warp == kKWarp || warp == kVWarp) {
        // ================= TMA producers: K tiles and V tiles =================
        const bool is_k = warp == kKWarp;
        const CUtensorMap *map = is_k ? &p.map_k : &p.map_v;
        const int boxes = kTok / p.box_rows, groups = p.box_rows / 8, page_groups = p.t.page_size / 8;
        const int no_group = p.t.physical_pages * page_groups;  // behind the pool: zeros
        uint32_t order = 0;  // tiles of the ring before the segment
        int tile_base = 0;
        bool ok = true;
        while (ok && walk.next(p.t, g)) {
            const int n = g.j1 - g.j0, ahead = NARROW || g.rows <= kSlotRows ? 2 : 1;
            BoxRows rows;
            rows.start(p.t, g, p.box_rows);
            for (int i = 0; ok && i < n; ++i) {
                const int first = (g.j0 + i) * boxes;
                rows.seek(first);
                const bool bad = rows.page == -1 || rows.page >= p.t.physical_pages;
                const int group = rows.page < 0 || bad ? no_group : rows.page * page_groups + (rows.in_page >> 3);
                if (is_k) {
                    uint32_t valid = 0xff;
                    const uint32_t all = __ballot_sync(0xffffffffu, bad) >> (first - rows.base);
                    if (all) {
                        for (int e = 0; e < 8; ++e)
                            if ((all >> (e * 16 / p.box_rows)) & 1 && e * 16 / p.box_rows < boxes) valid &= ~(1u << e);
                        if (lane == 0 && valid != 0xff) tree_report(p.t, FLAT_ERR_PAGE_OUT_OF_RANGE, g.seq);
                    }
                    if (lane == 0) valid_s[(tile_base + i) % kValidRing] = valid;
                }
                const uint32_t at = order + (is_k ? k_entry(i, ahead) : v_entry(i, n, ahead));
                const int s = at % C::kStages;
                if (!mbar_wait_warp(empty(s), ((at / C::kStages) & 1) ^ 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 100 + s);
                    ok = false;
                    break;
                }
                __syncwarp();
                const bool leader = elect_one();
                if (leader) mbar_expect_tx(full(s), C::kKvTile);
                const uint32_t dst = smem_u32(kv_s + s * C::kKvTile);
                for (int b = 0; b < boxes; ++b) {
                    const int from = __shfl_sync(0xffffffffu, group, first - rows.base + b);
                    if (leader) tma_load_5d(dst + b * groups * C::kGroup, map, from, g.kv_head, full(s));
                }
                if (!is_k && leader && is_tail(g, g.j0 + i)) mbar_arrive(to_fix(s));
            }
            order += 2 * n;
            tile_base += n;
        }
    } else if (warp == kMmaWarp) {
        // ================= all products =================
        if (elect_one()) {
            const uint32_t q_desc = (uint32_t)make_smem_desc(smem_u32(q_s), 0, 1024);
            const uint32_t k_desc = (uint32_t)make_smem_desc(smem_u32(kv_s), 0, C::kGroup);
            const uint32_t v_desc = (uint32_t)make_smem_desc(smem_u32(kv_s), 1024, C::kGroup);
            constexpr uint32_t kTile16 = C::kKvTile >> 4;
            uint32_t order = 0, fixed_phase = 0;
            int valued[2] = {0, 0};  // tiles per slot
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity, int where) {
                if (ok && !mbar_wait(bar, parity, abort_flag)) {
                    record_timeout(p, where);
                    ok = false;
                }
            };
            auto landed = [&](int entry) {  // waits for a tile of the segment; its stage
                const uint32_t at = order + entry;
                wait(full(at % C::kStages), (at / C::kStages) & 1, 210);
                return (int)(at % C::kStages);
            };
            auto scores = [&](int w, int q_slot, int s) {
                if (!ok) return;
                tc_fence_after();
                const uint32_t q = q_desc + q_slot * (2 * C::kQTile >> 4), kk = k_desc + s * kTile16, d = tmem_base + col_s(w);
#pragma unroll
                for (int h = 0; h < 2; ++h)  // the two summands of q
#pragma unroll
                    for (int e = 0; e < D / 16; ++e)
                        mma_scores<C::kGroup>(d, q + h * (C::kQTile >> 4) + (e >> 2) * (C::kQBox >> 4) + (e & 3) * 2,
                                              kk + (e >> 2) * (1024 >> 4) + (e & 3) * 2, p.idesc_qk, h > 0 || e > 0);
                tc_commit(s_full(w));
            };
            auto values = [&](int w, int s, bool first, bool last) {
                wait(p_full(w), valued[w]++ & 1, 240 + w);
                if (!ok) return;
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < kTok / 16; ++e)
                    mma_values<C::kGroup>(tmem_base + col_o(w), tmem_base + col_s(w) + e * 8, v_desc + s * kTile16 + e * (2 * C::kGroup >> 4), p.idesc_pv,
                                          !first || e > 0);
                if (last) tc_commit(o_final(w));
            };
            auto fixed_tile = [&](int v, int s) {
                if (!is_tail(g, g.j0 + v)) return;
                wait(fixed(s), (fixed_phase >> s) & 1, 230);
                fixed_phase ^= 1u << s;
            };
            for (int k = 0; ok && walk.next(p.t, g); ++k) {
                const int n = g.j1 - g.j0;
                wait(q_ready, k & 1, 200);
                if (NARROW || g.rows <= kSlotRows) {
                    for (int i = 0; i < min(n, 2); ++i) {
                        const int s = landed(k_entry(i, 2));
                        scores(i, 0, s);
                        if (ok) tc_commit(empty(s));
                    }
                    for (int v = 0; ok && v < n; ++v) {
                        const int w = v & 1, s = landed(v_entry(v, n, 2));
                        fixed_tile(v, s);
                        values(w, s, v < 2, v + 2 >= n);
                        if (ok) tc_commit(empty(s));
                        if (v + 2 < n) {
                            const int sk = landed(k_entry(v + 2, 2));
                            scores(w, 0, sk);
                            if (ok) tc_commit(empty(sk));
                        }
                    }
                } else {
                    int sk = landed(0);
                    scores(0, 0, sk);
                    scores(1, 1, sk);
                    if (ok) tc_commit(empty(sk));
                    for (int v = 0; ok && v < n; ++v) {
                        const int s = landed(v_entry(v, n, 1));
                        fixed_tile(v, s);
                        values(0, s, v == 0, v + 1 == n);
                        if (v + 1 < n) {
                            sk = landed(k_entry(v + 1, 1));
                            scores(0, 0, sk);
                        }
                        values(1, s, v == 0, v + 1 == n);
                        if (ok) tc_commit(empty(s));
                        if (v + 1 < n) {
                            scores(1, 1, sk);
                            if (ok) tc_commit(empty(sk));
                        }
                    }
                }
                order += 2 * n;
            }
        }
    } else {
        // ================= V tiles with drafted tokens or the end of a sequence; the next segment's queries into the L2 =================
        uint32_t order = 0, phase = 0;
        bool ok = true;
        Walk coming = walk;
        Segment c;
        bool more = coming.next(p.t, c);  // the first segment itself
        for (int k = 0; ok && walk.next(p.t, g); ++k) {
            const int n = g.j1 - g.j0, ahead = NARROW || g.rows <= kSlotRows ? 2 : 1;
            if (lane == 0) poison_s[k % kPoisonRing] = 0;
            __syncwarp();
            more = more && coming.next(p.t, c);
            if (more) {
                const int r0 = c.pair * kItemRows;
                for (int i = lane; i < c.rows * C::kBoxes; i += 32) {  // 128 bytes each
                    const int r = r0 + i / C::kBoxes;
                    const char *at = static_cast<const char *>(p.t.q) +
                                     ((int64_t)(c.s.first + r / p.t.group) * p.t.q_heads + c.kv_head * p.t.group + r % p.t.group) * (D * 2) + i % C::kBoxes * 128;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                }
            }
            // (to_fix tells that the tile before in this stage is used up, without which its phase could be taken for this one's)
            for (int v = max(0, min(g.s.len / kTok, g.tiles - 1) - g.j0); v < n; ++v) {
                const uint32_t at = order + v_entry(v, n, ahead);
                const int s = at % C::kStages;
                if (!mbar_wait_warp(to_fix(s), (phase >> s) & 1, abort_flag) || !mbar_wait_warp(full(s), (at / C::kStages) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 400);
                    ok = false;
                    break;
                }
                phase ^= 1u << s;
                const int t0 = (g.j0 + v) * kTok, from = max(0, min(g.s.len, g.s.tokens) - t0), live = g.s.tokens - t0;
                uint8_t *tile = kv_s + s * C::kKvTile;
                bool met = false;
#pragma unroll 2
                for (int i = lane; i < (kTok - from) * C::kBoxes * 8; i += 32) {
                    const int row = from + i / (C::kBoxes * 8), e8 = i % (C::kBoxes * 8);
                    uint4 *x = reinterpret_cast<uint4 *>(tile + (row >> 3) * C::kGroup + (e8 >> 3) * 1024 + (row & 7) * 128 + ((e8 & 7) << 4));
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
                if (__any_sync(0xffffffffu, met) && lane == 0) poison_s[k % kPoisonRing] = 1;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(fixed(s));
            }
            order += 2 * n;
        }
    }

    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // let copies in flight land before the CTA exits
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512);
    }
}

// Joins the parts of an item that begins in CTA blockIdx.x and ends in a later one, in CTA order: 32 rows a block, a row a warp.
template <int D> __global__ void __launch_bounds__(256) tree_sm100_merge_kernel(const __grid_constant__ KernelParams p) {
    grid_dependency_wait();
    grid_dependency_launch();
    const Record rec = p.records[blockIdx.x];
    if (rec.parts <= 0) return;
    const TreeSequence s = tree_sequence(p.t, rec.seq);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r_begin = rec.pair * kItemRows;
    const int rows = min(kItemRows, s.nodes * p.t.group - r_begin);
    constexpr int kPer = D / 32;
    for (int r = blockIdx.y * 32 + warp; r < min(rows, (int)blockIdx.y * 32 + 32); r += 8) {
        auto slot = [&](int i) { return (int64_t)((blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kItemRows + r; };
        float mx = -INFINITY;
        for (int i = lane; i < rec.parts; i += 32) mx = fmaxf(mx, p.part_ml[slot(i)].x);
#pragma unroll
        for (int d = 16; d >= 1; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        float sum = 0.f, o[kPer] = {};
#pragma unroll 4
        for (int i = 0; i < rec.parts; ++i) {
            const float2 ml = p.part_ml[slot(i)];
            const float *from = p.part_o + slot(i) * D + lane * kPer;
            float x[kPer];
            if constexpr (kPer == 4) {
                const float4 y = *reinterpret_cast<const float4 *>(from);
                x[0] = y.x, x[1] = y.y, x[2] = y.z, x[3] = y.w;
            } else {
                const float2 y = *reinterpret_cast<const float2 *>(from);
                x[0] = y.x, x[1] = y.y;
            }
            if (ml.y == 0.f) continue;  // a part in which the row has seen nothing; a NaN counts
            const float f = ex2(ml.x - mx);
            sum = fmaf(f, ml.y, sum);
#pragma unroll
            for (int e = 0; e < kPer; ++e) o[e] = fmaf(f, x[e], o[e]);
        }
        const bool nothing = sum == 0.f;
        const float inv = nothing ? 0.f : 1.0f / sum;
        const int row = r_begin + r;
        const int64_t out = (int64_t)(s.first + row / p.t.group) * p.t.q_heads + rec.kv_head * p.t.group + row % p.t.group;
        uint32_t *to = reinterpret_cast<uint32_t *>(static_cast<__nv_bfloat16 *>(p.t.o) + out * D + lane * kPer);
#pragma unroll
        for (int e = 0; e < kPer; e += 2) to[e / 2] = pack_bf16(o[e] * inv, o[e + 1] * inv);
        if (lane == 0) p.t.lse[out] = nothing ? -INFINITY : (mx + log2f(sum)) * kLn2;
    }
}

// 5-D map over (64 dims, token of 8, 64-dim block, group of 8 tokens, head) of a pool, with a box of one head's `box_rows` tokens.
int make_pool_map(flat_ctx *ctx, CUtensorMap *map, const void *base, int head_dim, uint64_t rows, int kv_heads, int box_rows) {
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

template <int D, bool NARROW> int launch(flat_ctx *ctx, const TreeParams &t) {
    using C = Cfg<D, NARROW>;
    KernelParams p{};
    p.t = t;
    p.box_rows = t.page_size % 128 == 0 ? 128 : t.page_size % 64 == 0 ? 64 : t.page_size % 32 == 0 ? 32 : 16;
    const uint64_t rows = (uint64_t)t.physical_pages * t.page_size;
    if (int st = make_pool_map(ctx, &p.map_k, t.k, D, rows, t.kv_heads, p.box_rows)) return st;
    if (int st = make_pool_map(ctx, &p.map_v, t.v, D, rows, t.kv_heads, p.box_rows)) return st;
    p.idesc_qk = make_idesc(kFmtBF16, kFmtBF16, 0, 0, kSlotRows, kTok);
    p.idesc_pv = make_idesc(kFmtBF16, kFmtBF16, 0, 1, kSlotRows, D);
    const int grid = ctx->sm_count;
    char *at = static_cast<char *>(ctx->paged_scratch) + kPagedPlanBytes;
    const uint64_t rows_held = (uint64_t)grid * 2 * kItemRows;
    const uint64_t o_bytes = rows_held * D * sizeof(float), ml_bytes = rows_held * sizeof(float2);
    if (o_bytes + ml_bytes + grid * sizeof(Record) > kPagedScratchBytes - kPagedPlanBytes)
        return fail(ctx, FLAT_ERR_EXECUTION, "the scratch does not hold the parts of %d CTAs", grid);
    p.part_o = reinterpret_cast<float *>(at);
    p.part_ml = reinterpret_cast<float2 *>(at + o_bytes);
    p.records = reinterpret_cast<Record *>(at + o_bytes + ml_bytes);
    FLAT_CUDA_OK(ctx, cudaFuncSetAttribute(tree_sm100_kernel<D, NARROW>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    {
        KernelTimer timer(ctx);
        FLAT_CUDA_OK(ctx, launch_dependent(may_overlap_previous(ctx), tree_sm100_kernel<D, NARROW>, dim3((unsigned)grid), kThreads, C::kSmem, ctx->stream, p));
    }
    ctx->launches += 1;
    const int chunks = (int)std::min<int64_t>(kMergeChunks, ((int64_t)t.max_nodes * t.group + 31) / 32);
    FLAT_CUDA_OK(ctx, launch_dependent(true, tree_sm100_merge_kernel<D>, dim3((unsigned)grid, (unsigned)chunks), 256, 0, ctx->stream, p));
    ctx->launches += 1;
    return FLAT_OK;
}

}  // namespace

bool tree_sm100_supported(int dtype, const TreeParams &p) {
    return dtype == FLAT_BF16 && (p.head_dim == 64 || p.head_dim == 128) && p.page_size % 16 == 0 &&
           ((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.o) % 16 == 0;
}

int launch_tree_sm100(flat_ctx *ctx, const TreeParams &p) {
    const bool narrow = (int64_t)p.max_nodes * p.group <= kSlotRows;
    if (p.head_dim == 128) return narrow ? launch<128, true>(ctx, p) : launch<128, false>(ctx, p);
    return narrow ? launch<64, true>(ctx, p) : launch<64, false>(ctx, p);
}

}  // namespace flat
