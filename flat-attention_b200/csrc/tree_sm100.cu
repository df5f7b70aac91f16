// Attention of drafted tokens over a paged cache on the tensor cores: bf16, head_dim 64 or 128, pages of a multiple of 16 tokens.
//
//   rows of one (sequence, KV head): (drafted token, head of the group), n * G of them, all against the same keys and values
//   S = Q K^T (SS MMA, 128 rows x 64 tokens)  ->  P = exp2(S - m)  ->  O += P V (A operand from TMEM)
//
// The bytes are those of K and V, read once; with many drafted tokens the products cost as much, so both are kept going at once: a
// producer streams tiles of 64 tokens by TMA, one box per page or 64 tokens, into a ring that holds six of them (twelve at D = 64)
// whatever item is at hand; one thread issues all products; two groups of four warps ("slots") each own a 128-row accumulator and
// work a softmax row per thread, without shuffles.
//   more than 128 rows: slot w has rows 128 w .. and both slots take every tile, which crosses into the SM once for 256 rows;
//   otherwise:          both slots have the same rows and take the tiles in turn, and their states are joined at the end.  A slot is
//                       a chain (scores, softmax, values), and one alone does not keep up with the memory.
// Each slot has two score tiles: the scores of its next tile are formed while it works on this one.  P lies over the scores it
// comes from; the products of one thread execute in order, so the next scores of that tile cannot overtake the product that reads P.
//
// Work: the tiles of all (sequence, KV head, 256 rows) items stand in one line, which is cut into equal spans, one per CTA, whatever
// the lengths are.  Every CTA adds the lengths up itself, so nothing is planned on the host.  An item that a span's end cuts is
// joined by a small second kernel from the parts, in order; everything else is written directly.
//
// Roundings: q enters as the sum of two bf16 numbers (the tensor core takes one type, and K is bf16; q alone would cost 2^-9 of the
// scores: 1.7 times the error of the bf16 result, where this way is 1.4 times it), P as bf16, sums and statistics are f32.
// The running maximum is followed only when it grows by more than 2^8, which keeps the accumulator out of the loop; P then reaches
// 2^8, sums stay far inside f32.
//
// Tokens that a row does not see: its score is replaced by -inf.  P = 0 alone would not do for V that is not finite, so a fourth
// role goes over the V tiles that hold drafted tokens or the end of a sequence before they are used: rows behind the end (whatever
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
constexpr int kTok = 64, kSlotRows = 128, kItemRows = 2 * kSlotRows;
constexpr int kSoftmaxWarps = 8, kProducerWarp = 8, kMmaWarp = 9, kFixWarp = 10;
constexpr int kThreads = 384;
constexpr int kValidRing = 32;   // tiles between the producer and the slowest softmax warp: the ring's and four more
constexpr int kPoisonRing = 16;  // segments between the fixing warp and the slowest softmax warp
constexpr int kMergeChunks = 8;  // blocks per item, 32 rows each

template <int D> struct Cfg {
    static constexpr int kBoxes = D / 64;
    static constexpr int kQBox = kSlotRows * 128, kQTile = kQBox * kBoxes;  // one of the two summands of a slot's queries
    static constexpr int kKvBox = kTok * 128, kKvTile = kKvBox * kBoxes;
    static constexpr int kStages = D == 128 ? 6 : 12;
    static constexpr int kSmem = 4 * kQTile + kStages * kKvTile + 1024;
};

struct Record {  // an item that begins in this CTA and ends in a later one
    int seq, kv_head, pair, parts;
};
struct KernelParams {
    TreeParams t;
    CUtensorMap map_k, map_v;
    uint32_t idesc_qk, idesc_pv;
    int box_rows;      // tokens of a TMA box: 16, 32 or 64, a divisor of the page size
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

// Which of the 64 tokens from t0 on drafted token `node` sees; valid: 16-token groups whose page is in the pool.
__device__ __forceinline__ uint64_t visible(const TreeParams &p, const TreeSequence &s, int node, int t0, uint32_t valid) {
    auto ones = [](int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
    const uint64_t live = ones(s.len - t0);
    uint64_t drafts = 0;
    if (t0 + kTok > s.len) {
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

template <int D> __global__ void __launch_bounds__(kThreads, 1) tree_sm100_kernel(const __grid_constant__ KernelParams p) {
    using C = Cfg<D>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *q_s = smem;                    // [slot][summand]
    uint8_t *kv_s = smem + 4 * C::kQTile;   // ring
    // slot 1's state, when the slots share rows: over its own queries, which are not there then, and over the shared ones, which no
    // product reads any more once slot 1's last value product is done
    float *join_o = reinterpret_cast<float *>(q_s + 2 * C::kQTile);
    float2 *join_ml = reinterpret_cast<float2 *>(q_s);
    __shared__ uint64_t bars[4 * C::kStages + 15];
    __shared__ uint64_t turns_s[D / 2];
    __shared__ uint32_t tmem_slot[1];
    __shared__ int abort_word;
    __shared__ uint32_t valid_s[kValidRing];
    __shared__ int poison_s[kPoisonRing];
    __shared__ int64_t sums_s[kThreads / 32];
    __shared__ int64_t start_s[2];
    volatile int *abort_flag = &abort_word;

    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](int s) { return bar0 + 8u * s; };                      // tile landed
    auto empty = [&](int s) { return bar0 + 8u * (C::kStages + s); };      // tile used
    auto fixed = [&](int s) { return bar0 + 8u * (2 * C::kStages + s); };  // V tile with drafted tokens gone over
    auto to_fix = [&](int s) { return bar0 + 8u * (3 * C::kStages + s); };  // such a tile has been requested
    auto s_full = [&](int w, int b) { return bar0 + 8u * (4 * C::kStages + 2 * w + b); };
    auto p_full = [&](int w, int b) { return bar0 + 8u * (4 * C::kStages + 4 + 2 * w + b); };
    auto pv_done = [&](int w, int b) { return bar0 + 8u * (4 * C::kStages + 8 + 2 * w + b); };
    const uint32_t q_ready = bar0 + 8u * (4 * C::kStages + 12);    // queries of the segment written
    const uint32_t q_free = bar0 + 8u * (4 * C::kStages + 13);     // a segment's queries and joined states are not needed any more
    const uint32_t join_full = bar0 + 8u * (4 * C::kStages + 14);  // slot 1's state written

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
        for (int i = 0; i < 4; ++i) {
            mbar_init(s_full(i >> 1, i & 1), 1);
            mbar_init(p_full(i >> 1, i & 1), 4);
            mbar_init(pv_done(i >> 1, i & 1), 1);
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
    auto col_s = [](int w, int b) { return (uint32_t)(2 * D + (2 * w + b) * kTok); };
    Walk walk{begin, end, start_s[1], (int)start_s[0]};
    Segment g;

    if (warp < kSoftmaxWarps) {
        // ================= queries, softmax, results =================
        const int w = warp >> 2, row = threadIdx.x & (kSlotRows - 1);
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's quarter of the TMEM lanes
        int count = 0;  // tiles of this slot so far
        int tile_base = 0;  // tiles of this CTA before the segment
        int joins = 0;
        bool ok = true;
        for (int k = 0; ok && walk.next(p.t, g); ++k) {
            const bool shared = g.rows <= kSlotRows;
            const int n = g.j1 - g.j0, r_begin = g.pair * kItemRows;
            if (k > 0 && !mbar_wait_warp(q_free, (k - 1) & 1, abort_flag)) {
                if (lane == 0) record_timeout(p, 330 + w);
                ok = false;
                break;
            }
            {
                const int node_lo = r_begin / p.t.group, node_hi = (r_begin + g.rows - 1) / p.t.group;
                const int tasks = (node_hi - node_lo + 1) * (D / 8);
                for (int i = threadIdx.x; i < tasks; i += kSoftmaxWarps * 32) {
                    const int node = node_lo + i / (D / 8), c = i % (D / 8);
                    const int position = p.t.positions[g.s.first + node];
                    float2 cs[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        cs[e] = turn_of(position, turns_s[c * 4 + e]);
                        cs[e].x *= p.t.scale * kLog2e;
                        cs[e].y *= p.t.scale * kLog2e;
                    }
                    const char *from = static_cast<const char *>(p.t.q) +
                                       (((int64_t)(g.s.first + node) * p.t.q_heads + g.kv_head * p.t.group) * D + c * 8) * 2;
                    const int r0 = node * p.t.group - r_begin;
#pragma unroll 4
                    for (int h = 0; h < p.t.group; ++h) {
                        const int r = r0 + h;
                        if (r < 0 || r >= g.rows) continue;
                        const uint4 raw = *reinterpret_cast<const uint4 *>(from + h * D * 2);
                        const uint32_t x[4] = {raw.x, raw.y, raw.z, raw.w};
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
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);

            const int r = r_begin + (shared ? 0 : w * kSlotRows) + row;  // of the (sequence, KV head)
            const bool live = r < r_begin + g.rows;
            const int node = live ? r / p.t.group : 0;
            const bool warp_live = (shared ? 0 : w * kSlotRows) + (warp & 3) * 32 < g.rows;
            float m = -INFINITY, l = 0.f;
            int mine = 0;  // tiles of this slot in this segment
            for (int i = shared ? w : 0; i < n; i += shared ? 2 : 1, ++mine, ++count) {
                const int b = count & 1;
                if (!mbar_wait_warp(s_full(w, b), (count >> 1) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 300 + w);
                    ok = false;
                    break;
                }
                if (warp_live) {
                    tc_fence_after();
                    uint32_t x[kTok];
                    tmem_ld32(tmem_base + lanes + col_s(w, b), x);
                    tmem_ld32(tmem_base + lanes + col_s(w, b) + 32, x + 32);
                    tc_wait_ld();
                    const int t0 = (g.j0 + i) * kTok;
                    const uint32_t valid = valid_s[(tile_base + i) % kValidRing];
                    if (t0 + kTok > g.s.len || valid != 0xf) {
                        const uint64_t on = visible(p.t, g.s, node, t0, valid);
                        const uint32_t on0 = (uint32_t)on, on1 = (uint32_t)(on >> 32);
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (!((on0 >> c) & 1)) x[c] = 0xff800000u;  // -inf
                            if (!((on1 >> c) & 1)) x[c + 32] = 0xff800000u;
                        }
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < kTok; ++c) mx[c & 3] = fmaxf(mx[c & 3], __uint_as_float(x[c]));
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    const bool grows = live && top > m + kRescaleThreshold;
                    if (__any_sync(0xffffffffu, grows)) {
                        const float now = grows ? top : m, f = grows ? ex2(m - now) : 1.f;  // m = -inf gives 0
                        m = now;
                        l *= f;
                        if (mine > 0) {
                            if (!mbar_wait_warp(pv_done(w, b ^ 1), ((count - 1) >> 1) & 1, abort_flag)) {
                                if (lane == 0) record_timeout(p, 310 + w);
                                ok = false;
                                break;
                            }
                            tc_fence_after();
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
#pragma unroll
                    for (int c = 0; c < kTok; c += 2) {
                        const float a = ex2(__uint_as_float(x[c]) - base), e = ex2(__uint_as_float(x[c + 1]) - base);
                        sum[(c >> 1) & 3] += a + e;
                        x[c >> 1] = pack_bf16(a, e);
                    }
                    l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    tmem_st32(tmem_base + lanes + col_s(w, b), x);
                    tc_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(w, b));
            }
            tile_base += n;
            if (!ok) break;
            if (mine > 0) {
                if (!mbar_wait_warp(pv_done(w, (count - 1) & 1), ((count - 1) >> 1) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 320 + w);
                    ok = false;
                    break;
                }
                tc_fence_after();
            }
            // ---- the slots' states, where they share rows, are joined by slot 0
            float keep = 1.f, add = 0.f;  // factors of this slot's and the other's accumulator
            if (shared) {
                if (w == 1) {
                    if (mine > 0) join_ml[row] = make_float2(m, l);
                    if (mine > 0 && warp_live) {
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem_base + lanes + col_o(1) + c, o);
                            tc_wait_ld();
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                *reinterpret_cast<uint4 *>(join_o + row * D + (((c / 4 + e) ^ (row & 7)) << 2)) =
                                    make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                        }
                    }
                }
                __syncwarp();
                if (w == 1) {
                    if (lane == 0) {
                        mbar_arrive(join_full);
                        mbar_arrive(q_free);
                    }
                    continue;
                }
                if (!mbar_wait_warp(join_full, joins++ & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 340);
                    ok = false;
                    break;
                }
                if (n > 1) {
                    const float2 other = join_ml[row];
                    const float mx = fmaxf(m, other.x);
                    keep = l == 0.f ? 0.f : ex2(m - mx);  // a slot that has seen nothing counts for nothing; a NaN counts
                    add = other.y == 0.f ? 0.f : ex2(other.x - mx);
                    l = (l == 0.f ? 0.f : keep * l) + (other.y == 0.f ? 0.f : add * other.y);
                    m = mx;
                }
            }
            const bool whole = g.j0 == 0 && g.j1 == g.tiles;
            const int64_t part = ((int64_t)blockIdx.x * 2 + (g.j0 == 0 ? 1 : 0)) * kItemRows + (r - r_begin);
            const int64_t out = (int64_t)(g.s.first + node) * p.t.q_heads + g.kv_head * p.t.group + (live ? r % p.t.group : 0);
            const bool nothing = l == 0.f;
            const float inv = whole ? (nothing ? 0.f : 1.0f / l) : 1.f;
            keep *= inv;
            add *= inv;
            const int poison = *reinterpret_cast<volatile int *>(&poison_s[k % kPoisonRing]);
            if (warp_live) {
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t raw[16];
                    float o[16];
                    tmem_ld16(tmem_base + lanes + col_o(w) + c, raw);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = nothing ? 0.f : __uint_as_float(raw[e]) * keep;
                    if (shared && n > 1 && add != 0.f) {
#pragma unroll
                        for (int e = 0; e < 16; e += 4) {
                            const float4 y = *reinterpret_cast<const float4 *>(join_o + row * D + (((c + e) / 4 ^ (row & 7)) << 2));
                            o[e] = fmaf(y.x, add, o[e]);
                            o[e + 1] = fmaf(y.y, add, o[e + 1]);
                            o[e + 2] = fmaf(y.z, add, o[e + 2]);
                            o[e + 3] = fmaf(y.w, add, o[e + 3]);
                        }
                    }
                    if (!live) continue;
                    if (poison) {  // drafted tokens of this segment whose V is not finite, as the rows that see them see them
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
                    if (whole) {
                        uint4 *to = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.t.o) + out * D + c);
                        to[0] = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
                        to[1] = make_uint4(pack_bf16(o[8], o[9]), pack_bf16(o[10], o[11]), pack_bf16(o[12], o[13]), pack_bf16(o[14], o[15]));
                    } else {
                        float4 *to = reinterpret_cast<float4 *>(p.part_o + part * D + c);
#pragma unroll
                        for (int e = 0; e < 4; ++e) to[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
                tc_fence_before();  // the next segment's first value product starts this accumulator anew
                if (live) {
                    if (whole) p.t.lse[out] = nothing ? -INFINITY : (m + log2f(l)) * kLn2;
                    else p.part_ml[part] = make_float2(m, l);
                }
            }
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
    } else if (warp == kProducerWarp) {
        // ================= TMA producer =================
        // Lane i fetches the id of the page of the tile's i-th box, a tile ahead of its load, and issues that box.
        const int boxes = kTok / p.box_rows;
        const uint32_t pool_rows = (uint32_t)p.t.physical_pages * (uint32_t)p.t.page_size;
        uint32_t order = 0;  // tiles requested so far
        int tile_base = 0;
        bool ok = true;
        while (ok && walk.next(p.t, g)) {
            const int n = g.j1 - g.j0, ahead = g.rows <= kSlotRows ? 2 : 1;
            const int32_t *table = p.t.page_tables + (int64_t)g.seq * p.t.max_pages;
            auto row_of = [&](int i) -> int {  // pool row of this lane's box; behind the pool: zeros.  -1: the page is none of the pool's
                const int t = (g.j0 + i) * kTok + lane * p.box_rows;
                if (lane >= boxes || i >= n || t >= g.s.tokens) return (int)pool_rows;
                const int page = table[t / p.t.page_size];
                if ((unsigned)page >= (unsigned)p.t.physical_pages) return -1;
                return page * p.t.page_size + t % p.t.page_size;
            };
            auto load = [&](const CUtensorMap *map, int at, bool fix) {
                const int s = order % C::kStages;
                if (!mbar_wait_warp(empty(s), ((order / C::kStages) & 1) ^ 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 100 + s);
                    ok = false;
                    return;
                }
                ++order;
                if (lane == 0) mbar_expect_tx(full(s), C::kKvTile);
                __syncwarp();
                const uint32_t dst = smem_u32(kv_s + s * C::kKvTile) + lane * p.box_rows * 128;
                if (lane < boxes)
                    for (int kb = 0; kb < C::kBoxes; ++kb)
                        tma_load_4d(dst + kb * C::kKvBox, map, kb * 64, at < 0 ? (int)pool_rows : at, g.kv_head, 0, full(s));
                if (fix && lane == 0) mbar_arrive(to_fix(s));
            };
            int now = row_of(0), last = 0, older = 0;
            for (int i = 0; ok && i < n + ahead; ++i) {
                const int next = row_of(i + 1);
                if (i < n) {
                    const uint32_t bad = __ballot_sync(0xffffffffu, now < 0);
                    uint32_t valid = 0xf;
                    if (bad) {
                        for (int e = 0; e < 4; ++e)
                            if ((bad >> (e * 16 / p.box_rows)) & 1) valid &= ~(1u << e);
                        if (lane == 0) tree_report(p.t, FLAT_ERR_PAGE_OUT_OF_RANGE, g.seq);
                    }
                    if (lane == 0) valid_s[(tile_base + i) % kValidRing] = valid;
                    load(&p.map_k, now, false);
                }
                if (i >= ahead && ok) load(&p.map_v, ahead == 2 ? older : last, is_tail(g, g.j0 + i - ahead));
                older = last;
                last = now;
                now = next;
            }
            tile_base += n;
        }
    } else if (warp == kMmaWarp) {
        // ================= all products =================
        if (elect_one()) {
            const uint32_t q_desc = (uint32_t)make_smem_desc(smem_u32(q_s), 0, 1024);
            const uint32_t k_desc = (uint32_t)make_smem_desc(smem_u32(kv_s), 0, 1024);
            const uint32_t v_desc = (uint32_t)make_smem_desc(smem_u32(kv_s), C::kKvBox, 1024);
            uint32_t order = 0, fixed_phase = 0;
            int scored[2] = {0, 0}, valued[2] = {0, 0};  // tiles per slot
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity, int where) {
                if (ok && !mbar_wait(bar, parity, abort_flag)) {
                    record_timeout(p, where);
                    ok = false;
                }
            };
            for (int k = 0; ok && walk.next(p.t, g); ++k) {
                const bool shared = g.rows <= kSlotRows;
                const int n = g.j1 - g.j0, ahead = shared ? 2 : 1;
                wait(q_ready, k & 1, 200);
                for (int i = 0; ok && i < n + ahead; ++i) {
                    if (i < n) {
                        const int s = order % C::kStages;
                        wait(full(s), (order / C::kStages) & 1, 210);
                        ++order;
                        if (!ok) break;
                        tc_fence_after();
                        for (int w = 0; w < 2; ++w) {
                            if (shared && (i & 1) != w) continue;
                            const int b = scored[w]++ & 1;
                            const uint32_t q = q_desc + (shared ? 0 : w) * (2 * C::kQTile >> 4), kk = k_desc + s * (C::kKvTile >> 4);
                            const uint32_t d = tmem_base + col_s(w, b);
#pragma unroll
                            for (int h = 0; h < 2; ++h)  // the two summands of q
#pragma unroll
                                for (int e = 0; e < D / 16; ++e)
                                    mma_ss_lo(d, q + h * (C::kQTile >> 4) + (e >> 2) * (C::kQBox >> 4), kk + (e >> 2) * (C::kKvBox >> 4),
                                              (e & 3) * 2, p.idesc_qk, h > 0 || e > 0);
                            tc_commit(s_full(w, b));
                        }
                        tc_commit(empty(s));
                    }
                    const int v = i - ahead;
                    if (v >= 0) {
                        const int s = order % C::kStages;
                        wait(full(s), (order / C::kStages) & 1, 220);
                        ++order;
                        if (is_tail(g, g.j0 + v)) {
                            wait(fixed(s), (fixed_phase >> s) & 1, 230);
                            fixed_phase ^= 1u << s;
                        }
                        for (int w = 0; w < 2; ++w) {
                            if (shared && (v & 1) != w) continue;
                            const int b = valued[w] & 1;
                            wait(p_full(w, b), (valued[w] >> 1) & 1, 240 + w);
                            if (!ok) break;
                            ++valued[w];
                            tc_fence_after();
                            const bool first = shared ? v < 2 : v == 0;
#pragma unroll
                            for (int e = 0; e < kTok / 16; ++e)
                                mma_ts_lo(tmem_base + col_o(w), tmem_base + col_s(w, b) + e * 8, v_desc + s * (C::kKvTile >> 4), e * (16 * 128 >> 4),
                                          p.idesc_pv, !first || e > 0);
                            tc_commit(pv_done(w, b));
                        }
                        if (ok) tc_commit(empty(s));
                    }
                }
            }
        }
    } else if (warp == kFixWarp) {
        // ================= V tiles with drafted tokens or the end of a sequence =================
        uint32_t order = 0, phase = 0;
        bool ok = true;
        for (int k = 0; ok && walk.next(p.t, g); ++k) {
            const int n = g.j1 - g.j0, ahead = g.rows <= kSlotRows ? 2 : 1;
            if (lane == 0) poison_s[k % kPoisonRing] = 0;
            __syncwarp();
            // (to_fix tells that the tile before in this stage is used up, without which its phase could be taken for this one's)
            for (int v = max(0, min(g.s.len / kTok, g.tiles - 1) - g.j0); v < n; ++v) {
                // V tile v is number v + min(n, v + 1 + ahead) of the segment
                const uint32_t at = order + v + min(n, v + 1 + ahead);
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
                for (int i = lane; i < (kTok - from) * C::kBoxes * 8; i += 32) {
                    const int row = from + i / (C::kBoxes * 8), c = i % (C::kBoxes * 8);
                    uint4 *x = reinterpret_cast<uint4 *>(tile + (c >> 3) * C::kKvBox + row * 128 + ((c & 7) << 4));
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

template <int D> int launch(flat_ctx *ctx, const TreeParams &t) {
    using C = Cfg<D>;
    KernelParams p{};
    p.t = t;
    p.box_rows = t.page_size % 64 == 0 ? 64 : t.page_size % 32 == 0 ? 32 : 16;
    const uint64_t rows = (uint64_t)t.physical_pages * t.page_size;
    const int64_t rs = (int64_t)t.kv_heads * D;
    if (int st = make_map(ctx, &p.map_k, false, t.k, D, rows, t.kv_heads, 1, rs, D, rs, p.box_rows)) return st;
    if (int st = make_map(ctx, &p.map_v, false, t.v, D, rows, t.kv_heads, 1, rs, D, rs, p.box_rows)) return st;
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
    FLAT_CUDA_OK(ctx, cudaFuncSetAttribute(tree_sm100_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    {
        KernelTimer timer(ctx);
        FLAT_CUDA_OK(ctx, launch_dependent(may_overlap_previous(ctx), tree_sm100_kernel<D>, dim3((unsigned)grid), kThreads, C::kSmem, ctx->stream, p));
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

int launch_tree_sm100(flat_ctx *ctx, const TreeParams &p) { return p.head_dim == 128 ? launch<128>(ctx, p) : launch<64>(ctx, p); }

}  // namespace flat
