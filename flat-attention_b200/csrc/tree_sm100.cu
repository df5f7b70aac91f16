// Attention of drafted tokens over a paged cache on the tensor cores: bf16, head_dim 64 or 128, pages of a multiple of 16 tokens.
//
//   rows of one (sequence, KV head): (drafted token, head of the group), n * G of them, all against the same keys and values
//   S = Q K^T (SS MMA, 64 or 128 rows x 64 tokens)  ->  P = exp2(S - m)  ->  O += P V (A operand from TMEM)
//
// Bound by the bytes of K and V, read once, and with hundreds of rows by the products; either way what counts is that nothing stands between
// two tiles.  The beginning and the end of an item (queries read, turned and written; the first scores; the last weights; results) are
// a chain of 10000 clk and more, and a load takes 2000 clk while K and V stream in.  So:
//   two CTAs share an SM, 112 KB and half the TMEM each;
//   K and V tiles of 64 tokens come by TMA, a box per page or tile, through a ring that runs on whatever item is at hand;
//   one warp plans: it walks the span two items ahead of the products and puts what the other warps have to know in shared memory;
//   two warps make the next item's queries as soon as the last scores of the item before are formed;
//   four warps work a softmax row per thread, without shuffles, and write results, while the next item's first scores are formed;
//   one thread issues all products.  Two score tiles alternate; P lies over the scores it comes from, and the products of one
//   thread execute in order, so the scores after next cannot overtake the product that reads that P.
// ROWS is 64 where max_nodes allows a sequence no more, otherwise 128, whatever the sequences have (the host does not know).  A product of
// 64 rows takes as long as one of 128, but half the power, and the power limit is what a long run meets: at head_dim 128 one drafted
// token against 32 x 4000 takes 92 us a call in a run of seconds, with products of 128 rows 104 (alone 90 and 94), 4 to 16 tokens
// against 32 x 512 to 8192 108 and 118 (101 and 104).  At head_dim 64, where the softmax counts for more and a warp of it has 16 rows
// instead of 32, one token takes 62 and 65 (alone 62 both), 4 to 16 tokens 82 and 79 (82 and 75), and 16 tokens against 32 x 4000, 64
// whole rows, 78 and 71 (74 and 62).  For the power too rows that are not there are zeros.  Of more than 128 rows, two blocks of 128 go
// to two CTAs that walk the same span, so that the second one finds K and V in the L2.
//
// Work: the tiles of all items, a block of ROWS rows of a (sequence, KV head) each, stand in one line, which is cut into equal spans,
// one per CTA, whatever the lengths are.  Every CTA adds the lengths up itself, so nothing is planned on the host.  An item that a span's end cuts is
// joined, from the parts in order, by the CTA that finds that they are all there; everything else is written directly.
//
// Roundings: q enters as the sum of two bf16 numbers (the tensor core takes one type, and K is bf16; q alone would cost 2^-8 of the
// scores: 1.7 times the error of the bf16 result, where this way is 1.4 times it), P as bf16 (a second summand of it would double the
// value products; against 64 bits O is off by 2.3e-3 in the 2-norm, with weights of 32 bits by 1.7e-3, which is the result's own
// rounding), sums and statistics are f32.
// The running maximum is followed only when it grows by more than 2^8, which keeps the accumulator out of the loop; P then
// reaches 2^8, sums stay far inside f32.
//
// Tokens that a row does not see: its score is replaced by -inf.  P = 0 alone would not do for V that is not finite, so another
// warp goes over the V tiles that hold drafted tokens or the end of a sequence before they are used: rows behind the end (whatever
// an earlier owner of the page left) become zero, and so do values of drafted tokens that are not finite; these are then added to
// the rows that see them at the end, where they were met at all.
#include "tree_tc.cuh"

namespace flat {
namespace {

using namespace tree_tc;

constexpr int kTok = 64, kAhead = 2;  // kAhead: score tiles
constexpr int kQWarps = 2, kCtasPerSm = 2;
constexpr int kThreads = 320;  // warps: softmax 4, queries 2, K, V, products, and one that goes over V tiles
constexpr int kSegRing = 4;      // see below, planning
constexpr int kValidRing = 16;   // tiles between the producer and the slowest softmax warp: the ring's and four more
constexpr int kPoisonRing = 16;  // segments between the fixing warp and the slowest softmax warp

// A K or V tile lies in shared memory as [8 tokens][64 dims of D][token of the 8][64 dims]: one TMA box of any number of tokens
// then writes all D dims.  Queries: [summand][64 dims of D][row][64 dims].
template <int D, int ROWS> struct Cfg {
    static constexpr int kSoftmaxWarps = 4, kWarpRows = ROWS / 4, kQWarp = kSoftmaxWarps, kKWarp = kQWarp + kQWarps, kVWarp = kKWarp + 1, kMmaWarp = kVWarp + 1;
    static constexpr int kQSteps = 3;                     // tokens of a thread of the query warps in flight, as many as the registers hold
    static constexpr int kBoxes = D / 64;
    static constexpr int kQBox = ROWS * 128, kQTile = kQBox * kBoxes;  // one of the two summands of the queries
    static constexpr int kGroup = 1024 * kBoxes;                        // 8 tokens
    static constexpr int kKvTile = kTok / 8 * kGroup;
    static constexpr int kControl = 1024, kSmem = (228 / kCtasPerSm - 1) * 1024;  // of an SM's 228 KB, 1 KB a CTA is the system's
    static constexpr int kStages = (kSmem - kControl - 2 * kQTile) / kKvTile;     // D = 128: 5 and 3, D = 64: 12 and 10
    static_assert(kStages >= 3 && 4 * kStages + 9 + kSegRing <= 64, "ring");
};

struct KernelParams {
    TreeParams t;
    CUtensorMap map_k, map_v;
    uint32_t idesc_qk, idesc_pv;
    int box_rows;      // tokens of a TMA box: 16, 32 or 64, a divisor of the page size
    int share;         // CTAs of a span: 2 where two blocks of rows share K and V
    int items;         // of the line, at most
    float4 *part_o;    // [2 per CTA][D / 4][ROWS], not normalised
    float2 *part_ml;   // [2 per CTA][ROWS] maximum (log2 domain) and sum
    unsigned *arrived; // [CTA]: warps that have written their part of the item that begins in this CTA and ends in a later one; 0 between calls
};

// A part of an item that one CTA works on.
struct Segment {
    TreeSequence s;
    int seq, kv_head;
    int row0, rows;    // of the (sequence, KV head)
    int j0, n, tiles;  // its first tile, its tiles (0: there are no more segments), the item's
    int parts, cta;    // of an item that is cut, and the CTA that it begins in; otherwise parts = 1
};

__device__ __forceinline__ int tiles_of(const TreeSequence &s) { return max(1, (s.tokens + kTok - 1) / kTok); }
template <int ROWS> __device__ __forceinline__ int blocks_of(const TreeParams &p, const TreeSequence &s) { return (s.nodes * p.group + ROWS - 1) / ROWS; }
// An item's place on the line, in tiles: whole multiples of `grain`.
__device__ __forceinline__ int pitch_of(int tiles, int grain) { return (int)(((unsigned)tiles + (unsigned)grain - 1) / (unsigned)grain) * grain; }
// What a sequence takes of the line: the places of its items, or of its pairs of items where two CTAs walk a span.
template <int ROWS> __device__ __forceinline__ int units_of(const KernelParams &p, const TreeSequence &s, int grain) {
    return s.nodes == 0 ? 0 : (blocks_of<ROWS>(p.t, s) * p.t.kv_heads + p.share - 1) / p.share * pitch_of(tiles_of(s), grain);
}

// A CTA's way along its span.
template <int ROWS> struct Walk {
    int at, end, seq_start, units, span, grain, seq;
    TreeSequence s;  // of seq
    __device__ __forceinline__ void next(const KernelParams &p, Segment &g) {
        g.n = 0;
        while (at < end) {
            if (at >= seq_start + units) {
                seq_start += units;
                s = tree_sequence(p.t, ++seq);
                units = units_of<ROWS>(p, s, grain);
                continue;
            }
            const int tiles = tiles_of(s), blocks = blocks_of<ROWS>(p.t, s), pitch = pitch_of(tiles, grain);
            const int pair = (int)((unsigned)(at - seq_start) / (unsigned)pitch), item_start = seq_start + pair * pitch;
            const int lane = p.share == 2 ? (int)blockIdx.x & 1 : 0, item = pair * p.share + lane;
            const int j0 = at - item_start, n = min(tiles - j0, end - at);
            at = min(end, item_start + pitch);
            if (n <= 0) continue;  // behind the item's last tile
            const int kv_head = (int)((unsigned)item / (unsigned)blocks);
            if (kv_head >= p.t.kv_heads) continue;  // an odd number of items: nothing for the second CTA
            g.s = s;
            g.seq = seq;
            g.kv_head = kv_head;
            g.row0 = (item - kv_head * blocks) * ROWS;
            g.rows = min(ROWS, s.nodes * p.t.group - g.row0);
            g.tiles = tiles;
            g.j0 = j0;
            g.n = n;
            g.parts = 1;
            g.cta = blockIdx.x;
            if (n < tiles) {
                const int first = (int)((unsigned)item_start / (unsigned)span);
                g.cta = first * p.share + lane;
                g.parts = (int)((unsigned)(item_start + tiles - 1) / (unsigned)span) - first + 1;
            }
            return;
        }
    }
};

__device__ __forceinline__ void record_timeout(const KernelParams &p, int where) {
    report_status(p.t.status, FLAT_ERR_DEVICE_WAIT_TIMEOUT, where);
}

// Whether tile j of the segment's item holds drafted tokens or is its last: its V tile is gone over before it is used.  (Every
// item has such a tile, so the warp that does it is never more than the ring ahead.)
__device__ __forceinline__ bool is_tail(const Segment &g, int j) { return (j + 1) * kTok > g.s.len || j + 1 == g.tiles; }

struct Join {  // an item whose parts are all there
    int first, kv_head, row0, rows, parts, cta;
};

// What the warps of a CTA share, at the start of its shared memory.
template <int ROWS, int STAGES> struct Control {
    uint64_t bars[4 * STAGES + 9 + kSegRing];
    union {
        Segment seg[kSegRing];
        struct {  // before the first is planned
            int sums[16], tops[16];  // of each warp
        } start;
    };
    uint32_t tmem;
    int abort;
    Walk<ROWS> walk;  // of the planning warp
    Segment coming;
    Join join[2];  // an item that ends here, and one that does not
    uint8_t valid[kValidRing], poison[kPoisonRing];
};

// Joins the parts of an item in CTA order, whichever came last: a row a thread and a share of the dims.
template <int D, int ROWS> __device__ __forceinline__ void join_parts(const KernelParams &p, const Join &item) {
    const int lanes = item.rows <= 32 ? 32 : item.rows <= 64 ? 64 : 128, r = threadIdx.x & (lanes - 1), g = threadIdx.x / lanes, groups = 256 / lanes;
    const int parts = item.parts;
    if (r >= item.rows || threadIdx.x >= 256) return;
    auto part = [&](int i) { return (int64_t)((item.cta + i * p.share) * 2 + (i == 0 ? 1 : 0)); };  // the first CTA's second, the others' first
    auto weight = [](float2 ml, float mx) { return ml.y == 0.f ? 0.f : ex2(ml.x - mx); };  // a part in which the row has seen nothing; a NaN counts
    float mx = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int base = 0; base < parts; base += 8) {
        float2 ml[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) ml[u] = base + u < parts ? __ldcg(&p.part_ml[part(base + u) * ROWS + r]) : make_float2(-INFINITY, 0.f);
        const float before = mx;
#pragma unroll
        for (int u = 0; u < 8; ++u) mx = fmaxf(mx, ml[u].x);
        sum *= before == -INFINITY ? 0.f : ex2(before - mx);
#pragma unroll
        for (int u = 0; u < 8; ++u) sum = fmaf(weight(ml[u], mx), ml[u].y, sum);
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    const int row = item.row0 + r, node = row / p.t.group;
    const int64_t out = (int64_t)(item.first + node) * p.t.q_heads + item.kv_head * p.t.group + row - node * p.t.group;
    if (g == 0) p.t.lse[out] = sum == 0.f ? -INFINITY : (mx + log2f(sum)) * kLn2;
#pragma unroll 1
    for (int d4 = g * 4; d4 < D / 4; d4 += groups * 4) {
        float4 o[4] = {};
#pragma unroll 1
        for (int base = 0; base < parts; base += 2) {
            float4 x[2][4];
            float2 ml[2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (base + u < parts) {
                    ml[u] = __ldcg(&p.part_ml[part(base + u) * ROWS + r]);
                    const float4 *from = p.part_o + (part(base + u) * (D / 4) + d4) * ROWS + r;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[u][e] = __ldcg(from + e * ROWS);
                }
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (base + u < parts) {
                    const float f = weight(ml[u], mx) * inv;
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[e] = make_float4(fmaf(f, x[u][e].x, o[e].x), fmaf(f, x[u][e].y, o[e].y), fmaf(f, x[u][e].z, o[e].z), fmaf(f, x[u][e].w, o[e].w));
                }
        }
        uint4 *to = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.t.o) + out * D + d4 * 4);
        to[0] = make_uint4(pack_bf16(o[0].x, o[0].y), pack_bf16(o[0].z, o[0].w), pack_bf16(o[1].x, o[1].y), pack_bf16(o[1].z, o[1].w));
        to[1] = make_uint4(pack_bf16(o[2].x, o[2].y), pack_bf16(o[2].z, o[2].w), pack_bf16(o[3].x, o[3].y), pack_bf16(o[3].z, o[3].w));
    }
}

__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

template <int D, int ROWS>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) tree_sm100_kernel(const __grid_constant__ KernelParams p) {
    using C = Cfg<D, ROWS>;
    using Ctl = Control<ROWS, C::kStages>;
    constexpr int kSoftmaxWarps = C::kSoftmaxWarps, kQWarp = C::kQWarp, kKWarp = C::kKWarp, kVWarp = C::kVWarp, kMmaWarp = C::kMmaWarp;
    constexpr int kQSteps = C::kQSteps;
    static_assert(kThreads == (kMmaWarp + 2) * 32, "warps");
    extern __shared__ __align__(1024) uint8_t smem[];
    Ctl &ctl = *reinterpret_cast<Ctl *>(smem);
    static_assert(sizeof(Ctl) <= C::kControl, "control block");
    uint8_t *q_s = smem + C::kControl;       // [summand]
    uint8_t *kv_s = q_s + 2 * C::kQTile;     // ring
    volatile int *abort_flag = &ctl.abort;

    const uint32_t bar0 = smem_u32(ctl.bars);
    auto full = [&](int s) { return bar0 + 8u * s; };                        // tile landed
    auto empty = [&](int s) { return bar0 + 8u * (C::kStages + s); };        // tile used
    auto fixed = [&](int s) { return bar0 + 8u * (2 * C::kStages + s); };    // V tile with drafted tokens gone over
    auto to_fix = [&](int s) { return bar0 + 8u * (3 * C::kStages + s); };   // such a tile has been requested
    auto s_full = [&](int b) { return bar0 + 8u * (4 * C::kStages + b); };       // scores in tile b
    auto p_full = [&](int b) { return bar0 + 8u * (4 * C::kStages + 2 + b); };   // P written over tile b
    auto pv_done = [&](int b) { return bar0 + 8u * (4 * C::kStages + 4 + b); };  // ... and used
    const uint32_t q_ready = bar0 + 8u * (4 * C::kStages + 6);                   // queries of the segment written
    const uint32_t q_empty = bar0 + 8u * (4 * C::kStages + 7);                   // ... and not needed any more
    const uint32_t go = bar0 + 8u * (4 * C::kStages + 8);                        // K and V may be asked for
    auto planned = [&](int k) { return bar0 + 8u * (4 * C::kStages + 9 + k % kSegRing); };  // segment k

    const int warp = warp_index_uniform(), lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        ctl.join[0].parts = ctl.join[1].parts = 0;
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
            mbar_init(fixed(s), 1);
            mbar_init(to_fix(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(s_full(b), 1);
            mbar_init(p_full(b), kSoftmaxWarps);
            mbar_init(pv_done(b), 1);
        }
        mbar_init(q_ready, kQWarps);
        mbar_init(q_empty, 1);
        mbar_init(go, kQWarps);
        for (int k = 0; k < kSegRing; ++k) mbar_init(planned(k), 1);
        mbar_fence_init();
        fence_proxy_async();
        tma_prefetch_desc(&p.map_k);
        tma_prefetch_desc(&p.map_v);
    }
    // rows that are not there are zeros, see above
    for (int i = threadIdx.x; i < 2 * C::kQTile / 16; i += kThreads) reinterpret_cast<uint4 *>(q_s)[i] = make_uint4(0, 0, 0, 0);
    fence_proxy_async();
    // TMEM behind the wait: a kernel before this one may still be about to allocate all of it.  The next kernel comes in behind
    // the barriers below, when this CTA has its own.
    grid_dependency_wait();
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(&ctl.tmem), 512 / kCtasPerSm);
        tmem_relinquish();
    }

    // The line's length, then the sequence that this CTA's span starts in: a scan over kThreads sequences at a time, the same once more
    // where there are more.  (What runs once is kept short here and below: instructions that are not in the cache yet come at a
    // tenth of the rate.)
    int span = 1, grain = 1, begin = 0, end = 0;
    {
        int total = 0, before = 0, longest = 0;
        bool counting = true;
#pragma unroll 1
        for (int base = 0;; base += kThreads) {
            TreeSequence mine{};
            int units = 0;
            if (base + (int)threadIdx.x < p.t.num_seqs) {
                mine = tree_sequence(p.t, base + threadIdx.x);
                units = units_of<ROWS>(p, mine, grain);
                if (mine.code && counting && blockIdx.x == 0) report_status(p.t.status, mine.code, base + threadIdx.x, kPlaceBound);
            }
            int upto = units;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += y;
            }
            const int top = (int)__reduce_max_sync(0xffffffffu, mine.nodes ? tiles_of(mine) : 0);
            if (lane == 31) {
                ctl.start.sums[warp] = upto;
                ctl.start.tops[warp] = top;
            }
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
            const int sums = lane < kThreads / 32 ? ctl.start.sums[lane] : 0;
            longest = max(longest, (int)__reduce_max_sync(0xffffffffu, lane < kThreads / 32 ? ctl.start.tops[lane] : 0));
            const int pass = (int)__reduce_add_sync(0xffffffffu, sums);
            upto += (int)__reduce_add_sync(0xffffffffu, lane < warp ? sums : 0);
            __syncthreads();  // the next pass's sums
            if (counting) {
                total += pass;
                if (base + kThreads < p.t.num_seqs) continue;
                counting = false;
                const unsigned spans = gridDim.x / p.share, line = blockIdx.x / p.share;
                // Few tiles are not spread over all CTAs: each part costs the end of its item about a third of what a tile takes, so that an
                // item of t tiles is done first with some sqrt(t / 3) tiles a part (one KV head, 16000 tokens: 90 -> 24 us; 8 heads, 700
                // tokens: 16.4 -> 14.8).
                const int least = (int)(sqrtf(0.35f * (float)longest) + 0.5f), even = (int)((unsigned)(total + spans - 1) / spans);
                span = max(max(least, 1), even);
                // A second item in a CTA's span costs it what four tiles take, so items get whole spans where that needs no more than
                // four tiles more a span (8 heads, 2000 tokens: 21.9 us -> 19; 16000: 36 -> 32), which takes another pass here (1 us) and
                // is left out where they do anyway.
                if (p.items > 1 && p.items < (int)spans && (longest % span || total != p.items * longest)) {
                    const int whole = max(max(least, 1), (int)((unsigned)max(total - p.items, 0) / (spans - p.items)) + 1);
                    if (whole <= span + 4) span = grain = whole;
                }
                begin = span * (int)line;
                end = begin + span;  // with a grain the line's length is a multiple of it
                if (grain == 1) {
                    begin = min(begin, total);
                    end = min(end, total);
                }
                if (base > 0 || grain > 1) {
                    base = -kThreads;
                    continue;
                }
            }
            upto += before;
            if (begin < upto && begin >= upto - units) {
                ctl.walk = Walk<ROWS>{begin, end, upto - units, units, span, grain, base + (int)threadIdx.x, mine};
            }
            before += pass;
            if (before > begin || base + kThreads >= p.t.num_seqs) {
                if (before <= begin) end = begin;  // behind the line's end: nothing to do
                break;
            }
        }
    }
    __syncthreads();
    grid_dependency_wait();  // long over: it stands here so that the rule, nothing is let in before one's own wait, can be seen
    grid_dependency_launch();
    const uint32_t tmem_base = ctl.tmem;
    auto col_s = [](int b) { return (uint32_t)(D + b * kTok); };  // O in columns 0 .. D - 1
    bool ok = true;
    auto segment = [&](int k) -> const Segment & {  // waits until it is planned
        if (!mbar_wait_warp(planned(k), (k / kSegRing) & 1, abort_flag)) {
            if (lane == 0) record_timeout(p, 500 + warp);
            ok = false;
        }
        return ctl.seg[k % kSegRing];
    };

    if (begin >= end) {  // nothing to do
    } else if (warp < kSoftmaxWarps) {
        // ================= softmax and results =================
        const uint32_t lanes = (uint32_t)warp << 21;  // this warp's quarter of the TMEM lanes
        // The accumulator's rows lie in lanes 0 .. 31 of each quarter of the TMEM lanes, of 64 rows in lanes 0 .. 15.
        const int row = lane < C::kWarpRows ? warp * C::kWarpRows + lane : ROWS;
        int count = 0;  // tiles so far
        for (int k = 0;; ++k) {
            const Segment &g = segment(k);
            if (!ok || g.n == 0) break;
            const int rows = g.rows, n = g.n, j0 = g.j0, all_see = min(g.s.len, g.s.tokens);  // live tokens that are not cut off
            const bool live = row < rows, warp_live = warp * C::kWarpRows < rows;
            const int node = live ? (g.row0 + row) / p.t.group : 0;
            uint32_t own0 = 0, own1 = 0;  // first mask bits
            if (p.t.mask && live) {
                const uint32_t *bits = p.t.mask + (int64_t)(g.s.first + node) * p.t.mask_words;
                own0 = bits[0];
                if (p.t.mask_words > 1) own1 = bits[1];
            }
            float m = -INFINITY, l = 0.f;
            for (int i = 0; i < n; ++i, ++count) {
                const int b = count & 1;
                if (!mbar_wait_warp(s_full(b), (count >> 1) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 300 + b);
                    ok = false;
                    break;
                }
                if (warp_live) {
                    tc_fence_after();
                    uint32_t x[kTok];
                    tmem_ld32(tmem_base + lanes + col_s(b), x);
                    tmem_ld32(tmem_base + lanes + col_s(b) + 32, x + 32);
                    const uint32_t valid = *reinterpret_cast<volatile uint8_t *>(&ctl.valid[count % kValidRing]);  // 16-token groups whose page is in the pool
                    const int t0 = (j0 + i) * kTok;
                    const bool masked = t0 + kTok > all_see || valid != 0xf;
                    uint64_t on = ~0ull;
                    if (masked) {
                        on = visible(p.t, g.s, node, t0, own0 | (uint64_t)own1 << 32);
                        for (int e = 0; e < 4; ++e)
                            if (!((valid >> e) & 1)) on &= ~(0xffffull << (16 * e));
                    }
                    tc_wait_ld();
                    if (masked) {
                        const uint32_t on0 = (uint32_t)on, on1 = (uint32_t)(on >> 32);
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            if (!((on0 >> e) & 1)) x[e] = 0xff800000u;  // -inf
                            if (!((on1 >> e) & 1)) x[32 + e] = 0xff800000u;
                        }
                    }
                    float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int e = 0; e < kTok; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(x[e]));
                    const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                    const bool grows = live && top > m + (i ? kRescaleThreshold : 0.f);
                    if (__any_sync(0xffffffffu, grows)) {
                        const float now = grows ? top : m, f = grows ? ex2(m - now) : 1.f;  // m = -inf gives 0
                        m = now;
                        l *= f;
                        if (i > 0) {  // the accumulator, which the value product before this tile still writes
                            if (!mbar_wait_warp(pv_done(b ^ 1), ((count - 1) >> 1) & 1, abort_flag)) {
                                if (lane == 0) record_timeout(p, 310 + b);
                                ok = false;
                                break;
                            }
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 16) {
                                uint32_t o[16];
                                tmem_ld16(tmem_base + lanes + c, o);
                                tc_wait_ld();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st16(tmem_base + lanes + c, o);
                            }
                        }
                    }
                    const float base = m == -INFINITY ? 0.f : m;
                    if (!live)  // P = 0
#pragma unroll
                        for (int e = 0; e < kTok; ++e) x[e] = 0xff800000u;
                    uint64_t sum2 = 0, sum3 = 0;
                    const uint64_t nbase = pack2(-base, -base);
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float pa, pb;
                            uint64_t t2, p2;
                            asm("mov.b64 %0, {%1, %2};" : "=l"(t2) : "r"(x[32 * h + e]), "r"(x[32 * h + e + 1]));
                            asm("add.rn.f32x2 %0, %0, %1;" : "+l"(t2) : "l"(nbase));
                            asm("mov.b64 {%0, %1}, %2;" : "=f"(pa), "=f"(pb) : "l"(t2));
                            pa = ex2(pa);
                            pb = ex2(pb);
                            asm("mov.b64 %0, {%1, %2};" : "=l"(p2) : "f"(pa), "f"(pb));
                            if (e & 2) asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum3) : "l"(p2));
                            else asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sum2) : "l"(p2));
                            x[32 * h + e / 2] = pack_bf16(pa, pb);
                        }
                        tmem_st16(tmem_base + lanes + col_s(b) + 16 * h, x + 32 * h);
                    }
                    {
                        float s0, s1, s2f, s3;
                        asm("mov.b64 {%0, %1}, %2;" : "=f"(s0), "=f"(s1) : "l"(sum2));
                        asm("mov.b64 {%0, %1}, %2;" : "=f"(s2f), "=f"(s3) : "l"(sum3));
                        l += (s0 + s1) + (s2f + s3);
                    }
                    tc_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(b));
            }
            if (!ok) break;
            // ---- results, while the next segment's first scores are formed
            if (!mbar_wait_warp(pv_done((count - 1) & 1), ((count - 1) >> 1) & 1, abort_flag)) {
                if (lane == 0) record_timeout(p, 320);
                ok = false;
                break;
            }
            tc_fence_after();
            if (warp_live) {
                const bool whole = g.parts == 1, nothing = l == 0.f;
                const int64_t part = (int64_t)blockIdx.x * 2 + (j0 == 0 ? 1 : 0);
                const int64_t out = (int64_t)(g.s.first + node) * p.t.q_heads + g.kv_head * p.t.group + (live ? g.row0 + row - node * p.t.group : 0);
                const float keep = nothing ? 0.f : whole ? 1.0f / l : 1.f;
                const int poison = *reinterpret_cast<volatile uint8_t *>(&ctl.poison[k % kPoisonRing]);
                if (live) {
                    if (whole) p.t.lse[out] = nothing ? -INFINITY : (m + log2f(l)) * kLn2;
                    else p.part_ml[part * ROWS + row] = make_float2(m, l);
                }
                uint4 *to = reinterpret_cast<uint4 *>(static_cast<__nv_bfloat16 *>(p.t.o) + out * D);
                float4 *to_part = p.part_o + part * (D / 4) * ROWS + row;
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t raw[16];
                    float o[16];
                    tmem_ld16(tmem_base + lanes + c, raw);
                    tc_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[e] = nothing ? 0.f : __uint_as_float(raw[e]) * keep;
                    if (!live) continue;
                    if (poison) add_not_finite(p.t, g.s, g.seq, g.kv_head, node, j0 * kTok, (j0 + n) * kTok, c, o);
                    if (whole) {
                        to[c / 8] = make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]), pack_bf16(o[6], o[7]));
                        to[c / 8 + 1] = make_uint4(pack_bf16(o[8], o[9]), pack_bf16(o[10], o[11]), pack_bf16(o[12], o[13]), pack_bf16(o[14], o[15]));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) to_part[(c / 4 + e) * ROWS] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
            }
            tc_fence_before();  // the next segment's first value product starts the accumulator anew, behind this warp's next P
            if (g.parts > 1) {
                __syncwarp();
                if (lane == 0) {
                    __threadfence();
                    if (atomicInc(&p.arrived[g.cta], kSoftmaxWarps * g.parts - 1) == kSoftmaxWarps * g.parts - 1u) {  // the last one's CTA joins
                        __threadfence();
                        ctl.join[j0 > 0 && !(j0 + n < g.tiles) ? 0 : 1] = Join{g.s.first, g.kv_head, g.row0, rows, g.parts, g.cta};
                    }
                }
            }
        }
    } else if (warp < kQWarp + kQWarps) {
        // ================= planning; queries =================
        // A segment is planned once the queries of the one two before it are not needed any more.  By then its last scores have been
        // asked for, and with them the value products of the segment before: no warp has to do with anything before that one, which is three
        // before the planned one, and the ring holds four.
        // (The way along the span and what is planned next lie in shared memory: there is no room for them beside the queries.)
        const bool plans = warp == kQWarp;
        bool more = plans;  // the end is not planned yet
        auto plan = [&]() {
            Walk<ROWS> walk = ctl.walk;
            Segment coming;
            walk.next(p, coming);
            __syncwarp();
            if (lane == 0) {
                ctl.walk = walk;
                ctl.coming = coming;
            }
            __syncwarp();
        };
        auto publish = [&](int k) {
            more = ctl.coming.n > 0;
            __syncwarp();
            if (lane == 0) {
                ctl.seg[k % kSegRing] = ctl.coming;
                mbar_arrive(planned(k));
            }
            __syncwarp();
        };
        if (plans) {
#pragma unroll 1
            for (int k = 0; k < 2 && more; ++k) {
                plan();
                publish(k);
            }
        }
        const int tid = threadIdx.x - kQWarp * 32, quads = (p.t.group + 3) / 4;
        static_assert(kQWarps * 32 % (D / 8) == 0, "a thread's dims");
        const int c = tid % (D / 8);  // its 8 dims, of whatever token
        uint64_t turns[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) turns[e] = p.t.freq.turns[c * 4 + e];
        for (int k = 0;; ++k) {
            const Segment &g = segment(k);
            if (!ok || g.n == 0) break;
            const int node0 = g.row0 / p.t.group, nodes = (g.row0 + g.rows - 1) / p.t.group + 1 - node0, row0 = g.row0 - node0 * p.t.group, rows = g.rows;
            const int tasks = nodes * quads * (D / 8), head0 = g.kv_head * p.t.group, first = g.s.first + node0;
            // A thread takes 8 dims of up to four heads of a drafted token, whose angles are the same, kQSteps tokens' at a time: all
            // loads of 64 rows (of groups of four) are in flight while the last scores of the segment before are formed.
            uint4 raw[kQSteps][4];
            int position[kQSteps];
            auto request = [&](int i, uint4 (&x)[4], int &at) {
                if (i >= tasks) return;
                const int nq = i / (D / 8), node = quads == 1 ? nq : nq / quads, h = (nq - node * quads) * 4;
                at = p.t.positions[first + node];
                const char *from = static_cast<const char *>(p.t.q) + (((int64_t)(first + node) * p.t.q_heads + head0 + h) * D + c * 8) * 2;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (h + e < p.t.group && (unsigned)(node * p.t.group + h + e - row0) < (unsigned)rows) x[e] = *reinterpret_cast<const uint4 *>(from + e * D * 2);
            };
            const bool planning = k > 0 && more;
            if (planning) plan();
#pragma unroll
            for (int u = 0; u < kQSteps; ++u) request(tid + u * kQWarps * 32, raw[u], position[u]);
            if (k > 0) {
                if (!mbar_wait_warp(q_empty, (k - 1) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 330);
                    ok = false;
                    break;
                }
                if (planning) publish(k + 1);
            } else {
                // The ring's first filling is 24 MB of the whole device: the first queries would arrive behind it, 7000 clk later.
                uint32_t seen = 0;
                if (tid < tasks) asm volatile("mov.b32 %0, %1;" : "=r"(seen) : "r"(raw[0][0].x));
                __syncwarp();
                if (lane == 0) mbar_arrive(go);
            }
#pragma unroll 1
            for (int i = tid; i < tasks; i += kQWarps * 32) {
                const int nq = i / (D / 8), node = quads == 1 ? nq : nq / quads, h = (nq - node * quads) * 4;
                float2 cs[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    cs[e] = turn_of_fast(position[0], turns[e]);
                    cs[e].x *= p.t.scale * kLog2e;
                    cs[e].y *= p.t.scale * kLog2e;
                }
#pragma unroll 1
                for (int r = node * p.t.group + h - row0, e = h; e < min(h + 4, p.t.group); ++e, ++r) {
                    if ((unsigned)r < (unsigned)rows) write_query<C::kQTile>(raw[0][0], cs, q_s + (c >> 3) * C::kQBox + r * 128 + (((c & 7) ^ (r & 7)) << 4));
                    raw[0][0] = raw[0][1], raw[0][1] = raw[0][2], raw[0][2] = raw[0][3];  // registers move so that the loops stay loops
                }
#pragma unroll
                for (int u = 0; u + 1 < kQSteps; ++u) {
                    position[u] = position[u + 1];
#pragma unroll
                    for (int e = 0; e < 4; ++e) raw[u][e] = raw[u + 1][e];
                }
                request(i + kQSteps * kQWarps * 32, raw[kQSteps - 1], position[kQSteps - 1]);
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready);
        }
    } else if (warp == kKWarp || warp == kVWarp) {
        // ================= TMA producers: K tiles and V tiles =================
        const bool is_k = warp == kKWarp;
        const CUtensorMap *map = is_k ? &p.map_k : &p.map_v;
        const int boxes = kTok / p.box_rows, groups = p.box_rows / 8, page_groups = p.t.page_size / 8;
        const int no_group = p.t.physical_pages * page_groups;  // behind the pool: zeros
        uint32_t order = 0;  // tiles of the ring before the segment
        int count = 0;
        for (int k = 0;; ++k) {
            const Segment g = segment(k);
            if (!ok || g.n == 0) break;
            BoxRows rows;
            rows.start(p.t, g.seq, g.s.tokens, g.j0 * kTok, p.box_rows);
            if (k == 0 && !mbar_wait_warp(go, 0, abort_flag)) {
                if (lane == 0) record_timeout(p, 110);
                ok = false;
                break;
            }
            for (int i = 0; i < g.n; ++i, ++count) {
                const int first = (g.j0 + i) * boxes;
                rows.seek(first);
                const bool bad = rows.page == -1 || rows.page >= p.t.physical_pages;
                const int group = rows.page < 0 || bad ? no_group : rows.page * page_groups + (rows.in_page >> 3);
                if (is_k) {
                    uint32_t valid = 0xf;
                    const uint32_t all = __ballot_sync(0xffffffffu, bad) >> (first - rows.base);
                    if (all) {
                        for (int e = 0; e < 4; ++e)
                            if ((all >> (e * 16 / p.box_rows)) & 1 && e * 16 / p.box_rows < boxes) valid &= ~(1u << e);
                        if (lane == 0 && valid != 0xf) report_status(p.t.status, FLAT_ERR_PAGE_OUT_OF_RANGE, g.seq);
                    }
                    if (lane == 0) ctl.valid[count % kValidRing] = (uint8_t)valid;
                }
                const uint32_t at = order + (is_k ? k_entry(i, kAhead) : v_entry(i, g.n, kAhead));
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
            if (!ok) break;
            order += 2 * g.n;
        }
    } else if (warp == kMmaWarp) {
        // ================= all products =================
        if (elect_one()) {
            const uint32_t q_desc = (uint32_t)make_smem_desc(smem_u32(q_s), 0, 1024);
            const uint32_t k_desc = (uint32_t)make_smem_desc(smem_u32(kv_s), 0, C::kGroup);
            const uint32_t v_desc = (uint32_t)make_smem_desc(smem_u32(kv_s), 1024, C::kGroup);
            constexpr uint32_t kTile16 = C::kKvTile >> 4;
            uint32_t order = 0, fixed_phase = 0;
            int done = 0;  // tiles of the segments before
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
            auto scores = [&](int i, int n) {
                const int b = (done + i) & 1, s = landed(k_entry(i, kAhead));
                if (!ok) return;
                tc_fence_after();
                const uint32_t kk = k_desc + s * kTile16, d = tmem_base + col_s(b);
#pragma unroll
                for (int h = 0; h < 2; ++h)  // the two summands of q
#pragma unroll
                    for (int e = 0; e < D / 16; ++e)
                        mma_scores<C::kGroup>(d, q_desc + h * (C::kQTile >> 4) + (e >> 2) * (C::kQBox >> 4) + (e & 3) * 2,
                                              kk + (e >> 2) * (1024 >> 4) + (e & 3) * 2, p.idesc_qk, h > 0 || e > 0);
                tc_commit(s_full(b));
                tc_commit(empty(s));
                if (i + 1 == n) tc_commit(q_empty);
            };
            auto values = [&](int v, const Segment &g) {
                const int b = (done + v) & 1, s = landed(v_entry(v, g.n, kAhead));
                if (is_tail(g, g.j0 + v)) {
                    wait(fixed(s), (fixed_phase >> s) & 1, 230);
                    fixed_phase ^= 1u << s;
                }
                wait(p_full(b), ((done + v) >> 1) & 1, 240 + b);
                if (!ok) return;
                tc_fence_after();
#pragma unroll
                for (int e = 0; e < kTok / 16; ++e)
                    mma_values<C::kGroup>(tmem_base, tmem_base + col_s(b) + e * 8, v_desc + s * kTile16 + e * (2 * C::kGroup >> 4), p.idesc_pv, v > 0 || e > 0);
                tc_commit(pv_done(b));
                tc_commit(empty(s));
            };
            for (int k = 0;; ++k) {
                wait(planned(k), (k / kSegRing) & 1, 506);
                if (!ok) break;
                const Segment g = ctl.seg[k % kSegRing];
                if (g.n == 0) break;
                wait(q_ready, k & 1, 200);
#pragma unroll 1
                for (int i = 0; ok && i < g.n + kAhead; ++i) {
                    if (i >= kAhead) values(i - kAhead, g);
                    if (i < g.n) scores(i, g.n);
                }
                if (!ok) break;
                done += g.n;
                order += 2 * g.n;
            }
        }
    } else {
        // ================= V tiles with drafted tokens or the end of a sequence =================
        uint32_t order = 0, phase = 0;
        for (int k = 0;; ++k) {
            const Segment g = segment(k);
            if (!ok || g.n == 0) break;
            if (lane == 0) ctl.poison[k % kPoisonRing] = 0;
            __syncwarp();
            // (to_fix tells that the tile before in this stage is used up, without which its phase could be taken for this one's)
            for (int v = max(0, min(g.s.len / kTok, g.tiles - 1) - g.j0); v < g.n; ++v) {
                const uint32_t at = order + v_entry(v, g.n, kAhead);
                const int s = at % C::kStages;
                if (!mbar_wait_warp(to_fix(s), (phase >> s) & 1, abort_flag) || !mbar_wait_warp(full(s), (at / C::kStages) & 1, abort_flag)) {
                    if (lane == 0) record_timeout(p, 400);
                    ok = false;
                    break;
                }
                phase ^= 1u << s;
                const int t0 = (g.j0 + v) * kTok;
                const bool met = clear_values<C::kBoxes, kTok>(kv_s + s * C::kKvTile, max(0, min(g.s.len, g.s.tokens) - t0), g.s.tokens - t0);
                if (__any_sync(0xffffffffu, met) && lane == 0) ctl.poison[k % kPoisonRing] = 1;
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(fixed(s));
            }
            if (!ok) break;
            order += 2 * g.n;
        }
    }

    if (*abort_flag) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);  // let copies in flight land before the CTA exits
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem_base, 512 / kCtasPerSm);
    }
#pragma unroll 1
    for (int i = 0; i < 2; ++i)
        if (ctl.join[i].parts) join_parts<D, ROWS>(p, ctl.join[i]);
}

template <int D, int ROWS> int launch(flat_ctx *ctx, const TreeParams &t) {
    using C = Cfg<D, ROWS>;
    KernelParams p{};
    p.t = t;
    p.share = (int64_t)t.max_nodes * t.group > ROWS ? 2 : 1;
    const int64_t blocks = ((int64_t)t.max_nodes * t.group + ROWS - 1) / ROWS;
    p.items = (int)((blocks * t.kv_heads + p.share - 1) / p.share * t.num_seqs);
    p.box_rows = t.page_size % 64 == 0 ? 64 : t.page_size % 32 == 0 ? 32 : 16;
    const uint64_t rows = (uint64_t)t.physical_pages * t.page_size;
    if (int st = make_pool_map(ctx, &p.map_k, t.k, D, rows, t.kv_heads, p.box_rows)) return st;
    if (int st = make_pool_map(ctx, &p.map_v, t.v, D, rows, t.kv_heads, p.box_rows)) return st;
    p.idesc_qk = make_idesc(kFmtBF16, kFmtBF16, 0, 0, ROWS, kTok);
    p.idesc_pv = make_idesc(kFmtBF16, kFmtBF16, 0, 1, ROWS, D);
    const int grid = ctx->sm_count * kCtasPerSm;
    static_assert(kCtasPerSm == 2, "the grid has to be even");
    char *at = static_cast<char *>(ctx->paged_scratch) + kPagedPlanBytes;
    const uint64_t rows_held = (uint64_t)grid * 2 * ROWS;
    const uint64_t o_bytes = rows_held * D * sizeof(float), ml_bytes = rows_held * sizeof(float2);
    if (o_bytes + ml_bytes > kPagedScratchBytes - kPagedPlanBytes || (uint64_t)grid > kPagedTickets)
        return fail(ctx, FLAT_ERR_EXECUTION, "the scratch does not hold the parts of %d CTAs", grid);
    p.part_o = reinterpret_cast<float4 *>(at);
    p.part_ml = reinterpret_cast<float2 *>(at + o_bytes);
    p.arrived = paged_tickets(ctx) + 1;
    FLAT_CUDA_OK(ctx, cudaFuncSetAttribute(tree_sm100_kernel<D, ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem));
    {
        KernelTimer timer(ctx);
        FLAT_CUDA_OK(ctx, launch_dependent(may_overlap_previous(ctx), tree_sm100_kernel<D, ROWS>, dim3((unsigned)grid), kThreads, C::kSmem, ctx->stream, p));
    }
    ctx->launches += 1;
    return FLAT_OK;
}

}  // namespace

bool tree_sm100_supported(int dtype, const TreeParams &p) {
    // the line's length is a 32-bit number
    const int64_t blocks = ((int64_t)p.max_nodes * p.group + 63) / 64, tiles = (std::min<int64_t>(p.max_context, (int64_t)p.max_pages * p.page_size) + kTok - 1) / kTok;
    return dtype == FLAT_BF16 && (p.head_dim == 64 || p.head_dim == 128) && p.page_size % 16 == 0 &&
           ((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v | (uintptr_t)p.o) % 16 == 0 && blocks * p.kv_heads * p.num_seqs < (1ll << 30) / tiles;
}

int launch_tree_sm100(flat_ctx *ctx, const TreeParams &p) {
    const bool few = (int64_t)p.max_nodes * p.group <= 64;
    if (p.head_dim == 128) return few ? launch<128, 64>(ctx, p) : launch<128, 128>(ctx, p);
    return few ? launch<64, 64>(ctx, p) : launch<64, 128>(ctx, p);
}

}  // namespace flat
