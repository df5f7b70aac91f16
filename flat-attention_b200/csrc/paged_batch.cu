// Page tables of a batch of sequences kept on the device: taking pages for new tokens with the slot of each (reserve), and giving
// pages back (release).  Nothing of it passes the host, so a step of a serving loop can be captured and replayed.
//
// Both are prefix sums over the sequences followed by a fill over tokens (pages):
//   need[s] = max(0, ceil((L + N) / page) - H),  e = exclusive sum of need;  page H + i of s is free[f - 1 - (e + i)]
//   gone[s] = H - min(H, ceil(keep / page)),     e = exclusive sum of gone;  free[f + e + i] is page H - 1 - i of s
// which makes the result a fixed function of the inputs, in sequence order, with no atomics on them.  The sums are held in 64 bits:
// lengths are whatever the device arrays say.  There is hardly anything to read or write, so the time is launches and chains of
// dependent loads.  Up to kBlockSeqs sequences every block makes the sums for itself, in shared memory, and fills its share of the
// tokens (pages): one launch and no second look at the arrays.  Inputs may be outputs (counts in place), so outputs per sequence are
// written by the block that finds that all others have read theirs.  More sequences are a scanning block and a fill of its own.
#include "common.h"

namespace flat {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kSegment = 256;  // tokens or pages that a warp of the large fill takes at a time
constexpr int kItems = 4;      // sequences of a thread where every block scans for itself; tokens (pages) of a thread in flight
constexpr int kBlockSeqs = kItems * kScanThreads;

// Inclusive sum over the block; `total` receives the block's sum.
__device__ __forceinline__ int64_t block_scan(int64_t x, int64_t *warp_sums, int64_t &total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int64_t y = warp_sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t z = __shfl_up_sync(0xffffffffu, y, d);
            if (lane >= d) y += z;
        }
        warp_sums[lane] = y;
    }
    __syncthreads();
    total = warp_sums[kScanThreads / 32 - 1];
    if (warp > 0) x += warp_sums[warp - 1];
    __syncthreads();  // the next scan writes warp_sums
    return x;
}

// The same for two numbers at once, once per kernel: each has sums of its own.
__device__ __forceinline__ void block_scan2(int64_t &x, int64_t &y, int64_t &total_x, int64_t &total_y) {
    __shared__ longlong2 sums[kScanThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto scan = [&](int64_t &a, int64_t &b) {
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t c = __shfl_up_sync(0xffffffffu, a, d), e = __shfl_up_sync(0xffffffffu, b, d);
            if (lane >= d) a += c, b += e;
        }
    };
    scan(x, y);
    if (lane == 31) sums[warp] = make_longlong2(x, y);
    __syncthreads();
    int64_t a = sums[lane].x, b = sums[lane].y;  // every warp for itself
    scan(a, b);
    const int64_t before_x = __shfl_sync(0xffffffffu, a, max(warp, 1) - 1), before_y = __shfl_sync(0xffffffffu, b, max(warp, 1) - 1);
    if (warp > 0) x += before_x, y += before_y;
    total_x = __shfl_sync(0xffffffffu, a, 31);
    total_y = __shfl_sync(0xffffffffu, b, 31);
}

// The sequence that entry i of a packed list belongs to: the last one that starts at or before i.
__device__ __forceinline__ int sequence_of(const int32_t *offsets, int num_seqs, int i) {
    int lo = 0, hi = num_seqs;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (offsets[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int clamped_free_count(const PagedBatchParams &p) {
    return min(max(*p.free_count, 0), p.physical_pages);
}

// Pages of n tokens, 0 <= n < 2^31: in 32 bits, a 64-bit division is some hundred instructions.
__device__ __forceinline__ int pages_of(const PagedBatchParams &p, int64_t n) {
    return (int)(((unsigned)n + (unsigned)p.page_size - 1) / (unsigned)p.page_size);
}

// Tokens that a row of the table holds; lengths are 32-bit numbers.
__device__ __forceinline__ int64_t most_tokens(const PagedBatchParams &p) {
    return min((int64_t)p.max_pages * p.page_size, (int64_t)0x7fffffff);
}

__device__ __forceinline__ void reserve_scan(const PagedBatchParams &p) {
    __shared__ int64_t warp_sums[kScanThreads / 32];
    const int f = clamped_free_count(p);
    if (threadIdx.x == 0 && f != *p.free_count) report_status(p.status, FLAT_ERR_CAPACITY_OVERFLOW, -1);
    int64_t tokens = 0, pages = 0;  // of the sequences before this pass
    int64_t taken = 0;              // pages that are really given out
    const int64_t most = most_tokens(p);
    for (int base = 0; base < p.num_seqs; base += kScanThreads) {
        const int s = base + threadIdx.x;
        const bool on = s < p.num_seqs;
        const int64_t L = on ? p.context_lens[s] : 0, asked = on ? p.lens[s] : 0, H = on ? p.page_counts[s] : 0;
        const int64_t N = asked > 0 ? asked : 0;
        int64_t sum;
        const int64_t upto = tokens + block_scan(N, warp_sums, sum);
        tokens += sum;
        const bool valid = on && L >= 0 && asked >= 0 && H <= p.max_pages && L <= H * p.page_size &&
                           L + N <= most && upto <= p.max_tokens;
        const int64_t want = valid ? pages_of(p, L + N) : 0;
        const int64_t need = want > H ? want - H : 0;
        const int64_t got = pages + block_scan(need, warp_sums, sum);
        pages += sum;
        const bool granted = valid && (need == 0 || got <= f);
        block_scan(granted ? need : 0, warp_sums, sum);
        taken += sum;
        if (on) {
            p.plan[s] = make_int4((int)L, (int)H, granted ? (int)(got - need) : 0, granted ? 1 : 0);
            p.offsets[s] = (int)min(upto - N, (int64_t)p.max_tokens);
            p.page_counts_out[s] = (int)(granted ? H + need : H);
            if (p.context_lens_out) p.context_lens_out[s] = (int)(granted ? L + N : L);
            if (!granted) report_status(p.status, valid ? FLAT_ERR_CAPACITY_EXCEEDED : FLAT_ERR_INVALID_CACHE_LENGTH, s);
        }
    }
    if (threadIdx.x == 0) {
        p.offsets[p.num_seqs] = (int)min(tokens, (int64_t)p.max_tokens);
        *p.plan_free_count = f;
        *p.free_count_out = f - (int)taken;
    }
}

// Slot and position of token i, and the table entry of the page that it is the first token of.  (A new page's first token is
// always a new token: the pages held cover all live ones.)
struct NewToken {
    int seq, page, in_page, position;
    int64_t entry;  // to write, < 0: none
};
__device__ __forceinline__ NewToken reserve_look(const PagedBatchParams &p, const int32_t *starts, const int4 *plans, int s, int i, int total, int f) {
    NewToken x{-1, -1, 0, 0, -1};
    if (i >= total) return x;
    const int4 plan = plans[s];
    if (!plan.w) return x;
    const int j = i - starts[s], t = plan.x + j;
    const int logical = t / p.page_size;
    const bool fresh = logical >= plan.y;
    const int64_t entry = (int64_t)s * p.max_pages + logical;
    x.seq = s;
    x.in_page = t - logical * p.page_size;
    x.page = fresh ? p.free_pages[f - 1 - (plan.z + logical - plan.y)] : p.page_tables[entry];
    x.position = plan.x + (p.depths ? p.depths[i] : j);
    if (fresh && x.in_page == 0) x.entry = entry;
    return x;
}
__device__ __forceinline__ int reserve_enter(const PagedBatchParams &p, NewToken x) {  // the token's slot
    if (x.seq >= 0 && (unsigned)x.page >= (unsigned)p.physical_pages) {
        report_status(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, x.seq, kPlacePages);
        x.page = -1;
    }
    if (x.entry >= 0) p.page_tables[x.entry] = x.page;
    return x.page >= 0 ? x.page * p.page_size + x.in_page : -1;
}

__device__ __forceinline__ void release_scan(const PagedBatchParams &p) {
    __shared__ int64_t warp_sums[kScanThreads / 32];
    const int f = clamped_free_count(p);
    if (threadIdx.x == 0 && f != *p.free_count) report_status(p.status, FLAT_ERR_CAPACITY_OVERFLOW, -1);
    const int64_t room = p.physical_pages - f;
    int64_t pages = 0;
    for (int base = 0; base < p.num_seqs; base += kScanThreads) {
        const int s = base + threadIdx.x;
        const bool on = s < p.num_seqs;
        const int64_t keep = on ? p.lens[s] : 0, H = on ? p.page_counts[s] : 0;
        const bool valid = on && H >= 0 && H <= p.max_pages && keep >= 0;
        const int64_t left = valid ? min(H, (int64_t)pages_of(p, keep)) : H;
        const int64_t gone = H - left;
        int64_t sum;
        const int64_t upto = pages + block_scan(gone, warp_sums, sum);
        pages += sum;
        if (on) {
            p.plan[s] = make_int4(0, (int)H, (int)left, 0);
            p.plan_offsets[s] = (int)min(upto - gone, room);
            p.page_counts_out[s] = (int)left;
            if (!valid) report_status(p.status, FLAT_ERR_INVALID_CACHE_LENGTH, s);
            else if (upto > room) report_status(p.status, FLAT_ERR_CAPACITY_OVERFLOW, s);
        }
    }
    if (threadIdx.x == 0) {
        p.plan_offsets[p.num_seqs] = (int)min(pages, room);
        *p.plan_free_count = f;
        *p.free_count_out = f + (int)min(pages, room);
    }
}

__device__ __forceinline__ void release_page(const PagedBatchParams &p, int i, int f) {
    const int s = sequence_of(p.plan_offsets, p.num_seqs, i);
    const int page = p.page_tables[(int64_t)s * p.max_pages + p.plan[s].y - 1 - (i - p.plan_offsets[s])];
    if ((unsigned)page >= (unsigned)p.physical_pages) report_status(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, s, kPlacePages);
    p.free_pages[f + i] = page;
}

template <bool RELEASE> __device__ __forceinline__ void fill(const PagedBatchParams &p, int first, int stride_warps, int segment) {
    const int lane = threadIdx.x & 31;
    const int f = *p.plan_free_count;
    const int total = RELEASE ? p.plan_offsets[p.num_seqs] : p.offsets[p.num_seqs];
    const int64_t end = RELEASE ? total : p.max_tokens;  // slots behind the last token are -1
    for (int64_t at = (int64_t)first * segment; at < end; at += (int64_t)stride_warps * segment)
        for (int64_t i = at + lane; i < min(at + segment, end); i += 32) {
            if (RELEASE) {
                release_page(p, (int)i, f);
            } else {
                const NewToken x = reserve_look(p, p.offsets, p.plan, sequence_of(p.offsets, p.num_seqs, (int)i), (int)i, total, f);
                p.slots[i] = reserve_enter(p, x);
                p.positions[i] = x.position;
            }
        }
}

// Scan and fill in one launch, for num_seqs <= kBlockSeqs.  Shared memory: a plan per sequence (as the scratch's, release without
// the unused fields' meaning) and where its tokens (pages) start.
template <bool RELEASE> __global__ void __launch_bounds__(kScanThreads) paged_batch_kernel(const __grid_constant__ PagedBatchParams p) {
    extern __shared__ int4 plan_s[];
    int32_t *starts_s = reinterpret_cast<int32_t *>(plan_s + p.num_seqs);
    __shared__ int last_s, taken_s;  // taken: pages that are given out
    if (threadIdx.x == 0) taken_s = 0;  // before the scan's barrier
    grid_dependency_wait();
    grid_dependency_launch();
    const int items = (p.num_seqs + kScanThreads - 1) / kScanThreads, s0 = threadIdx.x * items;
    const int given = *p.free_count, f = min(max(given, 0), p.physical_pages);
    int L[kItems], A[kItems], H[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
        const int s = s0 + i;
        const bool on = i < items && s < p.num_seqs;
        L[i] = on && !RELEASE ? p.context_lens[s] : 0;
        A[i] = on ? p.lens[s] : 0;
        H[i] = on ? p.page_counts[s] : 0;
    }
    int held[kItems], flags[kItems];  // pages afterwards; what to report
    int64_t total;                    // tokens (pages that go)
    if (RELEASE) {
        const int64_t room = p.physical_pages - f;
        int64_t gone = 0;
        int left[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            if (i >= items) break;
            const bool valid = H[i] >= 0 && H[i] <= p.max_pages && A[i] >= 0;
            left[i] = valid ? min(H[i], pages_of(p, A[i])) : H[i];
            flags[i] = valid ? FLAT_OK : FLAT_ERR_INVALID_CACHE_LENGTH;
            gone += H[i] - left[i];
        }
        int64_t upto = gone, none = 0, no_total;
        block_scan2(upto, none, total, no_total);
        upto -= gone;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int s = s0 + i;
            if (i >= items || s >= p.num_seqs) break;
            held[i] = left[i];
            plan_s[s] = make_int4(0, H[i], left[i], 0);
            starts_s[s] = (int)min(upto, room);
            upto += H[i] - left[i];
            if (flags[i] == FLAT_OK && upto > room) flags[i] = FLAT_ERR_CAPACITY_OVERFLOW;
        }
        total = min(total, room);
    } else {
        // Both sums at once: whether the tokens so far pass max_tokens does not enter the pages' sum, since all sequences behind the
        // first for which they do are refused anyway.
        const int64_t most = most_tokens(p);
        int64_t tokens = 0, needs = 0;
        int need[kItems];
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            if (i >= items) break;
            const int64_t N = max(A[i], 0);
            const bool valid = L[i] >= 0 && A[i] >= 0 && H[i] <= p.max_pages && L[i] <= (int64_t)H[i] * p.page_size && L[i] + N <= most;
            need[i] = valid ? max(pages_of(p, L[i] + N) - H[i], 0) : 0;
            flags[i] = valid ? FLAT_OK : FLAT_ERR_INVALID_CACHE_LENGTH;
            tokens += N;
            needs += need[i];
        }
        int64_t upto = tokens, before = needs, sum;
        block_scan2(upto, before, total, sum);
        upto -= tokens;
        before -= needs;
        int given_out = 0;
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int s = s0 + i;
            if (i >= items) break;
            if (s < p.num_seqs) starts_s[s] = (int)min(upto, (int64_t)p.max_tokens);
            upto += max(A[i], 0);
            if (upto > p.max_tokens) flags[i] = FLAT_ERR_INVALID_CACHE_LENGTH;
            if (flags[i] == FLAT_OK && need[i] > 0 && before + need[i] > f) flags[i] = FLAT_ERR_CAPACITY_EXCEEDED;
            const bool granted = flags[i] == FLAT_OK;
            if (s < p.num_seqs) plan_s[s] = make_int4(L[i], H[i], granted ? (int)before : 0, granted ? 1 : 0);
            before += need[i];
            held[i] = granted ? H[i] + need[i] : H[i];
            given_out += granted ? need[i] : 0;
        }
        given_out = __reduce_add_sync(0xffffffffu, given_out);  // f at most
        if ((threadIdx.x & 31) == 0 && given_out) atomicAdd(&taken_s, given_out);
        total = min(total, (int64_t)p.max_tokens);
    }
    if (threadIdx.x == 0) starts_s[p.num_seqs] = (int)total;
    __syncthreads();
    // All reads of what may be written in place are done: the block's scan has used them.  The answer comes during the fill.
    if (threadIdx.x == 0) {
        if (gridDim.x == 1) {
            last_s = 1;
        } else {
            __threadfence();
            last_s = atomicInc(p.plan_ticket, gridDim.x - 1) == gridDim.x - 1;
            __threadfence();
        }
    }
    // kItems tokens (pages) in a row for a thread: they mostly are the same sequence's, whose start is found once
    const int end = RELEASE ? (int)total : p.max_tokens;  // slots behind the last token are -1
    const bool vectors = !RELEASE && ((uintptr_t)p.slots | (uintptr_t)p.positions) % 16 == 0;
    for (int64_t at = ((int64_t)blockIdx.x * kScanThreads + threadIdx.x) * kItems; at < end; at += (int64_t)gridDim.x * kBlockSeqs) {
        const int i0 = (int)at, n = min(kItems, end - i0);
        int s = sequence_of(starts_s, p.num_seqs, i0);
        if (RELEASE) {
            int page[kItems], seq[kItems];
#pragma unroll
            for (int u = 0; u < kItems; ++u) {
                if (u >= n) break;
                if (u > 0 && starts_s[s + 1] <= i0 + u) s = sequence_of(starts_s, p.num_seqs, i0 + u);
                seq[u] = s;
                page[u] = p.page_tables[(int64_t)s * p.max_pages + plan_s[s].y - 1 - (i0 + u - starts_s[s])];
            }
#pragma unroll
            for (int u = 0; u < kItems; ++u) {
                if (u >= n) break;
                if ((unsigned)page[u] >= (unsigned)p.physical_pages) report_status(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, seq[u], kPlacePages);
                p.free_pages[f + i0 + u] = page[u];
            }
        } else {
            NewToken x[kItems];
#pragma unroll
            for (int u = 0; u < kItems; ++u) {
                if (u >= n) break;
                if (u > 0 && i0 + u < total && starts_s[s + 1] <= i0 + u) s = sequence_of(starts_s, p.num_seqs, i0 + u);
                x[u] = reserve_look(p, starts_s, plan_s, s, i0 + u, (int)total, f);
            }
            if (vectors && n == kItems) {
                int slot[kItems];
#pragma unroll
                for (int u = 0; u < kItems; ++u) slot[u] = reserve_enter(p, x[u]);
                *reinterpret_cast<int4 *>(p.slots + i0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
                *reinterpret_cast<int4 *>(p.positions + i0) = make_int4(x[0].position, x[1].position, x[2].position, x[3].position);
            } else {
#pragma unroll
                for (int u = 0; u < kItems; ++u) {
                    if (u >= n) break;
                    p.slots[i0 + u] = reserve_enter(p, x[u]);
                    p.positions[i0 + u] = x[u].position;
                }
            }
        }
    }
    __syncthreads();
    if (last_s) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int s = s0 + i;
            if (i >= items || s >= p.num_seqs) break;
            p.page_counts_out[s] = held[i];
            if (!RELEASE) {
                p.offsets[s] = starts_s[s];
                if (p.context_lens_out) p.context_lens_out[s] = flags[i] == FLAT_OK ? L[i] + A[i] : L[i];
            }
            if (flags[i] != FLAT_OK) report_status(p.status, flags[i], s);
        }
        if (threadIdx.x == 0) {
            if (!RELEASE) p.offsets[p.num_seqs] = (int)total;
            *p.free_count_out = RELEASE ? f + (int)total : f - taken_s;
            if (f != given) report_status(p.status, FLAT_ERR_CAPACITY_OVERFLOW, -1);
        }
    }
}

template <bool RELEASE> __global__ void __launch_bounds__(kScanThreads) paged_batch_scan_kernel(const __grid_constant__ PagedBatchParams p) {
    grid_dependency_wait();
    grid_dependency_launch();
    if (RELEASE) release_scan(p);
    else reserve_scan(p);
}

template <bool RELEASE> __global__ void __launch_bounds__(256) paged_batch_fill_kernel(const __grid_constant__ PagedBatchParams p) {
    grid_dependency_wait();
    grid_dependency_launch();
    fill<RELEASE>(p, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8, kSegment);
}

}  // namespace

int launch_paged_batch(flat_ctx *ctx, PagedBatchParams &p, bool release) {
    // what the fill goes over, at most; the host does not know how much of it there is
    const int64_t entries = release ? std::min<int64_t>((int64_t)p.num_seqs * p.max_pages, p.physical_pages) : p.max_tokens;
    const bool overlap = may_overlap_previous(ctx);
    if (p.num_seqs <= kBlockSeqs) {
        auto *kernel = release ? paged_batch_kernel<true> : paged_batch_kernel<false>;
        const size_t smem = (size_t)p.num_seqs * (sizeof(int4) + sizeof(int32_t)) + sizeof(int32_t);
        if (smem > 40 << 10) FLAT_CUDA_OK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 << 10));
        const int64_t blocks = std::min<int64_t>((entries + kBlockSeqs - 1) / kBlockSeqs, ctx->sm_count);
        FLAT_CUDA_OK(ctx, launch_dependent(overlap, kernel, dim3((unsigned)blocks), kScanThreads, smem, ctx->stream, p));
        ctx->launches += 1;
        return FLAT_OK;
    }
    auto *scan = release ? paged_batch_scan_kernel<true> : paged_batch_scan_kernel<false>;
    FLAT_CUDA_OK(ctx, launch_dependent(overlap, scan, dim3(1), kScanThreads, 0, ctx->stream, p));
    ctx->launches += 1;
    const int64_t blocks = std::min<int64_t>((entries + 8 * kSegment - 1) / (8 * kSegment), (int64_t)ctx->sm_count * 4);
    auto *filler = release ? paged_batch_fill_kernel<true> : paged_batch_fill_kernel<false>;
    FLAT_CUDA_OK(ctx, launch_dependent(true, filler, dim3((unsigned)blocks), 256, 0, ctx->stream, p));
    ctx->launches += 1;
    return FLAT_OK;
}

}  // namespace flat
