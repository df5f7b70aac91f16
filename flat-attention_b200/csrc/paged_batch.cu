// Page tables of a batch of sequences kept on the device: taking pages for new tokens with the slot of each (reserve), and giving
// pages back (release).  Nothing of it passes the host, so a step of a serving loop can be captured and replayed.
//
// Both are prefix sums over the sequences followed by a fill over tokens (pages):
//   need[s] = max(0, ceil((L + N) / page) - H),  e = exclusive sum of need;  page H + i of s is free[f - 1 - (e + i)]
//   gone[s] = H - min(H, ceil(keep / page)),     e = exclusive sum of gone;  free[f + e + i] is page H - 1 - i of s
// which makes the result a fixed function of the inputs, in sequence order, with no atomics.  The sums are held in 64 bits: lengths
// are whatever the device arrays say.  There is hardly anything to read or write, so the time is launches and chains of dependent
// loads: a small call is one block (scan, barrier, fill), a large one a scanning block and a fill over the whole device.
#include "common.h"

namespace flat {
namespace {

constexpr int kScanThreads = 1024;
constexpr int kSegment = 256;  // tokens or pages that a warp of the large fill takes at a time

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

__device__ __forceinline__ void flag(DeviceStatus *status, int code, int where) {
    status->code = code;
    status->where = where;
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

__device__ __forceinline__ void reserve_scan(const PagedBatchParams &p) {
    __shared__ int64_t warp_sums[kScanThreads / 32];
    const int f = clamped_free_count(p);
    if (threadIdx.x == 0 && f != *p.free_count) flag(p.status, FLAT_ERR_CAPACITY_OVERFLOW, -1);
    int64_t tokens = 0, pages = 0;  // of the sequences before this pass
    int64_t taken = 0;              // pages that are really given out
    for (int base = 0; base < p.num_seqs; base += kScanThreads) {
        const int s = base + threadIdx.x;
        const bool on = s < p.num_seqs;
        const int64_t L = on ? p.context_lens[s] : 0, asked = on ? p.lens[s] : 0, H = on ? p.page_counts[s] : 0;
        const int64_t N = asked > 0 ? asked : 0;
        int64_t sum;
        const int64_t upto = tokens + block_scan(N, warp_sums, sum);
        tokens += sum;
        const bool valid = on && L >= 0 && asked >= 0 && H <= p.max_pages && L <= H * p.page_size &&
                           L + N <= (int64_t)p.max_pages * p.page_size && upto <= p.max_tokens;
        const int64_t want = valid ? (L + N + p.page_size - 1) / p.page_size : 0;
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
            if (!granted) flag(p.status, valid ? FLAT_ERR_CAPACITY_EXCEEDED : FLAT_ERR_INVALID_CACHE_LENGTH, s);
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
__device__ __forceinline__ void reserve_token(const PagedBatchParams &p, int i, int total, int f) {
    int slot = -1, position = 0;
    if (i < total) {
        const int s = sequence_of(p.offsets, p.num_seqs, i);
        const int4 plan = p.plan[s];
        if (plan.w) {
            const int j = i - p.offsets[s], t = plan.x + j;
            const int logical = t / p.page_size, in_page = t - logical * p.page_size;
            const bool fresh = logical >= plan.y;
            const int64_t entry = (int64_t)s * p.max_pages + logical;
            int page = fresh ? p.free_pages[f - 1 - (plan.z + logical - plan.y)] : p.page_tables[entry];
            if ((unsigned)page >= (unsigned)p.physical_pages) {
                flag(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, s);
                page = -1;
            }
            if (fresh && in_page == 0) p.page_tables[entry] = page;
            if (page >= 0) slot = page * p.page_size + in_page;
            position = plan.x + (p.depths ? p.depths[i] : j);
        }
    }
    p.slots[i] = slot;
    p.positions[i] = position;
}

__device__ __forceinline__ void release_scan(const PagedBatchParams &p) {
    __shared__ int64_t warp_sums[kScanThreads / 32];
    const int f = clamped_free_count(p);
    if (threadIdx.x == 0 && f != *p.free_count) flag(p.status, FLAT_ERR_CAPACITY_OVERFLOW, -1);
    const int64_t room = p.physical_pages - f;
    int64_t pages = 0;
    for (int base = 0; base < p.num_seqs; base += kScanThreads) {
        const int s = base + threadIdx.x;
        const bool on = s < p.num_seqs;
        const int64_t keep = on ? p.lens[s] : 0, H = on ? p.page_counts[s] : 0;
        const bool valid = on && H >= 0 && H <= p.max_pages && keep >= 0;
        const int64_t left = valid ? min(H, (keep + p.page_size - 1) / p.page_size) : H;
        const int64_t gone = H - left;
        int64_t sum;
        const int64_t upto = pages + block_scan(gone, warp_sums, sum);
        pages += sum;
        if (on) {
            p.plan[s] = make_int4(0, (int)H, (int)left, 0);
            p.plan_offsets[s] = (int)min(upto - gone, room);
            p.page_counts_out[s] = (int)left;
            if (!valid) flag(p.status, FLAT_ERR_INVALID_CACHE_LENGTH, s);
            else if (upto > room) flag(p.status, FLAT_ERR_CAPACITY_OVERFLOW, s);
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
    if ((unsigned)page >= (unsigned)p.physical_pages) flag(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, s);
    p.free_pages[f + i] = page;
}

template <bool RELEASE> __device__ __forceinline__ void fill(const PagedBatchParams &p, int first, int stride_warps, int segment) {
    const int lane = threadIdx.x & 31;
    const int f = *p.plan_free_count;
    const int total = RELEASE ? p.plan_offsets[p.num_seqs] : p.offsets[p.num_seqs];
    const int64_t end = RELEASE ? total : p.max_tokens;  // slots behind the last token are -1
    for (int64_t at = (int64_t)first * segment; at < end; at += (int64_t)stride_warps * segment)
        for (int64_t i = at + lane; i < min(at + segment, end); i += 32) {
            if (RELEASE) release_page(p, (int)i, f);
            else reserve_token(p, (int)i, total, f);
        }
}

template <bool RELEASE> __global__ void __launch_bounds__(kScanThreads) paged_batch_kernel(const __grid_constant__ PagedBatchParams p) {
    grid_dependency_wait();
    grid_dependency_launch();
    if (RELEASE) release_scan(p);
    else reserve_scan(p);
    if (!p.fused) return;
    __syncthreads();
    fill<RELEASE>(p, threadIdx.x >> 5, kScanThreads / 32, 32);
}

template <bool RELEASE> __global__ void __launch_bounds__(256) paged_batch_fill_kernel(const __grid_constant__ PagedBatchParams p) {
    grid_dependency_wait();
    grid_dependency_launch();
    fill<RELEASE>(p, blockIdx.x * 8 + (threadIdx.x >> 5), gridDim.x * 8, kSegment);
}

}  // namespace

int launch_paged_batch(flat_ctx *ctx, PagedBatchParams &p, bool release) {
    // what the fill goes over, at most; the host does not know how much of it there is
    const int64_t entries = release ? (int64_t)p.num_seqs * p.max_pages : p.max_tokens;
    p.fused = entries <= 8192 ? 1 : 0;
    auto *kernel = release ? paged_batch_kernel<true> : paged_batch_kernel<false>;
    FLAT_CUDA_OK(ctx, launch_dependent(may_overlap_previous(ctx), kernel, dim3(1), kScanThreads, 0, ctx->stream, p));
    ctx->launches += 1;
    if (p.fused) return FLAT_OK;
    const int64_t blocks = std::min<int64_t>((entries + 8 * kSegment - 1) / (8 * kSegment), (int64_t)ctx->sm_count * 4);
    auto *filler = release ? paged_batch_fill_kernel<true> : paged_batch_fill_kernel<false>;
    FLAT_CUDA_OK(ctx, launch_dependent(true, filler, dim3((unsigned)blocks), 256, 0, ctx->stream, p));
    ctx->launches += 1;
    return FLAT_OK;
}

}  // namespace flat
