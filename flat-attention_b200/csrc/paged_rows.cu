// Rows of a paged K/V pool written through a slot map, and rows of accepted drafts moved to where they belong.
//
// Both are copies: each byte is read once and written once, 16 bytes a thread.  The write turns K on the way (neighbouring pairs of
// each head's slice, by position * theta^(-2j/D)); a block takes a few tokens, computes their (cos, sin) once for all heads while
// the rows are on their way, and keeps them in shared memory.
#include "common.h"
#include "turns.cuh"

namespace flat {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxBlockTokens = 8;

__device__ __forceinline__ uint4 load16(const void *p) {
    uint4 r;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p));
    return r;
}

__device__ __forceinline__ void turn_pair(float &x, float &y, float2 cs) {
    const float a = x * cs.x - y * cs.y, b = x * cs.y + y * cs.x;
    x = a;
    y = b;
}

template <typename T> __device__ __forceinline__ uint4 turn16(uint4 r, const float2 *cs);
template <> __device__ __forceinline__ uint4 turn16<float>(uint4 r, const float2 *cs) {
    float f[4] = {__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w)};
    turn_pair(f[0], f[1], cs[0]);
    turn_pair(f[2], f[3], cs[1]);
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}
template <> __device__ __forceinline__ uint4 turn16<__nv_bfloat16>(uint4 r, const float2 *cs) {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        float x = __uint_as_float(w[e] << 16), y = __uint_as_float(w[e] & 0xffff0000u);
        turn_pair(x, y, cs[e]);
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);  // the cache's type: one rounding
        w[e] = *reinterpret_cast<const uint32_t *>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Rows whose head slices are whole 16-byte vectors.
template <typename T>
__global__ void __launch_bounds__(kThreads) paged_write_kernel(const __grid_constant__ PagedWriteParams p) {
    constexpr int kPer = 16 / sizeof(T);
    constexpr int kFlight = 4;
    __shared__ float2 cs_s[kMaxBlockTokens][kMaxHeadDim / 2];
    __shared__ int64_t row_s[kMaxBlockTokens];
    grid_dependency_wait();
    grid_dependency_launch();
    const int half = p.head_dim / 2, vecs = p.row_elems / kPer;
    const int64_t first = (int64_t)blockIdx.x * p.block_tokens;
    const int n = (int)min((int64_t)p.block_tokens, p.tokens - first);
    if (threadIdx.x < n) {
        const int slot = p.slots[first + threadIdx.x];
        if (slot >= p.pool_rows) report_status(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, (int)(first + threadIdx.x), kPlaceSlot);
        row_s[threadIdx.x] = slot < p.pool_rows ? slot : -1;
    }
    const int total = n * vecs;
    uint4 k[kFlight], v[kFlight];
    auto request = [&](int base) {
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int i = base + u * kThreads;
            if (i < total) {
                k[u] = load16(static_cast<const char *>(p.k_src) + (first * vecs + i) * 16);
                v[u] = load16(static_cast<const char *>(p.v_src) + (first * vecs + i) * 16);
            }
        }
    };
    request(threadIdx.x);
    if (p.positions)
        for (int i = threadIdx.x; i < n * half; i += kThreads) {
            const int t = i / half;
            cs_s[t][i - t * half] = turn_of(p.positions[first + t], p.freq.turns[i - t * half]);
        }
    __syncthreads();
    for (int base = threadIdx.x; base < total; base += kFlight * kThreads) {
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int i = base + u * kThreads;
            if (i >= total) break;
            const int t = i / vecs, c = i - t * vecs;
            const int64_t row = row_s[t];
            if (row < 0) continue;
            const int64_t to = (row * vecs + c) * 16;
            *reinterpret_cast<uint4 *>(static_cast<char *>(p.k_dst) + to) =
                p.positions ? turn16<T>(k[u], &cs_s[t][(c * kPer % p.head_dim) / 2]) : k[u];
            *reinterpret_cast<uint4 *>(static_cast<char *>(p.v_dst) + to) = v[u];
        }
        if (base + kFlight * kThreads < total) request(base + kFlight * kThreads);
    }
}

// Any head_dim and alignment: a thread takes one pair of a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) paged_write_pairs_kernel(const __grid_constant__ PagedWriteParams p) {
    grid_dependency_wait();
    grid_dependency_launch();
    const int pairs = (p.row_elems + 1) / 2;
    const int64_t total = p.tokens * pairs;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        const int64_t t = i / pairs;
        const int e = (int)(i - t * pairs) * 2;
        const int64_t row = p.slots[t];
        if (row < 0) continue;
        if (row >= p.pool_rows) {
            if (e == 0) report_status(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, (int)t, kPlaceSlot);
            continue;
        }
        const bool two = e + 1 < p.row_elems;
        const T *ks = static_cast<const T *>(p.k_src) + t * p.row_elems + e, *vs = static_cast<const T *>(p.v_src) + t * p.row_elems + e;
        T *kd = static_cast<T *>(p.k_dst) + row * p.row_elems + e, *vd = static_cast<T *>(p.v_dst) + row * p.row_elems + e;
        if (p.positions) {  // head_dim is even: a pair never straddles two heads
            float x = to_float<T>(ks[0]), y = to_float<T>(ks[1]);
            turn_pair(x, y, turn_of(p.positions[t], p.freq.turns[(e % p.head_dim) / 2]));
            kd[0] = from_float<T>(x);
            kd[1] = from_float<T>(y);
        } else {
            kd[0] = ks[0];
            if (two) kd[1] = ks[1];
        }
        vd[0] = vs[0];
        if (two) vd[1] = vs[1];
    }
}

// Row j of a sequence's drafts := row path[j], j = 0, 1, ...  The path rises strictly, so path[j] >= j: a step's destination is never
// a later step's source, and what a step overwrites an earlier one has read, if each thread goes through the steps in order.  A
// block takes a sequence, a thread one 16-byte (otherwise one-element) column of its rows at a time, kFlight rows in flight, so no
// two threads touch the same bytes.  Which rows the steps mean is looked up once for the block, kSteps at a time.
template <typename V> __global__ void __launch_bounds__(kThreads) paged_accept_kernel(const __grid_constant__ PagedAcceptParams p) {
    constexpr int kFlight = 8, kSteps = kThreads;
    __shared__ int bad_s;
    __shared__ int64_t from_s[kSteps], to_s[kSteps];  // < 0 in from_s: stays
    grid_dependency_wait();
    grid_dependency_launch();
    const int seq = blockIdx.x;
    const int take = p.accept_lens[seq], len = p.context_lens[seq], held = min(p.page_counts[seq], p.max_pages);
    const int32_t *path = p.path + (int64_t)seq * p.max_accept;
    const int32_t *table = p.page_tables + (int64_t)seq * p.max_pages;
    auto row_of = [&](int node) -> int64_t {  // < 0: not a row that the sequence holds
        const unsigned t = (unsigned)len + (unsigned)node, logical = t / (unsigned)p.page_size;
        if (node < 0 || (int64_t)logical >= held) return -1;
        const int page = table[logical];
        return (unsigned)page < (unsigned)p.physical_pages ? (int64_t)page * p.page_size + (t - logical * (unsigned)p.page_size) : -1;
    };
    if (threadIdx.x == 0) bad_s = take < 0 || take > p.max_accept || len < 0;
    __syncthreads();
    // the whole path first, its beginning last: a sequence moves all of it or nothing
    auto look = [&](int base) {
        const int j = base + threadIdx.x;
        if (j >= take) return;
        const int node = path[j], before = j > 0 ? path[j - 1] : -1;
        const int64_t from = row_of(node), to = row_of(j);
        if (node < j || before >= node || from < 0 || to < 0) bad_s = 1;
        from_s[threadIdx.x] = node == j ? -1 : from;
        to_s[threadIdx.x] = to;
    };
    if (!bad_s)
        for (int base = (max(take, 1) - 1) / kSteps * kSteps; base >= 0; base -= kSteps) look(base);
    __syncthreads();
    const bool bad = bad_s != 0;
    if (threadIdx.x == 0) p.context_lens_out[seq] = bad ? len : len + take;  // may be context_lens: every thread has read the length
    if (bad) {
        if (threadIdx.x == 0) report_status(p.status, FLAT_ERR_LENGTH_MISMATCH, seq, kPlacePath);
        return;
    }
    for (int base = 0; base < take; base += kSteps) {
        if (base > 0) {
            __syncthreads();
            look(base);
            __syncthreads();
        }
        const int steps = min(kSteps, take - base);
        for (int64_t column = threadIdx.x; column < 2 * p.row_vecs; column += kThreads) {
            V *at = column < p.row_vecs ? static_cast<V *>(p.k) + column : static_cast<V *>(p.v) + (column - p.row_vecs);
            for (int j = 0; j < steps; j += kFlight) {
                V x[kFlight];
                bool moves[kFlight];
#pragma unroll
                for (int u = 0; u < kFlight; ++u) {
                    moves[u] = j + u < steps && from_s[j + u] >= 0;
                    if (moves[u]) x[u] = at[from_s[j + u] * p.row_vecs];
                }
#pragma unroll
                for (int u = 0; u < kFlight; ++u)
                    if (moves[u]) at[to_s[j + u] * p.row_vecs] = x[u];
            }
        }
    }
}

}  // namespace

int launch_paged_write(flat_ctx *ctx, int dtype, PagedWriteParams &p) {
    const int size = (int)dtype_size(dtype);
    const bool vectors = (int64_t)p.head_dim * size % 16 == 0 &&
                         ((uintptr_t)p.k_src | (uintptr_t)p.v_src | (uintptr_t)p.k_dst | (uintptr_t)p.v_dst) % 16 == 0;
    const bool overlap = may_overlap_previous(ctx);
    if (vectors) {
        const int64_t per = p.tokens >= (int64_t)ctx->sm_count * 32 ? kMaxBlockTokens : 4;
        p.block_tokens = (int)per;
        const int64_t blocks = (p.tokens + per - 1) / per;
        FLAT_CUDA_OK(ctx, launch_dependent(overlap, dtype == FLAT_BF16 ? paged_write_kernel<__nv_bfloat16> : paged_write_kernel<float>,
                                           dim3((unsigned)blocks), kThreads, 0, ctx->stream, p));
    } else {
        const int64_t blocks = std::min<int64_t>((p.tokens * ((p.row_elems + 1) / 2) + kThreads - 1) / kThreads, (int64_t)ctx->sm_count * 8);
        FLAT_CUDA_OK(ctx, launch_dependent(overlap, dtype == FLAT_BF16 ? paged_write_pairs_kernel<__nv_bfloat16> : paged_write_pairs_kernel<float>,
                                           dim3((unsigned)blocks), kThreads, 0, ctx->stream, p));
    }
    ctx->launches += 1;
    return FLAT_OK;
}

int launch_paged_accept(flat_ctx *ctx, int dtype, int64_t row_elems, PagedAcceptParams &p) {
    const int64_t bytes = row_elems * (int64_t)dtype_size(dtype);
    const bool vectors = bytes % 16 == 0 && ((uintptr_t)p.k | (uintptr_t)p.v) % 16 == 0;
    p.row_vecs = vectors ? bytes / 16 : row_elems;
    auto *kernel = vectors ? paged_accept_kernel<uint4> : dtype == FLAT_BF16 ? paged_accept_kernel<uint16_t> : paged_accept_kernel<uint32_t>;
    FLAT_CUDA_OK(ctx, launch_dependent(may_overlap_previous(ctx), kernel, dim3((unsigned)p.num_seqs), kThreads, 0, ctx->stream, p));
    ctx->launches += 1;
    return FLAT_OK;
}

}  // namespace flat
