// Attention of drafted tokens over a paged cache, any type, head_dim, group and page size, in 32-bit arithmetic.
//
//   query i of sequence s, turned at its position, sees the L live tokens and drafted token j (row L + j) iff its mask says so:
//   O = softmax(scale * q K^T) V,  LSE = log sum exp;  a query that sees nothing: O = 0, LSE = -inf
//
// A block takes one KV head of one sequence, 32 of its (drafted token, head of the group) rows and a chunk of the tokens; it goes
// over the chunk in tiles of 32 tokens that it holds in shared memory as f32, with the running maximum and sum of each row.  The
// chunks' results are joined by a second kernel.  Bound by the FMA pipe for many rows and by latency for few; each K and V byte is
// read once per 32 rows.  A masked token counts for nothing whatever its K and V hold: its score is replaced, not added to, and its
// product with V is left out rather than formed with weight 0.
#include "common.h"
#include "tree.cuh"
#include "turns.cuh"

namespace flat {
namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kRows = 32, kTokens = 32, kThreads = 128, kMaxSplits = 256;
constexpr float kMasked = -1.f;  // in place of a weight, which is never negative

// Four values from `at` on as f32, `left` of them there; vec: rows are whole aligned groups of four.
template <typename T> __device__ __forceinline__ float4 load4(const T *at, bool vec, int left);
template <> __device__ __forceinline__ float4 load4<float>(const float *at, bool vec, int left) {
    if (vec) return *reinterpret_cast<const float4 *>(at);
    return make_float4(at[0], left > 1 ? at[1] : 0.f, left > 2 ? at[2] : 0.f, left > 3 ? at[3] : 0.f);
}
template <> __device__ __forceinline__ float4 load4<__nv_bfloat16>(const __nv_bfloat16 *at, bool vec, int left) {
    if (vec) {
        const uint2 x = *reinterpret_cast<const uint2 *>(at);
        return make_float4(__uint_as_float(x.x << 16), __uint_as_float(x.x & 0xffff0000u), __uint_as_float(x.y << 16), __uint_as_float(x.y & 0xffff0000u));
    }
    return make_float4(to_float<__nv_bfloat16>(at[0]), left > 1 ? to_float<__nv_bfloat16>(at[1]) : 0.f, left > 2 ? to_float<__nv_bfloat16>(at[2]) : 0.f,
                       left > 3 ? to_float<__nv_bfloat16>(at[3]) : 0.f);
}

__device__ __forceinline__ TreeSequence span_of(const TreeParams &p, int seq) {
    const TreeSequence s = tree_sequence(p, seq);
    if (s.code && threadIdx.x == 0) report_status(p.status, s.code, seq, kPlaceBound);
    return s;
}

__device__ __forceinline__ bool sees(const TreeParams &p, const TreeSequence &s, int node, int token) {
    return token < s.len || (token - s.len < s.nodes && tree_sees(p, s, node, token - s.len));
}

// HALVES: of 64 dims (head_dim up to 64 or 128).
template <typename T, int HALVES> __global__ void __launch_bounds__(kThreads) tree_simt_kernel(const __grid_constant__ TreeParams p) {
    extern __shared__ __align__(16) float smem[];
    grid_dependency_wait();
    grid_dependency_launch();
    const int tid = threadIdx.x;
    const int D = p.head_dim, D4 = (D + 3) / 4 * 4, stride = D4 + 4;
    float *q_s = smem, *k_s = q_s + kRows * stride, *v_s = k_s + kTokens * stride, *p_s = v_s + kTokens * stride;
    float *m_s = p_s + kRows * (kTokens + 1), *l_s = m_s + kRows, *a_s = l_s + kRows;
    __shared__ int on_s[kTokens];  // whether the token is there
    const int tiles = (p.max_nodes * p.group + kRows - 1) / kRows;
    const int seq = blockIdx.z, kv_head = blockIdx.y / tiles, row0 = blockIdx.y % tiles * kRows, split = blockIdx.x;
    const TreeSequence s = span_of(p, seq);
    const int rows = min(kRows, s.nodes * p.group - row0);
    if (rows <= 0) return;
    const int begin = (int)min((int64_t)split * p.chunk, (int64_t)s.tokens), end = (int)min((int64_t)begin + p.chunk, (int64_t)s.tokens);
    if (begin >= end && split > 0) return;  // the merge leaves it out

    // K and V of a tile on their way: tokens rg + 8 i, dims cg * 4 (+ 64).  Asked for while the tile before is worked on, the first one
    // while the queries are turned.
    float4 k_next[HALVES][kTokens / 8], v_next[HALVES][kTokens / 8];
    bool there[kTokens / 8];
    auto request = [&](int t0) {
        int64_t at[kTokens / 8];
#pragma unroll
        for (int i = 0; i < kTokens / 8; ++i) {
            const int t = t0 + (tid >> 4) + 8 * i, logical = t / p.page_size;
            at[i] = -1;
            if (t < end) {
                const int page = p.page_tables[(int64_t)seq * p.max_pages + logical];
                if ((unsigned)page < (unsigned)p.physical_pages) {
                    at[i] = (((int64_t)page * p.page_size + t - logical * p.page_size) * p.kv_heads + kv_head) * D;
                } else if ((tid & 15) == 0) {  // never read: its tokens are left out and the call is flagged
                    report_status(p.status, FLAT_ERR_PAGE_OUT_OF_RANGE, seq);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kTokens / 8; ++i) {
            there[i] = at[i] >= 0;
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int e = (tid & 15) * 4 + h * 64;
                k_next[h][i] = v_next[h][i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at[i] < 0 || e >= D) continue;
                k_next[h][i] = load4<T>(static_cast<const T *>(p.k) + at[i] + e, p.vectors, D - e);
                v_next[h][i] = load4<T>(static_cast<const T *>(p.v) + at[i] + e, p.vectors, D - e);
            }
        }
    };
    request(begin);

    // the rows' queries, turned, with the softmax scale and log2(e): scores come out in the exp2 domain
    const int rg = tid >> 4, cg = tid & 15;  // rows rg * 4 .. + 3; tokens cg, cg + 16; dims cg * 4 and cg * 4 + 64
#pragma unroll
    for (int h = 0; h < HALVES; ++h) {
        const int e = cg * 4 + h * 64;
        if (e >= D4) break;
#pragma unroll 1
        for (int i = 0; i < kRows / 8; ++i) {
            const int r = rg + 8 * i;
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            if (r < rows) {
                const int node = s.first + (row0 + r) / p.group, head = kv_head * p.group + (row0 + r) % p.group;
                const float4 q = load4<T>(static_cast<const T *>(p.q) + ((int64_t)node * p.q_heads + head) * D + e, p.vectors, D - e);
                const int position = p.positions[node];
                const float scale = p.scale * kLog2e;
                const float2 c0 = turn_of(position, p.freq.turns[e / 2]), c1 = e + 2 < D ? turn_of(position, p.freq.turns[e / 2 + 1]) : make_float2(0.f, 0.f);
                x = make_float4((q.x * c0.x - q.y * c0.y) * scale, (q.x * c0.y + q.y * c0.x) * scale, (q.z * c1.x - q.w * c1.y) * scale,
                                (q.z * c1.y + q.w * c1.x) * scale);
            }
            *reinterpret_cast<float4 *>(q_s + r * stride + e) = x;
        }
    }
    if (tid < kRows) {
        m_s[tid] = -INFINITY;
        l_s[tid] = 0.f;
    }
    float acc[4][4 * HALVES];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < 4 * HALVES; ++e) acc[r][e] = 0.f;

    for (int t0 = begin; t0 < end; t0 += kTokens) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kTokens / 8; ++i) {
            if (cg == 0) on_s[rg + 8 * i] = there[i];
#pragma unroll
            for (int h = 0; h < HALVES; ++h) {
                const int e = cg * 4 + h * 64;
                if (e >= D4) break;
                *reinterpret_cast<float4 *>(k_s + (rg + 8 * i) * stride + e) = k_next[h][i];
                *reinterpret_cast<float4 *>(v_s + (rg + 8 * i) * stride + e) = v_next[h][i];
            }
        }
        if (t0 + kTokens < end) request(t0 + kTokens);
        __syncthreads();
        float x[4][2];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r][0] = x[r][1] = 0.f;
        for (int e = 0; e < D4; e += 4) {
            const float4 k0 = *reinterpret_cast<const float4 *>(k_s + cg * stride + e);
            const float4 k1 = *reinterpret_cast<const float4 *>(k_s + (cg + 16) * stride + e);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 q = *reinterpret_cast<const float4 *>(q_s + (rg * 4 + r) * stride + e);
                x[r][0] = fmaf(q.x, k0.x, fmaf(q.y, k0.y, fmaf(q.z, k0.z, fmaf(q.w, k0.w, x[r][0]))));
                x[r][1] = fmaf(q.x, k1.x, fmaf(q.y, k1.y, fmaf(q.z, k1.z, fmaf(q.w, k1.w, x[r][1]))));
            }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = rg * 4 + r, node = (row0 + row) / p.group;
            bool on[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int t = cg + 16 * c;
                on[c] = row < rows && on_s[t] && sees(p, s, node, t0 + t);
                if (!on[c]) x[r][c] = -INFINITY;
            }
            float top = fmaxf(x[r][0], x[r][1]);
#pragma unroll
            for (int w = 8; w >= 1; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
            const float before = m_s[row], now = fmaxf(before, top), base = now == -INFINITY ? 0.f : now;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float w = exp2f(x[r][c] - base);
                p_s[row * (kTokens + 1) + cg + 16 * c] = on[c] ? w : kMasked;
                if (on[c]) sum += w;
            }
#pragma unroll
            for (int w = 8; w >= 1; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
            __syncwarp();
            if (cg == 0) {
                const float a = exp2f(before - base);  // before = -inf gives 0
                m_s[row] = now;
                l_s[row] = l_s[row] * a + sum;
                a_s[row] = a;
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float a = a_s[rg * 4 + r];
#pragma unroll
            for (int e = 0; e < 4 * HALVES; ++e) acc[r][e] *= a;
        }
        for (int t = 0; t < kTokens; ++t) {
            float4 v[HALVES];
#pragma unroll
            for (int h = 0; h < HALVES; ++h)
                v[h] = cg * 4 + h * 64 < D4 ? *reinterpret_cast<const float4 *>(v_s + t * stride + cg * 4 + h * 64) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float w = p_s[(rg * 4 + r) * (kTokens + 1) + t];
                if (w < 0.f) continue;
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    acc[r][4 * h] = fmaf(w, v[h].x, acc[r][4 * h]);
                    acc[r][4 * h + 1] = fmaf(w, v[h].y, acc[r][4 * h + 1]);
                    acc[r][4 * h + 2] = fmaf(w, v[h].z, acc[r][4 * h + 2]);
                    acc[r][4 * h + 3] = fmaf(w, v[h].w, acc[r][4 * h + 3]);
                }
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int row = rg * 4 + r;
        if (row >= rows) continue;
        const float m = m_s[row], l = l_s[row];
        const bool empty = l == 0.f;  // a NaN counts
        const float inv = empty ? 0.f : 1.0f / l, lse = empty ? -INFINITY : (m + log2f(l)) * kLn2;
        const int64_t out = (int64_t)(s.first + (row0 + row) / p.group) * p.q_heads + kv_head * p.group + (row0 + row) % p.group;
        const int64_t part = (int64_t)split * p.max_q * p.q_heads + out;
#pragma unroll
        for (int e = 0; e < 4 * HALVES; ++e) {
            const int d = cg * 4 + (e & 3) + (e >> 2) * 64;
            if (d >= D) continue;
            const float o = empty ? 0.f : acc[r][e] * inv;
            if (p.splits > 1) p.partial_o[part * D + d] = o;
            else static_cast<T *>(p.o)[out * D + d] = from_float<T>(o);
        }
        if (cg == 0) (p.splits > 1 ? p.partial_lse[part] : p.lse[out]) = lse;
    }
}

// Joins the chunks of one drafted token's head: LSE = log sum exp(LSE_i), O = sum exp(LSE_i - LSE) O_i.  Threads take chunks for the
// weights; for the sum four dims each, and groups of threads every so many-th chunk, added up in a fixed order.
template <typename T> __global__ void __launch_bounds__(kThreads) tree_merge_kernel(const __grid_constant__ TreeParams p) {
    constexpr int kWarps = kThreads / 32;
    __shared__ float w[kMaxSplits], top_s[kWarps], sum_s[kWarps];
    __shared__ float4 o_s[kWarps][32];
    grid_dependency_wait();
    grid_dependency_launch();
    const int seq = blockIdx.z, node = blockIdx.y, head = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const TreeSequence s = tree_sequence(p, seq);
    if (node >= s.nodes) return;
    const int parts = max(1, (s.tokens + p.chunk - 1) / p.chunk), D = p.head_dim;
    const int64_t rows = (int64_t)p.max_q * p.q_heads, row = (int64_t)(s.first + node) * p.q_heads + head;
    auto larger = [](float a, float b) { return b > a || b != b ? b : a; };  // a NaN stays one
    float mx = -INFINITY, sum = 0.f;
    for (int i = threadIdx.x; i < parts; i += kThreads) {
        const float x = p.partial_lse[i * rows + row];
        w[i] = x;
        mx = larger(mx, x);
    }
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) mx = larger(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    if (lane == 0) top_s[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWarps; ++i) mx = larger(mx, top_s[i]);
    const float base = mx == -INFINITY ? 0.f : mx;
    for (int i = threadIdx.x; i < parts; i += kThreads) sum += w[i] = expf(w[i] - base);
#pragma unroll
    for (int d = 16; d >= 1; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sum_s[warp] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) sum += sum_s[i];
    const bool empty = sum == 0.f;
    const float inv = empty ? 0.f : 1.0f / sum;
    int width = 1;  // threads of a row
    while (width * 4 < D) width *= 2;
    const int groups = kThreads / width, d = threadIdx.x % width * 4;
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    if (d < D) {
        const bool vec = D % 4 == 0;  // the partial results' rows then are whole groups of four
#pragma unroll 8
        for (int i = threadIdx.x / width; i < parts; i += groups) {
            const float4 x = load4<float>(p.partial_o + (i * rows + row) * D + d, vec, D - d);
            const float f = w[i];
            o[0] = fmaf(f, x.x, o[0]);  // a chunk in which the row sees nothing holds zeros
            o[1] = fmaf(f, x.y, o[1]);
            o[2] = fmaf(f, x.z, o[2]);
            o[3] = fmaf(f, x.w, o[3]);
        }
    }
    for (int g = 16; g >= width; g /= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor_sync(0xffffffffu, o[e], g);
    o_s[warp][lane] = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    if (threadIdx.x < width) {  // 32 threads a row at most
#pragma unroll
        for (int i = 1; i < kWarps; ++i) {
            const float4 x = o_s[i][threadIdx.x];
            o[0] += x.x, o[1] += x.y, o[2] += x.z, o[3] += x.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (d + e < D) static_cast<T *>(p.o)[row * D + d + e] = from_float<T>(o[e] * inv);
    }
    if (threadIdx.x == 0) p.lse[row] = empty ? -INFINITY : base + logf(sum);
}

template <typename T> int launch(flat_ctx *ctx, TreeParams &p) {
    const int tiles = (int)(((int64_t)p.max_nodes * p.group + kRows - 1) / kRows);
    if ((int64_t)tiles * p.kv_heads > 65535)
        return fail(ctx, FLAT_ERR_DISPATCH_LIMIT, "%d drafted tokens of %d heads are more row tiles than one launch has", p.max_nodes, p.q_heads);
    // chunks of the longest context that fill the device about four times, a tile of 32 tokens at least, as many as the scratch holds; the
    // longest that the bound allows: where the sequences are far shorter they are few chunks of many tiles (18 us -> 117 us for
    // sequences of up to 1200 tokens under a bound of 32768)
    const int64_t rows = (int64_t)p.max_q * p.q_heads, units = (int64_t)tiles * p.kv_heads * p.num_seqs;
    const int64_t fit = (int64_t)((kPagedScratchBytes - kPagedPlanBytes) / (rows * (p.head_dim + 1) * sizeof(float)));
    int64_t splits = std::min<int64_t>({(p.max_context + kTokens - 1) / kTokens, std::max<int64_t>(1, (int64_t)ctx->sm_count * 4 / units), kMaxSplits, fit});
    if (splits < 1) splits = 1;
    p.chunk = (int)((p.max_context + splits - 1) / splits + kTokens - 1) / kTokens * kTokens;
    p.splits = (int)((p.max_context + p.chunk - 1) / p.chunk);
    p.vectors = p.head_dim % 4 == 0 && ((uintptr_t)p.q | (uintptr_t)p.k | (uintptr_t)p.v) % (4 * sizeof(T)) == 0;
    p.partial_o = reinterpret_cast<float *>(static_cast<char *>(ctx->paged_scratch) + kPagedPlanBytes);
    p.partial_lse = p.partial_o + p.splits * rows * p.head_dim;
    const int stride = (p.head_dim + 3) / 4 * 4 + 4;
    const size_t smem = ((kRows + 2 * kTokens) * stride + kRows * (kTokens + 1) + 3 * kRows) * sizeof(float);
    static_assert((32 + 64) * (kMaxHeadDim + 4) * 4 + 32 * 33 * 4 + 96 * 4 < 64 << 10, "shared memory of the largest head_dim");
    auto *kernel = p.head_dim <= 64 ? tree_simt_kernel<T, 1> : tree_simt_kernel<T, 2>;
    if (smem > 40 << 10) FLAT_CUDA_OK(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 << 10));
    {
        KernelTimer timer(ctx);
        FLAT_CUDA_OK(ctx, launch_dependent(may_overlap_previous(ctx), kernel, dim3((unsigned)p.splits, (unsigned)(tiles * p.kv_heads), (unsigned)p.num_seqs),
                                           kThreads, smem, ctx->stream, p));
    }
    ctx->launches += 1;
    if (p.splits > 1) {
        FLAT_CUDA_OK(ctx, launch_dependent(true, tree_merge_kernel<T>, dim3((unsigned)p.q_heads, (unsigned)p.max_nodes, (unsigned)p.num_seqs), kThreads, 0,
                                           ctx->stream, p));
        ctx->launches += 1;
    }
    return FLAT_OK;
}

}  // namespace

int launch_tree_simt(flat_ctx *ctx, int dtype, TreeParams &p) { return dtype == FLAT_BF16 ? launch<__nv_bfloat16>(ctx, p) : launch<float>(ctx, p); }

}  // namespace flat
