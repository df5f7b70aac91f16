// What the kernels of the attention of drafted tokens share: a sequence as they see it, and what a drafted token sees.
#pragma once

#include "common.h"

namespace flat {
#ifdef __CUDACC__

// The device arrays hold whatever they hold: the rows stay inside q and o, the tokens inside the pages that the sequence holds.
struct TreeSequence {
    int first, nodes, len, tokens;  // rows of q; drafted tokens (0: nothing to do); live tokens; tokens that there are pages for
    int code;                       // FLAT_OK or what the caller reports
};
__device__ __forceinline__ TreeSequence tree_sequence(const TreeParams &p, int seq) {
    TreeSequence s;
    s.first = p.q_offsets[seq];
    const int64_t nodes = (int64_t)p.q_offsets[seq + 1] - s.first;
    s.len = p.context_lens[seq];
    s.nodes = s.tokens = 0;
    s.code = FLAT_OK;
    if (s.first < 0 || nodes < 0 || nodes > p.max_nodes || nodes > p.max_q - (int64_t)s.first || s.len < 0) {
        s.code = FLAT_ERR_LENGTH_MISMATCH;
        return s;
    }
    if (nodes == 0) return s;
    s.nodes = (int)nodes;
    const int64_t room = (int64_t)min(max(p.page_counts[seq], 0), p.max_pages) * p.page_size, want = (int64_t)s.len + s.nodes;
    s.tokens = (int)min(min(want, room), (int64_t)p.max_context);
    if (s.tokens < want) s.code = FLAT_ERR_PAGE_OUT_OF_RANGE;
    return s;
}
// Whether drafted token `node` sees drafted token j of its sequence.
__device__ __forceinline__ bool tree_sees(const TreeParams &p, const TreeSequence &s, int node, int j) {
    if (!p.mask) return !p.causal || j <= node;
    return (p.mask[(int64_t)(s.first + node) * p.mask_words + (j >> 5)] >> (j & 31)) & 1u;
}

#endif
}  // namespace flat
