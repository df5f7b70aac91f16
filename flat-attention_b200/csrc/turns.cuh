// RoPE angles of far positions.  A frequency is held as the fraction of a turn that a position is worth, scaled by 2^64: the
// product with a position modulo 2^64 is then the exact fraction of a turn of that product, whatever the position (negative ones
// too), and its upper 32 bits, as a float, give the angle to 2^-26 of a turn (24 of 31 bits, worst near half a turn).  An angle that
// is formed as a 32-bit float of position times frequency is off by position * 2^-25 radians in the fastest pair, 4e-3 at position 131072.
#pragma once

#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "common.h"

namespace flat {

// theta^(-2j / D) / (2 pi) modulo 1, times 2^64
inline void fill_turns(flat_ctx *ctx, float theta, int head_dim, TurnTable *out) {
    if (ctx->turns_theta != theta || ctx->turns_dim != head_dim) {
        for (int j = 0; j < head_dim / 2; ++j) {
            const long double f = powl((long double)theta, -2.0L * j / head_dim) / 6.283185307179586476925286766559L;
            ctx->turns[j] = (uint64_t)((f - floorl(f)) * 18446744073709551616.0L);  // 2^64
        }
        ctx->turns_theta = theta;
        ctx->turns_dim = head_dim;
    }
    for (int j = 0; j < head_dim / 2; ++j) out->turns[j] = ctx->turns[j];
}

#ifdef __CUDACC__
// (cos, sin) of a position
__device__ __forceinline__ float2 turn_of(int32_t position, uint64_t turns) {
    const uint64_t phase = turns * (uint64_t)(int64_t)position + 0x80000000ull;
    float2 cs;
    sincospif((float)(int32_t)(phase >> 32) * 0x1p-31f, &cs.y, &cs.x);
    return cs;
}
// The same by the special-function unit, for queries that are rounded to 16 bits in two summands anyway.  Off by 2^-20 at most: 2^-21.2 for
// the function itself between -pi and pi, 2^-21.4 for the angle (2^-26 of a turn, the constant and the product in 32 bits)
__device__ __forceinline__ float2 turn_of_fast(int32_t position, uint64_t turns) {
    const uint64_t phase = turns * (uint64_t)(int64_t)position + 0x80000000ull;
    const float angle = (float)(int32_t)(phase >> 32) * (0x1p-31f * 3.14159265358979f);
    return make_float2(__cosf(angle), __sinf(angle));
}
#endif

}  // namespace flat
