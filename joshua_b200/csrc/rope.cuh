// Rotary positions from a table of (cosine, sine) pairs: the rotation of one value, given its partner.
#pragma once

#include "common.cuh"

namespace jq {

struct RopeArgs {
    const float2* table;  // [n_pos][rot / 2] (cosine, sine); NULL: nothing is rotated
    uint32_t n_pos, rot;  // positions in the table, rotated dimensions of a head (the first ones)
    uint32_t interleaved; // pairs (2 i, 2 i + 1); else (i, i + rot / 2)
    uint32_t vectors;     // rot is a multiple of 8 and the table 16-byte aligned
};

// (a cos - b sin, a sin + b cos), products and sums rounded one by one: the cache rounds its rows to a few bits, where a fused
// multiply-add would now and then give another code than the formula.
__device__ __forceinline__ float rope_rotate(bool first, float v, float partner, float2 cs) {
    return first ? __fsub_rn(__fmul_rn(v, cs.x), __fmul_rn(partner, cs.y)) : __fadd_rn(__fmul_rn(partner, cs.y), __fmul_rn(v, cs.x));
}

}  // namespace jq
