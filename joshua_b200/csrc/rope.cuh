// Rotary positions from a table of (cosine, sine) pairs: the rotation of one value, given its partner.
#pragma once

#include "common.cuh"

namespace jq {

struct RopeArgs {
    const float2* table;  // [n_pos][rot / 2] (cosine, sine); NULL: nothing is rotated
    uint32_t n_pos, rot;  // positions in the table, rotated dimensions of a head (the first ones)
    uint32_t interleaved; // pairs (2 i, 2 i + 1); else (i, i + rot / 2)
};

// Dimension d of a head, d < rot: the dimension it is paired with, and the pair's number.
__device__ __forceinline__ uint32_t rope_partner(const RopeArgs& r, uint32_t d) {
    const uint32_t half = r.rot / 2;
    return r.interleaved ? d ^ 1u : d < half ? d + half : d - half;
}
__device__ __forceinline__ uint32_t rope_pair(const RopeArgs& r, uint32_t d) {
    const uint32_t half = r.rot / 2;
    return r.interleaved ? d / 2 : d < half ? d : d - half;
}
__device__ __forceinline__ bool rope_first(const RopeArgs& r, uint32_t d) { return r.interleaved ? !(d & 1u) : d < r.rot / 2; }

// (a cos - b sin, a sin + b cos), products and sums rounded one by one: the cache rounds its rows to a few bits, where a fused
// multiply-add would now and then give another code than the formula.
__device__ __forceinline__ float rope_rotate(bool first, float v, float partner, float2 cs) {
    return first ? __fsub_rn(__fmul_rn(v, cs.x), __fmul_rn(partner, cs.y)) : __fadd_rn(__fmul_rn(partner, cs.y), __fmul_rn(v, cs.x));
}

}  // namespace jq
