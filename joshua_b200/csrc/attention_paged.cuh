// What the kernels of the attention over the paged cache share.
#pragma once

#include "kv_pages.cuh"

namespace jq {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
// a and b, and what f16 leaves of them
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    *hi = half2_bits(h), *lo = half2_bits(__floats2half2_rn(a - f.x, b - f.y));
}
// bytes b, b + 1 of w (codes + 128) as halves
template <int B>
__device__ __forceinline__ uint32_t codes8(uint32_t w) {
    return half2_bits(__hsub2(bits_half2(__byte_perm(w, 0x64646464u, B == 0 ? 0x4140 : 0x4342)), __float2half2_rn(1152.0f)));
}
// four-bit codes + 8 at bits 4 N .. and 16 + 4 N .. as halves
template <int N>
__device__ __forceinline__ uint32_t codes4(uint32_t w) {
    if constexpr (N >= 2) w >>= 8;
    if constexpr (N % 2 == 0)  // 1024 + n
        return half2_bits(__hsub2(bits_half2((w & 0x000F000Fu) | 0x64006400u), __float2half2_rn(1032.0f)));
    // 1024 + 16 n
    return half2_bits(__hfma2(bits_half2((w & 0x00F000F0u) | 0x64006400u), __float2half2_rn(0.0625f), __float2half2_rn(-72.0f)));
}

constexpr uint32_t LEAD_MOST = 8;  // partial results of the leading pages

struct PagedArgs {
    KvPages c;
    const float* q;
    uint64_t q_stride;
    const int32_t* len;
    uint32_t n_q, group, split;  // query heads; heads a kv head; warps' worth of them (each up to ROWS rows)
    float scale;
    uint32_t common, done;  // leading pages named by the first sequence; leading pages that the other kernel takes
    float* out;
    uint64_t out_stride;
    uint32_t* arrived;  // a counter a CTA, for the segment that goes on behind it; zero between calls
    float* part;        // [grid][2][ROWS (HD + 2)]
    const float* lead;  // done: [lead_splits][n_kv][batch * group][HD], then their maxima, then their sums
    uint32_t lead_splits;
    int32_t* bad_pos;
};

// Weight of a piece with maximum m under the joint maximum; equal ones are 1 (infinities too)
__device__ __forceinline__ float piece_weight(float m, float top) { return m == top ? 1.0f : ex2(m - top); }

// attention_lead.cu: the leading pages on the 5th-generation tensor cores, heads of 64 and 128.  grid (splits, blocks of 128 query
// rows, kv heads), `cluster` splits joined; lead: as PagedArgs has it.
cudaError_t launch_attention_lead_tiles(const PagedArgs& a, float* lead, uint32_t splits, uint32_t blocks, uint32_t cluster, int* error_flag,
                                        cudaStream_t s);

}  // namespace jq
