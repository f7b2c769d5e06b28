// Where a value stands in the paged key / value cache, and how blocks of 32 values are rounded to it.
//
// A page holds KV_PAGE positions of every kv head, a head's part in one run: key codes | key scales | value codes | value
// scales.  Kinds: halves (no scales); eight bits (code + 128, scale f16: amax / 127 of a block of 32 dimensions); four bits
// (code + 8, scale f16: m / -8, m the value of largest magnitude).  The codes stand in the order in which the lanes of a warp
// hold the operands of m16n8k16 products, so that a lane's share of a fragment is one aligned load and a warp's is one run of
// 512 bytes:
//   keys    A operand, rows = positions (lane / 4 and 8 behind it), columns = dimensions.  Any order of the dimensions within
//           a product will do if the query follows it: lane % 4 holds 8 consecutive ones of a block of 32.
//   values  A operand transposed, rows = dimensions (lane / 4 holds 4 consecutive ones of a block), columns = positions
//           (pairs 2 (lane % 4) of each half of 16).
// Four-bit codes share a byte with one of the same position, so a position is written without reading its neighbours.
#pragma once

#include <cuda_fp16.h>

#include "serving.cuh"

namespace jq {

constexpr uint32_t KV_PAGE = 64;
enum : uint32_t { KV_F16 = 1, KV_Q4_0 = 2, KV_Q8_0 = 8 };  // GGUF ids of the block types

__host__ __device__ constexpr uint32_t kv_code_bytes(uint32_t kind, uint32_t hd) {  // a head's keys (or values) in a page
    return kind == KV_F16 ? KV_PAGE * hd * 2 : kind == KV_Q8_0 ? KV_PAGE * hd : KV_PAGE * hd / 2;
}
__host__ __device__ constexpr uint32_t kv_scale_bytes(uint32_t kind, uint32_t hd) {
    return kind == KV_F16 ? 0 : KV_PAGE * (hd / 32) * 2;
}
__host__ __device__ constexpr uint32_t kv_head_bytes(uint32_t kind, uint32_t hd) {
    return 2 * (kv_code_bytes(kind, hd) + kv_scale_bytes(kind, hd));
}

// Byte of the first of four consecutive dimensions (dim a multiple of 4) of a position's key, and the distance of the bytes
// that follow: F16 four halves and Q8_0 four codes in one run; Q4_0 (dim, dim + 2) here, (dim + 1, dim + 3) two bytes behind.
template <uint32_t KIND, uint32_t HD>
__device__ __forceinline__ uint32_t kv_key_at(uint32_t pos, uint32_t dim) {
    constexpr uint32_t NB = HD / 32;
    const uint32_t a = pos / 16, h = pos / 8 % 2, r = pos % 8, b = dim / 32, c = dim % 32 / 8, s = dim % 8 / 4;
    if constexpr (KIND == KV_F16) return (((a * NB + b) * 2 + s) * 32 + r * 4 + c) * 16 + h * 8;
    if constexpr (KIND == KV_Q8_0) return ((a * NB + b) * 32 + r * 4 + c) * 16 + h * 8 + s * 4;
    return ((a * (NB / 2) + b / 2) * 32 + r * 4 + c) * 16 + b % 2 * 8 + s * 4 + h;
}
// The same of a value: dimensions dim .. dim + 3 stand at distances 0, x, m, m + x: F16 x = 4, m = 512; Q8_0 x = 2, m = 8;
// Q4_0 (dim, dim + 1) here, (dim + 2, dim + 3) m = 4 bytes behind.
template <uint32_t KIND, uint32_t HD>
__device__ __forceinline__ uint32_t kv_value_at(uint32_t pos, uint32_t dim) {
    constexpr uint32_t NB = HD / 32;
    const uint32_t a = pos / 16, h = pos / 8 % 2, c = pos % 8 / 2, e = pos % 2, b = dim / 32, r = dim % 32 / 4;
    if constexpr (KIND == KV_F16) return ((a * NB + b) * 2 * 32 + r * 4 + c) * 16 + h * 8 + e * 2;
    if constexpr (KIND == KV_Q8_0) return ((a * NB + b) * 32 + r * 4 + c) * 16 + h * 4 + e;
    return ((a * (NB / 2) + b / 2) * 32 + r * 4 + c) * 16 + b % 2 * 8 + e * 2 + h;
}
// Byte of a block's scale within the scales.
template <uint32_t HD>
__device__ __forceinline__ uint32_t kv_scale_at(uint32_t pos, uint32_t block) {
    return (((pos / 32 * 8 + pos % 8) * (HD / 32) + block) * 4 + pos % 32 / 8) * 2;
}

// Four consecutive values of a block of 32 that eight neighbouring lanes (a multiple of 8 on) hold between them -> what is
// stored.  A block with a value that is not finite gets a scale of NaN and reads as NaN; sizes past what a scale holds saturate.
// Each operation is rounded by itself (no fused multiply-adds), so the codes are those of the formulas.
struct KvQuad {
    uint32_t code[4];
    uint16_t scale;
};
template <uint32_t KIND>
__device__ __forceinline__ KvQuad kv_round(const float (&x)[4]) {
    KvQuad r;
    if constexpr (KIND == KV_F16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = fabsf(x[i]) < INFINITY ? fminf(fmaxf(x[i], -65504.0f), 65504.0f) : NAN;
            r.code[i] = __half_as_ushort(__float2half_rn(v));
        }
        r.scale = 0;
        return r;
    }
    bool finite = true;
    float hi = x[0], lo = x[0];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        finite &= fabsf(x[i]) < INFINITY;
        hi = fmaxf(hi, x[i]), lo = fminf(lo, x[i]);
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xFFFFFFFFu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xFFFFFFFFu, lo, o));
    }
    const uint32_t lane = threadIdx.x & 31;
    finite = (__ballot_sync(0xFFFFFFFFu, !finite) >> (lane & 24) & 0xFF) == 0;
    float d;
    if constexpr (KIND == KV_Q8_0)
        d = fminf(__fmul_rn(fmaxf(hi, -lo), 1.0f / 127.0f), 65504.0f);
    else
        d = fminf(fmaxf(__fmul_rn(hi > -lo ? hi : lo, -0.125f), -65504.0f), 65504.0f);
    const __half dh = __float2half_rn(d);
    const float f = __half2float(dh), inv = f != 0.0f ? __frcp_rn(f) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float c = finite ? rintf(__fmul_rn(x[i], inv)) : 0.0f;
        if constexpr (KIND == KV_Q8_0)
            r.code[i] = (uint32_t)(fminf(fmaxf(c, -127.0f), 127.0f) + 128.0f);
        else
            r.code[i] = (uint32_t)fminf(fmaxf(c + 8.0f, 0.0f), 15.0f);
    }
    r.scale = finite ? __half_as_ushort(dh) : (uint16_t)0x7FFF;
    return r;
}

// Bytes of the page of position p of sequence i; NULL if there is none.
__device__ __forceinline__ uint8_t* page_of(const KvPages& c, int32_t i, int32_t p, uint32_t head_bytes) {
    if (i < 0 || (uint32_t)i >= c.n_seq || p < 0 || (uint32_t)p >= c.table_stride * (uint64_t)KV_PAGE) return nullptr;
    const int32_t id = c.table[(uint64_t)i * c.table_stride + (uint32_t)p / KV_PAGE];
    if (id < 0 || (uint32_t)id >= c.n_pages) return nullptr;
    return c.pages + (uint64_t)id * c.n_kv * head_bytes;
}

// Four consecutive dimensions of a position's key or value; `part` begins at its codes.
template <uint32_t KIND, uint32_t HD, bool VALUES>
__device__ __forceinline__ float4 kv_load(const uint8_t* part, uint32_t pos, uint32_t d) {
    float v[4];
    if constexpr (KIND == KV_F16) {
        const uint8_t* at = part + (VALUES ? kv_value_at<KIND, HD>(pos, d) : kv_key_at<KIND, HD>(pos, d));
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e)
            v[e] = __half2float(*reinterpret_cast<const __half*>(at + (VALUES ? (e >> 1) * 512 + (e & 1) * 4 : 2 * e)));
    } else {
        const uint8_t* at = part + (VALUES ? kv_value_at<KIND, HD>(pos, d) : kv_key_at<KIND, HD>(pos, d));
        const float s = __half2float(*reinterpret_cast<const __half*>(part + kv_code_bytes(KIND, HD) + kv_scale_at<HD>(pos, d / 32)));
        if constexpr (KIND == KV_Q8_0) {
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = (float)((int)at[VALUES ? (e >> 1) * 8 + (e & 1) * 2 : e] - 128) * s;
        } else {
            const uint32_t one = at[0], two = at[VALUES ? 4 : 2];
            const uint32_t c[4] = {one & 15, VALUES ? one >> 4 : two & 15, VALUES ? two & 15 : one >> 4, two >> 4};
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] = (float)((int)c[e] - 8) * s;
        }
    }
    return make_float4(v[0], v[1], v[2], v[3]);
}

// f(kind, head dimension) as template arguments
template <class F>
cudaError_t for_kind(uint32_t kind, uint32_t hd, F f) {
#define JQ_KV_CASE(K, D) \
    if (kind == K && hd == D) return f.template operator()<K, D>();
    JQ_KV_CASE(KV_F16, 64)
    JQ_KV_CASE(KV_F16, 128)
    JQ_KV_CASE(KV_F16, 256)
    JQ_KV_CASE(KV_Q8_0, 64)
    JQ_KV_CASE(KV_Q8_0, 128)
    JQ_KV_CASE(KV_Q8_0, 256)
    JQ_KV_CASE(KV_Q4_0, 64)
    JQ_KV_CASE(KV_Q4_0, 128)
    JQ_KV_CASE(KV_Q4_0, 256)
#undef JQ_KV_CASE
    return cudaErrorInvalidValue;
}

}  // namespace jq
