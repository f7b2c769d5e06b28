// A page of the quantised cache as operands of the 5th-generation tensor cores: codes times scales in one or two f16 terms, keys and
// values in K-major tiles with the 128-byte swizzle.
#pragma once

#include "attention_paged.cuh"
#include "f32x2.cuh"
#include "tc5.cuh"

namespace jq {

namespace {

// Scores are multiplied and shifted by their maximum in one step, exact but for the shift itself: with maxima from here on, whose last bit
// may be worth more than the probabilities' terms have room for, they are rounded as the maximum was and shifted by it first, in a step
// of their own.
constexpr float FAR = 0x1p20f;

__device__ __forceinline__ void sts_v4(uint32_t addr, const uint32_t (&v)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// Four words a lane of four neighbouring lanes: word i of lane c becomes word c of lane i.
__device__ __forceinline__ void transpose4(uint32_t (&v)[4], uint32_t c) {
    const uint32_t a = __shfl_xor_sync(0xFFFFFFFFu, c & 1 ? v[0] : v[1], 1), b = __shfl_xor_sync(0xFFFFFFFFu, c & 1 ? v[2] : v[3], 1);
    if (c & 1)
        v[0] = a, v[2] = b;
    else
        v[1] = a, v[3] = b;
    const uint32_t d = __shfl_xor_sync(0xFFFFFFFFu, c & 2 ? v[0] : v[2], 2), e = __shfl_xor_sync(0xFFFFFFFFu, c & 2 ? v[1] : v[3], 2);
    if (c & 2)
        v[0] = d, v[1] = e;
    else
        v[2] = d, v[3] = e;
}
// code times scale as two terms: exact, a code has 8 bits at most and a scale 11
__device__ __forceinline__ void scaled_terms(uint32_t code, __half2 scale, uint32_t* hi, uint32_t* lo) {
    const __half2 c = bits_half2(code), h = __hmul2(c, scale);
    *hi = half2_bits(h), *lo = half2_bits(__hfma2(c, scale, __hneg2(h)));
}
// 2^n as f32
__device__ __forceinline__ float power(int n) { return __uint_as_float((uint32_t)(127 + n) << 23); }
// two scales (halves) times a power of two
__device__ __forceinline__ __half2 scaled(uint32_t w, float f) {
    const float2 s = __half22float2(bits_half2(w));
    return __floats2half2_rn(s.x * f, s.y * f);
}


template <uint32_t KIND, uint32_t HD>
struct PageTile {
    static constexpr uint32_t NB = HD / 32, TERMS = KIND == KV_F16 ? 1 : 2;
    static constexpr uint32_t HALVES = HD / 64;              // 64-dimension accumulators of a score
    static constexpr uint32_t K_PLANE = KV_PAGE * 128;       // 64 dimensions of the tile's keys, one term
    static constexpr uint32_t K_STAGE = TERMS * HALVES * K_PLANE;
    static constexpr uint32_t V_PLANE = HD * 128;            // the tile's keys of every dimension, one term
    static constexpr uint32_t V_STAGE = TERMS * V_PLANE;
    static constexpr uint32_t RAW = kv_head_bytes(KIND, HD) / 2;  // a page's keys or values of a head
    static_assert(RAW % 16 == 0, "bulk copies");
};

// The WARPS warps that turn whole pages into operands, both K-major.
template <uint32_t KIND, uint32_t HD, uint32_t WARPS>
struct PageConverter {
    using T = PageTile<KIND, HD>;
    static constexpr uint32_t NB = T::NB, CODES = kv_code_bytes(KIND, HD), K_LO = T::HALVES * T::K_PLANE, V_LO = T::V_PLANE;
    static constexpr int TOP = KIND == KV_Q4_0 ? 26 : 22;  // a scale below 2^(e - 14) times 2^(TOP - e) times a code stays below 2^15
    uint32_t cw, lane, r, c;

    __device__ __forceinline__ PageConverter(uint32_t warp, uint32_t lane_) : cw(warp), lane(lane_), r(lane_ / 4), c(lane_ % 4) {}
    // 16 bytes (8 halves) of a key row: dimensions 32 b + 8 c .., in the 128-byte swizzle
    __device__ __forceinline__ uint32_t key_at(uint32_t stage, uint32_t row, uint32_t b) const {
        return stage + (b / 2) * T::K_PLANE + row * 128 + ((((b % 2) * 4 + c) ^ (row & 7)) << 4);
    }
    // 16 bytes (8 keys: 8 chunk ..) of a dimension's row of values
    __device__ __forceinline__ static uint32_t value_at(uint32_t stage, uint32_t d, uint32_t chunk) { return stage + d * 128 + ((chunk ^ (d & 7)) << 4); }
    // a page's keys; *inverse: what their products are multiplied by
    __device__ __forceinline__ void keys(uint32_t st, const uint8_t* raw, float* inverse) const {
        if constexpr (KIND == KV_F16) {
#pragma unroll
            for (uint32_t i = cw; i < 4 * NB; i += WARPS) {
                const uint32_t g = i / NB, b = i % NB;
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 1024 + lane * 16), y = *reinterpret_cast<const uint4*>(raw + i * 1024 + 512 + lane * 16);
                sts_v4(key_at(st, 16 * g + r, b), {x.x, x.y, y.x, y.y});
                sts_v4(key_at(st, 16 * g + r + 8, b), {x.z, x.w, y.z, y.w});
            }
        } else {
            constexpr uint32_t BLOCKS = KIND == KV_Q8_0 ? 1 : 2;  // of a 16-byte vector
            uint32_t top = 0x04000400u;  // the page's largest scale
#pragma unroll
            for (uint32_t i = 0; i < NB / 2; ++i) {  // 8 bytes a position and block pair
                const uint2 v = *reinterpret_cast<const uint2*>(raw + CODES + (i * 32 + lane) * 8);
                top = __vmaxu2(top, __vmaxu2(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu));
            }
            const int e = (int)(__reduce_max_sync(0xFFFFFFFFu, max(top >> 16, top & 0xFFFFu)) >> 10);
            const float f = power(TOP - e);
            if (cw == 0 && lane == 0) *inverse = power(e - TOP);
#pragma unroll 2
            for (uint32_t i = cw; i < 4 * NB / BLOCKS; i += WARPS) {
                const uint32_t g = i / (NB / BLOCKS), b0 = i % (NB / BLOCKS) * BLOCKS;
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 512 + lane * 16);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                const uint8_t* scales = raw + CODES + (g / 2 * 8 + r) * NB * 8 + g % 2 * 4;  // of rows r and r + 8, by block
#pragma unroll
                for (uint32_t o = 0; o < BLOCKS; ++o) {
                    const float2 s = __half22float2(bits_half2(*reinterpret_cast<const uint32_t*>(scales + (b0 + o) * 8)));
                    const __half2 s0 = __float2half2_rn(s.x * f), s1 = __float2half2_rn(s.y * f);
                    uint32_t hi[2][4], lo[2][4];
                    if constexpr (KIND == KV_Q8_0) {
                        scaled_terms(codes8<0>(w[0]), s0, &hi[0][0], &lo[0][0]), scaled_terms(codes8<2>(w[0]), s0, &hi[0][1], &lo[0][1]);
                        scaled_terms(codes8<0>(w[1]), s0, &hi[0][2], &lo[0][2]), scaled_terms(codes8<2>(w[1]), s0, &hi[0][3], &lo[0][3]);
                        scaled_terms(codes8<0>(w[2]), s1, &hi[1][0], &lo[1][0]), scaled_terms(codes8<2>(w[2]), s1, &hi[1][1], &lo[1][1]);
                        scaled_terms(codes8<0>(w[3]), s1, &hi[1][2], &lo[1][2]), scaled_terms(codes8<2>(w[3]), s1, &hi[1][3], &lo[1][3]);
                    } else {
#pragma unroll
                        for (uint32_t q = 0; q < 2; ++q) {
                            const uint32_t u = w[2 * o + q];
                            scaled_terms(codes4<0>(u), s0, &hi[0][2 * q], &lo[0][2 * q]), scaled_terms(codes4<1>(u), s0, &hi[0][2 * q + 1], &lo[0][2 * q + 1]);
                            scaled_terms(codes4<2>(u), s1, &hi[1][2 * q], &lo[1][2 * q]), scaled_terms(codes4<3>(u), s1, &hi[1][2 * q + 1], &lo[1][2 * q + 1]);
                        }
                    }
                    const uint32_t at0 = key_at(st, 16 * g + r, b0 + o), at1 = key_at(st, 16 * g + r + 8, b0 + o);
                    sts_v4(at0, hi[0]), sts_v4(at0 + K_LO, lo[0]);
                    sts_v4(at1, hi[1]), sts_v4(at1 + K_LO, lo[1]);
                }
            }
        }
    }
    // values: keys run along a row of the tile, so four lanes' words are transposed: lane c then has eight keys of two
    // dimensions (halves: of one).  inverse: what the products of each block are multiplied by.
    __device__ __forceinline__ void values(uint32_t st, const uint8_t* raw, float* inverse) const {
        if constexpr (KIND == KV_F16) {
#pragma unroll
            for (uint32_t i = cw; i < 8 * NB; i += WARPS) {
                const uint32_t g = i / (2 * NB), b = i / 2 % NB, m = i % 2;
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 512 + lane * 16);
                uint32_t w[4] = {x.x, x.y, x.z, x.w};
                transpose4(w, c);
                sts_v4(value_at(st, 32 * b + 4 * r + 2 * m + c % 2, 2 * g + c / 2), w);
            }
        } else {
            constexpr uint32_t BLOCKS = KIND == KV_Q8_0 ? 1 : 2;
#pragma unroll 2
            for (uint32_t i = cw; i < 4 * NB / BLOCKS; i += WARPS) {
                const uint32_t g = i / (NB / BLOCKS), b0 = i % (NB / BLOCKS) * BLOCKS;
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 512 + lane * 16);
                uint32_t w[4] = {x.x, x.y, x.z, x.w};
                transpose4(w, c);
                // lanes 0 .. 15 (and again 16 .. 31) have the block's scales of positions 32 (lane / 8) + lane % 8 + 8 k
                __half2 mine[BLOCKS];  // of the group's positions: lane % 8 and that + 8, in the lanes of its 32 positions
#pragma unroll
                for (uint32_t o = 0; o < BLOCKS; ++o) {
                    const uint2 s = *reinterpret_cast<const uint2*>(raw + CODES + ((lane & 15) * NB + b0 + o) * 8);
                    const uint32_t t = __vmaxu2(__vmaxu2(s.x & 0x7FFF7FFFu, s.y & 0x7FFF7FFFu), 0x04000400u);
                    const int e = (int)(__reduce_max_sync(0xFFFFFFFFu, max(t >> 16, t & 0xFFFFu)) >> 10);
                    mine[o] = scaled(g % 2 ? s.y : s.x, power(TOP - e));
                    if (g == 0 && lane == 0) inverse[b0 + o] = power(e - TOP);
                }
                // two neighbouring positions' scales: of the half that a lane has (Q4_0: of both halves, of the lane's block)
                auto pair = [&](uint32_t q, uint32_t h) {  // positions 8 h + 2 q, 8 h + 2 q + 1
                    uint32_t u[2];
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        u[k] = __shfl_sync(0xFFFFFFFFu, half2_bits(mine[0]), g / 2 * 8 + 2 * q + k);
                        if constexpr (BLOCKS == 2) {
                            const uint32_t other = __shfl_sync(0xFFFFFFFFu, half2_bits(mine[BLOCKS - 1]), g / 2 * 8 + 2 * q + k);
                            u[k] = c / 2 ? other : u[k];
                        }
                    }
                    return bits_half2(h ? __byte_perm(u[0], u[1], 0x7632) : __byte_perm(u[0], u[1], 0x5410));
                };
                if constexpr (KIND == KV_Q8_0) {
                    uint32_t hi[2][4], lo[2][4];
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) {
                        const __half2 s = pair(q, c % 2);
                        scaled_terms(codes8<0>(w[q]), s, &hi[0][q], &lo[0][q]), scaled_terms(codes8<2>(w[q]), s, &hi[1][q], &lo[1][q]);
                    }
#pragma unroll
                    for (uint32_t y = 0; y < 2; ++y) {
                        const uint32_t at = value_at(st, 32 * b0 + 4 * r + 2 * (c / 2) + y, 2 * g + c % 2);
                        sts_v4(at, hi[y]), sts_v4(at + V_LO, lo[y]);
                    }
                } else {
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        uint32_t hi[2][4], lo[2][4];
#pragma unroll
                        for (uint32_t q = 0; q < 4; ++q) {
                            const __half2 s = pair(q, h);
                            scaled_terms(h ? codes4<2>(w[q]) : codes4<0>(w[q]), s, &hi[0][q], &lo[0][q]);
                            scaled_terms(h ? codes4<3>(w[q]) : codes4<1>(w[q]), s, &hi[1][q], &lo[1][q]);
                        }
#pragma unroll
                        for (uint32_t y = 0; y < 2; ++y) {
                            const uint32_t at = value_at(st, 32 * (b0 + c / 2) + 4 * r + 2 * (c % 2) + y, 2 * g + h);
                            sts_v4(at, hi[y]), sts_v4(at + V_LO, lo[y]);
                        }
                    }
                }
            }
        }
    }
};

}  // namespace

}  // namespace jq
