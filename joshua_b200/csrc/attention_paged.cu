// Attention of one new token per sequence over the pages of the quantised cache.
//
// out[b, head, :] = sum_t p_t V_t / sum_t p_t, p_t = 2^(s_t - max), s_t = scale log2(e) q . K_t, t = 0 .. len[b] - 1, in one
// pass with a running maximum and sum.  A warp takes STEP positions of a kv head and all query rows that share it:
//   scores   S^T = K Q^T as m16n8k16 products, keys (codes as they are: whole numbers or halves, exact in f16) the 16-row
//            operand, query rows the 8 columns, in two f16 terms under a power of two of their row (22 bits).  The accumulator
//            of a block of 32 dimensions is scaled by the block's factor and added in f32.
//            Codes of 8 and 4 bits stand in the low bits of a half as they are, 4-bit ones in bits 4 .. 7: a subnormal number, the
//            code plus its bias times 2^-24 (2^-20), which the products take exactly.  The bias times the sum of the query's terms
//            is where their sums begin.  (The products are aligned by their exponents before they are added, and a subnormal's
//            is that of 2^-14: with 4-bit codes in bits 0 .. 3 the result was off by 2.9e-6 of itself, so by 5e-7.)
//   output   O^T = V^T P^T, values the 16-row operand; probabilities times the value's scale of the block, under a power of two
//            of the step's largest scale, in two f16 terms (22 bits below the largest).  Accumulators hold a step, not the
//            sequence: the tensor core adds with truncation, the running output is added round-to-nearest.
// Up to four query rows stand as four pairs of columns (term, term): one product does both terms.
//
// Every code is read once and serves all query heads of its kv head.  Long batches are bound by memory: 64 sequences of up to
// 8192 positions, 32 heads on 8 of 128 in eight bits, 568 MB in 103 us (5.5 TB/s, 84% of a copy), with 48% of the issue slots.
// Four bits are bound by instructions (24 sequences of up to 16384, 32 heads on 4 of 128, 84 MB: 42 us; 50% of the issue slots by
// three warps a scheduler, whose chains of product, softmax and product leave the rest), short batches by the chain of one
// piece (one sequence of 1000: 10 us, of which about 1 the cut, 4 the steps, 5 the joining within and across CTAs).
#include <cooperative_groups.h>

#include "attention_paged.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;

__device__ __forceinline__ uint4 ld_stream(const uint8_t* p) {  // read once: not kept in L1
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ void prefetch_l2(const uint8_t* p, uint32_t bytes) {
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// d = A B + (c0, c1) in the columns of this lane
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1));
}
// the 8x8 transpose between the accumulator's layout (row = position) and the B operand's (row of lanes = column)
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t t;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(v));
    return t;
}
__device__ __forceinline__ uint32_t split1(float a) {  // (term, term)
    const float h = __half2float(__float2half_rn(a));
    return half2_bits(__floats2half2_rn(h, a - h));
}
template <uint32_t KIND_, uint32_t HD_>
struct Step {
    static constexpr uint32_t KIND = KIND_, HD = HD_, NB = HD / 32, BITS = KIND == KV_F16 ? 16 : KIND == KV_Q8_0 ? 8 : 4;
    static constexpr uint32_t HEAD = kv_head_bytes(KIND, HD);  // a head of a page
    // positions at a time: 4 KB of keys and of values, 32 registers a lane each (heads of 256 in halves: 64).  Four bits: 2 KB;
    // 64 positions spill (24 ragged sequences of up to 16384, 32 / 4 heads of 128: 49.1 us, with 32 positions 41.7)
    static constexpr uint32_t WANT = (KIND == KV_Q4_0 ? 32 : 64) * 128 * 4 / (HD * BITS), POS = WANT < 16 ? 16 : WANT > 64 ? 64 : WANT;
    static constexpr uint32_t GROUPS = POS / 16, VECS = POS * HD * BITS / 8 / 512;
    static constexpr uint32_t SW = KIND == KV_F16 ? 1 : POS / 16;  // words of two scales a block
};

// One step's keys or values, a lane's share: codes, scales of positions lane / 4 + 8 i by block.
template <class T>
struct Rows {
    uint4 c[T::VECS];
    uint32_t s[T::NB][T::SW];

    // KEEP: other warps of the SM read it too
    template <bool KEEP = false>
    __device__ __forceinline__ void load(const uint8_t* part, uint32_t at, uint32_t lane) {
        const uint8_t* p = part + at * (T::HD * T::BITS / 8) + lane * 16;
#pragma unroll
        for (uint32_t i = 0; i < T::VECS; ++i) c[i] = KEEP ? __ldg(reinterpret_cast<const uint4*>(p + i * 512)) : ld_stream(p + i * 512);
        if constexpr (T::KIND != KV_F16) {
            const uint8_t* q = part + kv_code_bytes(T::KIND, T::HD) + ((at / 32 * 8 + lane / 4) * T::NB) * 8;
            if constexpr (T::POS == 16) {
#pragma unroll
                for (uint32_t b = 0; b < T::NB; ++b) s[b][0] = __ldg(reinterpret_cast<const uint32_t*>(q + b * 8 + at % 32 / 4));
            } else {
#pragma unroll
                for (uint32_t h = 0; h < T::POS / 32; ++h)
#pragma unroll
                    for (uint32_t b = 0; b < T::NB; b += 2) {
                        const uint4 v = __ldg(reinterpret_cast<const uint4*>(q + h * (64 * T::NB) + b * 8));
                        s[b][2 * h] = v.x, s[b][2 * h + 1] = v.y, s[b + 1][2 * h] = v.z, s[b + 1][2 * h + 1] = v.w;
                    }
            }
        }
    }
    __device__ __forceinline__ uint32_t word(uint32_t vec, uint32_t i) const {
        return i == 0 ? c[vec].x : i == 1 ? c[vec].y : i == 2 ? c[vec].z : c[vec].w;
    }
    // scale of position lane / 4 + 8 i
    __device__ __forceinline__ float scale(uint32_t b, uint32_t i) const {
        const float2 f = __half22float2(bits_half2(s[b][i / 2]));
        return i % 2 ? f.y : f.x;
    }
    // A operand of 16 keys (group a) and 16 dimensions (half h of block b); codes with their bias, times 2^-KEY_SHIFT
    static constexpr int KEY_SHIFT = T::KIND == KV_Q8_0 ? 24 : T::KIND == KV_Q4_0 ? 20 : 0;
    __device__ __forceinline__ void key(uint32_t a, uint32_t b, uint32_t h, uint32_t (&r)[4]) const {
        if constexpr (T::KIND == KV_F16) {
            const uint32_t v = (a * T::NB + b) * 2 + h;
            r[0] = word(v, 0), r[1] = word(v, 2), r[2] = word(v, 1), r[3] = word(v, 3);
        } else if constexpr (T::KIND == KV_Q8_0) {
            const uint32_t v = a * T::NB + b, x = word(v, h), y = word(v, 2 + h);
            r[0] = __byte_perm(x, 0, 0x4140), r[1] = __byte_perm(y, 0, 0x4140);
            r[2] = __byte_perm(x, 0, 0x4342), r[3] = __byte_perm(y, 0, 0x4342);
        } else {
            const uint32_t x = word(a * (T::NB / 2) + b / 2, b % 2 * 2 + h);
            r[0] = x << 4 & 0x00F000F0u, r[1] = x >> 4 & 0x00F000F0u, r[2] = x & 0x00F000F0u, r[3] = x >> 8 & 0x00F000F0u;
        }
    }
    // A operand of 16 dimensions (tile m of block b) and 16 positions (group a)
    __device__ __forceinline__ void value(uint32_t a, uint32_t b, uint32_t m, uint32_t (&r)[4]) const {
        if constexpr (T::KIND == KV_F16) {
            const uint32_t v = (a * T::NB + b) * 2 + m;
            r[0] = word(v, 0), r[1] = word(v, 1), r[2] = word(v, 2), r[3] = word(v, 3);
        } else if constexpr (T::KIND == KV_Q8_0) {
            const uint32_t v = a * T::NB + b, x = word(v, 2 * m), y = word(v, 2 * m + 1);
            r[0] = codes8<0>(x), r[1] = codes8<2>(x), r[2] = codes8<0>(y), r[3] = codes8<2>(y);
        } else {
            const uint32_t x = word(a * (T::NB / 2) + b / 2, b % 2 * 2 + m);
            r[0] = codes4<0>(x), r[1] = codes4<1>(x), r[2] = codes4<2>(x), r[3] = codes4<3>(x);
        }
    }
};

// Query rows of a warp: NT tiles of eight columns.  PAIRS: four rows, (term, term) in neighbouring columns; else eight rows a
// tile, the terms as two products.  A lane's rows are those of its accumulator columns: lane % 4, or 8 t + 2 (lane % 4) + {0, 1}.
template <class T, uint32_t NT, bool PAIRS>
struct Queries {
    static constexpr uint32_t ROWS = PAIRS ? 4 : 8 * NT, MINE = PAIRS ? 1 : 2 * NT;
    // words in shared memory: the B operand, [tile][block half][term][lane] pairs (PAIRS: in registers), and what its sums begin
    // with, [tile][block][lane % 4] pairs
    static constexpr uint32_t OPERAND = PAIRS ? 0 : NT * (T::HD / 16) * 2 * 64, WORDS = OPERAND + NT * T::NB * 8;
};

template <class T, uint32_t NT, bool PAIRS>
struct Attend {
    using Q = Queries<T, NT, PAIRS>;
    static constexpr uint32_t HD = T::HD, NB = T::NB, GROUPS = T::GROUPS, MINE = Q::MINE, COLS = PAIRS ? 1 : 2;
    uint32_t qf[PAIRS ? 2 * NB : 1][2];  // B operand of the query rows, in registers (PAIRS)
    const uint32_t* q_shared;            // the rest of it
    float rf[MINE];                      // what a row's scores are multiplied by
    float mx[MINE], sum[MINE];           // running maximum; sum of this lane's positions
    float o[NB][2][NT][2 * COLS];        // dimensions 4 (lane / 4) + 2 m + {0, 1} of a block, by column

    __device__ __forceinline__ void reset() {
#pragma unroll
        for (uint32_t i = 0; i < MINE; ++i) mx[i] = -INFINITY, sum[i] = 0.0f;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b)
#pragma unroll
            for (uint32_t m = 0; m < 2; ++m)
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                    for (uint32_t i = 0; i < 2 * COLS; ++i) o[b][m][t][i] = 0.0f;
    }

    // `row(i)`: query row i as a pointer to HD floats, NULL for none.  With shared memory: all lanes of the warp write, and
    // other warps may read after a barrier.
    template <class F>
    __device__ __forceinline__ void load_queries(F row, float scale, uint32_t lane, uint32_t* shared) {
        const uint32_t n = lane / 4, c = lane % 4;
        q_shared = shared;
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t) {
            const float* src = row(PAIRS ? n / 2 : 8 * t + n);
            float x[NB][8], amax = 0.0f;
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                const float4 u = src ? *reinterpret_cast<const float4*>(src + 32 * b + 8 * c) : zero;
                const float4 v = src ? *reinterpret_cast<const float4*>(src + 32 * b + 8 * c + 4) : zero;
                const float w[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 8; ++i) x[b][i] = w[i], amax = fmaxf(amax, fabsf(w[i]));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
            // a power of two that puts the row's largest value just below 2^15
            const uint32_t e = __float_as_uint(amax) >> 23, bits = e == 255 ? 127u : min(254u, 268u - e);
            const float up = __uint_as_float(bits << 23);
            const float down = (bits == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((254u - bits) << 23)) * scale *
                               (1.44269504f * (float)(1 << Rows<T>::KEY_SHIFT));
#pragma unroll
            for (uint32_t b = 0; b < NB; ++b) {
                float sum = 0.0f;  // of the terms of this lane's column
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    uint32_t hi[2], lo[2];
                    split2(x[b][4 * h] * up, x[b][4 * h + 1] * up, &hi[0], &lo[0]);
                    split2(x[b][4 * h + 2] * up, x[b][4 * h + 3] * up, &hi[1], &lo[1]);
                    auto of = [](uint32_t w) {
                        const float2 f = __half22float2(bits_half2(w));
                        return f.x + f.y;
                    };
                    if constexpr (PAIRS) {
                        qf[2 * b + h][0] = n % 2 ? lo[0] : hi[0], qf[2 * b + h][1] = n % 2 ? lo[1] : hi[1];
                        sum += of(qf[2 * b + h][0]) + of(qf[2 * b + h][1]);
                    } else {
                        uint2* to = reinterpret_cast<uint2*>(shared) + ((t * 2 * NB + 2 * b + h) * 2) * 32 + lane;
                        to[0] = make_uint2(hi[0], hi[1]), to[32] = make_uint2(lo[0], lo[1]);
                        sum += of(hi[0]) + of(lo[0]) + of(hi[1]) + of(lo[1]);
                    }
                }
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 1);
                sum += __shfl_xor_sync(0xFFFFFFFFu, sum, 2);
                sum *= (T::KIND == KV_F16 ? 0.0f : T::KIND == KV_Q8_0 ? -128.0f : -8.0f) / (float)(1 << Rows<T>::KEY_SHIFT);
                const float b0 = __shfl_sync(0xFFFFFFFFu, sum, 8 * c), b1 = __shfl_sync(0xFFFFFFFFu, sum, 8 * c + 4);
                if (T::KIND != KV_F16 && n == 0)
                    *reinterpret_cast<float2*>(shared + Q::OPERAND + ((t * NB + b) * 4 + c) * 2) = make_float2(b0, b1);
            }
            if constexpr (PAIRS) {
                rf[0] = __shfl_sync(0xFFFFFFFFu, down, 8 * c);
            } else {
                rf[2 * t] = __shfl_sync(0xFFFFFFFFu, down, 8 * c), rf[2 * t + 1] = __shfl_sync(0xFFFFFFFFu, down, 8 * c + 4);
            }
        }
        __syncwarp();
    }

    // s[group][tile][...]: position lane / 4 (+ 8 in the upper half) by column
    __device__ __forceinline__ void scores(const Rows<T>& k, uint32_t lane, float (&s)[GROUPS][NT][2 * COLS]) const {
#pragma unroll
        for (uint32_t a = 0; a < GROUPS; ++a)
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                for (uint32_t i = 0; i < 2 * COLS; ++i) s[a][t][i] = 0.0f;
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            uint2 q[2][NT][PAIRS ? 1 : 2];
            float2 begin[NT];
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t) {
                if constexpr (T::KIND == KV_F16)
                    begin[t] = make_float2(0.0f, 0.0f);
                else
                    begin[t] = *reinterpret_cast<const float2*>(q_shared + Q::OPERAND + ((t * NB + b) * 4 + lane % 4) * 2);
            }
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t) {
                    if constexpr (PAIRS) {
                        q[h][t][0] = make_uint2(qf[2 * b + h][0], qf[2 * b + h][1]);
                    } else {
                        const uint2* from = reinterpret_cast<const uint2*>(q_shared) + ((t * 2 * NB + 2 * b + h) * 2) * 32 + lane;
                        q[h][t][0] = from[0], q[h][t][1] = from[32];
                    }
                }
#pragma unroll
            for (uint32_t a = 0; a < GROUPS; ++a) {
                uint32_t r[2][4];
                k.key(a, b, 0, r[0]), k.key(a, b, 1, r[1]);
                float up = 1.0f, down = 1.0f;
                if constexpr (T::KIND != KV_F16) up = k.scale(b, 2 * a), down = k.scale(b, 2 * a + 1);
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t) {
                    float d[4];
                    constexpr int LAST = PAIRS ? 0 : 1;
                    mma16816(d, r[0], q[0][t][LAST].x, q[0][t][LAST].y, begin[t].x, begin[t].y);
                    mma16816(d, r[1], q[1][t][LAST].x, q[1][t][LAST].y);
                    if constexpr (!PAIRS) mma16816(d, r[0], q[0][t][0].x, q[0][t][0].y), mma16816(d, r[1], q[1][t][0].x, q[1][t][0].y);
                    if constexpr (PAIRS) {
                        s[a][t][0] = fmaf(d[0] + d[1], up, s[a][t][0]), s[a][t][1] = fmaf(d[2] + d[3], down, s[a][t][1]);
                    } else {
                        s[a][t][0] = fmaf(d[0], up, s[a][t][0]), s[a][t][1] = fmaf(d[1], up, s[a][t][1]);
                        s[a][t][2] = fmaf(d[2], down, s[a][t][2]), s[a][t][3] = fmaf(d[3], down, s[a][t][3]);
                    }
                }
            }
        }
    }

    // scores -> probabilities under the new maximum; positions from `valid` on are nothing.  alpha: of what was before.
    __device__ __forceinline__ void softmax(float (&s)[GROUPS][NT][2 * COLS], uint32_t valid, uint32_t lane, float (&alpha)[MINE]) {
        float nm[MINE];
#pragma unroll
        for (uint32_t i = 0; i < MINE; ++i) nm[i] = mx[i];
#pragma unroll
        for (uint32_t a = 0; a < GROUPS; ++a)
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t c = 0; c < COLS; ++c) {
                        const uint32_t i = COLS * t + c;
                        float& x = s[a][t][COLS * h + c];
                        x = 16 * a + 8 * h + lane / 4 < valid ? x * rf[i] : -INFINITY;
                        nm[i] = fmaxf(nm[i], x);
                    }
#pragma unroll
        for (uint32_t i = 0; i < MINE; ++i) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) nm[i] = fmaxf(nm[i], __shfl_xor_sync(0xFFFFFFFFu, nm[i], o));
            alpha[i] = ex2(mx[i] - nm[i]);
            mx[i] = nm[i], sum[i] *= alpha[i];
        }
#pragma unroll
        for (uint32_t a = 0; a < GROUPS; ++a)
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t c = 0; c < COLS; ++c) {
                        const uint32_t i = COLS * t + c;
                        float& x = s[a][t][COLS * h + c];
                        x = ex2(x - nm[i]);
                        sum[i] += x;
                    }
    }

    // B operands of the probabilities times up[i], the factor of position lane / 4 + 8 i
    struct Terms {
        uint32_t b[GROUPS][NT][PAIRS ? 1 : 2][2];
    };
    __device__ __forceinline__ void terms(const float (&p)[GROUPS][NT][2 * COLS], const float (&up)[2 * GROUPS], Terms& w) const {
#pragma unroll
        for (uint32_t a = 0; a < GROUPS; ++a)
#pragma unroll
            for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h) {
                    if constexpr (PAIRS) {
                        w.b[a][t][0][h] = transpose8(split1(p[a][t][h] * up[2 * a + h]));
                    } else {
                        uint32_t hi, lo;
                        split2(p[a][t][2 * h] * up[2 * a + h], p[a][t][2 * h + 1] * up[2 * a + h], &hi, &lo);
                        w.b[a][t][0][h] = transpose8(hi), w.b[a][t][1][h] = transpose8(lo);
                    }
                }
    }

    __device__ __forceinline__ void output(const float (&p)[GROUPS][NT][2 * COLS], Rows<T>& v, uint32_t valid, uint32_t lane,
                                           const float (&alpha)[MINE]) {
        Terms w;
        float up[2 * GROUPS], down = 1.0f / 16384.0f;
        bool moved = false;
#pragma unroll
        for (uint32_t i = 0; i < MINE; ++i) moved |= alpha[i] != 1.0f;
        moved = __any_sync(0xFFFFFFFFu, moved);
        if constexpr (T::KIND == KV_F16) {
#pragma unroll
            for (uint32_t i = 0; i < 2 * GROUPS; ++i) up[i] = 16384.0f;
            terms(p, up, w);
            if (valid < T::POS) {  // what stands behind the last position may be no number
                const uint32_t c = lane % 4 * 2;
#pragma unroll
                for (uint32_t i = 0; i < T::VECS; ++i) {
                    const uint32_t first = i / (2 * NB) * 16 + c;
                    const uint32_t low = (first < valid ? 0xFFFFu : 0u) | (first + 1 < valid ? 0xFFFF0000u : 0u);
                    const uint32_t high = (first + 8 < valid ? 0xFFFFu : 0u) | (first + 9 < valid ? 0xFFFF0000u : 0u);
                    v.c[i].x &= low, v.c[i].y &= low, v.c[i].z &= high, v.c[i].w &= high;
                }
            }
        } else if (valid < T::POS) {
#pragma unroll
            for (uint32_t i = 0; i < 2 * GROUPS; i += 2) {
                const uint32_t at = 8 * i + lane / 4, keep = (at < valid ? 0xFFFFu : 0u) | (at + 8 < valid ? 0xFFFF0000u : 0u);
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b) v.s[b][i / 2] &= keep;
            }
        }
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            if constexpr (T::KIND != KV_F16) {
                uint32_t top = 0x04000400u;  // not below the smallest normal number
#pragma unroll
                for (uint32_t i = 0; i < T::SW; ++i) top = __vmaxu2(top, v.s[b][i] & 0x7FFF7FFFu);
                const uint32_t e = __reduce_max_sync(0xFFFFFFFFu, max(top >> 16, top & 0xFFFFu)) >> 10;
                const float f = __uint_as_float((156u - e) << 23);  // 2^(29 - e): the largest scale times f is below 2^15
                down = __uint_as_float((98u + e) << 23);
#pragma unroll
                for (uint32_t i = 0; i < 2 * GROUPS; ++i) up[i] = v.scale(b, i) * f;
                terms(p, up, w);
            }
#pragma unroll
            for (uint32_t m = 0; m < 2; ++m) {
                float d[NT][4];
#pragma unroll
                for (uint32_t a = 0; a < GROUPS; ++a) {
                    uint32_t r[4];
                    v.value(a, b, m, r);
#pragma unroll
                    for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
                        for (int term = PAIRS ? 0 : 1; term >= 0; --term) {
                            if (a == 0 && term == (PAIRS ? 0 : 1))
                                mma16816(d[t], r, w.b[a][t][term][0], w.b[a][t][term][1], 0.0f, 0.0f);
                            else
                                mma16816(d[t], r, w.b[a][t][term][0], w.b[a][t][term][1]);
                        }
                }
#pragma unroll
                for (uint32_t t = 0; t < NT; ++t) {
                    float (&x)[2 * COLS] = o[b][m][t];
                    if (moved) {
#pragma unroll
                        for (uint32_t i = 0; i < 2 * COLS; ++i) x[i] *= alpha[PAIRS ? 0 : 2 * t + i % 2];
                    }
                    if constexpr (PAIRS) {
                        x[0] = fmaf(d[t][0] + d[t][1], down, x[0]), x[1] = fmaf(d[t][2] + d[t][3], down, x[1]);
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) x[i] = fmaf(d[t][i], down, x[i]);
                    }
                }
            }
        }
    }

    // [ROWS][HD] sums, then maxima and sums of exponentials of the rows
    __device__ __forceinline__ void store(float* to, uint32_t lane) {
        const uint32_t g = lane / 4, c = lane % 4;
#pragma unroll
        for (uint32_t t = 0; t < NT; ++t)
#pragma unroll
            for (uint32_t i = 0; i < COLS; ++i) {
                const uint32_t row = PAIRS ? c : 8 * t + 2 * c + i, mine = PAIRS ? 0 : 2 * t + i;
#pragma unroll
                for (uint32_t b = 0; b < NB; ++b)
                    *reinterpret_cast<float4*>(to + row * HD + 32 * b + 4 * g) =
                        make_float4(o[b][0][t][i], o[b][0][t][COLS + i], o[b][1][t][i], o[b][1][t][COLS + i]);
                float l = sum[mine];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xFFFFFFFFu, l, x);
                if (g == 0) to[Q::ROWS * HD + row] = mx[mine], to[Q::ROWS * HD + Q::ROWS + row] = l;
            }
    }
};

// The pages of one sequence from page `first` on: ids of 32 at a time, a lane each, and a page's tile of a head requested from
// memory (into L2) one page ahead.
template <class T>
struct Pages {
    const PagedArgs& a;
    const int32_t* table;
    uint32_t kvh, lane, have, end;  // first page whose id is held; page behind the last one wanted
    int32_t ids;
    bool lost;  // some id is outside the cache

    __device__ __forceinline__ void fetch(uint32_t from) {
        const uint32_t p = from + lane;
        have = from;
        ids = p < end ? (p < a.common ? a.c.table : table)[p] : 0;
    }
    __device__ __forceinline__ const uint8_t* tile(uint32_t p) {
        if (p - have >= 32) fetch(p);
        const int32_t id = __shfl_sync(0xFFFFFFFFu, ids, p - have);
        const bool fine = id >= 0 && (uint32_t)id < a.c.n_pages;
        lost |= !fine;
        return a.c.pages + ((uint64_t)(fine ? id : 0) * a.c.n_kv + kvh) * T::HEAD;
    }
    // the tile, and the next one asked for
    __device__ __forceinline__ const uint8_t* enter(uint32_t p) {
        const uint8_t* t = tile(p);
        if (p + 1 < end) {
            const uint8_t* next = tile(p + 1);
            if (lane == 0) prefetch_l2(next, T::HEAD);
        }
        return t;
    }
};

// A row's joined pieces: lane i has dimensions 4 i .. 4 i + 3 (HD 256: also those 128 behind; HD 64: lanes 0 .. 15).
template <uint32_t HD>
struct Joined {
    static constexpr uint32_t N = HD <= 128 ? 1 : HD / 128;
    float4 x[N];
    float top, den;

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        top = -INFINITY, den = 0.0f;
    }
    // n more pieces by a warp: piece(i): [ROWS][HD] sums, maxima, sums of exponentials.  OTHERS: other CTAs have just written them.
    template <uint32_t ROWS, bool OTHERS, class F>
    __device__ __forceinline__ void add(uint32_t n, F piece, uint32_t row, uint32_t lane) {
        auto load = [](auto* q) { return OTHERS ? __ldcg(q) : *q; };
        for (uint32_t i0 = 0; i0 < n; i0 += 32) {
            const uint32_t cnt = min(32u, n - i0);
            const float* mine = piece(i0 + min(lane, cnt - 1));
            const float m = lane < cnt ? load(mine + ROWS * HD + row) : -INFINITY, l = lane < cnt ? load(mine + ROWS * HD + ROWS + row) : 0.0f;
            float t = fmaxf(top, m);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xFFFFFFFFu, t, o));
            const float old = piece_weight(top, t), w = lane < cnt ? piece_weight(m, t) : 0.0f;
            float d = w * l;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
            den = fmaf(den, old, d), top = t;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) x[k].x *= old, x[k].y *= old, x[k].z *= old, x[k].w *= old;
#pragma unroll 4
            for (uint32_t j = 0; j < cnt; ++j) {
                const float f = __shfl_sync(0xFFFFFFFFu, w, j);
                const float* from = piece(i0 + j) + row * HD + 4 * lane;
#pragma unroll
                for (uint32_t k = 0; k < N; ++k) {
                    const float4 v = HD >= 128 || lane < HD / 4 ? load(reinterpret_cast<const float4*>(from + 128 * k)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    x[k].x = fmaf(f, v.x, x[k].x), x[k].y = fmaf(f, v.y, x[k].y), x[k].z = fmaf(f, v.z, x[k].z), x[k].w = fmaf(f, v.w, x[k].w);
                }
            }
        }
    }
    // ... and those of the leading pages, four on their way together
    __device__ __forceinline__ void add_lead(const PagedArgs& a, uint32_t kvh, uint32_t row, uint32_t lane) {
        constexpr uint32_t AT_ONCE = 4;
        const uint64_t rows = (uint64_t)a.c.n_seq * a.group, stride = a.c.n_kv * rows, all = a.lead_splits * stride, at = kvh * rows + row;
        for (uint32_t j0 = 0; j0 < a.lead_splits; j0 += AT_ONCE) {
            float4 v[AT_ONCE][N];
            float m[AT_ONCE], l[AT_ONCE], t = top;
#pragma unroll
            for (uint32_t j = 0; j < AT_ONCE; ++j) {
                const bool is = j0 + j < a.lead_splits;
                const uint64_t from = at + (j0 + j) * stride;
#pragma unroll
                for (uint32_t k = 0; k < N; ++k)
                    v[j][k] = is && (HD >= 128 || lane < HD / 4) ? *reinterpret_cast<const float4*>(a.lead + from * HD + 4 * lane + 128 * k)
                                                                 : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                m[j] = is ? a.lead[all * HD + from] : -INFINITY, l[j] = is ? a.lead[all * HD + all + from] : 0.0f;
                t = fmaxf(t, m[j]);
            }
            const float old = piece_weight(top, t);
            den *= old, top = t;
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) x[k].x *= old, x[k].y *= old, x[k].z *= old, x[k].w *= old;
#pragma unroll
            for (uint32_t j = 0; j < AT_ONCE; ++j) {
                const float f = piece_weight(m[j], t);
                den = fmaf(f, l[j], den);
#pragma unroll
                for (uint32_t k = 0; k < N; ++k) {
                    x[k].x = fmaf(f, v[j][k].x, x[k].x), x[k].y = fmaf(f, v[j][k].y, x[k].y);
                    x[k].z = fmaf(f, v[j][k].z, x[k].z), x[k].w = fmaf(f, v[j][k].w, x[k].w);
                }
            }
        }
    }
    // the row of the result: nothing where there was nothing
    __device__ __forceinline__ void finish(const PagedArgs& a, uint32_t b, uint32_t kvh, uint32_t in_group, uint32_t lane) {
        if (a.lead_splits) add_lead(a, kvh, b * a.group + in_group, lane);
        const float inv = den == 0.0f ? 0.0f : 1.0f / den;
        float* to = a.out + b * a.out_stride + (uint64_t)(kvh * a.group + in_group) * HD + 4 * lane;
#pragma unroll
        for (uint32_t k = 0; k < N; ++k)
            if (HD >= 128 || lane < HD / 4)
                *reinterpret_cast<float4*>(to + 128 * k) = make_float4(x[k].x * inv, x[k].y * inv, x[k].z * inv, x[k].w * inv);
    }
};

// A segment's beginning and end in steps (1 / 2 / 3 / 4: 64 sequences of up to 8192 107.4 / 101.4 / 101.5 / 101.6 us, 512 of up to
// 200 45.2 / 41.2 / 42.0 / 43.6; its kernel alone).
constexpr uint32_t SEG_UNITS = 2;
// Where no segment has more than so many units for each warp of a CTA, CTAs take whole segments, and none is joined across CTAs (32
// heads on 8 of 128, 8-bit, 4 sequences of 500: 9.8 us, cut anywhere 11.0; 512 of up to 200 39.5 and 41.2; one of 300 7.9 and 7.5.
// With 3 units: 16 sequences of 1000 15.3 us, cut anywhere 13.5).
constexpr uint32_t WHOLE_UNITS = 2;

// Positions of a sequence's own (behind the leading pages), or -1 where its length is out of range.
__device__ __forceinline__ int32_t own_positions(const PagedArgs& a, uint32_t b) {
    const int32_t n = a.len[b];
    if (n < 0 || (uint32_t)n > a.c.table_stride * KV_PAGE || (n > 0 && (uint32_t)n < a.common * KV_PAGE)) return -1;
    return n == 0 ? 0 : n - (int32_t)(a.done * KV_PAGE);
}

// The sequences' work stands in one row of units: sequence by sequence, head group by head group, SEG_UNITS for beginning and
// ending a segment (its queries, its result), then its steps.  It is cut into equal pieces, one a warp, whatever the lengths (short
// segments: first into CTAs' whole ones); a CTA's warps have neighbouring pieces.  Pieces of one segment (sequence, head group) are
// joined within the CTA, then, where a segment spans CTAs, by the last one of them to arrive, in order.
template <class T, bool PAIRS, uint32_t WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) attention_paged_kernel(PagedArgs a) {
    using At = Attend<T, 1, PAIRS>;
    constexpr uint32_t HD = T::HD, ROWS = At::Q::ROWS, PIECE = ROWS * (HD + 2);
    extern __shared__ __align__(16) uint32_t s_mem[];
    __shared__ uint32_t s_seg[2 * WARPS], s_from[2 * WARPS], s_to[2 * WARPS], s_scan[WARPS], s_most[WARPS], s_last[2], s_first[2];
    uint32_t* s_cum = s_mem;                                                       // [batch + 1] units of a head group in front of a sequence
    float* s_piece = reinterpret_cast<float*>(s_mem + ((a.c.n_seq + 4) & ~3u));    // [WARPS][2][PIECE]
    uint32_t* s_q = reinterpret_cast<uint32_t*>(s_piece + WARPS * 2 * PIECE);      // [WARPS] query operands
    pdl_trigger_all();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, batch = a.c.n_seq, groups = a.c.n_kv * a.split;
    if (tid < 2 * WARPS) s_seg[tid] = 0xFFFFFFFFu;
    // running sum of the sequences' units, a run of sequences a thread
    const uint32_t per = (batch + WARPS * 32 - 1) / (WARPS * 32), b0 = min(batch, tid * per), b1 = min(batch, b0 + per);
    uint32_t mine = 0, most = 0;
    auto units_of = [&](uint32_t b) {
        const uint32_t steps = (uint32_t)(max(own_positions(a, b), 0) + T::POS - 1) / T::POS;
        return steps ? steps + SEG_UNITS : 0;
    };
    for (uint32_t b = b0; b < b1; ++b) {
        const uint32_t n = units_of(b);
        mine += n, most = max(most, n);
    }
    most = __reduce_max_sync(0xFFFFFFFFu, most);
    uint32_t run = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, run, o);
        run += lane >= o ? up : 0;
    }
    if (lane == 31) s_scan[warp] = run, s_most[warp] = most;
    __syncthreads();
    for (uint32_t w = 0; w < WARPS; ++w) run += w < warp ? s_scan[w] : 0, most = max(most, s_most[w]);
    run -= mine;
    for (uint32_t b = b0; b < b1; ++b) {
        s_cum[b] = run;
        run += units_of(b);
    }
    if (b1 == batch && (b0 < b1 || tid == 0)) s_cum[batch] = run;
    __syncthreads();

    const uint64_t total = (uint64_t)s_cum[batch] * groups;
    const uint64_t workers = min((uint64_t)gridDim.x * WARPS, total);
    auto sequence_at = [&](uint64_t x) {  // the last sequence that begins at or in front of unit x: it has units
        uint32_t lo = 0, hi = batch;
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            (uint64_t)s_cum[mid] * groups <= x ? lo = mid : hi = mid;
        }
        return lo;
    };
    uint64_t at = 0, end = 0;
    if (most <= WHOLE_UNITS * WARPS) {  // the same in all CTAs; units fit 32 bits then
        static_assert((uint64_t)ATTENTION_MAX_BATCH * 4096 * WHOLE_UNITS * WARPS < 0xFFFFFFFFull, "units of 4096 heads a sequence");
        const uint32_t n = (uint32_t)total, each = n / gridDim.x, more = n % gridDim.x;
        auto begins = [&](uint32_t cta) {  // the segment that its first unit is in
            const uint32_t x = cta * each + cta * more / gridDim.x;
            if (x >= n) return n;
            const uint32_t b = sequence_at(x), first = s_cum[b] * groups, all = s_cum[b + 1] - s_cum[b];
            return first + (x - first) / all * all;
        };
        const uint32_t c0 = begins(blockIdx.x), units = begins(blockIdx.x + 1) - c0, warps = min(WARPS, units);
        if (warp < warps) at = c0 + warp * units / warps, end = c0 + (warp + 1) * units / warps;
    } else {
        const uint64_t me = (uint64_t)blockIdx.x * WARPS + warp;
        if (me < workers) at = me * total / workers, end = (me + 1) * total / workers;
    }
    At w;
    bool first_piece = true;
    // a piece of work: steps u0 .. u1 (perhaps none) of the `steps` of a sequence and head group
    struct Piece {
        uint32_t b, hg, u0, u1, steps, units;
    };
    auto piece_at = [&](uint64_t x, uint32_t b) {  // of the segment that unit x is in; b: at or in front of its sequence
        while (s_cum[b + 1] == s_cum[b] || (uint64_t)s_cum[b + 1] * groups <= x) ++b;
        const uint32_t all = s_cum[b + 1] - s_cum[b];
        const uint64_t in_seq = x - (uint64_t)s_cum[b] * groups;
        const uint32_t hg = (uint32_t)(in_seq / all), at0 = (uint32_t)(in_seq - (uint64_t)hg * all), at1 = (uint32_t)min((uint64_t)all, at0 + (end - x));
        auto step = [](uint32_t u) { return u > SEG_UNITS ? u - SEG_UNITS : 0; };
        return Piece{b, hg, step(at0), step(at1), all - SEG_UNITS, at1 - at0};
    };
    constexpr uint32_t PER_PAGE = KV_PAGE / T::POS;
    Pages<T> pages{a, a.c.table, 0, lane, 0, 0, 0, false};
    Rows<T> k, v;
    const uint8_t* tile = nullptr;
    auto begin = [&](const Piece& p) {  // its first keys on their way
        pages.table = a.c.table + (uint64_t)p.b * a.c.table_stride, pages.kvh = p.hg / a.split;
        pages.end = a.done + (p.u1 - 1) / PER_PAGE + 1, pages.lost = false;
        pages.fetch(a.done + p.u0 / PER_PAGE);
        tile = pages.enter(a.done + p.u0 / PER_PAGE);
        k.load(tile, p.u0 % PER_PAGE * T::POS, lane);
        // and its queries, into L1
        const uint32_t first = p.hg % a.split * ROWS, lines = min(ROWS, a.group - first) * (HD / 32);
        const float* q = a.q + p.b * a.q_stride + (uint64_t)(pages.kvh * a.group + first) * HD;
        for (uint32_t i = lane; i < lines; i += 32) asm volatile("prefetch.global.L1 [%0];" ::"l"(q + 32 * i));
    };
    // the next piece with steps, from unit `at` on, which moves behind it
    auto take = [&](uint32_t b) {
        Piece p{};
        while (at < end && p.u0 == p.u1) p = piece_at(at, b), at += p.units, b = p.b;
        return p;
    };
    Piece p{};
    if (at < end) {
        p = take(sequence_at(at));
        if (p.u0 < p.u1) begin(p);
    }
    while (p.u0 < p.u1) {
        const uint32_t kvh = p.hg / a.split, first = p.hg % a.split * ROWS, own = (uint32_t)own_positions(a, p.b);
        const float* q = a.q + p.b * a.q_stride + (uint64_t)(kvh * a.group + first) * HD;
        w.load_queries([&](uint32_t i) -> const float* { return first + i < a.group ? q + i * HD : nullptr; }, a.scale, lane,
                       s_q + warp * At::Q::WORDS);
        w.reset();
        Piece next{};
        bool lost = false;
        for (uint32_t u = p.u0; u < p.u1; ++u) {
            const uint32_t valid = min(own - u * T::POS, T::POS);
            v.load(tile + T::HEAD / 2, u % PER_PAGE * T::POS, lane);
            float s[T::GROUPS][1][2 * At::COLS], alpha[At::MINE];
            w.scores(k, lane, s);
            if (u + 1 < p.u1) {
                if ((u + 1) % PER_PAGE == 0) tile = pages.enter(a.done + (u + 1) / PER_PAGE);
                k.load(tile, (u + 1) % PER_PAGE * T::POS, lane);
            } else {
                lost = pages.lost;
                next = take(p.b);
                if (next.u0 < next.u1) begin(next);
            }
            w.softmax(s, valid, lane, alpha);
            w.output(s, v, valid, lane, alpha);
        }
        if (lost) {
#pragma unroll
            for (uint32_t i = 0; i < At::MINE; ++i) w.sum[i] = NAN;
            if (lane == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
        }
        const uint32_t slot = 2 * warp + (first_piece ? 0 : 1);
        float* to = s_piece + slot * PIECE;
        __syncwarp();
        w.store(to, lane);
        __syncwarp();
        if (p.u0 == 0 && p.u1 == p.steps) {
#pragma unroll 2
            for (uint32_t row = 0; row < min(ROWS, a.group - first); ++row) {
                Joined<HD> y;
                y.clear();
                y.template add<ROWS, false>(1, [&](uint32_t) { return to; }, row, lane);
                y.finish(a, p.b, kvh, first + row, lane);
            }
        } else {
            if (lane == 0) s_seg[slot] = p.b * groups + p.hg, s_from[slot] = p.u0, s_to[slot] = p.u1;
            first_piece = false;
        }
        p = next;
    }
    __syncthreads();
    // Pieces of segments that no warp has whole.  They stand in order, a segment's one after another; a warp joins a row of one.
    // What the CTA has whole is done; of others (its first and its last at most) the joined pieces go to memory, and the last CTA
    // to bring some joins them all.
    static_assert(2 * WARPS <= 32, "a lane a slot");
    const uint32_t seg_of = lane < 2 * WARPS ? s_seg[lane] : 0xFFFFFFFFu;
    const uint32_t held = __ballot_sync(0xFFFFFFFFu, seg_of != 0xFFFFFFFFu);
    // the held slots' numbers in order, one a lane
    const uint32_t n_held = __popc(held);
    uint32_t slot_of = 0;
    for (uint32_t m = held, i = 0; m; m &= m - 1, ++i) slot_of = lane == i ? __ffs(m) - 1 : slot_of;
    const uint32_t seg = __shfl_sync(0xFFFFFFFFu, seg_of, slot_of);  // of the lane-th held slot
    const uint32_t before = __shfl_up_sync(0xFFFFFFFFu, seg, 1);
    const uint32_t starts = __ballot_sync(0xFFFFFFFFu, lane < n_held && (lane == 0 || seg != before));
    const uint32_t n_seg = __popc(starts);
    uint32_t open = 0, open_seg[2] = {0, 0};  // 1: a segment that begins in an earlier CTA, 2: one that begins here and goes on
    for (uint32_t i = 0, m = starts; i < n_seg; ++i, m &= m - 1) {
        const uint32_t first = __ffs(m) - 1, behind = m & (m - 1) ? __ffs(m & (m - 1)) - 1 : n_held, n = behind - first;
        const uint32_t sg = __shfl_sync(0xFFFFFFFFu, seg, first), sb = sg / groups, hg = sg % groups, steps = s_cum[sb + 1] - s_cum[sb] - SEG_UNITS;
        const bool begins = s_from[__shfl_sync(0xFFFFFFFFu, slot_of, first)] == 0;
        const bool whole = begins && s_to[__shfl_sync(0xFFFFFFFFu, slot_of, behind - 1)] == steps;
        if (!whole) open |= 1u << begins, open_seg[begins] = sg;
        for (uint32_t row = (warp + WARPS - i * ROWS % WARPS) % WARPS; row < ROWS; row += WARPS) {  // segments in turn to different warps
            const uint32_t kvh = hg / a.split, in_group = hg % a.split * ROWS + row;
            Joined<HD> y;
            y.clear();
            y.template add<ROWS, false>(
                n, [&](uint32_t j) { return (const float*)(s_piece + __shfl_sync(0xFFFFFFFFu, slot_of, first + j) * PIECE); }, row, lane);
            if (whole) {
                if (in_group < a.group) y.finish(a, sb, kvh, in_group, lane);
            } else {
                float* dst = a.part + ((uint64_t)blockIdx.x * 2 + begins) * PIECE;
#pragma unroll
                for (uint32_t k = 0; k < Joined<HD>::N; ++k)
                    if (HD >= 128 || lane < HD / 4) __stcg(reinterpret_cast<float4*>(dst + row * HD + 4 * lane + 128 * k), y.x[k]);
                if (lane == 0) __stcg(dst + ROWS * HD + row, y.top), __stcg(dst + ROWS * HD + ROWS + row, y.den);
            }
        }
    }
    if (open) {  // the same in all threads
        __threadfence();
        __syncthreads();
        // CTAs that have a piece of it, from c0 on.  Of the segments whose first step is a CTA's only its last goes on behind it, so c0
        // tells open segments apart.
        auto owners = [&](uint32_t sg, uint32_t* c0) {
            const uint32_t sb = sg / groups, units = s_cum[sb + 1] - s_cum[sb];
            const uint64_t x = (uint64_t)s_cum[sb] * groups + (uint64_t)(sg % groups) * units, x0 = x + SEG_UNITS, x1 = x + units - 1;
            *c0 = (uint32_t)(((x0 + 1) * workers - 1) / total / WARPS);
            return (uint32_t)(((x1 + 1) * workers - 1) / total / WARPS) - *c0 + 1;
        };
        if (tid < 2) {
            s_last[tid] = 0;
            if (open >> tid & 1) {
                uint32_t c0;
                const uint32_t sg = open_seg[tid], n = owners(sg, &c0);
                if (atomicAdd(a.arrived + c0, 1) == n - 1) a.arrived[c0] = 0, s_last[tid] = n, s_first[tid] = c0;
            }
            __threadfence();
        }
        __syncthreads();
        for (uint32_t i = warp; i < 2 * ROWS; i += WARPS) {
            const uint32_t which = i / ROWS, row = i % ROWS, n = s_last[which], c0 = s_first[which];
            if (n == 0) continue;
            const uint32_t sg = open_seg[which], hg = sg % groups, in_group = hg % a.split * ROWS + row;
            if (in_group >= a.group) continue;
            Joined<HD> y;
            y.clear();
            y.template add<ROWS, true>(
                n, [&](uint32_t j) { return (const float*)(a.part + ((uint64_t)(c0 + j) * 2 + (j == 0)) * PIECE); }, row, lane);
            y.finish(a, sg / groups, hg / a.split, in_group, lane);
        }
    }
    // sequences without steps of their own
    for (uint32_t sb = blockIdx.x; sb < batch; sb += gridDim.x) {
        if (s_cum[sb + 1] != s_cum[sb]) continue;
        const int32_t own = own_positions(a, sb);
        if (own < 0 && tid == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
        if (own < 0 || a.len[sb] == 0) {
            for (uint32_t i = tid; i < a.n_q * HD; i += WARPS * 32) a.out[sb * a.out_stride + i] = own < 0 ? NAN : 0.0f;
        } else {
            for (uint32_t i = warp; i < a.n_q; i += WARPS) {
                Joined<HD> y;
                y.clear();
                y.finish(a, sb, i / a.group, i % a.group, lane);
            }
        }
    }
}

// The leading pages, once for all sequences: query rows of the batch (of one kv head) are the columns, NT * 8 a warp.  A CTA's
// warps take `sets` sets of rows and WARPS / sets parts of the CTA's share of the pages.  Bound by instructions, as the kernel
// above: a pass of 16 rows takes 2.6 times as long as a sequence's own pass of four over the same positions, and serves more
// (7 sequences of 32 heads on 8 of 128 in halves, 1024 pages: 101 us, by themselves 299).
template <class T, uint32_t NT, uint32_t WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) attention_lead_kernel(PagedArgs a, float* __restrict__ lead, uint32_t sets) {
    using At = Attend<T, NT, false>;
    constexpr uint32_t HD = T::HD, ROWS = At::Q::ROWS, PIECE = ROWS * (HD + 2), AREA = PIECE > At::Q::WORDS ? PIECE : At::Q::WORDS;
    constexpr uint32_t PER_PAGE = KV_PAGE / T::POS;
    extern __shared__ __align__(16) uint32_t s_mem[];  // [WARPS][AREA]: query operands, then the warps' sums
    pdl_trigger_all();
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, set = warp % sets, part = warp / sets, parts = WARPS / sets;
    const uint32_t split = blockIdx.x, kvh = blockIdx.z, rows = a.c.n_seq * a.group, first = (blockIdx.y * sets + set) * ROWS;
    const uint32_t p0 = (uint32_t)((uint64_t)split * a.done / gridDim.x), p1 = (uint32_t)((uint64_t)(split + 1) * a.done / gridDim.x);
    const uint32_t steps = (p1 - p0) * PER_PAGE, u0 = part * steps / parts, u1 = (part + 1) * steps / parts;
    At w;
    w.load_queries(
        [&](uint32_t i) -> const float* {
            const uint32_t row = first + i;
            return row < rows ? a.q + row / a.group * a.q_stride + (uint64_t)(kvh * a.group + row % a.group) * HD : nullptr;
        },
        a.scale, lane, s_mem + warp * AREA);
    w.reset();
    if (u0 < u1) {
        Pages<T> pages{a, a.c.table, kvh, lane, 0, p0 + (u1 - 1) / PER_PAGE + 1, 0, false};
        pages.fetch(p0 + u0 / PER_PAGE);
        const uint8_t* tile = pages.enter(p0 + u0 / PER_PAGE);
        Rows<T> k, v;
        k.template load<true>(tile, u0 % PER_PAGE * T::POS, lane);
        for (uint32_t u = u0; u < u1; ++u) {
            v.template load<true>(tile + T::HEAD / 2, u % PER_PAGE * T::POS, lane);
            float s[T::GROUPS][NT][2 * At::COLS], alpha[At::MINE];
            w.scores(k, lane, s);
            if (u + 1 < u1) {
                if ((u + 1) % PER_PAGE == 0) tile = pages.enter(p0 + (u + 1) / PER_PAGE);
                k.template load<true>(tile, (u + 1) % PER_PAGE * T::POS, lane);
            }
            w.softmax(s, T::POS, lane, alpha);
            w.output(s, v, T::POS, lane, alpha);
        }
        if (pages.lost) {
#pragma unroll
            for (uint32_t i = 0; i < At::MINE; ++i) w.sum[i] = NAN;
            if (lane == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
        }
    }
    __syncthreads();  // the query operands have been read
    float* pieces = reinterpret_cast<float*>(s_mem);
    w.store(pieces + warp * AREA, lane);
    // the parts of the CTA's warps and of the cluster's CTAs (page splits of the same rows) are joined, a share of the rows a CTA
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), n = sets * ROWS * (HD / 4);
    const uint64_t all = (uint64_t)(gridDim.x / ctas) * a.c.n_kv * rows, base = ((uint64_t)(split / ctas) * a.c.n_kv + kvh) * rows;
    const uint32_t i1 = (rank + 1) * n / ctas;
    for (uint32_t i = rank * n / ctas + tid; i < i1; i += WARPS * 32) {
        const uint32_t d = i % (HD / 4) * 4, r = i / (HD / 4) % ROWS, st = i / (HD / 4) / ROWS;
        const uint32_t row = (blockIdx.y * sets + st) * ROWS + r;
        if (row >= rows) continue;
        float top = -INFINITY, den = 0.0f;
        for (uint32_t c = 0; c < ctas; ++c)
            for (uint32_t j = 0; j < parts; ++j) top = fmaxf(top, cluster.map_shared_rank(pieces, c)[(j * sets + st) * AREA + ROWS * HD + r]);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t c = 0; c < ctas; ++c)
            for (uint32_t j = 0; j < parts; ++j) {
                const float* p = cluster.map_shared_rank(pieces, c) + (j * sets + st) * AREA;
                const float f = piece_weight(p[ROWS * HD + r], top);
                const float4 y = *reinterpret_cast<const float4*>(p + r * HD + d);
                sum.x = fmaf(f, y.x, sum.x), sum.y = fmaf(f, y.y, sum.y), sum.z = fmaf(f, y.z, sum.z), sum.w = fmaf(f, y.w, sum.w);
                den = fmaf(f, p[ROWS * HD + ROWS + r], den);
            }
        *reinterpret_cast<float4*>(lead + (base + row) * HD + d) = sum;
        if (d == 0) lead[all * HD + base + row] = top, lead[all * HD + all + base + row] = den;
    }
    cluster.sync();  // the others have read this CTA's pieces
}

constexpr uint32_t LEAD_WARPS = 8;
// Warps of a CTA, one a SM, by the registers that a step needs (64 sequences of up to 8192, heads of 128: 10 warps 108.9 us, 12
// 106.0, 16, which spill, 120.9).
constexpr uint32_t ap_warps(uint32_t hd) { return hd == 256 ? 8 : 12; }
constexpr uint32_t lead_tiles(uint32_t hd) { return hd == 256 ? 1 : 2; }  // columns of a warp / 8, by its registers too

// From so many query rows of a kv head on, the leading pages' kernel is the one of attention_lead.cu, whose time hardly depends
// on them up to 128 (32 query heads on 8 of 128, 8-bit, 64 pages, the whole call with 100 positions of each sequence's own, the pages
// taken once on either side: 16 rows 22.7 us, by attention_lead_kernel 21.9; 24 rows 22.7 and 23.4; 32 rows 23.2 and 24.4; 64 rows
// 23.9 and 29.8; 128 rows 26.0 and 42.4; 512 rows 56 and 113.  16 heads on 8, four bits, 200 pages: 16 rows 36.7 and 29.8, 24 rows
// 37.1 and 36.4, 32 rows 37.4 and 37.5, 48 rows 38.3 and 52.0).
constexpr uint32_t LEAD_TILE_ROWS = 32;
// Leading pages are taken once for all sequences where that saves so many elements of keys (positions times dimensions, over all
// passes) that the launch more and its joining, about 8 us, are won back; below, every sequence reads them by itself, most of it
// from L2.  32 heads on 8 of 128, 8-bit, 64 pages, batch 8: once 23.7 us, by themselves 19.3; batch 12: 24.0 and 24.3; 16: 24.3
// and 27.6; 32: 26.0 and 43.6.  Batch 128: 4 pages 34.3 and 27.3, 8 pages 35.8 and 35.0.  Heads of 256 (16 on 4, 64 pages): batch
// 32 54.0 and 48.8, 64 85.8 and 90.4, 128 149 and 169.
constexpr double LEAD_SAVES = 32e6;

// How a call is cut up: the same for its scratch and its launches.
struct PagedPlan {
    uint32_t group, split, rows, grid;       // of the kernel over the sequences' own pages
    uint32_t lead, sets, blocks, splits;     // of the leading pages' kernel: pages, row sets of a CTA, row blocks, page splits
    bool tiles;                              // it is the one of attention_lead.cu
    uint32_t cluster;                        // splits that one cluster joins
    size_t part_at, lead_at, bytes;
};
PagedPlan plan(uint32_t batch, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t shared) {
    PagedPlan p{};
    p.group = n_q / n_kv;
    p.rows = p.group <= 4 ? 4 : 8;
    p.split = (p.group + p.rows - 1) / p.rows;
    p.grid = std::min((uint32_t)num_sms(), ATTENTION_MOST_CTAS);
    const uint32_t rows = batch * p.group, tiles = (rows + 8 * lead_tiles(hd) - 1) / (8 * lead_tiles(hd));
    p.tiles = hd <= 128 && rows >= LEAD_TILE_ROWS;
    // passes over the leading pages: a sequence's own is the unit, 128 rows of attention_lead.cu take as long as 5, 16 (heads of
    // 256: 8) rows of attention_lead_kernel as 2.6 (1.56)
    const double own = (double)batch * p.split, once = p.tiles ? 5.0 * ((rows + 127) / 128) : (hd == 256 ? 1.56 : 2.6) * tiles;
    p.lead = (own - once) * n_kv * hd * KV_PAGE * shared >= LEAD_SAVES ? shared : 0;
    if (p.lead) {
        p.sets = 1, p.cluster = 4;
        while (p.sets < LEAD_WARPS && p.sets < tiles) p.sets *= 2;
        p.blocks = p.tiles ? (rows + 127) / 128 : (tiles + p.sets - 1) / p.sets;
        // one wave of one CTA a SM.  Clusters of four: of eight, SMs of the GPU's groups stay idle, and 16 of them took two waves (16
        // heads on 4 of 128, batch 32, 256 pages: 54.6 us, 12 of eight 37.2, 32 of four 32.1)
        const uint32_t fit = std::max(1u, std::min(p.lead, (uint32_t)num_sms() / std::max(1u, p.blocks * n_kv)));
        while (p.cluster > fit) p.cluster /= 2;
        p.splits = std::min(fit, LEAD_MOST * p.cluster) / p.cluster * p.cluster;
    }
    // the counters in one place for all calls: what one writes behind them is no other one's counter
    p.part_at = ATTENTION_MOST_CTAS * 4;
    p.lead_at = p.part_at + ((size_t)p.grid * 2 * p.rows * (hd + 2) * 4 + 255) / 256 * 256;
    p.bytes = p.lead_at + (p.lead ? (size_t)(p.splits / p.cluster) * n_q * batch * (hd + 2) * 4 : 0);
    return p;
}

struct LaunchPaged {
    PagedArgs a;
    const PagedPlan& p;
    float* lead;
    int* error_flag;
    cudaStream_t s;

    template <class T, bool PAIRS>
    cudaError_t own() const {
        using At = Attend<T, 1, PAIRS>;
        constexpr uint32_t WARPS = ap_warps(T::HD), BYTES = WARPS * (2 * At::Q::ROWS * (T::HD + 2) + At::Q::WORDS) * 4;
        auto kern = attention_paged_kernel<T, PAIRS, WARPS>;
        static bool configured[MAX_DEVICES] = {};
        if (cudaError_t e = set_max_smem_once(kern, BYTES + (ATTENTION_MAX_BATCH + 4) * 4, configured); e != cudaSuccess) return e;
        return launch_pdl(kern, dim3(p.grid), WARPS * 32, BYTES + ((a.c.n_seq + 4) & ~3u) * 4, s, a);
    }
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        using T = Step<KIND, HD>;
        if (p.lead && p.tiles) {
            cudaError_t e = launch_attention_lead_tiles(a, lead, p.splits, p.blocks, p.cluster, error_flag, s);
            if (e != cudaSuccess) return e;
        } else if (p.lead) {
            using At = Attend<T, lead_tiles(HD), false>;
            constexpr uint32_t PIECE = At::Q::ROWS * (HD + 2), AREA = PIECE > At::Q::WORDS ? PIECE : At::Q::WORDS;
            auto kern = attention_lead_kernel<T, lead_tiles(HD), LEAD_WARPS>;
            static bool configured[MAX_DEVICES] = {};
            if (cudaError_t e = set_max_smem_once(kern, LEAD_WARPS * AREA * 4, configured); e != cudaSuccess) return e;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(p.splits, p.blocks, a.c.n_kv);
            cfg.blockDim = dim3(LEAD_WARPS * 32);
            cfg.dynamicSmemBytes = LEAD_WARPS * AREA * 4;
            cfg.stream = s;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = p.cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
            attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 2;
            cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a, lead, p.sets);
            if (e != cudaSuccess) return e;
        }
        return p.rows == 4 ? own<T, true>() : own<T, false>();
    }
};

}  // namespace

size_t attention_paged_scratch_bytes(uint32_t batch, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t shared) {
    return plan(batch, n_q, n_kv, hd, shared).bytes;
}

cudaError_t launch_attention_paged(const KvPages& c, const float* q, uint64_t q_stride, const int32_t* len, uint32_t n_q, float scale,
                                   uint32_t shared, float* out, uint64_t out_stride, void* scratch, int32_t* bad_pos, int* error_flag,
                                   cudaStream_t s) {
    const PagedPlan p = plan(c.n_seq, n_q, c.n_kv, c.hd, shared);
    uint8_t* mem = static_cast<uint8_t*>(scratch);
    float* lead = reinterpret_cast<float*>(mem + p.lead_at);
    const PagedArgs a{c, q, q_stride, len, n_q, p.group, p.split, scale, shared, p.lead, out, out_stride,
                      reinterpret_cast<uint32_t*>(mem), reinterpret_cast<float*>(mem + p.part_at), lead, p.lead ? p.splits / p.cluster : 0, bad_pos};
    cudaError_t e = for_kind(c.kind, c.hd, LaunchPaged{a, p, lead, error_flag, s});
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
