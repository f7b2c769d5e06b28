// Attention of chunks of new tokens over the quantised cache on the 5th-generation tensor cores.
//
// A tile is up to 128 query rows: the heads of a kv head of consecutive tokens of a sequence, token by token.  It goes over the pages
// that some of its tokens see, a page at a time, running maximum and sum in f32.  Terms as in attention_lead.cu: queries two f16 terms
// under a power of two of their row; codes times scales as two f16 terms (halves: one) under powers of two of a page's largest scale;
// probabilities two terms; of a product of two terms each the smallest of the four is left out.  Accumulators hold a score or one page
// of the output; the running output lives in registers.  Scores of positions that a row does not see become nothing
// before the maximum, their probabilities zeros; values behind the tile's last position are zeros in the products, and those that are
// not finite too: they are added at the end, to the rows that see them.
//
// The tiles' work stands in one row of units, tile by tile, kv head by kv head, SEG_UNITS for beginning and ending one, then its
// pages.  It is cut into equal pieces, one a CTA, none smaller than the join of a tile's parts makes worth while; what several CTAs have
// of a tile is joined by the last of them to arrive, in order.
//
// Warps: 0 .. 3 softmax, a thread a query row; 4 .. 7 add up the output, the same; 8 .. 15 first cut the work, then turn the pages' codes
// into swizzled tiles, two stages (half of them keys, half values); 16 issues the products; 17 copies the pages.  Tensor memory: the
// query's terms (the A operand of the scores), scores and probabilities (A of the output) of two pages, output of one: scores of a page
// are under way while the softmax has the one before and the output the one before that.
//
// What bounds it: three products of f16 terms a page and tile, 1.14 us at the rate of a library product.  512 tokens behind 3584, 32 heads on
// 8 of 128, eight bits: 99 us, 59 of them products (the tensor pipe 42% of the time, half of the issue slots, 930 W); 4096 behind 8192
// 1.74 to 1.78 ms, 1.26 of them (985 W, the power limit: 84% of the rate that a library product has under it); four tokens of 32
// sequences 116 us, 1.1 us a page, for tiles of 16 rows take the products of 128; four prompts of 500, heads of 64 in halves 45 us, half of
// it the tiles' beginnings and ends (with divisions for the rows' tokens 47.7).
//
// Every wait on an mbarrier is bounded.  A warp whose wait ran out waits for none any more, hands nothing on, and goes through the
// rest of its work so, which brings it to every barrier that others expect it at; the status flag is raised and the rows become NaN.
#include <algorithm>

#include "attention_chunk.cuh"
#include "attention_tiles.cuh"

namespace jq {

namespace {

constexpr uint32_t CQ = CHUNK_TILE_ROWS;     // query rows of a tile
constexpr uint32_t C_SOFT = 4, C_SUM = 4, C_CONV = 8;  // warps
constexpr uint32_t C_FIRST_CONV = C_SOFT + C_SUM, C_ISSUE = C_FIRST_CONV + C_CONV, C_LOAD = C_ISSUE + 1;
constexpr int UP = 6;                        // probabilities stand times 2^UP ..
constexpr float LAZY = 8.0f;                 // .. and are up to 2^LAZY: below 2^15
constexpr uint32_t C_HALF = C_CONV / 2;                // of the converters: for keys, the others for values
constexpr uint32_t C_THREADS = (C_ISSUE + 4) * 32;  // whole warpgroups: they trade registers
// Registers a thread: the launch has 640 x 96 = 61440, of which the issuer's warpgroup keeps 128 x 32, the softmax threads (32 scores, 32
// terms) 128 x 112, the converters 256 x 64 and those that add up the output (128 running sums, 32 new ones) 128 x 208: all of it.  With
// heads of 64 the latter have half the sums and leave the converters more.
// No role may spill in its loop: the tiles leave so little L1 that spills come back from L2 (512 tokens behind 3584: 108 -> 171 us).
constexpr int C_REGS_ISSUE = 32, C_REGS_SOFT = 112;
constexpr int c_regs_conv(uint32_t hd) { return hd == 64 ? 72 : 64; }
constexpr int c_regs_sum(uint32_t hd) { return hd == 64 ? 192 : 208; }
constexpr bool c_regs_fit(uint32_t hd) {
    return 128 * C_REGS_ISSUE + C_CONV * 32 * c_regs_conv(hd) + C_SOFT * 32 * C_REGS_SOFT + C_SUM * 32 * c_regs_sum(hd) <= C_THREADS * 96;
}
static_assert(c_regs_fit(64) && c_regs_fit(128), "registers");

constexpr uint32_t SEG_UNITS = 2;   // a tile's beginning and end in pages
// What joining a part takes the last CTA, in pages (16 tokens, 8 heads on one of 128: 8000 positions cut over all CTAs 148 us, with 0.7 / 1 /
// 1.5 / 3 here 46.6 / 46.9 / 50.5 / 55.1; 32 on 8, 1000 positions 41.2 and 32.0 / 31.6 / 33.9 / 36.1; 16000 62.0 and 64.6 / 67.8 / 65.3 / 69.8).
constexpr float JOIN_UNITS = 1.0f;
constexpr uint32_t C_PIECES = 96;   // pieces of a CTA at a time
constexpr uint32_t C_STAGE = 5;     // 16-byte vectors a row of the stage, one of them empty: no bank conflicts

// Pages first .. end - 1 of the list of pages that a tile sees: those of the sinks, then those from its window's first on.
struct ChunkPiece {
    uint32_t seq, row0, pos0;        // the sequence, its tile's first row and that one's position
    uint32_t tokens, kvh, head0;     // tokens of the tile, kv head, its first query head
    uint32_t first, end;
    uint32_t sinks, skip;            // pages of sinks; pages left out behind them
    uint32_t parts, owner;           // CTAs that have a part of the tile (1: it is whole here), the first of them
};

// what the warps share beside the tiles
struct ChunkShared {
    float ks[4];              // inverse scale of the keys, by page % 4
    float vs[4][4];           // inverse scales of the values' blocks, by page % 4 (halves: 1)
    uint8_t odd[4][C_HALF];   // values that are not finite, by page % 4 and converter
    uint8_t lost[16];         // a page id outside the cache, by page % 16
    float alpha[4][CQ];       // what the sums before are worth under the new maximum, by page % 4
    float stat[4][2][CQ];     // maxima and sums of a finished piece, by its last page % 4
    // page % 2: what the products wait for (operands in place, the result before read), that they are through
    uint64_t s_go[2], s_done[2], o_go[2], o_done[2], q_full;
    uint64_t rk_full[2], rk_empty[2], rv_full[2], rv_empty[2];  // the raw pages
    uint64_t drained;         // the products of a CTA that gives up
    uint32_t tmem_slot;
    int abort_flag;
    uint32_t last;            // this CTA was the last one to bring its part of a tile
    uint32_t scan[2][C_CONV], first_seg, end_seg;
    uint32_t named[C_SOFT], named_too[C_CONV];  // rows of all sequences, by warp: of the softmax, of the converters
    uint32_t pieces, batches;  // pieces of this batch; batches
    float4 stage[2][4][32][C_STAGE];  // of the softmax warps and of the output's: 16 dimensions of 32 rows on their way between lanes
    ChunkPiece piece[C_PIECES];
};

template <uint32_t V>
struct Constant {
    static constexpr uint32_t value = V;
};

// The WARPS warps that turn pages into operands: keys K-major (dimensions along a row), values MN-major (the same), so that no lane
// needs another's codes.  Only the first `valid` positions of a page are anyone's: what stands behind them does not count for the
// page's scales, and values there, or not finite, become zeros.  Scales are looked over once a page for what is not finite; the path
// without any has no masks.
template <uint32_t KIND, uint32_t HD, uint32_t WARPS>
struct ChunkConverter {
    using T = PageTile<KIND, HD>;
    static constexpr uint32_t NB = T::NB, CODES = kv_code_bytes(KIND, HD), K_LO = T::HALVES * T::K_PLANE, V_LO = T::V_PLANE;
    static constexpr uint32_t BLOCKS = KIND == KV_Q4_0 ? 2 : 1, COLS = NB / BLOCKS, ITEMS = 4 * COLS;  // blocks of a lane's 16 bytes
    static constexpr int TOP = KIND == KV_Q4_0 ? 26 : 22;  // a scale below 2^(e - 14) times 2^(TOP - e) times a code stays below 2^15
    static_assert(WARPS % COLS == 0, "a warp has blocks of its own");
    static_assert(CODES % 16 == 0 && K_LO % 1024 == 0 && V_LO % 1024 == 0 && TOP / 2 < 15, "vectors of codes, the swizzle's period, Up's factors");
    uint32_t cw, lane, r, c, b0;
    uint32_t key_to, value_to[2];  // places in a stage: keys of row r, values of positions 2 c and 2 c + 1

    __device__ __forceinline__ ChunkConverter(uint32_t warp, uint32_t lane_)
        : cw(warp), lane(lane_), r(lane_ / 4), c(lane_ % 4), b0(warp % COLS * BLOCKS) {
        key_to = b0 / 2 * T::K_PLANE + r * 128 + (((b0 % 2 * 4 + c) ^ r) << 4);
        for (uint32_t e = 0; e < 2; ++e)
            value_to[e] = b0 / 2 * (KV_PAGE * 128) + (2 * c + e) * 128 + (((b0 % 2 * 4 + r / 2) ^ (2 * c + e)) << 4) + r % 2 * 8;
    }
    // halfwords of positions at and at + 8 that are there; those of finite numbers
    __device__ __forceinline__ static uint32_t there(uint32_t at, uint32_t valid) {
        return (at < valid ? 0xFFFFu : 0u) | (at + 8 < valid ? 0xFFFF0000u : 0u);
    }
    __device__ __forceinline__ static uint32_t finite(uint32_t w) { return __vcmpltu2(w & 0x7FFF7FFFu, 0x7C007C00u); }
    // the largest magnitude of scales (four of a position unit in 8 bytes: positions at + 8 k), as bits; first those not finite too
    template <uint32_t N>
    __device__ __forceinline__ static uint32_t largest(uint2 (&v)[N], const uint32_t (&at)[N], uint32_t valid, bool* odd) {
        if (valid < KV_PAGE) {
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) v[i].x &= there(at[i], valid), v[i].y &= there(at[i] + 16, valid);
        }
        auto top_of = [&] {
            uint32_t t = 0x04000400u;  // not below the smallest normal number
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) t = __vmaxu2(t, __vmaxu2(v[i].x & 0x7FFF7FFFu, v[i].y & 0x7FFF7FFFu));
            return __reduce_max_sync(0xFFFFFFFFu, max(t >> 16, t & 0xFFFFu));
        };
        uint32_t top = top_of();
        *odd = top >= 0x7C00u;
        if (*odd) {
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) v[i].x &= finite(v[i].x), v[i].y &= finite(v[i].y);
            top = top_of();
        }
        return top;
    }
    // factors whose product is 2^(TOP - e)
    struct Up {
        __half2 a, b;
        __device__ __forceinline__ explicit Up(int e) {
            const int n = TOP - e, half = n >> 1;
            const uint32_t x = (uint32_t)(15 + half) << 10, y = (uint32_t)(15 + n - half) << 10;
            a = bits_half2(x | x << 16), b = bits_half2(y | y << 16);
        }
        __device__ __forceinline__ uint32_t of(uint32_t s) const { return half2_bits(__hmul2(__hmul2(bits_half2(s), a), b)); }
    };
    __device__ __forceinline__ static __half2 low(uint32_t s) { return bits_half2(__byte_perm(s, 0, 0x1010)); }
    __device__ __forceinline__ static __half2 high(uint32_t s) { return bits_half2(__byte_perm(s, 0, 0x3232)); }

    // a page's keys; *inverse: what their products are multiplied by
    __device__ __forceinline__ void keys(uint32_t stage, const uint8_t* raw, uint32_t valid, float* inverse) const {
        if constexpr (KIND == KV_F16) {
#pragma unroll 1
            for (uint32_t i = cw; i < ITEMS; i += WARPS) {
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 1024 + lane * 16);
                const uint4 y = *reinterpret_cast<const uint4*>(raw + i * 1024 + 512 + lane * 16);
                const uint32_t to = stage + key_to + i / COLS * 2048;
                sts_v4(to, {x.x, x.y, y.x, y.y}), sts_v4(to + 1024, {x.z, x.w, y.z, y.w});
            }
        } else {
            constexpr uint32_t N = NB / 2;  // 8-byte units of a lane
            uint2 v[N];
            uint32_t at[N];
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
                const uint32_t unit = lane * N + i;
                v[i] = *reinterpret_cast<const uint2*>(raw + CODES + unit * 8), at[i] = unit / NB / 8 * 32 + unit / NB % 8;
            }
            bool odd;
            const int e = (int)(largest(v, at, valid, &odd) >> 10);
            const Up up(e);
            if (cw == 0 && lane == 0) *inverse = power(e - TOP);
#pragma unroll 1
            for (uint32_t i = cw; i < ITEMS; i += WARPS) {
                const uint32_t g = i / COLS, to = stage + key_to + g * 2048;
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 512 + lane * 16);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
                const uint8_t* scales = raw + CODES + (g / 2 * 8 + r) * NB * 8 + g % 2 * 4 + b0 * 8;  // of rows r and r + 8, by block
#pragma unroll
                for (uint32_t o = 0; o < BLOCKS; ++o) {
                    const uint32_t s = up.of(*reinterpret_cast<const uint32_t*>(scales + o * 8));
                    const __half2 s0 = low(s), s1 = high(s);
                    uint32_t hi[2][4], lo[2][4];
                    if constexpr (KIND == KV_Q8_0) {
#pragma unroll
                        for (uint32_t q = 0; q < 2; ++q) {
                            scaled_terms(codes8<0>(w[q]), s0, &hi[0][2 * q], &lo[0][2 * q]);
                            scaled_terms(codes8<2>(w[q]), s0, &hi[0][2 * q + 1], &lo[0][2 * q + 1]);
                            scaled_terms(codes8<0>(w[2 + q]), s1, &hi[1][2 * q], &lo[1][2 * q]);
                            scaled_terms(codes8<2>(w[2 + q]), s1, &hi[1][2 * q + 1], &lo[1][2 * q + 1]);
                        }
                    } else {
#pragma unroll
                        for (uint32_t q = 0; q < 2; ++q) {
                            const uint32_t u = w[2 * o + q];
                            scaled_terms(codes4<0>(u), s0, &hi[0][2 * q], &lo[0][2 * q]);
                            scaled_terms(codes4<1>(u), s0, &hi[0][2 * q + 1], &lo[0][2 * q + 1]);
                            scaled_terms(codes4<2>(u), s1, &hi[1][2 * q], &lo[1][2 * q]);
                            scaled_terms(codes4<3>(u), s1, &hi[1][2 * q + 1], &lo[1][2 * q + 1]);
                        }
                    }
                    const uint32_t block = to ^ o << 6;  // the second block of a pair stands four 16-byte pieces on, in the swizzle
                    sts_v4(block, hi[0]), sts_v4(block + K_LO, lo[0]);
                    sts_v4(block + 1024, hi[1]), sts_v4(block + 1024 + K_LO, lo[1]);
                }
            }
        }
    }
    __device__ __forceinline__ static void sts_v2(uint32_t addr, uint32_t a, uint32_t b) {
        asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(addr), "r"(a), "r"(b) : "memory");
    }
    // Two dimensions (x = 0, 1) of the position of half h and place e: of a word of Q8_0 codes [x][e], of Q4_0 codes [e][h].
    template <uint32_t E, uint32_t H>
    __device__ __forceinline__ static uint32_t value_codes(uint32_t w) {
        if constexpr (KIND == KV_Q8_0) {
            return half2_bits(__hsub2(bits_half2(__byte_perm(w, 0x64646464u, E ? 0x4341 : 0x4240)), __float2half2_rn(1152.0f)));
        } else {  // 1024 + n and 1024 + 16 n
            constexpr uint32_t BYTE = 2 * E + H;
            const uint32_t t = __byte_perm(w, 0x64646464u, 0x4040 | BYTE << 8 | BYTE) & 0xFFF0FF0Fu;
            return half2_bits(__hfma2(bits_half2(t), __halves2half2(__float2half_rn(1.0f), __float2half_rn(0.0625f)),
                                      __halves2half2(__float2half_rn(-1032.0f), __float2half_rn(-72.0f))));
        }
    }
    // a page's values; inverse: what the products of each block are multiplied by.  True: some value that is there is not finite.
    __device__ __forceinline__ bool values(uint32_t stage, const uint8_t* raw, uint32_t valid, float* inverse) const {
        if constexpr (KIND == KV_F16) {
            bool odd = false;
#pragma unroll 1
            for (uint32_t i = cw; i < ITEMS; i += WARPS) {
                const uint32_t g = i / COLS;
                uint32_t w[2][4];
                __half2 zero = __float2half2_rn(0.0f);
                if (valid < KV_PAGE) zero = __float2half2_rn(NAN);  // looked at one by one
#pragma unroll
                for (uint32_t m = 0; m < 2; ++m) {
                    const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 1024 + m * 512 + lane * 16);
                    w[m][0] = x.x, w[m][1] = x.y, w[m][2] = x.z, w[m][3] = x.w;
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k) zero = __hfma2(bits_half2(w[m][k]), __float2half2_rn(0.0f), zero);
                }
                if (__any_sync(0xFFFFFFFFu, (half2_bits(zero) & 0x7FFF7FFFu) != 0)) {
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) {  // positions 16 g + 8 (k / 2 % 2) + 2 c and the next
                        uint32_t& x = w[k / 4][k % 4];
                        const uint32_t at = 16 * g + k / 2 % 2 * 8 + 2 * c;
                        x &= (at < valid ? 0xFFFFu : 0u) | (at + 1 < valid ? 0xFFFF0000u : 0u);
                        const uint32_t fine = finite(x);
                        odd |= fine != 0xFFFFFFFFu, x &= fine;
                    }
                }
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        const uint32_t order = e ? 0x7632 : 0x5410;
                        sts_v2(stage + value_to[e] + g * 2048 + h * 1024, __byte_perm(w[0][2 * h], w[0][2 * h + 1], order),
                               __byte_perm(w[1][2 * h], w[1][2 * h + 1], order));
                    }
            }
            return odd;
        } else {
            // lanes 0 .. 15 (and again 16 .. 31) have the block's scales of positions 32 (lane / 8) + lane % 8 + 8 k
            bool odd[BLOCKS], careful = valid < KV_PAGE;
            int e[BLOCKS];
#pragma unroll
            for (uint32_t o = 0; o < BLOCKS; ++o) {
                uint2 v[1] = {*reinterpret_cast<const uint2*>(raw + CODES + ((lane & 15) * NB + b0 + o) * 8)};
                const uint32_t at[1] = {(lane & 15) / 8 * 32 + lane % 8};
                e[o] = (int)(largest(v, at, valid, &odd[o]) >> 10);
                if (cw < COLS && lane == 0) inverse[b0 + o] = power(e[o] - TOP);
                careful |= odd[o];
            }
#pragma unroll 1
            for (uint32_t i = cw; i < ITEMS; i += WARPS) {
                const uint32_t g = i / COLS;
                const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 512 + lane * 16);
                const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (uint32_t o = 0; o < BLOCKS; ++o) {
                    const Up up(e[o]);
                    uint32_t s[2];  // of places e: halves h
#pragma unroll
                    for (uint32_t p = 0; p < 2; ++p) {
                        s[p] = *reinterpret_cast<const uint32_t*>(raw + CODES + ((g / 2 * 8 + 2 * c + p) * NB + b0 + o) * 8 + g % 2 * 4);
                        if (careful) s[p] &= there(16 * g + 2 * c + p, valid) & finite(s[p]);
                        s[p] = up.of(s[p]);
                    }
                    auto put = [&](auto place, auto half) {
                        constexpr uint32_t E = decltype(place)::value, H = decltype(half)::value;
                        const __half2 f = H ? high(s[E]) : low(s[E]);
                        uint32_t hi[2], lo[2];
#pragma unroll
                        for (uint32_t m = 0; m < 2; ++m)
                            scaled_terms(value_codes<E, H>(KIND == KV_Q8_0 ? w[2 * m + H] : w[2 * o + m]), f, &hi[m], &lo[m]);
                        const uint32_t to = (stage + value_to[E] + g * 2048 + H * 1024) ^ o << 6;
                        sts_v2(to, hi[0], hi[1]), sts_v2(to + V_LO, lo[0], lo[1]);
                    };
                    put(Constant<0>{}, Constant<0>{}), put(Constant<0>{}, Constant<1>{});
                    put(Constant<1>{}, Constant<0>{}), put(Constant<1>{}, Constant<1>{});
                }
            }
            bool some = odd[0];
            if constexpr (BLOCKS == 2) some |= odd[1];
            return some;
        }
    }
};

// Rows of a tile: `heads` (up to 128) places a token.
struct TileRows {
    uint32_t heads, inverse;
    __device__ __forceinline__ explicit TileRows(const PagedArgs& a) : heads(min(a.group, CQ)), inverse((65536 + heads - 1) / heads) {}
    __device__ __forceinline__ uint32_t token(uint32_t row) const { return row * inverse >> 16; }  // exact: row and heads are below 2^8
};

// Values: 64 dimensions along a row of 128 bytes, keys from row to row; 8 keys 1024 bytes apart, the next 64 dimensions a page of rows on.
__device__ __forceinline__ uint64_t umma_desc_values(uint32_t smem_addr) {
    return umma_desc(smem_addr) - ((uint64_t)1 << 16) + ((uint64_t)(KV_PAGE * 128 >> 4) << 16);
}


template <uint32_t KIND, uint32_t HD>
struct ChunkTile : PageTile<KIND, HD> {
    using P = PageTile<KIND, HD>;
    using P::HALVES, P::K_STAGE, P::RAW, P::V_STAGE;
    static constexpr uint32_t TILES = 2 * (K_STAGE + V_STAGE);
    static constexpr uint32_t SMEM = TILES + 4 * RAW + sizeof(ChunkShared);  // and the tiles in front of every sequence
    static_assert(SMEM + (ATTENTION_MAX_BATCH + 1) * 4 <= 227 * 1024, "shared memory");
    // tensor memory columns
    static constexpr uint32_t Q_HI = 0, Q_LO = HD / 2, S0 = HD, P0 = S0 + 2 * KV_PAGE, O = P0 + 2 * KV_PAGE;  // scores and probabilities of two pages
    static_assert(O + HD <= 512, "tensor memory");
};

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// The tiles of a sequence, and what one of them sees.
struct ChunkTiles {
    uint32_t per_tile, tiles, heads, blocks;  // tokens a tile; tiles; query heads of a tile, blocks of them a kv head

    __device__ __forceinline__ ChunkTiles(const PagedArgs& a, uint32_t rows) {
        heads = min(a.group, CQ), blocks = (a.group + CQ - 1) / CQ, per_tile = CQ / heads, tiles = (rows + per_tile - 1) / per_tile;
    }
};
struct TilePages {
    uint32_t sinks, skip, n;
    __device__ __forceinline__ TilePages(const SpanArgs& s, uint32_t pos0, uint32_t tokens) {
        const Sight see(s, pos0);
        const uint32_t low = see.low / KV_PAGE, end = (pos0 + tokens + KV_PAGE - 1) / KV_PAGE;
        sinks = min((uint32_t)(((uint64_t)see.sinks + KV_PAGE - 1) / KV_PAGE), low), skip = low - sinks, n = end - skip;
    }
};
// rows of a sequence that this kernel takes
__device__ __forceinline__ uint32_t tile_rows(const PagedArgs& a, const SequenceRows& s) { return s.n <= a.span.few || s.len <= 0 ? 0 : s.n; }

template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(C_THREADS, 1) attention_chunk_tiles_kernel(PagedArgs a, int* error_flag) {
    using T = ChunkTile<KIND, HD>;
    constexpr uint32_t HEAD = kv_head_bytes(KIND, HD);
    constexpr uint32_t PART = CHUNK_TILE_ROWS * (HD + 2);                  // floats of a part of a tile
    extern __shared__ __align__(1024) uint8_t smem[];  // K and V stages | raw keys, raw values | ChunkShared | s_tiles
    const uint32_t k_base = smem_u32(smem), v_base = k_base + 2 * T::K_STAGE;
    uint8_t* raw_k = smem + T::TILES;
    uint8_t* raw_v = raw_k + 2 * T::RAW;
    ChunkShared& sh = *reinterpret_cast<ChunkShared*>(raw_v + 2 * T::RAW);
    uint32_t* s_tiles = reinterpret_cast<uint32_t*>(&sh + 1);  // [batch + 1] tiles in front of a sequence

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, batch = a.c.n_seq;
    const bool aligned = k_base % 1024 == 0;  // the swizzle's period; no static shared memory stands in front
    if (KIND == KV_F16 && tid < 16) sh.vs[tid / 4][tid % 4] = 1.0f;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_go[i], C_HALF + C_SOFT);
            mbar_init(&sh.s_done[i], 1);
            mbar_init(&sh.o_go[i], C_HALF + C_SOFT + C_SUM);
            mbar_init(&sh.o_done[i], 1);
            mbar_init(&sh.rk_full[i], 1);
            mbar_init(&sh.rv_full[i], 1);
            mbar_init(&sh.rk_empty[i], C_HALF);
            mbar_init(&sh.rv_empty[i], C_HALF);
        }
        mbar_init(&sh.drained, 1);
        mbar_init(&sh.q_full, C_SOFT);
        sh.abort_flag = !aligned;
        mbar_fence_init();
    }
    if (warp == C_ISSUE) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_slot)), "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_slot;
    pdl_trigger();
    pdl_wait();
    bool ok = aligned;  // the same in all lanes of a warp; once false, the warp waits for nothing more
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        if (ok) ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
        return ok;
    };
    // Where all warps meet: in front of a batch of pieces and behind it.
    auto meet = [&] {
        if (!ok && lane == 0) *static_cast<volatile int*>(&sh.abort_flag) = 1;
        tc_fence_before();
        asm volatile("bar.sync 6, %0;" ::"n"(C_THREADS) : "memory");
        tc_fence_after();
    };

    if (warp < C_SOFT) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C_REGS_SOFT));
        // rows of sequences without positions, or with ones out of range
        uint32_t named = 0;
        for (uint32_t b = tid; b < batch; b += C_SOFT * 32) named += sequence_rows(a, b).n;
        named = __reduce_add_sync(0xFFFFFFFFu, named);
        if (lane == 0) sh.named[warp] = named;
        asm volatile("bar.sync 4, %0;" ::"n"(C_SOFT * 32) : "memory");
        named = 0;
        for (uint32_t w = 0; w < C_SOFT; ++w) named += sh.named[w];
        const bool fit = rows_fit(a, named);
        for (uint32_t b = blockIdx.x; b < batch; b += gridDim.x) {
            const SequenceRows sq = sequence_rows(a, b);
            if ((!fit || sq.lost || sq.len < 0) && tid == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
            if (!fit || sq.n <= a.span.few || sq.len > 0) continue;
            for (uint32_t k = 0; k < sq.n; ++k)
                for (uint32_t i = tid; i < a.n_q * HD; i += C_SOFT * 32) a.out[(sq.row + k) * a.out_stride + i] = sq.len < 0 ? NAN : 0.0f;
        }
        // ── softmax: a thread a query row ──
        const uint32_t row = tid, lanes = tmem + ((warp * 32) << 16);
        uint32_t g = 0;   // pages so far
        float rf = 0.0f;  // inverse scale of the query row, times log2(e) and the softmax scale
        // Rows come 16 dimensions of 8 rows a load, four lanes a row (a row a lane asks the cache for 32 lines a load: 128 rows of 128
        // took 4 us), and go to their lanes through the stage.
        const TileRows rows(a);
        auto rows_of = [&](const ChunkPiece& p, uint32_t i) -> const float4* {  // of row 8 i + lane / 4 of the warp, its lane % 4-th vector
            const uint32_t r = warp * 32 + 8 * i + lane / 4, t = rows.token(r), h = r - t * rows.heads;
            if (t >= p.tokens || p.head0 + h >= (p.kvh + 1) * a.group) return nullptr;
            return reinterpret_cast<const float4*>(a.q + (uint64_t)(p.row0 + t) * a.q_stride + (uint64_t)(p.head0 + h) * HD) + lane % 4;
        };
        auto load = [](const float4* from, uint32_t at) { return from ? from[at] : make_float4(0.0f, 0.0f, 0.0f, 0.0f); };
        // The largest magnitude of the thread's row, asked for a piece ahead: the row itself then comes from L2.
        auto largest = [&](const ChunkPiece& p) {
            float amax[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const float4* from = rows_of(p, i);
                amax[i] = 0.0f;
#pragma unroll
                for (uint32_t c = 0; c < HD / 16; ++c) {
                    const float4 v = load(from, 4 * c);
                    amax[i] = fmaxf(amax[i], fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                }
            }
            float mine = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                float x = amax[i];
                x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 1));
                x = fmaxf(x, __shfl_xor_sync(0xFFFFFFFFu, x, 2));
                x = __shfl_sync(0xFFFFFFFFu, x, lane % 8 * 4);
                mine = lane / 8 == i ? x : mine;
            }
            return mine;
        };
        // a piece's queries into tensor memory; the scores before have been worked out
        auto query = [&](const ChunkPiece& p, float amax) {
            // a power of two that puts the row's largest value just below 2^15, with the sign of the scale: the row's maximum is
            // looked for before the scores are multiplied by rf, which must not turn their order round
            const uint32_t e = __float_as_uint(amax) >> 23, bits = e == 255 ? 127u : min(254u, 268u - e);
            const float sc = copysignf(__uint_as_float(bits << 23), a.scale);
            rf = (bits == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((254u - bits) << 23)) * (fabsf(a.scale) * 1.44269504f);
            const float4* from[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) from[i] = rows_of(p, i);
            float4 (&stage)[32][C_STAGE] = sh.stage[0][warp];
            float4 v[4], next[4];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) next[i] = load(from[i], 0);
#pragma unroll 1
            for (uint32_t c = 0; c < HD / 16; ++c) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) v[i] = next[i];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                    if (c + 1 < HD / 16) next[i] = load(from[i], 4 * (c + 1));
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) stage[8 * i + lane / 4][lane % 4] = v[i];
                __syncwarp();
                uint32_t hi[8], lo[8];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float4 x = stage[lane][i];
                    split2(x.x * sc, x.y * sc, &hi[2 * i], &lo[2 * i]), split2(x.z * sc, x.w * sc, &hi[2 * i + 1], &lo[2 * i + 1]);
                }
                __syncwarp();
                tmem_st8(lanes + T::Q_HI + 8 * c, hi);
                tmem_st8(lanes + T::Q_LO + 8 * c, lo);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full);  // the first scores wait for the query's terms
        };
        float mx = -INFINITY;
        f32x2 sums = 0;  // sum and outputs times 2^UP, as the probabilities are
        // The probabilities of page g into tensor memory, when the products before the last have read theirs; seen (EDGE): the positions
        // that the row sees, a bit each.  Returns what the sums before are worth under the new maximum.
        auto page = [&](auto edge, uint32_t seen0, uint32_t seen1) {
            constexpr bool EDGE = decltype(edge)::value;
            const uint32_t from = lanes + T::S0 + (g & 1) * KV_PAGE, to = lanes + T::P0 + (g & 1) * KV_PAGE;
            float cms[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
            for (uint32_t c = 0; c < 2; ++c) {  // one copy of the code: what all warps do at a time has to stay in the instruction cache
                uint32_t r[32];
                tmem_ld32(from + 32 * c, r);
                const uint32_t seen = c ? seen1 : seen0;
#pragma unroll
                for (uint32_t i = 0; i < 32; i += 2) {
                    const float x = EDGE && !(seen >> i & 1) ? -INFINITY : __uint_as_float(r[i]);
                    const float y = EDGE && !(seen >> (i + 1) & 1) ? -INFINITY : __uint_as_float(r[i + 1]);
                    cms[i / 2 % 4] = max3(cms[i / 2 % 4], x, y);
                }
            }
            const float cm = fmaxf(max3(cms[0], cms[1], cms[2]), cms[3]);
            float f = KIND == KV_F16 ? rf : rf * sh.ks[g & 3], alpha = 1.0f;
            const float top = __fmul_rn(cm, f);
            if (top - mx > LAZY) alpha = ex2(mx - top), mx = top;  // 0 on the first page with something to see (mx = -inf)
            float base = (float)UP - (mx > -INFINITY ? mx : 0.0f);
            if (__any_sync(0xFFFFFFFFu, fabsf(base) >= FAR)) {
                const float less = mx > -INFINITY ? mx : 0.0f;
#pragma unroll 1
                for (uint32_t c = 0; c < KV_PAGE; c += 8) {
                    uint32_t r[8];
                    tmem_ld8(from + c, r);
#pragma unroll
                    for (uint32_t i = 0; i < 8; ++i) r[i] = __float_as_uint(__fsub_rn(__fmul_rn(__uint_as_float(r[i]), f), less));
                    tmem_st8(from + c, r);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                f = 1.0f, base = (float)UP;
            }
            const f32x2 ff = pair(f, f), shift = pair(base, base);
            f32x2 ps = 0;
            wait_all(&sh.o_done[g & 1], ((g >> 1) & 1) ^ 1);
            tc_fence_after();
#pragma unroll 1
            for (uint32_t c = 0; c < 2; ++c) {
                uint32_t r[32], w0[16], w1[16];
                tmem_ld32(from + 32 * c, r);
                const uint32_t seen = c ? seen1 : seen0;
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) {
                    const float2 y = both(fma2(pair(r[2 * i], r[2 * i + 1]), ff, shift));
                    float x0 = ex2(y.x), x1 = ex2(y.y);
                    if constexpr (EDGE) x0 = seen >> (2 * i) & 1 ? x0 : 0.0f, x1 = seen >> (2 * i + 1) & 1 ? x1 : 0.0f;
                    const f32x2 both_p = pair(x0, x1);
                    ps = add2(ps, both_p);
                    const __half2 h = __floats2half2_rn(x0, x1);
                    const float2 hf = __half22float2(h);
                    const float2 rest = both(fma2(pair(hf.x, hf.y), pair(-1.0f, -1.0f), both_p));
                    w0[i] = half2_bits(h), w1[i] = half2_bits(__floats2half2_rn(rest.x, rest.y));
                }
                tmem_st16(to + 16 * c, w0);
                tmem_st16(to + 32 + 16 * c, w1);
            }
            sums = fma2(sums, pair(alpha, alpha), ps);
            return alpha;
        };
        if (lane == 0) mbar_arrive(&sh.s_go[0]), mbar_arrive(&sh.s_go[1]);  // nothing to read in front of the first two
        meet();
        for (uint32_t turn = 0; turn < sh.batches; ++turn) {
            const uint32_t pieces = sh.pieces;
            float amax = pieces ? largest(sh.piece[0]) : 0.0f;
            for (uint32_t k = 0; k < pieces; ++k) {
                const ChunkPiece& p = sh.piece[k];
                query(p, amax);
                if (k + 1 < pieces) amax = largest(sh.piece[k + 1]);
                const uint32_t n = p.end - p.first;
                const Sight see(a.span, p.pos0 + rows.token(row)), last_see(a.span, p.pos0 + p.tokens - 1);
                mx = -INFINITY, sums = 0;
                for (uint32_t j = 0; j < n; ++j, ++g) {
                    const uint32_t u = p.first + j, base = (u < p.sinks ? u : u + p.skip) * KV_PAGE;
                    wait_all(&sh.s_done[g & 1], (g >> 1) & 1);
                    tc_fence_after();
                    float alpha;
                    if (base + KV_PAGE > p.pos0 + 1 || (base < last_see.low && base + KV_PAGE > last_see.sinks)) {
                        auto seen = [&](uint32_t t0) {  // of 32 positions
                            auto below = [&](uint32_t x) { return x <= t0 ? 0u : x - t0 >= 32 ? 0xFFFFFFFFu : (1u << (x - t0)) - 1; };
                            return below(see.end) & (~below(see.low) | below(see.sinks));
                        };
                        alpha = page(Constant<1>{}, seen(base), seen(base + 32));
                    } else {
                        alpha = page(Constant<0>{}, 0, 0);
                    }
                    sh.alpha[g & 3][row] = alpha;
                    if (j + 1 == n) {
                        const float2 two = both(sums);
                        sh.stat[g & 3][0][row] = mx, sh.stat[g & 3][1][row] = ok ? two.x + two.y : NAN;
                    }
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive(&sh.s_go[g & 1]);
                        if (ok) mbar_arrive(&sh.o_go[g & 1]);
                    }
                }
            }
            meet();
            meet();
        }
    } else if (warp < C_FIRST_CONV) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(c_regs_sum(HD)));
        // ── the output: a thread a query row ──
        const uint32_t row = tid - C_SOFT * 32, lanes = tmem + (((warp - C_SOFT) * 32) << 16);
        uint32_t g = 0;
        f32x2 o[HD / 2];  // times 2^UP, as the probabilities are
        if (lane == 0) mbar_arrive(&sh.o_go[0]);  // nothing to read in front of the first one
        meet();
        for (uint32_t turn = 0; turn < sh.batches; ++turn) {
            const uint32_t pieces = sh.pieces;
            for (uint32_t k = 0; k < pieces; ++k) {
                const ChunkPiece& p = sh.piece[k];
                const uint32_t n = p.end - p.first;
                uint32_t odd_first = 0xFFFFFFFFu, odd_end = 0;
                bool lost = false;
#pragma unroll
                for (uint32_t i = 0; i < HD / 2; ++i) o[i] = 0;
                for (uint32_t j = 0; j < n; ++j, ++g) {
                    wait_all(&sh.o_done[g & 1], (g >> 1) & 1);
                    tc_fence_after();
                    const float alpha = sh.alpha[g & 3][row];
                    if (__any_sync(0xFFFFFFFFu, alpha != 1.0f)) {
#pragma unroll
                        for (uint32_t i = 0; i < HD / 2; ++i) o[i] = mul2(o[i], pair(alpha, alpha));
                    }
                    if (*reinterpret_cast<const uint32_t*>(sh.odd[g & 3]) != 0) odd_first = min(odd_first, p.first + j), odd_end = p.first + j + 1;
                    lost |= sh.lost[g & 15] != 0;
#pragma unroll
                    for (uint32_t c = 0; c < HD / 32; ++c) {
                        uint32_t r[32];
                        tmem_ld32(lanes + T::O + 32 * c, r);
                        const float f = sh.vs[g & 3][c];
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) {
                            f32x2& x = o[16 * c + i];
                            x = fma2(pair(r[2 * i], r[2 * i + 1]), pair(f, f), x);
                        }
                    }
                    if (j + 1 < n) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.o_go[(g + 1) & 1]);
                    }
                }
                const TileRows rows(a);  // here: the loop has no register left
                const uint32_t t = rows.token(row);
                const float mx = sh.stat[(g - 1) & 3][0][row];
                float sum = sh.stat[(g - 1) & 3][1][row];
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.o_go[g & 1]);
                if (!ok || lost) sum = NAN;
                if (lost && row == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
                const Sight see(a.span, p.pos0 + t);
                const bool live = t < p.tokens && p.head0 + row - t * rows.heads < (p.kvh + 1) * a.group;
                // Values that are not finite stood as zeros in the products: they go where a row sees them, and nowhere else; at(d): where
                // this row's dimension d stands.
                auto add_odd = [&](auto at) {
                    if (!live) return;
#pragma unroll 1
                    for (uint32_t u = odd_first; u < odd_end; ++u) {
                        const uint32_t number = u < p.sinks ? u : u + p.skip;
                        const int32_t id = a.c.table[(uint64_t)p.seq * a.c.table_stride + number];
                        if (id < 0 || (uint32_t)id >= a.c.n_pages) continue;
                        const uint8_t* values = a.c.pages + ((uint64_t)id * a.c.n_kv + p.kvh) * HEAD + HEAD / 2;
#pragma unroll 1
                        for (uint32_t i = 0; i < KV_PAGE; ++i) {
                            const uint32_t t = number * KV_PAGE + i;
                            if (t >= see.end || (t < see.low && t >= see.sinks)) continue;
#pragma unroll 1
                            for (uint32_t d = 0; d < HD; d += 4) {
                                const float4 v = kv_load<KIND, HD, true>(values, i, d);
                                if (!(fabsf(v.x) < INFINITY)) *at(d) += v.x;
                                if (!(fabsf(v.y) < INFINITY)) *at(d + 1) += v.y;
                                if (!(fabsf(v.z) < INFINITY)) *at(d + 2) += v.z;
                                if (!(fabsf(v.w) < INFINITY)) *at(d + 3) += v.w;
                            }
                        }
                    }
                };
                auto store = [&](float den) {  // through the stage, as the queries came
                    const float inv = 1.0f / den;
                    float4 (&stage)[32][C_STAGE] = sh.stage[1][warp - C_SOFT];
                    float4* to[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const uint32_t r = (warp - C_SOFT) * 32 + 8 * i + lane / 4, tok = rows.token(r), h = r - tok * rows.heads;
                        to[i] = tok < p.tokens && p.head0 + h < (p.kvh + 1) * a.group
                                    ? reinterpret_cast<float4*>(a.out + (uint64_t)(p.row0 + tok) * a.out_stride + (uint64_t)(p.head0 + h) * HD) + lane % 4
                                    : nullptr;
                    }
#pragma unroll
                    for (uint32_t c = 0; c < HD / 16; ++c) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            const float2 x = both(o[8 * c + 2 * i]), y = both(o[8 * c + 2 * i + 1]);
                            stage[lane][i] = make_float4(x.x * inv, x.y * inv, y.x * inv, y.y * inv);
                        }
                        __syncwarp();
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            if (to[i]) to[i][4 * c] = stage[8 * i + lane / 4][lane % 4];
                        __syncwarp();
                    }
                };
                if (p.parts == 1) {
                    store(sum);
                    if (odd_end != 0) {
                        float* out = a.out + (uint64_t)(p.row0 + t) * a.out_stride + (uint64_t)(p.head0 + row - t * rows.heads) * HD;
                        add_odd([&](uint32_t d) { return out + d; });
                    }
                } else {
                    // [HD / 4][CQ] outputs of four dimensions, then maxima, then sums
                    float* mine = a.part + ((uint64_t)blockIdx.x * 2 + (p.first == 0)) * PART;
#pragma unroll
                    for (uint32_t i = 0; i < HD / 4; ++i) {
                        const float2 x = both(o[2 * i]), y = both(o[2 * i + 1]);
                        __stcg(reinterpret_cast<float4*>(mine) + i * CQ + row, make_float4(x.x, x.y, y.x, y.y));
                    }
                    __stcg(mine + HD * CQ + row, mx), __stcg(mine + (HD + 1) * CQ + row, sum);
                    if (odd_end != 0) add_odd([&](uint32_t d) { return mine + (d / 4 * CQ + row) * 4 + d % 4; });
                    asm volatile("bar.sync 5, %0;" ::"n"(C_SUM * 32) : "memory");
                    if (row == 0) {
                        __threadfence();  // behind the barrier: for all of the CTA's stores
                        const bool last = atomicAdd(a.arrived + p.owner, 1) == p.parts - 1;
                        if (last) a.arrived[p.owner] = 0;
                        __threadfence();
                        sh.last = last;
                    }
                    asm volatile("bar.sync 5, %0;" ::"n"(C_SUM * 32) : "memory");
                    if (sh.last) {
                        auto part_of = [&](uint32_t i) { return a.part + ((uint64_t)(p.owner + i) * 2 + (i == 0)) * PART; };
                        float best = -INFINITY, den = 0.0f;
                        for (uint32_t i = 0; i < p.parts; ++i) best = fmaxf(best, __ldcg(part_of(i) + HD * CQ + row));
#pragma unroll
                        for (uint32_t i = 0; i < HD / 2; ++i) o[i] = 0;
                        for (uint32_t i = 0; i < p.parts; ++i) {
                            const float* from = part_of(i);
                            const float w = piece_weight(__ldcg(from + HD * CQ + row), best);
                            den = fmaf(w, __ldcg(from + (HD + 1) * CQ + row), den);
#pragma unroll
                            for (uint32_t d = 0; d < HD / 4; d += 8) {  // eight on their way: more take the loops' registers
                                float4 v[8];
#pragma unroll
                                for (uint32_t k = 0; k < 8; ++k) v[k] = __ldcg(reinterpret_cast<const float4*>(from) + (d + k) * CQ + row);
#pragma unroll
                                for (uint32_t k = 0; k < 8; ++k) {
                                    f32x2 &x = o[2 * (d + k)], &y = o[2 * (d + k) + 1];
                                    x = fma2(pair(v[k].x, v[k].y), pair(w, w), x), y = fma2(pair(v[k].z, v[k].w), pair(w, w), y);
                                }
                                asm volatile("" ::: "memory");
                            }
                        }
                        store(den);
                    }
                }
            }
            meet();
            meet();
        }
    } else if (warp < C_ISSUE) {
        // ── converters; first they cut the work ──
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(c_regs_conv(HD)));
        const uint32_t ct = tid - C_FIRST_CONV * 32, cw = warp - C_FIRST_CONV;
        auto scan = [&](uint32_t x, uint32_t which, uint32_t* total) {  // sum of the threads in front
            uint32_t run = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(0xFFFFFFFFu, run, o);
                run += lane >= o ? up : 0;
            }
            if (lane == 31) sh.scan[which][cw] = run;
            asm volatile("bar.sync 7, %0;" ::"n"(C_CONV * 32) : "memory");
            uint32_t all = 0;
            for (uint32_t w = 0; w < C_CONV; ++w) run += w < cw ? sh.scan[which][w] : 0, all += sh.scan[which][w];
            *total = all;
            return run - x;
        };
        // tiles in front of every sequence
        uint32_t n_tiles = 0, total = 0;
        {
            const uint32_t per = (batch + C_CONV * 32 - 1) / (C_CONV * 32), b0 = min(batch, ct * per), b1 = min(batch, b0 + per);
            uint32_t mine = 0, named = 0;
            for (uint32_t b = b0; b < b1; ++b) {
                const SequenceRows s = sequence_rows(a, b);
                named += s.n, mine += ChunkTiles(a, tile_rows(a, s)).tiles;
            }
            named = __reduce_add_sync(0xFFFFFFFFu, named);
            if (lane == 0) sh.named_too[cw] = named;
            uint32_t run = scan(mine, 0, &n_tiles);
            named = 0;
            for (uint32_t w = 0; w < C_CONV; ++w) named += sh.named_too[w];
            const bool fit = rows_fit(a, named);
            if (!fit) run = n_tiles = 0;  // nobody has tiles
            for (uint32_t b = b0; b < b1; ++b) s_tiles[b] = run, run += fit ? ChunkTiles(a, tile_rows(a, sequence_rows(a, b))).tiles : 0;
            if (ct == 0) s_tiles[batch] = n_tiles, sh.first_seg = 0, sh.end_seg = 0;
            asm volatile("bar.sync 7, %0;" ::"n"(C_CONV * 32) : "memory");
        }
        // a run of tiles a thread, and the units in front of it
        const uint32_t per = (n_tiles + C_CONV * 32 - 1) / (C_CONV * 32), t0 = min(n_tiles, ct * per), t1 = min(n_tiles, t0 + per);
        auto sequence_at = [&](uint32_t t) {  // the sequence that tile t is of
            uint32_t lo = 0, hi = batch;
            while (hi - lo > 1) {
                const uint32_t mid = (lo + hi) / 2;
                s_tiles[mid] <= t ? lo = mid : hi = mid;
            }
            return lo;
        };
        const uint32_t b0 = t0 < t1 ? sequence_at(t0) : 0;
        // f(tile's number, sequence, its rows, first token, tokens, pages): the thread's tiles
        auto each_tile = [&](auto f) {
            uint32_t b = b0;
            for (uint32_t i = t0; i < t1; ++i) {
                while (s_tiles[b + 1] <= i) ++b;
                const SequenceRows sq = sequence_rows(a, b);
                const ChunkTiles of(a, sq.n);
                const uint32_t token = (i - s_tiles[b]) * of.per_tile, tokens = min(of.per_tile, sq.n - token);
                f(i, b, sq, token, tokens, TilePages(a.span, (uint32_t)sq.len - sq.n + token, tokens));
            }
        };
        uint32_t mine = 0;
        each_tile([&](uint32_t, uint32_t, const SequenceRows&, uint32_t, uint32_t, const TilePages& pages) { mine += pages.n + SEG_UNITS; });
        const uint32_t in_front = scan(mine, 1, &total);
        const uint32_t heads = min(a.group, CQ), blocks = (a.group + CQ - 1) / CQ, segments = a.c.n_kv * blocks;  // of a tile
        const uint64_t units = (uint64_t)total * segments;
        // of a tile of n units, pieces of sqrt(JOIN_UNITS n) end first: smaller ones wait for the join
        const uint32_t least = max(1u, (uint32_t)sqrtf(JOIN_UNITS * (float)total / (float)max(n_tiles, 1u)));
        const uint64_t workers = units >= (uint64_t)gridDim.x * least ? gridDim.x : ((uint32_t)units + least - 1) / least;
        const uint64_t x0 = blockIdx.x < workers ? blockIdx.x * units / workers : 0;
        const uint64_t x1 = blockIdx.x < workers ? (blockIdx.x + 1) * units / workers : 0;
        auto cta_at = [&](uint64_t x) { return (uint32_t)(((x + 1) * workers - 1) / units); };
        // segments of which [x0, x1) has pages: from the one that x0 is in to the last one of which it has more than the beginning
        uint32_t run = in_front;
        each_tile([&](uint32_t i, uint32_t, const SequenceRows&, uint32_t, uint32_t, const TilePages& pages) {
            const uint32_t cost = pages.n + SEG_UNITS;
            const uint64_t begin = (uint64_t)run * segments, end = begin + (uint64_t)cost * segments;
            run += cost;
            if (x0 < x1 && x0 >= begin && x0 < end) {
                const uint32_t s = (uint32_t)((x0 - begin) / cost);
                sh.first_seg = i * segments + s;
            }
            if (x0 < x1 && x1 - 1 >= begin && x1 - 1 < end) {
                const uint32_t s = (uint32_t)((x1 - 1 - begin) / cost), in = (uint32_t)(x1 - 1 - begin - (uint64_t)s * cost);
                sh.end_seg = i * segments + s + (in >= SEG_UNITS);
            }
        });
        asm volatile("bar.sync 7, %0;" ::"n"(C_CONV * 32) : "memory");
        const uint32_t first_seg = sh.first_seg, end_seg = sh.end_seg;
        const uint32_t batches = end_seg > first_seg ? (end_seg - first_seg + C_PIECES - 1) / C_PIECES : 0;
        const ChunkConverter<KIND, HD, C_HALF> convert(cw % C_HALF, lane);
        uint32_t g = 0;
        auto list = [&](uint32_t turn) {
            const uint32_t from = first_seg + turn * C_PIECES, to = min(end_seg, from + C_PIECES);
            uint32_t run = in_front;
            each_tile([&](uint32_t i, uint32_t b, const SequenceRows& sq, uint32_t token, uint32_t tokens, const TilePages& pages) {
                const uint32_t cost = pages.n + SEG_UNITS;
                const uint64_t begin = (uint64_t)run * segments;
                run += cost;
                const uint32_t s0 = max(from, i * segments), s1 = min(to, (i + 1) * segments);
                for (uint32_t s = s0; s < s1; ++s) {
                    const uint32_t of = s - i * segments;
                    const uint64_t at = begin + (uint64_t)of * cost, page0 = at + SEG_UNITS, end = at + cost;
                    ChunkPiece p;
                    p.seq = b, p.row0 = sq.row + token, p.pos0 = (uint32_t)sq.len - sq.n + token, p.tokens = tokens;
                    p.kvh = of / blocks, p.head0 = p.kvh * a.group + of % blocks * heads;
                    p.first = x0 > page0 ? (uint32_t)(x0 - page0) : 0, p.end = x1 < end ? (uint32_t)(x1 - page0) : pages.n;
                    p.sinks = pages.sinks, p.skip = pages.skip;
                    p.owner = cta_at(page0), p.parts = cta_at(end - 1) - p.owner + 1;
                    sh.piece[s - from] = p;
                }
            });
            if (ct == 0) sh.pieces = to - from, sh.batches = batches;
        };
        if (batches) list(0);
        else if (ct == 0) sh.pieces = 0, sh.batches = 0;
        meet();
        for (uint32_t turn = 0; turn < batches; ++turn) {
            const uint32_t pieces = sh.pieces;
            for (uint32_t k = 0; k < pieces; ++k) {
                const ChunkPiece& p = sh.piece[k];
                const uint32_t n = p.end - p.first, behind = p.pos0 + p.tokens;
                for (uint32_t j = 0; j < n; ++j, ++g) {
                    const uint32_t st = g & 1, half = (g >> 1) & 1, u = p.first + j, base = (u < p.sinks ? u : u + p.skip) * KV_PAGE;
                    const uint32_t valid = min(KV_PAGE, behind - base);
                    if (cw < C_HALF) {
                        wait_all(&sh.s_done[st], half ^ 1);
                        if (!wait_all(&sh.rk_full[st], half)) continue;
                        convert.keys(k_base + st * T::K_STAGE, raw_k + st * T::RAW, valid, &sh.ks[g & 3]);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.s_go[st]), mbar_arrive(&sh.rk_empty[st]);
                    } else {
                        wait_all(&sh.o_done[st], half ^ 1);
                        if (!wait_all(&sh.rv_full[st], half)) continue;
                        const bool odd = __any_sync(0xFFFFFFFFu, convert.values(v_base + st * T::V_STAGE, raw_v + st * T::RAW, valid, sh.vs[g & 3]));
                        if (lane == 0) sh.odd[g & 3][cw - C_HALF] = odd;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.o_go[st]), mbar_arrive(&sh.rv_empty[st]);
                    }
                }
            }
            meet();
            if (turn + 1 < batches) list(turn + 1);
            meet();
        }
    } else {
        // ── issuer (one warp issues, one copies, two have nothing to do) ──
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C_REGS_ISSUE));
        uint32_t g = 0, q_phase = 0, k_sent = 0, v_sent = 0;
        meet();
        const uint32_t batches = sh.batches;
        for (uint32_t turn = 0; turn < batches; ++turn) {
            const uint32_t pieces = sh.pieces;
            if (warp == C_ISSUE) {
                // one warp issues both, batch after batch
                constexpr uint32_t idesc_s = umma_idesc_f16(KV_PAGE), idesc_o = umma_idesc_f16(HD) | 1u << 16;  // values MN-major
                const uint64_t dk = umma_desc(k_base), dv = umma_desc_values(v_base);
                // scores of page j in one accumulator, small products first; `begins`: of a piece's first, the queries are in place
                auto scores = [&](uint32_t j, bool begins) {
                    if (begins) wait_all(&sh.q_full, q_phase), q_phase ^= 1;
                    if (!wait_all(&sh.s_go[j & 1], (j >> 1) & 1)) return;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t d0 = dk + (uint64_t)(j & 1) * (T::K_STAGE >> 4);
                        const uint32_t d = tmem + T::S0 + (j & 1) * KV_PAGE;
#pragma unroll
                        for (uint32_t kk = 0; kk < HD / 16; ++kk) {
                            const uint64_t hi = d0 + kk / 4 * (T::K_PLANE >> 4) + kk % 4 * 2, lo = hi + T::HALVES * (T::K_PLANE >> 4);
                            umma_f16_ts(d, tmem + T::Q_LO + 8 * kk, hi, idesc_s, kk != 0);
                            if constexpr (T::TERMS == 2) umma_f16_ts(d, tmem + T::Q_HI + 8 * kk, lo, idesc_s, 1);
                        }
#pragma unroll
                        for (uint32_t kk = 0; kk < HD / 16; ++kk)
                            umma_f16_ts(d, tmem + T::Q_HI + 8 * kk, d0 + kk / 4 * (T::K_PLANE >> 4) + kk % 4 * 2, idesc_s, 1);
                        umma_commit(&sh.s_done[j & 1]);
                    }
                    __syncwarp();
                };
                uint32_t all = 0, k = 0, left = 0;  // pages; the piece whose scores come next, pages left of it
                for (uint32_t i = 0; i < pieces; ++i) all += sh.piece[i].end - sh.piece[i].first;
                auto next = [&] {
                    const bool begins = left == 0;
                    if (begins) left = sh.piece[k].end - sh.piece[k].first, ++k;
                    --left;
                    return begins;
                };
                if (all) scores(g, next());
                for (uint32_t j = 0; j < all; ++j, ++g) {
                    const bool more = j + 1 < all, begins = more && next();
                    if (more && !begins) scores(g + 1, false);
                    if (wait_all(&sh.o_go[g & 1], (g >> 1) & 1)) {
                        tc_fence_after();
                        if (elect_one()) {
                            const uint64_t hi = dv + (uint64_t)(g & 1) * (T::V_STAGE >> 4), lo = hi + (T::V_PLANE >> 4);
                            const uint32_t d = tmem + T::O, p_hi = tmem + T::P0 + (g & 1) * KV_PAGE, p_lo = p_hi + 32;
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; ++kk) {
                                umma_f16_ts(d, p_lo + 8 * kk, hi + 128 * kk, idesc_o, kk != 0);
                                if constexpr (T::TERMS == 2) umma_f16_ts(d, p_hi + 8 * kk, lo + 128 * kk, idesc_o, 1);
                            }
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; ++kk) umma_f16_ts(d, p_hi + 8 * kk, hi + 128 * kk, idesc_o, 1);
                            umma_commit(&sh.o_done[g & 1]);
                        }
                        __syncwarp();
                    }
                    if (begins) scores(g + 1, true);  // behind the products of the piece before: its rows bring the next queries
                }
            } else if (warp == C_LOAD) {
                // ── loader: a page's keys, or values, of a head are one run of memory; page ids 32 at a time, a lane each ──
                for (uint32_t k = 0; k < pieces; ++k) {
                    const ChunkPiece& p = sh.piece[k];
                    const uint32_t n = p.end - p.first;
                    const int32_t* table = a.c.table + (uint64_t)p.seq * a.c.table_stride;
                    int32_t ids = 0;
                    for (uint32_t j = 0; j < n; ++j, ++g) {
                        if (j % 32 == 0) {
                            const uint32_t u = p.first + min(j + lane, n - 1);
                            ids = table[u < p.sinks ? u : u + p.skip];
                        }
                        const int32_t id = __shfl_sync(0xFFFFFFFFu, ids, j % 32);
                        const bool fine = id >= 0 && (uint32_t)id < a.c.n_pages;
                        const uint8_t* src = a.c.pages + ((uint64_t)(fine ? id : 0) * a.c.n_kv + p.kvh) * HEAD;
                        const uint32_t st = g & 1, freed = ((g >> 1) & 1) ^ 1;
                        if (wait_all(&sh.rk_empty[st], freed)) {
                            ++k_sent;
                            if (lane == 0) {
                                sh.lost[g & 15] = !fine;
                                mbar_arrive_expect_tx(&sh.rk_full[st], T::RAW);
                                bulk_g2s(raw_k + st * T::RAW, src, T::RAW, &sh.rk_full[st]);
                            }
                        }
                        if (wait_all(&sh.rv_empty[st], freed)) {
                            ++v_sent;
                            if (lane == 0) {
                                mbar_arrive_expect_tx(&sh.rv_full[st], T::RAW);
                                bulk_g2s(raw_v + st * T::RAW, src + T::RAW, T::RAW, &sh.rv_full[st]);
                            }
                        }
                    }
                }
            }
            meet();
            meet();
        }
        if (!ok && warp == C_ISSUE) {  // products in flight still use tensor memory and the tiles
            if (elect_one()) umma_commit(&sh.drained);
            __syncwarp();
            mbar_wait(&sh.drained, 0);
        }
        if (!ok && warp == C_LOAD) {  // copies in flight still write to shared memory
            for (uint32_t back = 1; back <= 2; ++back) {
                if (k_sent >= back) mbar_wait(&sh.rk_full[(k_sent - back) & 1], ((k_sent - back) >> 1) & 1);
                if (v_sent >= back) mbar_wait(&sh.rv_full[(v_sent - back) & 1], ((v_sent - back) >> 1) & 1);
            }
        }
    }
    meet();
    if (tid == 0 && sh.abort_flag && error_flag) *reinterpret_cast<volatile int*>(error_flag) = 1;
    if (warp == C_ISSUE)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

struct LaunchTiles {
    const PagedArgs& a;
    uint32_t grid;
    int* error_flag;
    cudaStream_t s;
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        if constexpr (HD > 128) {
            return cudaErrorInvalidValue;
        } else {
            auto kern = attention_chunk_tiles_kernel<KIND, HD>;
            constexpr uint32_t BYTES = ChunkTile<KIND, HD>::SMEM;
            static bool configured[MAX_DEVICES] = {};
            if (cudaError_t e = set_max_smem_once(kern, BYTES + (ATTENTION_MAX_BATCH + 1) * 4, configured); e != cudaSuccess) return e;
            return launch_pdl(kern, dim3(grid), C_THREADS, BYTES + (a.c.n_seq + 1) * 4, s, a, error_flag);
        }
    }
};

}  // namespace

cudaError_t launch_attention_chunk_tiles(const PagedArgs& a, uint32_t grid, int* error_flag, cudaStream_t s) {
    return for_kind(a.c.kind, a.c.hd, LaunchTiles{a, grid, error_flag, s});
}

}  // namespace jq
