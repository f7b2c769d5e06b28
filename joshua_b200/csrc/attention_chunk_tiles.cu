// Attention of chunks of new tokens over the quantised cache on the 5th-generation tensor cores.
//
// A tile is up to 128 query rows: the heads of a kv head of consecutive tokens of a sequence, token by token.  It goes over the pages
// that some of its tokens sees, a page at a time, running maximum and sum in f32.  Terms as in attention_lead.cu: queries two f16 terms
// under a power of two of their row; codes times scales as two f16 terms (halves: one) under powers of two of a page's largest scale;
// probabilities two terms; of a product of two terms each the smallest of the four is left out.  Accumulators hold 64 dimensions of a
// score or one page of the output; the running output lives in registers.  Scores of positions that a row does not see become nothing
// before the maximum, their probabilities zeros; values behind the tile's last position are zeros in the products, and those that are
// not finite too: they are added at the end, to the rows that see them.
//
// The tiles' work stands in one row of units, tile by tile, kv head by kv head, SEG_UNITS for beginning and ending one, then its
// pages.  It is cut into equal pieces, one a CTA; pieces of a tile that several CTAs have are joined by the last of them to arrive, in order.
//
// Warps: 0 .. 15 softmax, four threads a query row (16 keys and a quarter of the output dimensions each); 16 .. 23 first cut the work,
// then turn the pages' codes into swizzled K-major tiles, two stages; 24 issues the products; 25 copies the pages.  Tensor memory: the
// query's terms (the A operand of the scores), scores, probabilities (A of the output), output of a page.
//
// Every wait on an mbarrier is bounded.  A warp whose wait ran out waits for none any more, hands nothing on, and goes through the
// rest of its work so, which brings it to every barrier that others expect it at; the status flag is raised and the rows become NaN.
#include <algorithm>

#include "attention_chunk.cuh"
#include "attention_tiles.cuh"

namespace jq {

namespace {

constexpr uint32_t CQ = CHUNK_TILE_ROWS;     // query rows of a tile
constexpr uint32_t C_SOFT = 16, C_CONV = 8;  // warps
constexpr uint32_t C_PARTS = C_SOFT / 4;     // threads a row
constexpr uint32_t C_KEYS = KV_PAGE / C_PARTS;
constexpr int UP = 6;                        // probabilities stand times 2^UP ..
constexpr float LAZY = 8.0f;                 // .. and are up to 2^LAZY: below 2^15
constexpr uint32_t C_THREADS = (C_SOFT + C_CONV + 4) * 32;  // whole warpgroups: they trade registers
// Registers a thread: the launch has 896 x 72 = 64512, of which the issuer's warpgroup keeps 128 x 32, the converters 256 x 56 and the
// softmax threads (32 running outputs, 16 scores, 16 terms) 512 x 88.
constexpr int C_REGS_ISSUE = 32, C_REGS_CONV = 56, C_REGS_SOFT = 88;
static_assert(128 * C_REGS_ISSUE + C_CONV * 32 * C_REGS_CONV + C_SOFT * 32 * C_REGS_SOFT <= C_THREADS * 72, "registers");

constexpr uint32_t SEG_UNITS = 2;   // a tile's beginning and end in pages
constexpr uint32_t C_PIECES = 96;   // pieces of a CTA at a time

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
    float vs[4][4];           // inverse scales of the values' blocks, by page % 4
    uint8_t odd[4][C_CONV];   // values that are not finite, by page % 4 and converter
    uint8_t lost[8];          // a page id outside the cache, by page % 8
    float row[2][C_PARTS][CQ];
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full, s_free, p_full, o_full;
    uint64_t rk_full[2], rk_empty[2], rv_full[2], rv_empty[2];  // the raw pages
    uint64_t drained;         // the products of a CTA that gives up
    uint32_t tmem_slot;
    int abort_flag;
    uint32_t last;            // this CTA was the last one to bring its part of a tile
    uint32_t scan[2][C_CONV], first_seg, end_seg;
    uint32_t pieces, batches;  // pieces of this batch; batches
    ChunkPiece piece[C_PIECES];
};

template <uint32_t KIND, uint32_t HD>
struct ChunkTile : PageTile<KIND, HD> {
    using P = PageTile<KIND, HD>;
    using P::HALVES, P::K_STAGE, P::RAW, P::V_STAGE;
    static constexpr uint32_t TILES = 2 * (K_STAGE + V_STAGE);
    static constexpr uint32_t SMEM = TILES + 4 * RAW + sizeof(ChunkShared);  // and the tiles in front of every sequence
    static_assert(SMEM + (ATTENTION_MAX_BATCH + 1) * 4 <= 227 * 1024, "shared memory");
    // tensor memory columns
    static constexpr uint32_t Q_HI = 0, Q_LO = HD / 2, S0 = HD, P0 = S0 + 64 * HALVES, O = P0 + 64;
    static_assert(O + HD <= 512, "tensor memory");
};

// Scores of a row: 16 columns at a, with HALVES = 2 also 16 at b, one wait for both.
__device__ __forceinline__ void tmem_ld16_pair(uint32_t a, uint32_t b, uint32_t (&x)[16], uint32_t (&y)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%32];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        "{%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%33];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(x[0]), "=&r"(x[1]), "=&r"(x[2]), "=&r"(x[3]), "=&r"(x[4]), "=&r"(x[5]), "=&r"(x[6]), "=&r"(x[7]), "=&r"(x[8]), "=&r"(x[9]),
          "=&r"(x[10]), "=&r"(x[11]), "=&r"(x[12]), "=&r"(x[13]), "=&r"(x[14]), "=&r"(x[15]), "=&r"(y[0]), "=&r"(y[1]), "=&r"(y[2]), "=&r"(y[3]),
          "=&r"(y[4]), "=&r"(y[5]), "=&r"(y[6]), "=&r"(y[7]), "=&r"(y[8]), "=&r"(y[9]), "=&r"(y[10]), "=&r"(y[11]), "=&r"(y[12]), "=&r"(y[13]),
          "=&r"(y[14]), "=&r"(y[15])
        : "r"(a), "r"(b)
        : "memory");
}
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
// sequences of this kernel: its rows, or none
__device__ __forceinline__ SequenceRows tile_rows(const PagedArgs& a, uint32_t b) {
    SequenceRows s = sequence_rows(a, b);
    if (s.n <= a.span.few || s.len <= 0) s.n = 0;
    return s;
}

template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(C_THREADS, 1) attention_chunk_tiles_kernel(PagedArgs a, int* error_flag) {
    using T = ChunkTile<KIND, HD>;
    constexpr uint32_t HEAD = kv_head_bytes(KIND, HD), DN = HD / C_PARTS;  // dimensions of a softmax thread
    constexpr uint32_t PART = CHUNK_TILE_ROWS * (HD + 2);                  // floats of a part of a tile
    extern __shared__ __align__(1024) uint8_t smem[];  // K and V stages | raw keys, raw values | ChunkShared | s_tiles
    const uint32_t k_base = smem_u32(smem), v_base = k_base + 2 * T::K_STAGE;
    uint8_t* raw_k = smem + T::TILES;
    uint8_t* raw_v = raw_k + 2 * T::RAW;
    ChunkShared& sh = *reinterpret_cast<ChunkShared*>(raw_v + 2 * T::RAW);
    uint32_t* s_tiles = reinterpret_cast<uint32_t*>(&sh + 1);  // [batch + 1] tiles in front of a sequence

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, batch = a.c.n_seq;
    const bool aligned = k_base % 1024 == 0;  // the swizzle's period; no static shared memory stands in front
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], C_CONV);
            mbar_init(&sh.v_full[i], C_CONV);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.rk_full[i], 1);
            mbar_init(&sh.rv_full[i], 1);
            mbar_init(&sh.rk_empty[i], C_CONV);
            mbar_init(&sh.rv_empty[i], C_CONV);
        }
        mbar_init(&sh.s_full, 1);
        mbar_init(&sh.s_free, C_SOFT);
        mbar_init(&sh.p_full, C_SOFT);
        mbar_init(&sh.o_full, 1);
        mbar_init(&sh.drained, 1);
        sh.abort_flag = !aligned;
        mbar_fence_init();
    }
    if (warp == C_SOFT + C_CONV) {
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
        for (uint32_t b = blockIdx.x; b < batch; b += gridDim.x) {
            const SequenceRows sq = sequence_rows(a, b);
            if ((sq.lost || sq.len < 0) && tid == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
            if (sq.n <= a.span.few || sq.len > 0) continue;
            for (uint32_t k = 0; k < sq.n; ++k)
                for (uint32_t i = tid; i < a.n_q * HD; i += C_SOFT * 32) a.out[(sq.row + k) * a.out_stride + i] = sq.len < 0 ? NAN : 0.0f;
        }
        // ── softmax: thread = (query row, part) ──
        const uint32_t quarter = warp & 3, part = warp >> 2, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((quarter * 32) << 16);
        uint32_t phase = 0, g = 0;  // of the exchange between a row's threads; pages so far
        auto exchange = [&](float x) -> const float* {  // [part * CQ]: x of the row's threads
            float* at = &sh.row[phase][0][row];
            phase ^= 1;
            at[part * CQ] = x;
            asm volatile("bar.sync %0, 128;" ::"r"(1 + quarter) : "memory");
            return at;
        };
        auto share_max = [&](float x) {
            const float* v = exchange(x);
            return fmaxf(fmaxf(v[0], v[CQ]), fmaxf(v[2 * CQ], v[3 * CQ]));
        };
        float rf = 0.0f;  // inverse scale of the query row, times log2(e) and the softmax scale
        // a piece's queries into tensor memory; the scores before have been worked out
        auto query = [&](const ChunkPiece& p) {
            const uint32_t heads = min(a.group, CQ), t = row / heads, h = row % heads;
            const bool live = t < p.tokens && (p.head0 + h) / a.group == p.kvh;
            const float4* src = reinterpret_cast<const float4*>(a.q + (uint64_t)(p.row0 + (live ? t : 0)) * a.q_stride +
                                                                (uint64_t)(p.head0 + (live ? h : 0)) * HD + part * DN);
            auto load = [&](uint32_t i) { return live ? src[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f); };
            float amax = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < DN / 4; ++i) {
                const float4 v = load(i);
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
            amax = share_max(amax);
            // a power of two that puts the row's largest value just below 2^15, with the sign of the scale: the row's maximum is
            // looked for before the scores are multiplied by rf, which must not turn their order round
            const uint32_t e = __float_as_uint(amax) >> 23, bits = e == 255 ? 127u : min(254u, 268u - e);
            const float sc = copysignf(__uint_as_float(bits << 23), a.scale);
            rf = (bits == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((254u - bits) << 23)) * (fabsf(a.scale) * 1.44269504f);
#pragma unroll
            for (uint32_t c = 0; c < DN / 16; ++c) {
                uint32_t hi[8], lo[8];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    const float4 v = load(4 * c + i);
                    split2(v.x * sc, v.y * sc, &hi[2 * i], &lo[2 * i]), split2(v.z * sc, v.w * sc, &hi[2 * i + 1], &lo[2 * i + 1]);
                }
                tmem_st8(lanes + T::Q_HI + part * (DN / 2) + 8 * c, hi);
                tmem_st8(lanes + T::Q_LO + part * (DN / 2) + 8 * c, lo);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_free);  // the first scores wait for the query's terms
        };
        f32x2 o[DN / 2];
        uint32_t odd_first = 0xFFFFFFFFu, odd_end = 0;
        bool lost = false;
        // o = o * alpha + the page's output; u: its place in the piece's list
        auto add_page = [&](uint32_t j, float alpha, uint32_t u) {
            if (__any_sync(0xFFFFFFFFu, alpha != 1.0f)) {
#pragma unroll
                for (uint32_t i = 0; i < DN / 2; ++i) o[i] = mul2(o[i], pair(alpha, alpha));
            }
            if (!wait_all(&sh.o_full, j & 1)) return;
            tc_fence_after();
            if (*reinterpret_cast<const uint64_t*>(sh.odd[j & 3]) != 0) odd_first = min(odd_first, u), odd_end = u + 1;
            lost |= sh.lost[j & 7] != 0;
#pragma unroll
            for (uint32_t c = 0; c < DN / 16; ++c) {
                uint32_t r[16];
                tmem_ld16(lanes + T::O + part * DN + 16 * c, r);
                const float f = KIND == KV_F16 ? 1.0f : sh.vs[j & 3][(part * DN + 16 * c) / 32];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    f32x2& x = o[8 * c + i];
                    x = KIND == KV_F16 ? add2(x, pair(r[2 * i], r[2 * i + 1])) : fma2(pair(r[2 * i], r[2 * i + 1]), pair(f, f), x);
                }
            }
        };
        meet();
        for (uint32_t turn = 0; turn < sh.batches; ++turn) {
            const uint32_t pieces = sh.pieces;
            if (pieces) query(sh.piece[0]);
            for (uint32_t k = 0; k < pieces; ++k) {
                const ChunkPiece& p = sh.piece[k];
                const uint32_t heads = min(a.group, CQ), t = row / heads, n = p.end - p.first;
                const Sight see(a.span, p.pos0 + t), last_see(a.span, p.pos0 + p.tokens - 1);
                const float my_rf = rf;
#pragma unroll
                for (uint32_t i = 0; i < DN / 2; ++i) o[i] = 0;
                float mx = -INFINITY, alpha_prev = 0.0f;
                f32x2 sums = 0;  // sum and outputs times 2^UP, as the probabilities are
                odd_first = 0xFFFFFFFFu, odd_end = 0, lost = false;
                for (uint32_t j = 0; j < n; ++j, ++g) {
                    const uint32_t u = p.first + j, base = (u < p.sinks ? u : u + p.skip) * KV_PAGE;
                    f32x2 sc[C_KEYS / 2];
                    wait_all(&sh.s_full, g & 1);
                    tc_fence_after();
                    {
                        uint32_t r[16];
                        if constexpr (T::HALVES == 2) {
                            uint32_t r2[16];
                            tmem_ld16_pair(lanes + T::S0 + part * C_KEYS, lanes + T::S0 + 64 + part * C_KEYS, r, r2);
#pragma unroll
                            for (int i = 0; i < 8; ++i) sc[i] = add2(pair(r[2 * i], r[2 * i + 1]), pair(r2[2 * i], r2[2 * i + 1]));
                        } else {
                            tmem_ld16(lanes + T::S0 + part * C_KEYS, r);
#pragma unroll
                            for (int i = 0; i < 8; ++i) sc[i] = pair(r[2 * i], r[2 * i + 1]);
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (j + 1 < n && lane == 0) mbar_arrive(&sh.s_free);  // behind the last page: when the next queries are in place
                    const float f = KIND == KV_F16 ? my_rf : my_rf * sh.ks[g & 3];
                    // positions of this thread's that the row sees, a bit each
                    uint32_t seen = 0xFFFFu;
                    const bool edge = base + KV_PAGE > p.pos0 + 1 || (base < last_see.low && base + KV_PAGE > last_see.sinks);
                    if (edge) {
                        const uint32_t t0 = base + part * C_KEYS;
                        auto below = [&](uint32_t x) { return x <= t0 ? 0u : x - t0 >= C_KEYS ? 0xFFFFu : (1u << (x - t0)) - 1; };
                        seen = below(see.end) & (~below(see.low) | below(see.sinks));
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float2 v = both(sc[i]);
                            sc[i] = pair(seen >> (2 * i) & 1 ? v.x : -INFINITY, seen >> (2 * i + 1) & 1 ? v.y : -INFINITY);
                        }
                    }
                    float cm = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 v = both(sc[i]);
                        cm = max3(cm, v.x, v.y);
                    }
                    const float top = share_max(cm) * f;
                    float alpha = 1.0f;
                    if (top > mx + LAZY) alpha = ex2(mx - top), mx = top;  // 0 on the first page with something to see (mx = -inf)
                    const float from = (float)UP - (mx > -INFINITY ? mx : 0.0f);
                    const f32x2 ff = pair(f, f), shift = pair(from, from);
                    f32x2 ps = 0;
                    uint32_t w0[8], w1[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 y = both(fma2(sc[i], ff, shift));
                        float x0 = ex2(y.x), x1 = ex2(y.y);
                        if (edge) x0 = seen >> (2 * i) & 1 ? x0 : 0.0f, x1 = seen >> (2 * i + 1) & 1 ? x1 : 0.0f;
                        const f32x2 both_p = pair(x0, x1);
                        ps = add2(ps, both_p);
                        const __half2 h = __floats2half2_rn(x0, x1);
                        const float2 hf = __half22float2(h);
                        const float2 rest = both(fma2(pair(hf.x, hf.y), pair(-1.0f, -1.0f), both_p));
                        w0[i] = half2_bits(h), w1[i] = half2_bits(__floats2half2_rn(rest.x, rest.y));
                    }
                    sums = fma2(sums, pair(alpha, alpha), ps);
                    if (j > 0) add_page(g - 1, alpha_prev, u - 1);  // its products have read the probabilities before these
                    alpha_prev = alpha;
                    tmem_st8(lanes + T::P0 + part * 8, w0);
                    tmem_st8(lanes + T::P0 + 32 + part * 8, w1);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (ok && lane == 0) mbar_arrive(&sh.p_full);
                }
                if (k + 1 < pieces) query(sh.piece[k + 1]);
                add_page(g - 1, alpha_prev, p.end - 1);
                const float2 two = both(sums);
                const float* all_sums = exchange(two.x + two.y);
                float sum = (all_sums[0] + all_sums[CQ]) + (all_sums[2 * CQ] + all_sums[3 * CQ]);
                if (!ok || lost) sum = NAN;
                if (lost && row == 0 && part == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
                const bool live = t < p.tokens && (p.head0 + row % heads) / a.group == p.kvh;
                if (odd_end != 0 && live) {
                    // values that are not finite stood as zeros in the products: they go where a row sees them, and nowhere else
                    for (uint32_t u = odd_first; u < odd_end; ++u) {
                        const uint32_t page = u < p.sinks ? u : u + p.skip;
                        const int32_t id = a.c.table[(uint64_t)p.seq * a.c.table_stride + page];
                        if (id < 0 || (uint32_t)id >= a.c.n_pages) continue;
                        const uint8_t* values = a.c.pages + ((uint64_t)id * a.c.n_kv + p.kvh) * HEAD + HEAD / 2;
                        for (uint32_t i = 0; i < KV_PAGE; ++i) {
                            const uint32_t at = page * KV_PAGE + i;
                            if (at >= see.end || (at < see.low && at >= see.sinks)) continue;
#pragma unroll
                            for (uint32_t d = 0; d < DN; d += 4) {
                                const float4 v = kv_load<KIND, HD, true>(values, i, part * DN + d);
                                auto odd = [](float x) { return fabsf(x) < INFINITY ? 0.0f : x; };
                                o[d / 2] = add2(o[d / 2], pair(odd(v.x), odd(v.y))), o[d / 2 + 1] = add2(o[d / 2 + 1], pair(odd(v.z), odd(v.w)));
                            }
                        }
                    }
                }
                float* to = a.out + (uint64_t)(p.row0 + t) * a.out_stride + (uint64_t)(p.head0 + row % heads) * HD + part * DN;
                auto store = [&](float den) {
                    if (!live) return;
                    const float inv = 1.0f / den;
#pragma unroll
                    for (uint32_t i = 0; i < DN / 4; ++i) {
                        const float2 x = both(o[2 * i]), y = both(o[2 * i + 1]);
                        *reinterpret_cast<float4*>(to + 4 * i) = make_float4(x.x * inv, x.y * inv, y.x * inv, y.y * inv);
                    }
                };
                if (p.parts == 1) {
                    store(sum);
                } else {
                    // [HD / 4][CQ] outputs of four dimensions, then maxima, then sums
                    float* mine = a.part + ((uint64_t)blockIdx.x * 2 + (p.first == 0)) * PART;
#pragma unroll
                    for (uint32_t i = 0; i < DN / 4; ++i) {
                        const float2 x = both(o[2 * i]), y = both(o[2 * i + 1]);
                        __stcg(reinterpret_cast<float4*>(mine) + (part * (DN / 4) + i) * CQ + row, make_float4(x.x, x.y, y.x, y.y));
                    }
                    if (part == 0) __stcg(mine + HD * CQ + row, mx), __stcg(mine + (HD + 1) * CQ + row, sum);
                    __threadfence();
                    asm volatile("bar.sync 5, %0;" ::"n"(C_SOFT * 32) : "memory");
                    if (tid == 0) {
                        const bool last = atomicAdd(a.arrived + p.owner, 1) == p.parts - 1;
                        if (last) a.arrived[p.owner] = 0;
                        __threadfence();
                        sh.last = last;
                    }
                    asm volatile("bar.sync 5, %0;" ::"n"(C_SOFT * 32) : "memory");
                    if (sh.last) {
                        __threadfence();
                        auto part_of = [&](uint32_t i) { return a.part + ((uint64_t)(p.owner + i) * 2 + (i == 0)) * PART; };
                        float best = -INFINITY, den = 0.0f;
                        for (uint32_t i = 0; i < p.parts; ++i) best = fmaxf(best, __ldcg(part_of(i) + HD * CQ + row));
#pragma unroll
                        for (uint32_t i = 0; i < DN / 2; ++i) o[i] = 0;
                        for (uint32_t i = 0; i < p.parts; ++i) {
                            const float* from = part_of(i);
                            const float w = piece_weight(__ldcg(from + HD * CQ + row), best);
                            den = fmaf(w, __ldcg(from + (HD + 1) * CQ + row), den);
#pragma unroll
                            for (uint32_t d = 0; d < DN / 4; ++d) {
                                const float4 v = __ldcg(reinterpret_cast<const float4*>(from) + (part * (DN / 4) + d) * CQ + row);
                                o[2 * d] = fma2(pair(v.x, v.y), pair(w, w), o[2 * d]), o[2 * d + 1] = fma2(pair(v.z, v.w), pair(w, w), o[2 * d + 1]);
                            }
                        }
                        store(den);
                    }
                }
            }
            meet();
            meet();
        }
    } else if (warp < C_SOFT + C_CONV) {
        // ── converters; first they cut the work ──
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C_REGS_CONV));
        const uint32_t ct = tid - C_SOFT * 32, cw = warp - C_SOFT;
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
            uint32_t mine = 0;
            for (uint32_t b = b0; b < b1; ++b) mine += ChunkTiles(a, tile_rows(a, b).n).tiles;
            uint32_t run = scan(mine, 0, &n_tiles);
            for (uint32_t b = b0; b < b1; ++b) s_tiles[b] = run, run += ChunkTiles(a, tile_rows(a, b).n).tiles;
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
        const uint64_t units = (uint64_t)total * segments, workers = min((uint64_t)gridDim.x, units);
        const uint64_t x0 = blockIdx.x < workers ? blockIdx.x * units / workers : 0, x1 = blockIdx.x < workers ? (blockIdx.x + 1) * units / workers : 0;
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
        const uint32_t first_seg = sh.first_seg, end_seg = sh.end_seg, batches = end_seg > first_seg ? (end_seg - first_seg + C_PIECES - 1) / C_PIECES : 0;
        const PageConverter<KIND, HD, C_CONV, true> convert(cw, lane);
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
                    wait_all(&sh.k_empty[st], half ^ 1);
                    if (wait_all(&sh.rk_full[st], half)) {
                        convert.keys(k_base + st * T::K_STAGE, raw_k + st * T::RAW, valid, &sh.ks[g & 3]);
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.k_full[st]), mbar_arrive(&sh.rk_empty[st]);
                    }
                    wait_all(&sh.v_empty[st], half ^ 1);
                    if (wait_all(&sh.rv_full[st], half)) {
                        const bool odd = __any_sync(0xFFFFFFFFu, convert.values(v_base + st * T::V_STAGE, raw_v + st * T::RAW, valid, sh.vs[g & 3]));
                        if (lane == 0) sh.odd[g & 3][cw] = odd;
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.v_full[st]), mbar_arrive(&sh.rv_empty[st]);
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
        uint32_t g = 0, k_sent = 0, v_sent = 0;
        meet();
        const uint32_t batches = sh.batches;
        for (uint32_t turn = 0; turn < batches; ++turn) {
            const uint32_t pieces = sh.pieces;
            if (warp == C_SOFT + C_CONV) {
                constexpr uint32_t idesc_s = umma_idesc_f16(KV_PAGE), idesc_o = umma_idesc_f16(HD);
                const uint64_t dk = umma_desc(k_base), dv = umma_desc(v_base);
                auto scores = [&](uint32_t j) {  // one accumulator per 64 dimensions, small products first
                    // the scores before have been read (the first of a piece: the queries are in place)
                    wait_all(&sh.s_free, j & 1);
                    if (!wait_all(&sh.k_full[j & 1], (j >> 1) & 1)) return;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t d0 = dk + (uint64_t)(j & 1) * (T::K_STAGE >> 4);
#pragma unroll
                        for (uint32_t h = 0; h < T::HALVES; ++h) {
                            const uint64_t hi = d0 + h * (T::K_PLANE >> 4), lo = hi + T::HALVES * (T::K_PLANE >> 4);
                            const uint32_t d = tmem + T::S0 + 64 * h, a_hi = tmem + T::Q_HI + 32 * h, a_lo = tmem + T::Q_LO + 32 * h;
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; ++kk) {
                                umma_f16_ts(d, a_lo + 8 * kk, hi + 2 * kk, idesc_s, kk != 0);
                                if constexpr (T::TERMS == 2) umma_f16_ts(d, a_hi + 8 * kk, lo + 2 * kk, idesc_s, 1);
                            }
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; ++kk) umma_f16_ts(d, a_hi + 8 * kk, hi + 2 * kk, idesc_s, 1);
                        }
                        umma_commit(&sh.k_empty[j & 1]);
                        umma_commit(&sh.s_full);
                    }
                    __syncwarp();
                };
                uint32_t all = 0;
                for (uint32_t k = 0; k < pieces; ++k) all += sh.piece[k].end - sh.piece[k].first;
                if (all) scores(g);
                for (uint32_t j = 0; j < all; ++j, ++g) {
                    if (j + 1 < all) scores(g + 1);
                    // the probabilities are in place, the output before has been read
                    wait_all(&sh.v_full[g & 1], (g >> 1) & 1);
                    if (!wait_all(&sh.p_full, g & 1)) continue;
                    tc_fence_after();
                    if (elect_one()) {
                        const uint64_t hi = dv + (uint64_t)(g & 1) * (T::V_STAGE >> 4), lo = hi + (T::V_PLANE >> 4);
                        const uint32_t d = tmem + T::O, p_hi = tmem + T::P0, p_lo = p_hi + 32;
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; ++kk) {
                            umma_f16_ts(d, p_lo + 8 * kk, hi + 2 * kk, idesc_o, kk != 0);
                            if constexpr (T::TERMS == 2) umma_f16_ts(d, p_hi + 8 * kk, lo + 2 * kk, idesc_o, 1);
                        }
#pragma unroll
                        for (uint32_t kk = 0; kk < 4; ++kk) umma_f16_ts(d, p_hi + 8 * kk, hi + 2 * kk, idesc_o, 1);
                        umma_commit(&sh.v_empty[g & 1]);
                        umma_commit(&sh.o_full);
                    }
                    __syncwarp();
                }
            } else if (warp == C_SOFT + C_CONV + 1) {
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
                                sh.lost[g & 7] = !fine;
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
        if (!ok && warp == C_SOFT + C_CONV) {  // products in flight still use tensor memory and the tiles
            if (elect_one()) umma_commit(&sh.drained);
            __syncwarp();
            mbar_wait(&sh.drained, 0);
        }
        if (!ok && warp == C_SOFT + C_CONV + 1) {  // copies in flight still write to shared memory
            for (uint32_t back = 1; back <= 2; ++back) {
                if (k_sent >= back) mbar_wait(&sh.rk_full[(k_sent - back) & 1], ((k_sent - back) >> 1) & 1);
                if (v_sent >= back) mbar_wait(&sh.rv_full[(v_sent - back) & 1], ((v_sent - back) >> 1) & 1);
            }
        }
    }
    meet();
    if (tid == 0 && sh.abort_flag && error_flag) *reinterpret_cast<volatile int*>(error_flag) = 1;
    if (warp == C_SOFT + C_CONV)
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
