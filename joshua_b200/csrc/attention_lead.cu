// The leading pages of a batch that shares them, on the 5th-generation tensor cores: the batch's query rows of a kv head against
// the pages, once for all sequences (attention_paged.cu joins the result with each sequence's own pages).
//
// One CTA per (128 query rows, kv head, split of the pages), a page at a time, running maximum and sum in f32.  Queries are two
// f16 terms under a power of two of their row.  Keys and values are the code times the block's scale, 19 bits at most (halves: 11),
// as two f16 terms (halves: one), keys under a power of two of the page's largest scale, values under one of the page's largest
// scale of the block of 32 dimensions: exact for scales of at least 2^-21 (four bits: 2^-25) of that largest one; smaller scales are
// rounded by up to 2^-32 (2^-36) of it.  Probabilities are two terms.  A product of two terms each leaves out the smallest of the
// four.  Accumulators hold 64 dimensions of a score or one page of the output, the running output lives in registers and is added
// round-to-nearest.
//
// What bounds it is the chain of a tile (scores' product, maximum of the row, exponentials, probabilities' product), not the
// products: 1.65 us a page with heads of 128 in eight bits, 0.9 with heads of 64 in halves, of which the tensor pipe is busy 19%
// and 28%; the softmax threads have half of an SM's registers, so a second tile cannot run beside the first.  32 sequences, 32
// heads on 8 of 128, 64 pages: 22 us alone and cold for 128 CTAs of four pages each, about 10 of them launch, queries and joining; the
// whole call with 100 positions of each sequence's own 26 us, with attention_lead_kernel in its place 42.
//
// Warps: 0 .. 7 softmax, two threads a query row (32 keys and half of the output dimensions each); 8 .. 15 turn the pages' codes
// into swizzled K-major tiles, two stages; 16 issues the products; 17 copies the pages.  Tensor memory: the query's terms (the A
// operand of the scores), scores, probabilities (A of the output), output of a page.
//
// Every wait on an mbarrier is bounded.  A warp whose wait ran out hands nothing on but still comes to every barrier that others
// expect it at, so that all warps reach the common exit, where tensor memory is released; the status flag is raised and the rows
// of the CTA become NaN.
#include "attention_paged.cuh"
#include "tc5.cuh"

namespace jq {

namespace {

constexpr uint32_t LQ = 128, LK = KV_PAGE;   // query rows and keys of a tile
constexpr uint32_t L_SOFT = 8, L_CONV = 8;   // warps
constexpr int UP = 6;                        // probabilities stand times 2^UP ..
constexpr float LAZY = 8.0f;                 // .. and are up to 2^LAZY: below 2^15
constexpr uint32_t L_THREADS = (L_SOFT + L_CONV + 4) * 32;  // whole warpgroups: they trade registers
// Registers a thread: the launch has 640 x 96 = 61440, of which the issuer's warpgroup keeps 128 x 32, the converters 256 x 80
// and the softmax threads (64 running outputs, 32 scores, 32 terms) 256 x 144: all of it.
constexpr int L_REGS_ISSUE = 32, L_REGS_CONV = 80, L_REGS_SOFT = 144;
static_assert(128 * L_REGS_ISSUE + L_CONV * 32 * L_REGS_CONV + L_SOFT * 32 * L_REGS_SOFT <= L_THREADS * 96, "registers");

// what the warps share beside the tiles
struct LeadShared {
    float ks[4];              // inverse scale of the keys, by tile % 4
    float vs[4][8];           // inverse scales of the values' blocks, by tile % 4
    float row[2][2][LQ];      // row maxima of the two halves
    float stat[2][LQ];        // maxima and sums of the rows
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full, s_free, p_full, o_full;
    uint64_t rk_full[2], rk_empty[2], rv_full[2], rv_empty[2];  // the raw pages
    uint64_t drained;         // the products of a CTA that gives up
    uint32_t tmem_slot;
    int abort_flag, lost;     // lost: a page id outside the cache
};

// two f32 operations in one
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair(float a, float b) {
    f32x2 v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ f32x2 pair(uint32_t a, uint32_t b) { return pair(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 both(f32x2 v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <uint32_t KIND, uint32_t HD>
struct LeadTile {
    static constexpr uint32_t NB = HD / 32, TERMS = KIND == KV_F16 ? 1 : 2;
    static constexpr uint32_t HALVES = HD / 64;              // 64-dimension accumulators of a score
    static constexpr uint32_t K_PLANE = LK * 128;            // 64 dimensions of the tile's keys, one term
    static constexpr uint32_t K_STAGE = TERMS * HALVES * K_PLANE;
    static constexpr uint32_t V_PLANE = HD * 128;            // the tile's keys of every dimension, one term
    static constexpr uint32_t V_STAGE = TERMS * V_PLANE;
    static constexpr uint32_t RAW = kv_head_bytes(KIND, HD) / 2;  // a page's keys or values of a head
    static constexpr uint32_t TILES = 2 * (K_STAGE + V_STAGE), PITCH = HD + 4;  // rows of the result in the tiles' place
    static constexpr uint32_t SMEM = TILES + 4 * RAW + sizeof(LeadShared);
    static_assert(SMEM <= 227 * 1024 && LQ * PITCH * 4 <= TILES + 4 * RAW && RAW % 16 == 0, "shared memory");
    // tensor memory columns
    static constexpr uint32_t Q_HI = 0, Q_LO = HD / 2, S0 = HD, P0 = S0 + 64 * HALVES, O = P0 + 64;
    static_assert(O + HD <= 512, "tensor memory");
};

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
__global__ void __launch_bounds__(L_THREADS, 1) attention_lead_tiles_kernel(PagedArgs a, float* __restrict__ lead, int* __restrict__ error_flag) {
    using T = LeadTile<KIND, HD>;
    constexpr uint32_t NB = T::NB, HEAD = kv_head_bytes(KIND, HD), CODES = kv_code_bytes(KIND, HD);
    constexpr int TOP = KIND == KV_Q4_0 ? 26 : 22;  // a scale below 2^(e - 14) times 2^(TOP - e) times a code stays below 2^15
    extern __shared__ __align__(1024) uint8_t smem[];  // K and V stages | raw keys, raw values | LeadShared
    const uint32_t k_base = smem_u32(smem), v_base = k_base + 2 * T::K_STAGE;
    uint8_t* raw_k = smem + T::TILES;
    uint8_t* raw_v = raw_k + 2 * T::RAW;
    LeadShared& sh = *reinterpret_cast<LeadShared*>(raw_v + 2 * T::RAW);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool aligned = k_base % 1024 == 0;  // the swizzle's period; no static shared memory stands in front
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.k_full[i], L_CONV);
            mbar_init(&sh.v_full[i], L_CONV);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.rk_full[i], 1);
            mbar_init(&sh.rv_full[i], 1);
            mbar_init(&sh.rk_empty[i], L_CONV);
            mbar_init(&sh.rv_empty[i], L_CONV);
        }
        mbar_init(&sh.s_full, 1);
        mbar_init(&sh.s_free, L_SOFT);
        mbar_init(&sh.p_full, L_SOFT);
        mbar_init(&sh.o_full, 1);
        mbar_init(&sh.drained, 1);
        sh.abort_flag = !aligned, sh.lost = 0;
        mbar_fence_init();
    }
    if (warp == L_SOFT + L_CONV) {
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
    const uint32_t split = blockIdx.x, kvh = blockIdx.z, rows = a.c.n_seq * a.group, row0 = blockIdx.y * LQ;
    const uint32_t p0 = (uint32_t)((uint64_t)split * a.done / gridDim.x), p1 = (uint32_t)((uint64_t)(split + 1) * a.done / gridDim.x);
    const uint32_t n_tiles = aligned ? p1 - p0 : 0;
    bool ok = true;  // the same in all lanes of a warp; once false, the warp waits for nothing more
    auto wait_all = [&](uint64_t* bar, uint32_t parity) {
        return ok = __all_sync(0xFFFFFFFFu, mbar_wait(bar, parity));
    };
    // The common exit, where all warps meet: whether some wait of the CTA ran out.
    auto leave = [&] {
        if (!ok && lane == 0) *static_cast<volatile int*>(&sh.abort_flag) = 1;
        tc_fence_before();
        asm volatile("bar.sync 6, %0;" ::"n"(L_THREADS) : "memory");
        return *static_cast<volatile int*>(&sh.abort_flag) != 0;
    };

    if (warp < L_SOFT) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L_REGS_SOFT));
        // ── softmax: thread = (query row, half) ──
        const uint32_t quarter = warp & 3, half = warp >> 2, row = quarter * 32 + lane, at = row0 + row;
        const uint32_t lanes = tmem + ((quarter * 32) << 16);
        constexpr uint32_t DN = HD / 2;  // dimensions of this thread
        float rf;                        // inverse scale of the query row, times log2(e) and the softmax scale
        auto pair_bar = [&] { asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory"); };
        f32x2 o[DN / 2];
        {
            const bool live = at < rows;
            const float4* src = reinterpret_cast<const float4*>(
                a.q + (live ? at / a.group : 0) * a.q_stride + (uint64_t)(kvh * a.group + (live ? at % a.group : 0)) * HD + half * DN);
            float amax = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < DN / 4; ++i) {
                const float4 v = live ? src[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                o[2 * i] = pair(v.x, v.y), o[2 * i + 1] = pair(v.z, v.w);
                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
            }
            sh.row[1][half][row] = amax;
            pair_bar();
            amax = fmaxf(amax, sh.row[1][half ^ 1][row]);
            // a power of two that puts the row's largest value just below 2^15, with the sign of the scale: the row's maximum is
            // looked for before the scores are multiplied by rf, which must not turn their order round
            const uint32_t e = __float_as_uint(amax) >> 23, bits = e == 255 ? 127u : min(254u, 268u - e);
            const float sc = copysignf(__uint_as_float(bits << 23), a.scale);
            rf = (bits == 254 ? __uint_as_float(0x00400000u) : __uint_as_float((254u - bits) << 23)) * (fabsf(a.scale) * 1.44269504f);
#pragma unroll
            for (uint32_t c = 0; c < DN / 32; ++c) {
                uint32_t hi[16], lo[16];
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) {
                    const float2 v = both(o[16 * c + i]);
                    split2(v.x * sc, v.y * sc, &hi[i], &lo[i]);
                }
                tmem_st16(lanes + T::Q_HI + half * (DN / 2) + 16 * c, hi);
                tmem_st16(lanes + T::Q_LO + half * (DN / 2) + 16 * c, lo);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_free);  // the first scores wait for the query's terms
        }
#pragma unroll
        for (uint32_t i = 0; i < DN / 2; ++i) o[i] = 0;
        float mx = -INFINITY, alpha_prev = 0.0f;
        f32x2 sums = 0;  // sum and outputs times 2^UP, as the probabilities are
        // o = o * alpha + the tile's output
        auto add_tile = [&](uint32_t j, float alpha) {
            if (__any_sync(0xFFFFFFFFu, alpha != 1.0f)) {
#pragma unroll
                for (uint32_t i = 0; i < DN / 2; ++i) o[i] = mul2(o[i], pair(alpha, alpha));
            }
            if (!wait_all(&sh.o_full, j & 1)) return;
            tc_fence_after();
#pragma unroll
            for (uint32_t c = 0; c < DN / 32; ++c) {
                uint32_t r[32];
                tmem_ld32(lanes + T::O + half * DN + 32 * c, r);
                const float f = KIND == KV_F16 ? 1.0f : sh.vs[j & 3][half * (DN / 32) + c];
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) {
                    f32x2& x = o[16 * c + i];
                    x = KIND == KV_F16 ? add2(x, pair(r[2 * i], r[2 * i + 1])) : fma2(pair(r[2 * i], r[2 * i + 1]), pair(f, f), x);
                }
            }
        };
        uint32_t j = 0;  // tiles whose barrier this warp has come to
        while (j < n_tiles) {
            f32x2 sc[16];
            if (!wait_all(&sh.s_full, j & 1)) break;
            tc_fence_after();
            {
                uint32_t r[32];
                tmem_ld32(lanes + T::S0 + half * 32, r);
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = pair(r[2 * i], r[2 * i + 1]);
                if constexpr (T::HALVES == 2) {
                    tmem_ld32(lanes + T::S0 + 64 + half * 32, r);
#pragma unroll
                    for (int i = 0; i < 16; ++i) sc[i] = add2(sc[i], pair(r[2 * i], r[2 * i + 1]));
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.s_free);
            const float f = KIND == KV_F16 ? rf : rf * sh.ks[j & 3];
            float cm = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 v = both(sc[i]);
                cm = max3(cm, v.x, v.y);
            }
            sh.row[j & 1][half][row] = cm;
            pair_bar();
            const float t = fmaxf(cm, sh.row[j & 1][half ^ 1][row]) * f;
            float alpha = 1.0f;
            if (t > mx + LAZY) alpha = ex2(mx - t), mx = t;  // 0 on the first tile (mx = -inf)
            const f32x2 ff = pair(f, f), shift = pair((float)UP - mx, (float)UP - mx);
            f32x2 ps = 0;
            uint32_t w0[16], w1[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float2 y = both(fma2(sc[i], ff, shift));
                const float p = ex2(y.x), q = ex2(y.y);
                const f32x2 both_p = pair(p, q);
                ps = add2(ps, both_p);
                const __half2 h = __floats2half2_rn(p, q);
                const float2 g = __half22float2(h);
                const float2 rest = both(fma2(pair(g.x, g.y), pair(-1.0f, -1.0f), both_p));
                w0[i] = half2_bits(h), w1[i] = half2_bits(__floats2half2_rn(rest.x, rest.y));
            }
            sums = fma2(sums, pair(alpha, alpha), ps);
            if (j++ > 0) add_tile(j - 2, alpha_prev);  // its products have read the probabilities before these
            if (!ok) break;
            alpha_prev = alpha;
            tmem_st16(lanes + T::P0 + half * 16, w0);
            tmem_st16(lanes + T::P0 + 32 + half * 16, w1);
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full);
        }
        for (; j < n_tiles; ++j) pair_bar();  // the other half of the rows may not have given up
        if (ok && n_tiles) add_tile(n_tiles - 1, alpha_prev);
        const float2 two = both(sums);
        const float sum = two.x + two.y;
        sh.row[n_tiles & 1][half][row] = sum;
        pair_bar();
        const float all = sum + sh.row[n_tiles & 1][half ^ 1][row];
        const bool bad = leave() || sh.lost != 0;
        // the rows in the tiles' place, then those of the cluster's CTAs (splits of the same rows) joined, a share of the rows a CTA
        float* stage = reinterpret_cast<float*>(smem);
#pragma unroll
        for (uint32_t i = 0; i < DN / 4; ++i) {
            const float2 u = both(o[2 * i]), v = both(o[2 * i + 1]);
            *reinterpret_cast<float4*>(stage + row * T::PITCH + half * DN + 4 * i) =
                make_float4(u.x * power(-UP), u.y * power(-UP), v.x * power(-UP), v.y * power(-UP));
        }
        if (half == 0) sh.stat[0][row] = mx, sh.stat[1][row] = bad ? NAN : all * power(-UP);
        __syncwarp();
        cluster_sync_all();
        uint32_t ctas, rank;
        asm volatile("mov.u32 %0, %cluster_nctarank;" : "=r"(ctas));
        asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
        const uint64_t every = (uint64_t)(gridDim.x / ctas) * a.c.n_kv * rows, base = ((uint64_t)(split / ctas) * a.c.n_kv + kvh) * rows;
        const uint32_t stage_at = smem_u32(stage), stat_at = smem_u32(&sh.stat[0][0]), share = LQ / ctas;
        // the weight of every CTA's part of a row, a thread each, first those of the row's maximum
        constexpr uint32_t MOST = 8;  // CTAs
        float* weight = &sh.row[0][0][0];  // [share][ctas]
        const uint32_t r = rank * share + tid / 2 % share;  // two threads a row, half of the CTAs each
        if (tid < 2 * share) {
            float m[MOST / 2], l[MOST / 2], top = -INFINITY, den = 0.0f;
#pragma unroll
            for (uint32_t k = 0; k < MOST / 2; ++k) {
                const uint32_t c = 2 * k + tid % 2;
                m[k] = c < ctas ? ld_cluster_f32(stat_at + r * 4, c) : -INFINITY, l[k] = c < ctas ? ld_cluster_f32(stat_at + (LQ + r) * 4, c) : 0.0f;
            }
#pragma unroll
            for (uint32_t k = 0; k < MOST / 2; ++k) top = fmaxf(top, m[k]);
            top = fmaxf(top, __shfl_xor_sync(__activemask(), top, 1));
#pragma unroll
            for (uint32_t k = 0; k < MOST / 2; ++k) {
                const uint32_t c = 2 * k + tid % 2;
                const float f = piece_weight(m[k], top);
                if (c < ctas) weight[tid / 2 * ctas + c] = f, den = fmaf(f, l[k], den);
            }
            den += __shfl_xor_sync(__activemask(), den, 1);
            if (tid % 2 == 0 && row0 + r < rows) lead[every * HD + base + row0 + r] = top, lead[every * HD + every + base + row0 + r] = den;
        }
        asm volatile("bar.sync 5, %0;" ::"n"(L_SOFT * 32) : "memory");
#pragma unroll 2
        for (uint32_t i = tid; i < share * (HD / 4); i += L_SOFT * 32) {
            const uint32_t k = i / (HD / 4), d = i % (HD / 4) * 4, at_row = rank * share + k;
            float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
            for (uint32_t c = 0; c < ctas; ++c) {
                uint32_t from;
                float4 y;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(from) : "r"(stage_at + (at_row * T::PITCH + d) * 4), "r"(c));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(from));
                const float f = weight[k * ctas + c];
                x.x = fmaf(f, y.x, x.x), x.y = fmaf(f, y.y, x.y), x.z = fmaf(f, y.z, x.z), x.w = fmaf(f, y.w, x.w);
            }
            if (row0 + at_row < rows) *reinterpret_cast<float4*>(lead + (base + row0 + at_row) * HD + d) = x;
        }
    } else if (warp < L_SOFT + L_CONV) {
        // ── converters ──
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L_REGS_CONV));
        const uint32_t cw = warp - L_SOFT, r = lane / 4, c = lane % 4;
        auto publish = [&](uint64_t* bar) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // 16 bytes (8 halves) of a key row: dimensions 32 b + 8 c .., in the 128-byte swizzle
        auto key_at = [&](uint32_t st, uint32_t row, uint32_t b) {
            return k_base + st * T::K_STAGE + (b / 2) * T::K_PLANE + row * 128 + ((((b % 2) * 4 + c) ^ (row & 7)) << 4);
        };
        // 16 bytes (8 keys: 8 chunk ..) of a dimension's row of values
        auto value_at = [&](uint32_t st, uint32_t d, uint32_t chunk) { return v_base + st * T::V_STAGE + d * 128 + ((chunk ^ (d & 7)) << 4); };
        constexpr uint32_t K_LO = T::HALVES * T::K_PLANE, V_LO = T::V_PLANE;

        auto convert_keys = [&](uint32_t j, uint32_t st, const uint8_t* raw) {
            if constexpr (KIND == KV_F16) {
#pragma unroll
                for (uint32_t i = cw; i < 4 * NB; i += L_CONV) {
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
                if (cw == 0 && lane == 0) sh.ks[j & 3] = power(e - TOP);
#pragma unroll 2
                for (uint32_t i = cw; i < 4 * NB / BLOCKS; i += L_CONV) {
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
        };
        // values: keys run along a row of the tile, so four lanes' words are transposed: lane c then has eight keys of two
        // dimensions (halves: of one)
        auto convert_values = [&](uint32_t j, uint32_t st, const uint8_t* raw) {
            if constexpr (KIND == KV_F16) {
#pragma unroll
                for (uint32_t i = cw; i < 8 * NB; i += L_CONV) {
                    const uint32_t g = i / (2 * NB), b = i / 2 % NB, m = i % 2;
                    const uint4 x = *reinterpret_cast<const uint4*>(raw + i * 512 + lane * 16);
                    uint32_t w[4] = {x.x, x.y, x.z, x.w};
                    transpose4(w, c);
                    sts_v4(value_at(st, 32 * b + 4 * r + 2 * m + c % 2, 2 * g + c / 2), w);
                }
            } else {
                constexpr uint32_t BLOCKS = KIND == KV_Q8_0 ? 1 : 2;
#pragma unroll 2
                for (uint32_t i = cw; i < 4 * NB / BLOCKS; i += L_CONV) {
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
                        if (g == 0 && lane == 0) sh.vs[j & 3][b0 + o] = power(e - TOP);
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
        };
        for (uint32_t j = 0; j < n_tiles; ++j) {
            const uint32_t st = j & 1, turn = (j >> 1) & 1;
            if (!wait_all(&sh.k_empty[st], turn ^ 1) || !wait_all(&sh.rk_full[st], turn)) break;
            convert_keys(j, st, raw_k + st * T::RAW);
            publish(&sh.k_full[st]);
            if (lane == 0) mbar_arrive(&sh.rk_empty[st]);
            if (!wait_all(&sh.v_empty[st], turn ^ 1) || !wait_all(&sh.rv_full[st], turn)) break;
            convert_values(j, st, raw_v + st * T::RAW);
            publish(&sh.v_full[st]);
            if (lane == 0) mbar_arrive(&sh.rv_empty[st]);
        }
        leave();
        __syncwarp();
        cluster_sync_all();
    } else {
        // ── issuer (one warp issues, one copies, two have nothing to do) ──
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L_REGS_ISSUE));
        if (warp == L_SOFT + L_CONV) {
            constexpr uint32_t idesc_s = umma_idesc_f16(LK), idesc_o = umma_idesc_f16(HD);
            const uint64_t dk = umma_desc(k_base), dv = umma_desc(v_base);
            auto scores = [&](uint32_t j) {  // one accumulator per 64 dimensions, small products first
                // the scores before have been read (the first: the query is in place)
                if (!wait_all(&sh.s_free, j & 1) || !wait_all(&sh.k_full[j & 1], (j >> 1) & 1)) return;
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
            if (n_tiles) scores(0);
            for (uint32_t j = 0; j < n_tiles && ok; ++j) {
                if (j + 1 < n_tiles) scores(j + 1);
                // the probabilities are in place, the output before has been read
                if (!ok || !wait_all(&sh.v_full[j & 1], (j >> 1) & 1) || !wait_all(&sh.p_full, j & 1)) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t hi = dv + (uint64_t)(j & 1) * (T::V_STAGE >> 4), lo = hi + (T::V_PLANE >> 4);
                    const uint32_t d = tmem + T::O, p_hi = tmem + T::P0, p_lo = p_hi + 32;
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk) {
                        umma_f16_ts(d, p_lo + 8 * kk, hi + 2 * kk, idesc_o, kk != 0);
                        if constexpr (T::TERMS == 2) umma_f16_ts(d, p_hi + 8 * kk, lo + 2 * kk, idesc_o, 1);
                    }
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk) umma_f16_ts(d, p_hi + 8 * kk, hi + 2 * kk, idesc_o, 1);
                    umma_commit(&sh.v_empty[j & 1]);
                    umma_commit(&sh.o_full);
                }
                __syncwarp();
            }
            if (!ok) {  // products in flight still use tensor memory and the tiles
                if (elect_one()) umma_commit(&sh.drained);
                __syncwarp();
                mbar_wait(&sh.drained, 0);
            }
        } else if (warp == L_SOFT + L_CONV + 1) {
            // ── loader: a page's keys, or values, of a head are one run of memory; page ids 32 at a time, a lane each ──
            uint32_t k_sent = 0, v_sent = 0;
            int32_t ids = 0;
            for (uint32_t j = 0; j < n_tiles && ok; ++j) {
                if (j % 32 == 0) ids = j + lane < n_tiles ? a.c.table[p0 + j + lane] : 0;
                const int32_t id = __shfl_sync(0xFFFFFFFFu, ids, j % 32);
                const bool fine = id >= 0 && (uint32_t)id < a.c.n_pages;
                if (!fine && lane == 0) sh.lost = 1;
                const uint8_t* src = a.c.pages + ((uint64_t)(fine ? id : 0) * a.c.n_kv + kvh) * HEAD;
                const uint32_t st = j & 1, freed = ((j >> 1) & 1) ^ 1;
                if (!wait_all(&sh.rk_empty[st], freed)) break;
                ++k_sent;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh.rk_full[st], T::RAW);
                    bulk_g2s(raw_k + st * T::RAW, src, T::RAW, &sh.rk_full[st]);
                }
                if (!wait_all(&sh.rv_empty[st], freed)) break;
                ++v_sent;
                if (lane == 0) {
                    mbar_arrive_expect_tx(&sh.rv_full[st], T::RAW);
                    bulk_g2s(raw_v + st * T::RAW, src + T::RAW, T::RAW, &sh.rv_full[st]);
                }
            }
            if (!ok) {  // copies in flight still write to shared memory
                for (uint32_t back = 1; back <= 2; ++back) {
                    if (k_sent >= back) mbar_wait(&sh.rk_full[(k_sent - back) & 1], ((k_sent - back) >> 1) & 1);
                    if (v_sent >= back) mbar_wait(&sh.rv_full[(v_sent - back) & 1], ((v_sent - back) >> 1) & 1);
                }
            }
        }
        leave();
        __syncwarp();
        cluster_sync_all();
    }
    if (tid == 0) {
        if (sh.abort_flag && error_flag) *reinterpret_cast<volatile int*>(error_flag) = 1;
        if (sh.lost && a.bad_pos) atomicExch(a.bad_pos, 1);
    }
    __syncwarp();
    tc_fence_after();
    if (warp == L_SOFT + L_CONV)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    __syncwarp();
    cluster_sync_all();  // the others have read this CTA's rows
}

struct LaunchLead {
    const PagedArgs& a;
    float* lead;
    uint32_t splits, blocks, cluster;
    int* error_flag;
    cudaStream_t s;
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        if constexpr (HD > 128) {
            return cudaErrorInvalidValue;
        } else {
            auto kern = attention_lead_tiles_kernel<KIND, HD>;
            static bool configured[MAX_DEVICES] = {};
            if (cudaError_t e = set_max_smem_once(kern, LeadTile<KIND, HD>::SMEM, configured); e != cudaSuccess) return e;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(splits, blocks, a.c.n_kv);
            cfg.blockDim = dim3(L_THREADS);
            cfg.dynamicSmemBytes = LeadTile<KIND, HD>::SMEM;
            cfg.stream = s;
            cudaLaunchAttribute attr[2];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = cluster, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
            attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[1].val.programmaticStreamSerializationAllowed = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 2;
            return cudaLaunchKernelEx(&cfg, kern, a, lead, error_flag);
        }
    }
};

}  // namespace

cudaError_t launch_attention_lead_tiles(const PagedArgs& a, float* lead, uint32_t splits, uint32_t blocks, uint32_t cluster, int* error_flag,
                                        cudaStream_t s) {
    return for_kind(a.c.kind, a.c.hd, LaunchLead{a, lead, splits, blocks, cluster, error_flag, s});
}

}  // namespace jq
