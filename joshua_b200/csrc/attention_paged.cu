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

#include "attention_steps.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;


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
            w.softmax(s, Below{T::POS}, lane, alpha);
            w.output(s, v, Below{T::POS}, lane, alpha);
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
        auto kern = attention_paged_kernel<T, PAIRS, WARPS, false>;
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
