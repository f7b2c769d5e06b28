// Attention of some new tokens of every sequence over the pages of the quantised cache, causal, with a window and sinks if wanted.
//
// Rows first[b] .. first[b + 1] - 1 of q are the last positions of sequence b.  Row r at position p: out[r, head, :] =
// sum_t e_t V_t / sum_t e_t, e_t = exp(scale q . K_t - max), over t <= p with (no window, or p - t < window, or t < sinks).
// Sequences of few rows, and all with heads of 256, are taken row by row, each as a sequence of its own by attention_paged_kernel
// (attention_steps.cuh), cut into equal pieces of work whatever the lengths: the codes of its positions are read once a row.  (So a prompt
// with heads of 256 takes as long as its rows: 2000 behind 2000, 16 heads on 4 in eight bits, 2.27 ms; 8 on 2 in halves 0.97.)  The
// others go to the tiles of attention_chunk_tiles.cu.  Which are which is known on the device alone where `first` tells: both are
// launched then, one after the other, and each leaves the other's sequences (four tokens of 32 sequences: 122 us, with `first` 137).
#include <algorithm>

#include "attention_chunk.cuh"
#include "attention_steps.cuh"

namespace jq {

namespace {

// Passes over a sequence's pages, rows times warps' worth of heads, up to which its rows are taken one by one: a tile takes as long as
// three to four of them (16 sequences of up to 4000 positions, two / three / four rows one by one and eight in tiles: 32 heads on 8 of
// 128 in eight bits 29 / 45 / 56 and 60 us, in halves 32 / 49 / 73 and 64, 32 heads on 4 27 / 41 / 47 and 41).  Several tokens a pass in
// attention_paged_kernel, 16 query rows, was no faster than one by one: its products are the bound.
constexpr uint32_t CHUNK_FEW = 3;

struct ChunkPlan {
    uint32_t group, rows, split, grid;  // query heads a kv head; of a warp; warps' worth of them; CTAs
    uint32_t few;                       // rows of a sequence that are taken one by one
    bool tiles;                         // some sequence may have more
    size_t part_at, bytes;
};
ChunkPlan plan(uint32_t rows, uint32_t n_q, uint32_t n_kv, uint32_t hd) {
    ChunkPlan p{};
    p.group = n_q / n_kv;
    p.rows = p.group <= 4 ? 4 : 8;
    p.split = (p.group + p.rows - 1) / p.rows;
    p.grid = std::min((uint32_t)num_sms(), ATTENTION_MOST_CTAS);
    p.part_at = ATTENTION_MOST_CTAS * 4;
    p.few = hd <= 128 ? std::max(1u, CHUNK_FEW / p.split) : 0xFFFFFFFFu;
    p.tiles = rows > p.few;
    p.bytes = p.part_at + (size_t)p.grid * 2 * (p.tiles ? CHUNK_TILE_ROWS : p.rows) * (hd + 2) * 4;
    return p;
}

struct LaunchChunk {
    const PagedArgs& a;
    const ChunkPlan& p;
    cudaStream_t s;

    template <class T, bool PAIRS>
    cudaError_t rows() const {
        using At = Attend<T, 1, PAIRS>;
        constexpr uint32_t WARPS = ap_warps(T::HD), BYTES = WARPS * (2 * At::Q::ROWS * (T::HD + 2) + At::Q::WORDS) * 4;
        auto kern = attention_paged_kernel<T, PAIRS, WARPS, true>;
        static bool configured[MAX_DEVICES] = {};
        if (cudaError_t e = set_max_smem_once(kern, BYTES + (ATTENTION_MAX_BATCH + 4) * 4, configured); e != cudaSuccess) return e;
        return launch_pdl(kern, dim3(p.grid), WARPS * 32, BYTES + ((a.c.n_seq + 4) & ~3u) * 4, s, a);
    }
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        using T = Step<KIND, HD>;
        return p.rows == 4 ? rows<T, true>() : rows<T, false>();
    }
};

}  // namespace

size_t attention_chunk_scratch_bytes(uint32_t rows, uint32_t n_q, uint32_t n_kv, uint32_t hd) { return plan(rows, n_q, n_kv, hd).bytes; }

cudaError_t launch_attention_chunk(const KvPages& c, const float* q, uint64_t q_stride, const int32_t* first, const int32_t* len, uint32_t rows,
                                   uint32_t n_q, float scale, uint32_t window, uint32_t sinks, float* out, uint64_t out_stride,
                                   void* scratch, int32_t* bad_pos, int* error_flag, cudaStream_t s) {
    const ChunkPlan p = plan(rows, n_q, c.n_kv, c.hd);
    uint8_t* mem = static_cast<uint8_t*>(scratch);
    PagedArgs a{c, q, q_stride, len, n_q, p.group, p.split, scale, 0, 0, out, out_stride,
                reinterpret_cast<uint32_t*>(mem), reinterpret_cast<float*>(mem + p.part_at), nullptr, 0, bad_pos};
    a.span = SpanArgs{first, rows, first ? 0 : rows / c.n_seq, p.few, window, sinks};
    if (first ? p.tiles : a.span.each > p.few) {
        cudaError_t e = launch_attention_chunk_tiles(a, p.grid, error_flag, s);
        if (e != cudaSuccess || !first) return e != cudaSuccess ? e : cudaGetLastError();
    }
    cudaError_t e = for_kind(c.kind, c.hd, LaunchChunk{a, p, s});
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
