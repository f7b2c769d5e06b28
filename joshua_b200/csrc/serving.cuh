// Launchers of the serving operators: rotary positions, paged cache, attention over it, sampling.
#pragma once

#include <algorithm>

#include "common.cuh"
#include "pipe.cuh"
#include "rope.cuh"

namespace jq {

// The first two statements of a kernel whose predecessor in the stream may still run.  What that one may have written is then read
// by plain loads: read-only ones (__ldg, or plain ones through const __restrict__) may be moved above the wait, unless their address
// comes from such a plain load.
__device__ __forceinline__ void pdl_trigger_all() {
    pdl_trigger();
    pdl_wait();
}

constexpr uint32_t ROPE_MAX_ROT = 256;
struct RopeFrequencies {
    double f[ROPE_MAX_ROT / 2];
    double scale;  // of cosines and sines
};
cudaError_t launch_rope_table(const RopeFrequencies& f, uint32_t rot, uint32_t n_pos, float* table, cudaStream_t s);
cudaError_t launch_rope(const RopeArgs& r, const float* x, uint64_t x_stride, const int32_t* pos, uint32_t rows, uint32_t heads,
                        uint32_t hd, bool inverse, float* out, uint64_t out_stride, int32_t* bad_pos, cudaStream_t s);

// A paged cache and the pages of some sequences: position p of sequence i stands in page table[i * table_stride + p / 64].
struct KvPages {
    uint8_t* pages;
    uint32_t n_pages, n_kv, kind, hd;
    const int32_t* table;
    uint32_t n_seq, table_stride;
};
cudaError_t launch_kv_append(const KvPages& c, const RopeArgs& r, const float* qkv, uint64_t stride, const int32_t* pos,
                             const int32_t* seq, uint32_t rows, uint32_t n_q, const float* q_norm, const float* k_norm, float eps,
                             float* q_out, int32_t* bad_pos, cudaStream_t s);
cudaError_t launch_kv_read(const KvPages& c, const int32_t* pos, const int32_t* seq, uint32_t rows, float* k, float* v,
                           uint64_t row_stride, uint64_t head_stride, int32_t* bad_pos, cudaStream_t s);
// One query row a sequence and head over positions 0 .. len - 1; the first `shared` pages of sequence 0 are everybody's.
constexpr uint32_t ATTENTION_MAX_BATCH = 4096, ATTENTION_MOST_CTAS = 256;  // the scratch begins with a counter a CTA
size_t attention_paged_scratch_bytes(uint32_t batch, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t shared);
cudaError_t launch_attention_paged(const KvPages& c, const float* q, uint64_t q_stride, const int32_t* len, uint32_t n_q, float scale,
                                   uint32_t shared, float* out, uint64_t out_stride, void* scratch, int32_t* bad_pos, int* error_flag,
                                   cudaStream_t s);

// Rows first[i] .. first[i + 1] - 1 (NULL: rows / n_seq each) of q are the last positions of sequence i, which has len[i]; window 0: a
// row sees all positions up to its own, else that many and the first `sinks`.
constexpr uint32_t ATTENTION_MAX_ROWS = 65536;
// The kernels count steps of 16 positions (and a little for each row), and rows times heads, in 32 bits.
constexpr uint64_t SPAN_MOST_SEGMENTS = 1u << 27;  // rows of a call times query heads
__host__ __device__ constexpr bool span_rows_fit(uint64_t rows, uint32_t table_stride, uint32_t n_q) {
    return rows * (4 * (uint64_t)table_stride + 8) <= 0xFFFFFFFFull && rows * n_q <= SPAN_MOST_SEGMENTS;
}
size_t attention_chunk_scratch_bytes(uint32_t rows, uint32_t n_q, uint32_t n_kv, uint32_t hd);
cudaError_t launch_attention_chunk(const KvPages& c, const float* q, uint64_t q_stride, const int32_t* first, const int32_t* len, uint32_t rows,
                                   uint32_t n_q, float scale, uint32_t window, uint32_t sinks, float* out, uint64_t out_stride,
                                   void* scratch, int32_t* bad_pos, int* error_flag, cudaStream_t s);

struct SampleArgs {
    const float* logits;
    uint64_t stride;
    uint32_t vocab;
    const float* uniform;
    const float* temperature;  // NULL: 1
    const int32_t* top_k;      // NULL: off
    const float* top_p;        // NULL: off
    const float* min_p;        // NULL: off
    float penalty;
    int32_t* window;           // NULL: no penalty
    int32_t* window_state;
    int32_t* token;
    float* prob;               // NULL: not wanted
    int32_t* pos;              // NULL: no positions to advance
};
// Log probability of a token of every row, entropy, the `top` likeliest tokens.
struct LogProbArgs {
    const float* logits;
    uint64_t stride;
    uint32_t vocab;
    const int32_t* token;
    uint32_t top;           // at most LOG_PROBS_MOST
    float* log_prob;
    float* entropy;         // NULL: not wanted
    int32_t* top_token;     // [rows][top]
    float* top_log_prob;
};
constexpr uint32_t LOG_PROBS_MOST = 32;
cudaError_t launch_log_probs(const LogProbArgs& a, uint32_t rows, cudaStream_t s);

constexpr uint32_t SAMPLE_MAX_VOCAB = 8 * 49152;
cudaError_t launch_sample(const SampleArgs& a, uint32_t rows, cudaStream_t s);

}  // namespace jq
