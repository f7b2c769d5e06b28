// C ABI of the serving operators.  Declarations are in include/joshua_b200.h.
#include <cmath>

#include "handles.cuh"
#include "kv_pages.cuh"
#include "serving.cuh"

namespace {

int32_t bad(const char* who, const std::string& why) { return jq_fail(jq::E_INVALID, std::string(who) + ": " + why); }

bool unaligned(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
    return (reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
            reinterpret_cast<uintptr_t>(d)) % 16 != 0;
}

int32_t check_rope(const char* who, const jq_rope* r, uint32_t head_dim, jq::RopeArgs* out) {
    *out = jq::RopeArgs{};
    if (!r) return jq::OK;
    if (!r->table || reinterpret_cast<uintptr_t>(r->table) % 8 != 0) return bad(who, "the rope table must be set and 8-byte aligned");
    if (r->rot_dim == 0 || r->rot_dim % 2 || r->rot_dim > head_dim)
        return bad(who, "rot_dim " + std::to_string(r->rot_dim) + " must be even, above 0 and at most head_dim " + std::to_string(head_dim));
    if (r->interleaved != 0 && r->interleaved != 1) return bad(who, "interleaved must be 0 or 1");
    *out = jq::RopeArgs{reinterpret_cast<const float2*>(r->table), r->n_pos, r->rot_dim, (uint32_t)r->interleaved,
                        r->rot_dim % 8 == 0 && !unaligned(r->table)};
    return jq::OK;
}

int32_t check_cache(const char* who, const jq_kv_cache* c, const int32_t* table, uint32_t n_seq, uint32_t stride, jq::KvPages* out) {
    if (!c || !c->pages || !table) return bad(who, "NULL cache, pages or page table");
    if (jq_kv_page_bytes(c->type, c->n_kv, c->head_dim) == 0)
        return bad(who, "need a type of JQ_KV_F16, JQ_KV_Q8_0 or JQ_KV_Q4_0, head_dim 64, 128 or 256 and 1 to 1024 kv heads");
    if (unaligned(c->pages)) return bad(who, "pages must be 16-byte aligned");
    if (c->n_pages == 0 || c->n_pages > 0x7FFFFFFFu || n_seq == 0 || n_seq > 0x7FFFFFFFu || stride == 0 || stride > 0x7FFFFFFFu / JQ_KV_PAGE)
        return bad(who, "a cache without pages, a page table without entries, or more positions than 32 bits count");
    *out = jq::KvPages{static_cast<uint8_t*>(c->pages), c->n_pages, c->n_kv, c->type, c->head_dim, table, n_seq, stride};
    return jq::OK;
}

// n query heads on the cache's kv heads
int32_t check_heads(const char* who, const jq_kv_cache* c, uint32_t n_q) {
    if (n_q != 0 && n_q % c->n_kv == 0 && n_q <= 4096) return jq::OK;
    return bad(who, std::to_string(n_q) + " query heads on " + std::to_string(c->n_kv) + " kv heads");
}
// whether rows of `width` floats share any: a's and b's, `rows` of each
bool rows_meet(const float* a, uint64_t a_stride, const float* b, uint64_t b_stride, uint32_t rows, uint64_t width) {
    const uint64_t x = reinterpret_cast<uintptr_t>(a) / 4, y = reinterpret_cast<uintptr_t>(b) / 4;
    if (x + (rows - 1) * a_stride + width <= y || y + (rows - 1) * b_stride + width <= x) return false;
    if (rows == 1 || a_stride != b_stride) return true;  // side by side only as columns of one buffer
    const uint64_t ahead = x <= y ? (y - x) % a_stride : (a_stride - (x - y) % a_stride) % a_stride;
    return ahead < width || ahead > a_stride - width;
}

}  // namespace

extern "C" {

int32_t jq_rope_table_dev(const jq_rope_config* cfg, const float* freq_factors, uint32_t rot_dim, uint32_t n_pos, float* table_dev,
                          void* stream) {
    constexpr const char* who = "jq_rope_table_dev";
    if (!cfg || !table_dev) return bad(who, "NULL argument");
    if (rot_dim == 0 || rot_dim % 2 || rot_dim > jq::ROPE_MAX_ROT) return bad(who, "rot_dim must be even and in 2 .. 256");
    if (reinterpret_cast<uintptr_t>(table_dev) % 8 != 0) return bad(who, "the table must be 8-byte aligned");
    if (!(cfg->theta > 0.0) || !std::isfinite(cfg->theta)) return bad(who, "theta must be positive");
    if (cfg->scaling < JQ_ROPE_NONE || cfg->scaling > JQ_ROPE_YARN) return bad(who, "unknown scaling");
    if (cfg->scaling != JQ_ROPE_NONE && (!(cfg->factor > 0.0f) || !std::isfinite(cfg->factor))) return bad(who, "the factor must be positive");
    if (!(cfg->mscale >= 0.0f) || !std::isfinite(cfg->mscale)) return bad(who, "mscale must not be negative");
    double low = 0.0, high = 0.0;
    const uint32_t half = rot_dim / 2;
    if (cfg->scaling == JQ_ROPE_YARN) {
        if (cfg->orig_ctx == 0 || !(cfg->beta_slow > 0.0f) || !(cfg->beta_fast > cfg->beta_slow) || !std::isfinite(cfg->beta_fast) ||
            cfg->theta <= 1.0)
            return bad(who, "YaRN needs orig_ctx, beta_fast > beta_slow > 0 and theta > 1");
        // the pair that makes `turns` turns in orig_ctx positions
        auto pair_of = [&](double turns) {
            return rot_dim * std::log(cfg->orig_ctx / (turns * 2.0 * 3.14159265358979323846)) / (2.0 * std::log(cfg->theta));
        };
        low = std::max(std::floor(pair_of(cfg->beta_fast)), 0.0);
        high = std::min(std::ceil(pair_of(cfg->beta_slow)), rot_dim - 1.0);
        if (std::fabs(low - high) < 1.1920929e-07) high += 0.001;
    }
    jq::RopeFrequencies f{};
    f.scale = cfg->mscale == 0.0f ? 1.0 : cfg->mscale;
    for (uint32_t i = 0; i < half; ++i) {
        double v = std::pow(cfg->theta, -2.0 * i / rot_dim);
        if (freq_factors) {
            if (!(freq_factors[i] > 0.0f) || !std::isfinite(freq_factors[i])) return bad(who, "frequency factors must be positive");
            v /= freq_factors[i];
        }
        if (cfg->scaling == JQ_ROPE_LINEAR) v /= cfg->factor;
        if (cfg->scaling == JQ_ROPE_YARN) {
            const double r = 1.0 - std::min(std::max((i - low) / (high - low), 0.0), 1.0);
            v = v * (1.0 - r) / cfg->factor + v * r;
        }
        f.f[i] = v;
    }
    if (n_pos == 0) return jq::OK;
    JQ_CUDA(jq::launch_rope_table(f, rot_dim, n_pos, table_dev, static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

int32_t jq_rope_dev(const jq_rope* rope, const float* x, uint64_t x_stride, const int32_t* pos, uint32_t rows, uint32_t heads,
                    uint32_t head_dim, int32_t inverse, float* out, uint64_t out_stride, int32_t* bad_pos_dev, void* stream) {
    constexpr const char* who = "jq_rope_dev";
    jq::RopeArgs r;
    if (!rope) return bad(who, "NULL rope");
    if (head_dim == 0 || head_dim % 4 || head_dim > 1024) return bad(who, "head_dim must be a multiple of 4, at most 1024");
    if (int32_t rc = check_rope(who, rope, head_dim, &r)) return rc;
    if (rows == 0 || heads == 0) return jq::OK;
    if (!x || !pos || !out) return bad(who, "NULL buffer");
    const uint64_t width = (uint64_t)heads * head_dim;
    if (width > 0x7FFFFFFFu || x_stride < width || out_stride < width || x_stride % 4 || out_stride % 4 || unaligned(x, out))
        return bad(who, "rows of heads * head_dim floats must not overlap, on 16-byte boundaries");
    JQ_CUDA(jq::launch_rope(r, x, x_stride, pos, rows, heads, head_dim, inverse != 0, out, out_stride, bad_pos_dev,
                            static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

uint64_t jq_kv_page_bytes(uint32_t type, uint32_t n_kv, uint32_t head_dim) {
    if (type != JQ_KV_F16 && type != JQ_KV_Q8_0 && type != JQ_KV_Q4_0) return 0;
    if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || n_kv == 0 || n_kv > 1024) return 0;
    return (uint64_t)n_kv * jq::kv_head_bytes(type, head_dim);
}

int32_t jq_kv_append_dev(const jq_kv_cache* cache, const jq_rope* rope, const float* qkv, uint64_t qkv_stride, const int32_t* pos,
                         const int32_t* seq, const int32_t* page_table, uint32_t n_seq, uint32_t table_stride, uint32_t rows,
                         uint32_t n_q, const float* q_norm_w, const float* k_norm_w, float qk_eps, float* q_out,
                         int32_t* bad_pos_dev, void* stream) {
    constexpr const char* who = "jq_kv_append_dev";
    jq::KvPages c;
    jq::RopeArgs r;
    if (int32_t rc = check_cache(who, cache, page_table, n_seq, table_stride, &c)) return rc;
    if (int32_t rc = check_heads(who, cache, n_q)) return rc;
    if (int32_t rc = check_rope(who, rope, cache->head_dim, &r)) return rc;
    if (rows == 0) return jq::OK;
    if (!qkv || !pos || !q_out) return bad(who, "NULL buffer");
    if (rows > 0x7FFFFFFFu) return bad(who, "too many rows");
    if ((q_norm_w == nullptr) != (k_norm_w == nullptr)) return bad(who, "q and k norm weights go together");
    if (qkv_stride < (uint64_t)(n_q + 2 * cache->n_kv) * cache->head_dim || qkv_stride % 4 || unaligned(qkv, q_out, q_norm_w, k_norm_w))
        return bad(who, "rows of (n_q + 2 n_kv) * head_dim floats must not overlap; 16-byte boundaries");
    JQ_CUDA(jq::launch_kv_append(c, r, qkv, qkv_stride, pos, seq, rows, n_q, q_norm_w, k_norm_w, qk_eps, q_out, bad_pos_dev,
                                 static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

int32_t jq_kv_read_dev(const jq_kv_cache* cache, const int32_t* pos, const int32_t* seq, const int32_t* page_table, uint32_t n_seq,
                       uint32_t table_stride, uint32_t rows, float* k_out, float* v_out, uint64_t row_stride, uint64_t head_stride,
                       int32_t* bad_pos_dev, void* stream) {
    constexpr const char* who = "jq_kv_read_dev";
    jq::KvPages c;
    if (int32_t rc = check_cache(who, cache, page_table, n_seq, table_stride, &c)) return rc;
    if (rows == 0) return jq::OK;
    if (!pos || !k_out || !v_out) return bad(who, "NULL buffer");
    if (rows > 0x7FFFFFFFu) return bad(who, "too many rows");
    if (row_stride < cache->head_dim || head_stride < cache->head_dim || row_stride % 4 || head_stride % 4 || unaligned(k_out, v_out))
        return bad(who, "strides must be multiples of 4 floats and at least head_dim; 16-byte boundaries");
    JQ_CUDA(jq::launch_kv_read(c, pos, seq, rows, k_out, v_out, row_stride, head_stride, bad_pos_dev, static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

uint64_t jq_attention_paged_scratch_bytes(uint32_t batch, uint32_t n_q, uint32_t n_kv, uint32_t head_dim, uint32_t shared_pages) {
    if (batch == 0 || batch > JQ_ATTENTION_MAX_BATCH || n_kv == 0 || n_q == 0 || n_q % n_kv) return 0;
    return jq::attention_paged_scratch_bytes(batch, n_q, n_kv, head_dim, shared_pages);
}

int32_t jq_attention_paged_dev(const jq_kv_cache* cache, const float* q, uint64_t q_stride, const int32_t* len,
                               const int32_t* page_table, uint32_t batch, uint32_t table_stride, uint32_t n_q, float scale,
                               uint32_t shared_pages, float* out, uint64_t out_stride, void* scratch, int32_t* bad_pos_dev,
                               void* stream) {
    constexpr const char* who = "jq_attention_paged_dev";
    if (batch == 0) return jq::OK;
    jq::KvPages c;
    if (int32_t rc = check_cache(who, cache, page_table, batch, table_stride, &c)) return rc;
    if (int32_t rc = check_heads(who, cache, n_q)) return rc;
    if (!q || !len || !out || !scratch) return bad(who, "NULL buffer");
    static_assert(JQ_ATTENTION_MAX_BATCH == jq::ATTENTION_MAX_BATCH && JQ_ATTENTION_SCRATCH_ZEROED == 4 * jq::ATTENTION_MOST_CTAS, "header");
    if (batch > JQ_ATTENTION_MAX_BATCH) return jq_fail(jq::E_TOO_LARGE, "jq_attention_paged_dev: more than JQ_ATTENTION_MAX_BATCH sequences");
    if ((uint64_t)batch * table_stride > 1u << 28) return bad(who, "a page table of more than 2^28 entries");
    if (shared_pages > table_stride) return bad(who, "more shared pages than a page table row has entries");
    if (!std::isfinite(scale)) return bad(who, "the scale must be finite");
    const uint64_t width = (uint64_t)n_q * cache->head_dim;
    if (q_stride < width || out_stride < width || q_stride % 4 || out_stride % 4 || unaligned(q, out, scratch))
        return bad(who, "rows of n_q * head_dim floats must not overlap; 16-byte boundaries");
    if (scale == 0.0f) scale = 1.0f / std::sqrt((float)cache->head_dim);
    JQ_CUDA(jq::launch_attention_paged(c, q, q_stride, len, n_q, scale, shared_pages, out, out_stride, scratch, bad_pos_dev,
                                       jq_entry_status_flag(), static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

uint64_t jq_attention_chunk_scratch_bytes(uint32_t batch, uint32_t rows, uint32_t n_q, uint32_t n_kv, uint32_t head_dim) {
    if (batch == 0 || batch > JQ_ATTENTION_MAX_BATCH || rows == 0 || rows > JQ_ATTENTION_MAX_ROWS || n_kv == 0 || n_q == 0 || n_q % n_kv)
        return 0;
    return jq::attention_chunk_scratch_bytes(rows, n_q, n_kv, head_dim);
}

int32_t jq_attention_chunk_dev(const jq_kv_cache* cache, const float* q, uint64_t q_stride, const int32_t* first, const int32_t* len,
                               const int32_t* page_table, uint32_t batch, uint32_t table_stride, uint32_t rows, uint32_t n_q, float scale,
                               uint32_t window, uint32_t sinks, float* out, uint64_t out_stride, void* scratch, int32_t* bad_pos_dev,
                               void* stream) {
    constexpr const char* who = "jq_attention_chunk_dev";
    if (batch == 0 || rows == 0) return jq::OK;
    jq::KvPages c;
    if (int32_t rc = check_cache(who, cache, page_table, batch, table_stride, &c)) return rc;
    if (int32_t rc = check_heads(who, cache, n_q)) return rc;
    if (!q || !len || !out || !scratch) return bad(who, "NULL buffer");
    static_assert(JQ_ATTENTION_MAX_ROWS == jq::ATTENTION_MAX_ROWS, "header");
    if (batch > JQ_ATTENTION_MAX_BATCH) return jq_fail(jq::E_TOO_LARGE, "jq_attention_chunk_dev: more than JQ_ATTENTION_MAX_BATCH sequences");
    if (rows > JQ_ATTENTION_MAX_ROWS) return jq_fail(jq::E_TOO_LARGE, "jq_attention_chunk_dev: more than JQ_ATTENTION_MAX_ROWS rows");
    if (!first && rows % batch) return bad(who, "rows that do not divide into equal parts need `first`");
    if ((uint64_t)batch * table_stride > 1u << 28) return bad(who, "a page table of more than 2^28 entries");
    if (!jq::span_rows_fit(rows, table_stride, n_q))
        return jq_fail(jq::E_TOO_LARGE, "jq_attention_chunk_dev: rows times positions, or rows times heads, are too many");
    if (!std::isfinite(scale)) return bad(who, "the scale must be finite");
    const uint64_t width = (uint64_t)n_q * cache->head_dim;
    if (q_stride < width || out_stride < width || q_stride % 4 || out_stride % 4 || unaligned(q, out, scratch))
        return bad(who, "rows of n_q * head_dim floats must not overlap; 16-byte boundaries");
    if (rows_meet(q, q_stride, out, out_stride, rows, width)) return bad(who, "q and out must not overlap");
    if (scale == 0.0f) scale = 1.0f / std::sqrt((float)cache->head_dim);
    const uint32_t most = table_stride * JQ_KV_PAGE;
    if (window >= most) window = 0;
    JQ_CUDA(jq::launch_attention_chunk(c, q, q_stride, first, len, rows, n_q, scale, window, window ? std::min(sinks, most) : 0, out,
                                       out_stride, scratch, bad_pos_dev, jq_entry_status_flag(), static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

int32_t jq_sample_dev(const float* logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float* uniform,
                      const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                      float repetition_penalty, int32_t* window, int32_t* window_state, int32_t* token, float* prob, int32_t* pos,
                      void* stream) {
    constexpr const char* who = "jq_sample_dev";
    static_assert(JQ_SAMPLE_MAX_VOCAB == jq::SAMPLE_MAX_VOCAB && JQ_SAMPLE_WINDOW == 64, "header");
    if (rows == 0) return jq::OK;
    if (!logits || !uniform || !token || vocab == 0 || row_stride < vocab || rows > 65535) return bad(who, "bad argument");
    if (vocab > JQ_SAMPLE_MAX_VOCAB) return jq_fail(jq::E_TOO_LARGE, "jq_sample_dev: vocab above JQ_SAMPLE_MAX_VOCAB");
    if ((window == nullptr) != (window_state == nullptr)) return bad(who, "window and window_state go together");
    if (!(repetition_penalty > 0.0f)) return bad(who, "the penalty must be positive");
    jq::SampleArgs a{logits, row_stride, vocab, uniform, temperature, top_k, top_p, min_p, repetition_penalty, window, window_state,
                     token, prob, pos};
    JQ_CUDA(jq::launch_sample(a, rows, static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

int32_t jq_log_probs_dev(const float* logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const int32_t* token, uint32_t top,
                         float* log_prob, float* entropy, int32_t* top_token, float* top_log_prob, void* stream) {
    constexpr const char* who = "jq_log_probs_dev";
    static_assert(JQ_LOG_PROBS_MOST == jq::LOG_PROBS_MOST, "header");
    if (rows == 0) return jq::OK;
    if (!logits || !token || !log_prob) return bad(who, "NULL buffer");
    if (vocab == 0 || vocab > 0x7FFFFFFFu || row_stride < vocab) return bad(who, "rows of 1 to 2^31 - 1 logits must not overlap");
    if (rows > 1u << 24) return jq_fail(jq::E_TOO_LARGE, "jq_log_probs_dev: more than 2^24 rows");
    if (top > JQ_LOG_PROBS_MOST) return jq_fail(jq::E_TOO_LARGE, "jq_log_probs_dev: more than JQ_LOG_PROBS_MOST tokens of a row");
    if (top && (!top_token || !top_log_prob)) return bad(who, "NULL buffer of the likeliest tokens");
    jq::LogProbArgs a{logits, row_stride, vocab, token, top, log_prob, entropy, top_token, top_log_prob};
    JQ_CUDA(jq::launch_log_probs(a, rows, static_cast<cudaStream_t>(stream)));
    return jq::OK;
}

}  // extern "C"
