// Attention of one new token per sequence over the pages of the quantised cache.
//
// out[b, head, :] = sum_t p_t V_t / sum_t p_t with p_t = exp(scale q . K_t - max), t = 0 .. len[b] - 1.  Pages are independent:
// one CTA a page and query head gives the page's sum with its own maximum, a second kernel joins them in order.
#include "kv_pages.cuh"

namespace jq {

namespace {

// part[b, head, page]: HD sums, the maximum, the sum of exponentials
template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(128) attention_page_kernel(KvPages c, const float* __restrict__ q, uint64_t q_stride,
                                                             const int32_t* __restrict__ len, uint32_t n_q, float scale,
                                                             uint32_t shared, float* __restrict__ part) {
    constexpr uint32_t HEAD = kv_head_bytes(KIND, HD);
    __shared__ float s_q[HD], s_p[KV_PAGE], s_red[4];
    pdl_trigger_all();
    const uint32_t page = blockIdx.x, head = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t n = len[b];
    if (n <= 0 || (uint32_t)n > c.table_stride * (uint64_t)KV_PAGE || page * KV_PAGE >= (uint32_t)n) return;
    float* dst = part + (((uint64_t)b * n_q + head) * c.table_stride + page) * (HD + 2);
    const uint32_t cnt = min(KV_PAGE, (uint32_t)n - page * KV_PAGE);
    const int32_t id = c.table[(uint64_t)(page < shared ? 0 : b) * c.table_stride + page];
    if (id < 0 || (uint32_t)id >= c.n_pages) {
        for (uint32_t i = threadIdx.x; i < HD + 2; i += 128) dst[i] = NAN;
        return;
    }
    const uint8_t* tile = c.pages + ((uint64_t)id * c.n_kv + head / (n_q / c.n_kv)) * HEAD;
    for (uint32_t i = threadIdx.x; i < HD; i += 128) s_q[i] = q[b * q_stride + head * HD + i];
    __syncthreads();
    float mx = -INFINITY;
    for (uint32_t t = warp; t < cnt; t += 4) {
        float acc = 0.0f;
        for (uint32_t d = 4 * lane; d < HD; d += 128) {
            const float4 k = kv_load<KIND, HD, false>(tile, t, d);
            acc = fmaf(s_q[d], k.x, fmaf(s_q[d + 1], k.y, fmaf(s_q[d + 2], k.z, fmaf(s_q[d + 3], k.w, acc))));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xFFFFFFFFu, acc, o);
        if (lane == 0) s_p[t] = acc * scale;
        mx = fmaxf(mx, acc * scale);
    }
    if (lane == 0) s_red[warp] = mx;
    __syncthreads();
    mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    for (uint32_t t = threadIdx.x; t < cnt; t += 128) s_p[t] = expf(s_p[t] - mx);
    __syncthreads();
    float sum = 0.0f;
    for (uint32_t t = 0; t < cnt; ++t) sum += s_p[t];
    for (uint32_t d = 4 * threadIdx.x; d < HD; d += 512) {
        float4 o = make_float4(0, 0, 0, 0);
        for (uint32_t t = 0; t < cnt; ++t) {
            const float4 v = kv_load<KIND, HD, true>(tile + HEAD / 2, t, d);
            const float p = s_p[t];
            o.x = fmaf(p, v.x, o.x), o.y = fmaf(p, v.y, o.y), o.z = fmaf(p, v.z, o.z), o.w = fmaf(p, v.w, o.w);
        }
        dst[d] = o.x, dst[d + 1] = o.y, dst[d + 2] = o.z, dst[d + 3] = o.w;
    }
    if (threadIdx.x == 0) dst[HD] = mx, dst[HD + 1] = sum;
}

__global__ void __launch_bounds__(128) attention_page_merge_kernel(const float* __restrict__ part, const int32_t* __restrict__ len,
                                                                   uint32_t n_q, uint32_t hd, uint32_t stride, uint32_t shared,
                                                                   float* __restrict__ out, uint64_t out_stride,
                                                                   int32_t* __restrict__ bad_pos) {
    pdl_trigger_all();
    const uint32_t head = blockIdx.x, b = blockIdx.y;
    const int32_t n = len[b];
    float* dst = out + b * out_stride + (uint64_t)head * hd;
    const bool bad = n < 0 || (uint32_t)n > stride * (uint64_t)KV_PAGE || (n > 0 && (uint32_t)n < shared * KV_PAGE);
    const uint32_t pages = bad ? 0 : ((uint32_t)n + KV_PAGE - 1) / KV_PAGE;
    if (bad && head == 0 && threadIdx.x == 0 && bad_pos) atomicExch(bad_pos, 1);
    const float* src = part + ((uint64_t)b * n_q + head) * stride * (hd + 2);
    float mx = -INFINITY, den = 0.0f;
    bool lost = bad;
    for (uint32_t i = 0; i < pages; ++i) {
        const float m = src[(uint64_t)i * (hd + 2) + hd];
        lost |= m != m;
        mx = fmaxf(mx, m);
    }
    if (lost && !bad && head == 0 && threadIdx.x == 0 && bad_pos) atomicExch(bad_pos, 1);
    for (uint32_t i = 0; i < pages; ++i) den += expf(src[(uint64_t)i * (hd + 2) + hd] - mx) * src[(uint64_t)i * (hd + 2) + hd + 1];
    for (uint32_t d = threadIdx.x; d < hd; d += 128) {
        float acc = 0.0f;
        for (uint32_t i = 0; i < pages; ++i) acc = fmaf(expf(src[(uint64_t)i * (hd + 2) + hd] - mx), src[(uint64_t)i * (hd + 2) + d], acc);
        dst[d] = lost ? NAN : pages ? acc / den : 0.0f;
    }
}

struct LaunchPages {
    const KvPages& c;
    const float* q;
    uint64_t q_stride;
    const int32_t* len;
    uint32_t n_q;
    float scale;
    uint32_t shared;
    float* part;
    cudaStream_t s;
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        return launch_pdl(attention_page_kernel<KIND, HD>, dim3(c.table_stride, n_q, c.n_seq), 128, 0, s, c, q, q_stride, len, n_q, scale,
                          shared, part);
    }
};

}  // namespace

size_t attention_paged_scratch_bytes(uint32_t batch, uint32_t n_q, uint32_t n_kv, uint32_t hd, uint32_t table_stride, uint32_t shared) {
    return (size_t)batch * n_q * table_stride * (hd + 2) * 4;
}

cudaError_t launch_attention_paged(const KvPages& c, const float* q, uint64_t q_stride, const int32_t* len, uint32_t n_q, float scale,
                                   uint32_t shared, float* out, uint64_t out_stride, void* scratch, int32_t* bad_pos, cudaStream_t s) {
    float* part = static_cast<float*>(scratch);
    cudaError_t e = for_kind(c.kind, c.hd, LaunchPages{c, q, q_stride, len, n_q, scale, shared, part, s});
    if (e != cudaSuccess) return e;
    e = launch_pdl(attention_page_merge_kernel, dim3(n_q, c.n_seq), 128, 0, s, part, len, n_q, c.hd, c.table_stride, shared, out, out_stride,
                   bad_pos);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
