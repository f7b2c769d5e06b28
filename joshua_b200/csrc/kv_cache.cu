// The paged cache: new positions' keys and values rounded into their pages, keys and queries rotated on the way; positions
// read back as f32 rows.
#include "kv_pages.cuh"
#include "serving.cuh"

namespace jq {

namespace {

// One row of qkv [(n_q + 2 n_kv), HD] per blockIdx.x, a group of min(32, HD / 4) lanes a head, 4 (HD 256: 8) dimensions a lane.
template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(256) kv_append_kernel(KvPages c, RopeArgs r, const float* __restrict__ qkv, uint64_t stride,
                                                        const int32_t* __restrict__ pos, const int32_t* __restrict__ seq, uint32_t n_q,
                                                        const float* __restrict__ q_norm, const float* __restrict__ k_norm, float eps,
                                                        float* __restrict__ q_out, int32_t* __restrict__ bad_pos) {
    constexpr uint32_t LANES = HD / 4 < 32 ? HD / 4 : 32, QUADS = HD / 4 / LANES, HPW = 32 / LANES;
    constexpr uint32_t CODES = kv_code_bytes(KIND, HD), SCALES = kv_scale_bytes(KIND, HD), HEAD = kv_head_bytes(KIND, HD);
    __shared__ __align__(16) float s_head[8 * HPW][HD];
    pdl_trigger_all();
    const uint32_t row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / LANES, li = lane % LANES;
    const uint32_t heads = n_q + 2 * c.n_kv, head = (blockIdx.y * 8 + warp) * HPW + group;
    const bool live = head < heads;
    const int32_t p = pos[row];
    uint8_t* page = page_of(c, seq ? seq[row] : (int32_t)row, p, HEAD);
    if (page == nullptr || (r.table != nullptr && (uint32_t)p >= r.n_pos)) {  // the same in the whole row
        if (blockIdx.y == 0 && threadIdx.x == 0 && bad_pos) atomicExch(bad_pos, 1);
        return;
    }
    float x[QUADS][4];
    const float* src = qkv + row * stride + (uint64_t)head * HD;
#pragma unroll
    for (uint32_t i = 0; i < QUADS; ++i) {
        const float4 v = live ? *reinterpret_cast<const float4*>(src + 4 * (i * LANES + li)) : make_float4(0, 0, 0, 0);
        x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
    }
    const bool is_v = head >= n_q + c.n_kv, is_q = head < n_q;
    const float* nw = is_q ? q_norm : k_norm;
    if (nw != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(x[i][e], x[i][e], ss);
#pragma unroll
        for (uint32_t o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        const float sc = rsqrtf(ss / (float)HD + eps);
        if (!is_v) {
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][e] = x[i][e] * sc * nw[4 * (i * LANES + li) + e];
        }
    }
    if (r.table != nullptr) {  // values pass through shared memory too, and stay as they are
        float* mine = s_head[warp * HPW + group];
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i)
            *reinterpret_cast<float4*>(mine + 4 * (i * LANES + li)) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
        __syncwarp();
        if (!is_v) {
#pragma unroll
            for (uint32_t i = 0; i < QUADS; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t d = 4 * (i * LANES + li) + e;
                    if (d < r.rot)
                        x[i][e] = rope_rotate(rope_first(r, d), x[i][e], mine[rope_partner(r, d)],
                                              r.table[(uint64_t)p * (r.rot / 2) + rope_pair(r, d)]);
                }
        }
    }
    const uint32_t kvh = is_v ? head - n_q - c.n_kv : head - n_q, in_page = (uint32_t)p % KV_PAGE;
    uint8_t* part = page + (uint64_t)kvh * HEAD + (is_v ? CODES + SCALES : 0);
#pragma unroll
    for (uint32_t i = 0; i < QUADS; ++i) {
        const uint32_t d = 4 * (i * LANES + li);
        const KvQuad q = kv_round<KIND>(x[i]);
        if (!live) continue;
        if (is_q) {
            *reinterpret_cast<float4*>(q_out + ((uint64_t)row * n_q + head) * HD + d) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
            continue;
        }
        if (is_v) {
            uint8_t* at = part + kv_value_at<KIND, HD>(in_page, d);
            if constexpr (KIND == KV_F16) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) *reinterpret_cast<uint16_t*>(at + (e >> 1) * 512 + (e & 1) * 4) = (uint16_t)q.code[e];
            } else if constexpr (KIND == KV_Q8_0) {
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) at[(e >> 1) * 8 + (e & 1) * 2] = (uint8_t)q.code[e];
            } else {
                at[0] = (uint8_t)(q.code[0] | q.code[1] << 4), at[4] = (uint8_t)(q.code[2] | q.code[3] << 4);
            }
        } else {
            uint8_t* at = part + kv_key_at<KIND, HD>(in_page, d);
            if constexpr (KIND == KV_F16)
                *reinterpret_cast<uint2*>(at) = make_uint2(q.code[0] | q.code[1] << 16, q.code[2] | q.code[3] << 16);
            else if constexpr (KIND == KV_Q8_0)
                *reinterpret_cast<uint32_t*>(at) = q.code[0] | q.code[1] << 8 | q.code[2] << 16 | q.code[3] << 24;
            else
                at[0] = (uint8_t)(q.code[0] | q.code[2] << 4), at[2] = (uint8_t)(q.code[1] | q.code[3] << 4);
        }
        if (KIND != KV_F16 && li % 8 == 0)
            *reinterpret_cast<uint16_t*>(part + CODES + kv_scale_at<HD>(in_page, d / 32)) = q.scale;
    }
}

// A warp a row and kv head, keys and values.
template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(256) kv_read_kernel(KvPages c, const int32_t* __restrict__ pos, const int32_t* __restrict__ seq,
                                                      float* __restrict__ k, float* __restrict__ v, uint64_t row_stride,
                                                      uint64_t head_stride, int32_t* __restrict__ bad_pos) {
    constexpr uint32_t HEAD = kv_head_bytes(KIND, HD);
    pdl_trigger_all();
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 31, head = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (head >= c.n_kv) return;
    const int32_t p = pos[row];
    const uint8_t* page = page_of(c, seq ? seq[row] : (int32_t)row, p, HEAD);
    if (page == nullptr && head == 0 && lane == 0 && bad_pos) atomicExch(bad_pos, 1);
    const uint8_t* part = page + (uint64_t)head * HEAD;
    const uint64_t to = row * row_stride + head * head_stride;
    for (uint32_t d = 4 * lane; d < HD; d += 128) {
        const float4 bad = make_float4(NAN, NAN, NAN, NAN);
        *reinterpret_cast<float4*>(k + to + d) = page ? kv_load<KIND, HD, false>(part, (uint32_t)p % KV_PAGE, d) : bad;
        *reinterpret_cast<float4*>(v + to + d) = page ? kv_load<KIND, HD, true>(part + HEAD / 2, (uint32_t)p % KV_PAGE, d) : bad;
    }
}

struct LaunchAppend {
    const KvPages& c;
    const RopeArgs& r;
    const float* qkv;
    uint64_t stride;
    const int32_t *pos, *seq;
    uint32_t rows, n_q;
    const float *q_norm, *k_norm;
    float eps;
    float* q_out;
    int32_t* bad_pos;
    cudaStream_t s;
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        const uint32_t per_cta = 8 * (HD < 128 ? 2 : 1), heads = n_q + 2 * c.n_kv;
        return launch_pdl(kv_append_kernel<KIND, HD>, dim3(rows, (heads + per_cta - 1) / per_cta), 256, 0, s, c, r, qkv, stride, pos,
                          seq, n_q, q_norm, k_norm, eps, q_out, bad_pos);
    }
};
struct LaunchRead {
    const KvPages& c;
    const int32_t *pos, *seq;
    uint32_t rows;
    float *k, *v;
    uint64_t row_stride, head_stride;
    int32_t* bad_pos;
    cudaStream_t s;
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        return launch_pdl(kv_read_kernel<KIND, HD>, dim3(rows, (c.n_kv + 7) / 8), 256, 0, s, c, pos, seq, k, v, row_stride, head_stride,
                          bad_pos);
    }
};

}  // namespace

cudaError_t launch_kv_append(const KvPages& c, const RopeArgs& r, const float* qkv, uint64_t stride, const int32_t* pos,
                             const int32_t* seq, uint32_t rows, uint32_t n_q, const float* q_norm, const float* k_norm, float eps,
                             float* q_out, int32_t* bad_pos, cudaStream_t s) {
    cudaError_t e = for_kind(c.kind, c.hd, LaunchAppend{c, r, qkv, stride, pos, seq, rows, n_q, q_norm, k_norm, eps, q_out, bad_pos, s});
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_kv_read(const KvPages& c, const int32_t* pos, const int32_t* seq, uint32_t rows, float* k, float* v,
                           uint64_t row_stride, uint64_t head_stride, int32_t* bad_pos, cudaStream_t s) {
    cudaError_t e = for_kind(c.kind, c.hd, LaunchRead{c, pos, seq, rows, k, v, row_stride, head_stride, bad_pos, s});
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
