// Rotary positions: the table of cosines and sines, and the rotation of the heads of some rows.
#include "rope.cuh"
#include "serving.cuh"

namespace jq {

namespace {

// table[p][i] = m (cos, sin)(p f_i) in 64 bits, rounded once: a position of 100000 times a frequency of 1 has lost ten bits of
// its angle in 32.
__global__ void __launch_bounds__(256) rope_table_kernel(RopeFrequencies f, uint32_t half, uint32_t n_pos, float2* __restrict__ table) {
    pdl_trigger_all();
    const uint64_t n = (uint64_t)n_pos * half;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < n; i += gridDim.x * 256ull) {
        double s, c;
        sincos((double)(i / half) * f.f[i % half], &s, &c);
        table[i] = make_float2((float)(c * f.scale), (float)(s * f.scale));
    }
}

// Eight dimensions a thread and head: four pairs and their table entries, read once for all heads that the thread takes (the
// row's heads are spread over the threads of a CTA and over blockIdx.y).  Bound by memory: 2048 rows of 40 heads of 128 read and
// written in 15.7 us (5.3 TB/s; 9.7 where they are still in L2), one row of 40 heads 1.7.
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs r, const float* x, uint64_t x_stride, const int32_t* pos, uint32_t heads,
                                                   uint32_t hd, float sign, float* out, uint64_t out_stride, int32_t* bad_pos) {
    pdl_trigger_all();
    const uint32_t row = blockIdx.x, per_head = hd / 8, j = threadIdx.x % per_head;
    const uint32_t step = blockDim.x / per_head * gridDim.y, h0 = blockIdx.y * (blockDim.x / per_head) + threadIdx.x / per_head;
    const int32_t p = pos[row];
    if (p < 0 || (uint32_t)p >= r.n_pos) {
        if (threadIdx.x == 0 && blockIdx.y == 0 && bad_pos) atomicExch(bad_pos, 1);
        return;
    }
    const bool turns = 8 * j < r.rot;
    // the two runs of four dimensions: a run and its partners, or neighbours
    const uint32_t a = turns && !r.interleaved ? 4 * j : 8 * j, b = turns && !r.interleaved ? a + r.rot / 2 : a + 4;
    float2 cs[4];
    if (turns) {
        const float4* t = reinterpret_cast<const float4*>(r.table + (uint64_t)p * (r.rot / 2) + 4 * j);
        const float4 u = __ldg(t), v = __ldg(t + 1);
        cs[0] = make_float2(u.x, u.y * sign), cs[1] = make_float2(u.z, u.w * sign);
        cs[2] = make_float2(v.x, v.y * sign), cs[3] = make_float2(v.z, v.w * sign);
    }
    const float* src = x + row * x_stride;
    float* dst = out + row * out_stride;
    for (uint32_t h = h0; h < heads; h += step) {  // out may be x: a thread stores what it alone has loaded
        float4 u = *reinterpret_cast<const float4*>(src + h * hd + a), v = *reinterpret_cast<const float4*>(src + h * hd + b);
        if (turns) {
            float* first[4] = {&u.x, &u.y, &u.z, &u.w};
            float* second[4] = {&v.x, &v.y, &v.z, &v.w};
            if (r.interleaved) first[1] = &u.z, first[2] = &v.x, first[3] = &v.z, second[0] = &u.y, second[1] = &u.w, second[2] = &v.y;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float va = *first[i], vb = *second[i];
                *first[i] = rope_rotate(true, va, vb, cs[i]), *second[i] = rope_rotate(false, vb, va, cs[i]);
            }
        }
        *reinterpret_cast<float4*>(dst + h * hd + a) = u, *reinterpret_cast<float4*>(dst + h * hd + b) = v;
    }
}

// The same for heads or rotated parts that are no multiple of 8, two dimensions a thread.
__global__ void __launch_bounds__(256) rope_pairs_kernel(RopeArgs r, const float* x, uint64_t x_stride, const int32_t* pos, uint32_t heads,
                                                         uint32_t hd, float sign, float* out, uint64_t out_stride, int32_t* bad_pos) {
    pdl_trigger_all();
    const uint32_t row = blockIdx.x, half = r.rot / 2;
    const int32_t p = pos[row];
    if (p < 0 || (uint32_t)p >= r.n_pos) {
        if (threadIdx.x == 0 && bad_pos) atomicExch(bad_pos, 1);
        return;
    }
    for (uint32_t t = threadIdx.x; t < heads * (hd / 2); t += blockDim.x) {
        const uint32_t head = t / (hd / 2), i = t % (hd / 2);
        // pairs first, then the dimensions behind the rotated ones two by two
        const uint32_t a = i >= half || r.interleaved ? 2 * i : i, b = i >= half || r.interleaved ? a + 1 : a + half;
        const float* src = x + row * x_stride + head * hd;
        float* dst = out + row * out_stride + head * hd;
        float va = src[a], vb = src[b];
        if (i < half) {
            float2 cs = r.table[(uint64_t)p * half + i];
            cs.y *= sign;
            const float ra = rope_rotate(true, va, vb, cs), rb = rope_rotate(false, vb, va, cs);
            va = ra, vb = rb;
        }
        dst[a] = va, dst[b] = vb;
    }
}

}  // namespace

cudaError_t launch_rope_table(const RopeFrequencies& f, uint32_t rot, uint32_t n_pos, float* table, cudaStream_t s) {
    const uint64_t n = (uint64_t)n_pos * (rot / 2);
    cudaError_t e = launch_pdl(rope_table_kernel, (unsigned)std::min<uint64_t>((n + 255) / 256, 148 * 8), 256, 0, s, f, rot / 2, n_pos,
                               reinterpret_cast<float2*>(table));
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_rope(const RopeArgs& r, const float* x, uint64_t x_stride, const int32_t* pos, uint32_t rows, uint32_t heads,
                        uint32_t hd, bool inverse, float* out, uint64_t out_stride, int32_t* bad_pos, cudaStream_t s) {
    const float sign = inverse ? -1.0f : 1.0f;
    cudaError_t e;
    if (hd % 8 == 0 && r.vectors) {
        // four heads a thread, fewer where the rows alone do not fill the GPU (40 heads of 128, from L2: one row 2.3 us with four
        // heads a thread, 1.7 with one; 2048 rows 9.7 and 10.8)
        const uint32_t at_once = std::max(1u, 256 / (hd / 8)), threads = at_once * (hd / 8);
        const uint32_t most = (heads + at_once - 1) / at_once, few = (most + 3) / 4;
        const uint32_t parts = std::min(most, std::max(few, (uint32_t)(8 * num_sms()) / rows));
        e = launch_pdl(rope_kernel, dim3(rows, parts), threads, 0, s, r, x, x_stride, pos, heads, hd, sign, out, out_stride, bad_pos);
    } else {
        e = launch_pdl(rope_pairs_kernel, dim3(rows), 256, 0, s, r, x, x_stride, pos, heads, hd, sign, out, out_stride, bad_pos);
    }
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
