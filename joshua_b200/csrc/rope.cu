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

// A thread takes the four dimensions 4 i .. 4 i + 3 of a head of a row, and reads those of their partners.
__global__ void __launch_bounds__(256) rope_kernel(RopeArgs r, const float* __restrict__ x, uint64_t x_stride, const int32_t* __restrict__ pos,
                                                   uint32_t rows, uint32_t heads, uint32_t hd, float sign, float* __restrict__ out,
                                                   uint64_t out_stride, int32_t* __restrict__ bad_pos) {
    pdl_trigger_all();
    const uint32_t per_row = heads * (hd / 2);
    const uint64_t n = (uint64_t)rows * per_row;
    for (uint64_t t = blockIdx.x * 256ull + threadIdx.x; t < n; t += gridDim.x * 256ull) {
        const uint32_t row = (uint32_t)(t / per_row), in_row = (uint32_t)(t % per_row), head = in_row / (hd / 2), i = in_row % (hd / 2);
        const int32_t p = pos[row];
        if (p < 0 || (uint32_t)p >= r.n_pos) {
            if (in_row == 0 && bad_pos) atomicExch(bad_pos, 1);
            continue;
        }
        // pairs first, then the dimensions behind the rotated ones two by two
        const uint32_t half = r.rot / 2, a = i >= half ? 2 * i : r.interleaved ? 2 * i : i, b = i >= half || r.interleaved ? a + 1 : a + half;
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
    const uint64_t n = (uint64_t)rows * heads * (hd / 2);
    cudaError_t e = launch_pdl(rope_kernel, (unsigned)std::min<uint64_t>((n + 255) / 256, 148 * 16), 256, 0, s, r, x, x_stride, pos, rows,
                               heads, hd, inverse ? -1.0f : 1.0f, out, out_stride, bad_pos);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
