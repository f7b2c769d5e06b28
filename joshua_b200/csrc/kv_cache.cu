// The paged cache: new positions' keys and values rounded into their pages, keys and queries rotated on the way; positions
// read back as f32 rows.
//
// A block of 32 dimensions x becomes codes rint(x / d) under one scale d (kv_round), queries and keys (a cos - b sin, a sin + b
// cos) before.  Each f32 row is read once, queries written once, codes once: many rows are bound by memory (4096 rows of 32
// query heads on 8 of 64 in halves, 92 MB in 21.8 us; 1000 rows of 32 on 4 of 128 in four bits, 12.0), few by the chain from a row's
// position to its page (32 rows 3.2 us, launch included).
#include "kv_pages.cuh"
#include "serving.cuh"

namespace jq {

namespace {

// A group of min(32, HD / 4) lanes has a head of a row, 4 (HD 256: 8) dimensions a lane.
template <uint32_t HD>
struct HeadLanes {
    static constexpr uint32_t LANES = HD / 4 < 32 ? HD / 4 : 32, QUADS = HD / 4 / LANES, PER_WARP = 32 / LANES;
    float x[QUADS][4];

    __device__ __forceinline__ static uint32_t dim(uint32_t i) { return 4 * (i * LANES + threadIdx.x % LANES); }
    __device__ __forceinline__ void load(const float* src, bool live) {
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i) {
            const float4 v = live ? *reinterpret_cast<const float4*>(src + dim(i)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
        }
    }
    __device__ __forceinline__ void store(float* dst) const {
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i) *reinterpret_cast<float4*>(dst + dim(i)) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
    }
    __device__ __forceinline__ void norm(const float* w, float eps) {
        float ss = 0.0f;
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(x[i][e], x[i][e], ss);
#pragma unroll
        for (uint32_t o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        const float sc = rsqrtf(ss / (float)HD + eps);
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i][e] = x[i][e] * sc * w[dim(i) + e];
    }
    // to position p; `mine`: HD floats of shared memory of these lanes
    __device__ __forceinline__ void turn(const RopeArgs& r, uint32_t p, float* mine) {
        const uint32_t half = r.rot / 2;
        const float2* t = r.table + (uint64_t)p * half;
        if (!r.interleaved) {
            __syncwarp();
            store(mine);
            __syncwarp();
        }
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i) {
            const uint32_t d = dim(i);
            if (d >= r.rot) continue;
            float (&v)[4] = x[i];
            if (r.vectors) {  // rot a multiple of 8: four dimensions turn together, their table entries are whole vectors
                if (r.interleaved) {
                    const float4 cs = __ldg(reinterpret_cast<const float4*>(t + d / 2));
                    const float y[4] = {v[0], v[1], v[2], v[3]};
                    v[0] = rope_rotate(true, y[0], y[1], make_float2(cs.x, cs.y)), v[1] = rope_rotate(false, y[1], y[0], make_float2(cs.x, cs.y));
                    v[2] = rope_rotate(true, y[2], y[3], make_float2(cs.z, cs.w)), v[3] = rope_rotate(false, y[3], y[2], make_float2(cs.z, cs.w));
                } else {
                    const bool first = d < half;
                    const float4* cs = reinterpret_cast<const float4*>(t + (first ? d : d - half));
                    const float4 c0 = __ldg(cs), c1 = __ldg(cs + 1), y = *reinterpret_cast<const float4*>(mine + (first ? d + half : d - half));
                    // the second of a pair: a sin + b cos = b cos - a (-sin), rounded alike
                    const float s = first ? 1.0f : -1.0f;
                    v[0] = rope_rotate(true, v[0], y.x, make_float2(c0.x, c0.y * s)), v[1] = rope_rotate(true, v[1], y.y, make_float2(c0.z, c0.w * s));
                    v[2] = rope_rotate(true, v[2], y.z, make_float2(c1.x, c1.y * s)), v[3] = rope_rotate(true, v[3], y.w, make_float2(c1.z, c1.w * s));
                }
            } else {
                const float y[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                    const uint32_t at = d + e;
                    const bool first = r.interleaved ? e % 2 == 0 : at < half;
                    if (at >= r.rot) continue;
                    const float other = r.interleaved ? y[e ^ 1] : mine[first ? at + half : at - half];
                    v[e] = rope_rotate(first, y[e], other, __ldg(t + (r.interleaved ? at / 2 : first ? at : at - half)));
                }
            }
        }
    }
    // a key's or value's codes as position `pos` of `codes`, its scales as position `in_page` of `scales`; all lanes of the warp,
    // those with `live` store
    template <uint32_t KIND>
    __device__ __forceinline__ void put(uint8_t* codes, uint32_t pos, uint8_t* scales, uint32_t in_page, bool is_v, bool live) const {
#pragma unroll
        for (uint32_t i = 0; i < QUADS; ++i) {
            const uint32_t d = dim(i);
            const KvQuad q = kv_round<KIND>(x[i]);
            if (!live) continue;
            if (is_v) {
                uint8_t* at = codes + kv_value_at<KIND, HD>(pos, d);
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
                uint8_t* at = codes + kv_key_at<KIND, HD>(pos, d);
                if constexpr (KIND == KV_F16)
                    *reinterpret_cast<uint2*>(at) = make_uint2(q.code[0] | q.code[1] << 16, q.code[2] | q.code[3] << 16);
                else if constexpr (KIND == KV_Q8_0)
                    *reinterpret_cast<uint32_t*>(at) = q.code[0] | q.code[1] << 8 | q.code[2] << 16 | q.code[3] << 24;
                else
                    at[0] = (uint8_t)(q.code[0] | q.code[2] << 4), at[2] = (uint8_t)(q.code[1] | q.code[3] << 4);
            }
            if (KIND != KV_F16 && dim(0) % 32 == 0)
                *reinterpret_cast<uint16_t*>(scales + kv_scale_at<HD>(in_page, d / 32)) = q.scale;
        }
    }
};

struct AppendArgs {
    KvPages c;
    RopeArgs r;
    const float* qkv;
    uint64_t stride;
    const int32_t *pos, *seq;
    uint32_t rows, n_q;
    const float *q_norm, *k_norm;
    float eps;
    float* q_out;
    int32_t* bad_pos;

    __device__ __forceinline__ int32_t seq_of(uint32_t row) const { return seq ? seq[row] : (int32_t)row; }
    // the page of a row's position, NULL if it has no place
    __device__ __forceinline__ uint8_t* page(uint32_t row, uint32_t head_bytes) const {
        const int32_t p = pos[row];
        uint8_t* at = page_of(c, seq_of(row), p, head_bytes);
        return r.table != nullptr && (uint32_t)p >= r.n_pos ? nullptr : at;
    }
    // a key's or value's head in a page
    __device__ __forceinline__ uint8_t* part(uint8_t* page, uint32_t head, uint32_t head_bytes) const {
        return head < c.n_kv ? page + (uint64_t)head * head_bytes : page + (uint64_t)(head - c.n_kv) * head_bytes + head_bytes / 2;
    }
};

// The 16 rows that a warp or CTA of the kernels below takes, first + j (j = 0 .. 15): rows are grouped by the first row's position.
struct RowGroup {
    int64_t first;           // row of j = 0 (may be in front of the first row)
    uint32_t first_j, rows;  // live ones: j = first_j .. first_j + rows - 1
    bool runs;               // they stand at consecutive positions of one sequence, within a group of 16 of a page,
    int32_t p0;              // from p0 on

    __device__ __forceinline__ RowGroup(const int32_t* pos, uint32_t n, uint32_t block) {
        first = (int64_t)block * 16 - (pos[0] & 15);
        first_j = first < 0 ? (uint32_t)-first : 0;
        rows = (uint32_t)(min((int64_t)n, first + 16) - first) - first_j;
        if (first + first_j >= n) rows = 0;
    }
    __device__ __forceinline__ bool has(uint32_t j) const { return j >= first_j && j < first_j + rows; }
    __device__ __forceinline__ void look(const int32_t* pos, const int32_t* seq) {  // sets runs
        const uint32_t j = threadIdx.x & 15;
        const bool live = has(j);
        const int32_t p = live ? pos[first + j] : 0, s = live ? seq ? seq[first + j] : (int32_t)(first + j) : 0;
        const int32_t s0 = __shfl_sync(0xFFFFFFFFu, s, first_j & 15);
        p0 = __shfl_sync(0xFFFFFFFFu, p, first_j & 15) - (int32_t)first_j;
        runs = p0 >= 0 && p0 % 16 == 0 && __all_sync(0xFFFFFFFFu, !live || (p == p0 + (int32_t)j && s == s0));
    }
};

// A key's or value's head of a row (keys are heads 0 .. n_kv - 1, values those behind them), its codes to `run` as one of 16
// positions if that is given.
template <uint32_t KIND, uint32_t HD>
__device__ __forceinline__ void append_head(const AppendArgs& a, HeadLanes<HD>& x, uint32_t row, uint8_t* page, uint32_t p, uint32_t head,
                                            float* mine, uint8_t* run = nullptr) {
    constexpr uint32_t CODES = kv_code_bytes(KIND, HD), HEAD = kv_head_bytes(KIND, HD);
    if (page == nullptr) {  // the same in the warp
        if (head == 0 && threadIdx.x % 32 == 0 && a.bad_pos) atomicExch(a.bad_pos, 1);
        return;
    }
    const bool live = head < 2 * a.c.n_kv, is_v = head >= a.c.n_kv;
    if (__any_sync(0xFFFFFFFFu, !is_v)) {  // two heads a warp: a value's lanes go along, and stay as they were
        const HeadLanes<HD> y = x;
        if (a.k_norm) x.norm(a.k_norm, a.eps);
        if (a.r.table) x.turn(a.r, p, mine);
        if (is_v) x = y;
    }
    uint8_t* part = live ? a.part(page, head, HEAD) : page;
    x.template put<KIND>(run ? run : part, run ? p % 16 : p % KV_PAGE, part + CODES, p % KV_PAGE, is_v, live);
}

// Queries: a warp has a row and `turns` times as many heads as HD / 8 lanes each leave it, four dimensions and the four that they
// turn with a lane, so that a pair is one thread's and the row's cosines and sines serve all of its heads.
template <uint32_t HD>
__device__ __forceinline__ void append_queries(const AppendArgs& a, uint32_t item, uint32_t turns, float* s_warp) {
    constexpr uint32_t LANES = HD / 8, AT_ONCE = 32 / LANES;
    const uint32_t chunks = (a.n_q + turns * AT_ONCE - 1) / (turns * AT_ONCE), row = item / chunks;
    if (row >= a.rows) return;
    const uint32_t head0 = item % chunks * turns * AT_ONCE, end = min(a.n_q, head0 + turns * AT_ONCE);
    const float* src = a.qkv + row * a.stride;
    float* dst = a.q_out + (uint64_t)row * a.n_q * HD;
    const RopeArgs& r = a.r;
    if (r.table != nullptr && !r.vectors) {  // pairs that are no whole vectors
        using Lanes = HeadLanes<HD>;
        if (a.page(row, 0) == nullptr) return;
        const uint32_t p = (uint32_t)a.pos[row], group = (threadIdx.x & 31) / Lanes::LANES;
        for (uint32_t h = head0; h < end; h += Lanes::PER_WARP) {
            const bool live = h + group < end;
            Lanes x;
            x.load(src + (uint64_t)(h + group) * HD, live);
            if (a.q_norm) x.norm(a.q_norm, a.eps);
            x.turn(r, p, s_warp + group * HD);
            if (live) x.store(dst + (uint64_t)(h + group) * HD);
        }
        return;
    }
    const uint32_t l = (threadIdx.x & 31) % LANES, group = (threadIdx.x & 31) / LANES, half = r.rot / 2;
    const bool turned = r.table != nullptr && 8 * l < r.rot, split = turned && !r.interleaved;
    const uint32_t at_u = split ? 4 * l : 8 * l, at_v = split ? half + 4 * l : 8 * l + 4;
    // heads a lane has on their way (4096 rows of 32 and 2 x 4 heads of 128: one 33.9 us, two 31.7, three 32.2, four, which spill, 32.6)
    constexpr uint32_t AHEAD = 2;
    float4 next_u[AHEAD], next_v[AHEAD];
    auto request = [&](uint32_t first) {
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            const uint32_t head = first + i * AT_ONCE + group;
            const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            next_u[i] = head < end ? *reinterpret_cast<const float4*>(src + (uint64_t)head * HD + at_u) : zero;
            next_v[i] = head < end ? *reinterpret_cast<const float4*>(src + (uint64_t)head * HD + at_v) : zero;
        }
    };
    request(head0);
    if (a.page(row, 0) == nullptr) return;
    float4 cs0 = make_float4(1.0f, 0.0f, 1.0f, 0.0f), cs1 = cs0;
    if (turned) {
        const float4* t = reinterpret_cast<const float4*>(r.table + (uint64_t)(uint32_t)a.pos[row] * half + 4 * l);
        cs0 = __ldg(t), cs1 = __ldg(t + 1);
    }
    for (uint32_t first = head0; first < end; first += AHEAD * AT_ONCE) {
        if (first != head0) request(first);
#pragma unroll
        for (uint32_t i = 0; i < AHEAD; ++i) {
            if (first + i * AT_ONCE >= end) break;  // the same in the warp
            const uint32_t h = first + i * AT_ONCE + group;
            float u[4] = {next_u[i].x, next_u[i].y, next_u[i].z, next_u[i].w}, v[4] = {next_v[i].x, next_v[i].y, next_v[i].z, next_v[i].w};
            if (a.q_norm) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) ss = fmaf(u[e], u[e], fmaf(v[e], v[e], ss));
#pragma unroll
                for (uint32_t o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                const float4 wu = __ldg(reinterpret_cast<const float4*>(a.q_norm + at_u)), wv = __ldg(reinterpret_cast<const float4*>(a.q_norm + at_v));
                const float sc = rsqrtf(ss / (float)HD + a.eps);
                u[0] = u[0] * sc * wu.x, u[1] = u[1] * sc * wu.y, u[2] = u[2] * sc * wu.z, u[3] = u[3] * sc * wu.w;
                v[0] = v[0] * sc * wv.x, v[1] = v[1] * sc * wv.y, v[2] = v[2] * sc * wv.z, v[3] = v[3] * sc * wv.w;
            }
            if (turned) {
                const float2 cs[4] = {make_float2(cs0.x, cs0.y), make_float2(cs0.z, cs0.w), make_float2(cs1.x, cs1.y), make_float2(cs1.z, cs1.w)};
                auto turn = [](float& x, float& y, float2 by) {
                    const float first = rope_rotate(true, x, y, by);
                    y = rope_rotate(false, y, x, by), x = first;
                };
                if (split) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) turn(u[e], v[e], cs[e]);
                } else {
                    turn(u[0], u[1], cs[0]), turn(u[2], u[3], cs[1]), turn(v[0], v[1], cs[2]), turn(v[2], v[3], cs[3]);
                }
            }
            if (h >= end) continue;
            *reinterpret_cast<float4*>(dst + (uint64_t)h * HD + at_u) = make_float4(u[0], u[1], u[2], u[3]);
            *reinterpret_cast<float4*>(dst + (uint64_t)h * HD + at_v) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

// Keys and values in the first CTAs, queries in the rest.  RUNS: four warps have a key's or value's head of 16 rows, four rows
// each, their loads on their way together; where the 16 are a whole run of positions, the codes are put together in shared
// memory as they stand in the page and stored from there in whole lines: a position's codes alone are 4 bytes and fewer to a
// sector of 32.  Else a warp has one row's.
template <uint32_t KIND, uint32_t HD, bool RUNS>
__global__ void __launch_bounds__(256, 4) kv_append_kernel(AppendArgs a, uint32_t kv_blocks, uint32_t turns) {
    using Lanes = HeadLanes<HD>;
    constexpr uint32_t HPW = Lanes::PER_WARP, CODES = kv_code_bytes(KIND, HD), HEAD = kv_head_bytes(KIND, HD), RUN = CODES / 4;
    constexpr uint32_t EACH = RUNS ? 4 : 1, AT_ONCE = 2 * HPW;  // rows a warp, heads a CTA of runs
    __shared__ __align__(16) float s_head[8 * HPW][HD];
    __shared__ __align__(16) uint8_t s_run[RUNS ? AT_ONCE : 1][RUNS ? RUN : 16];
    pdl_trigger_all();
    const uint32_t warp = threadIdx.x >> 5, group = (threadIdx.x & 31) / Lanes::LANES;
    if (blockIdx.x >= kv_blocks) {
        append_queries<HD>(a, (blockIdx.x - kv_blocks) * 8 + warp, turns, s_head[warp * HPW]);
        return;
    }
    const uint32_t heads = 2 * a.c.n_kv;  // keys, then values
    if constexpr (!RUNS) {
        const uint32_t parts = (heads + HPW - 1) / HPW, item = blockIdx.x * 8 + warp, row = item / parts;
        if (row >= a.rows) return;
        const uint32_t head = item % parts * HPW + group;
        Lanes x;
        x.load(a.qkv + row * a.stride + (uint64_t)(a.n_q + head) * HD, head < heads);
        append_head<KIND, HD>(a, x, row, a.page(row, HEAD), (uint32_t)a.pos[row], head, s_head[warp * HPW + group]);
    } else {
        const uint32_t parts = (heads + AT_ONCE - 1) / AT_ONCE, first = blockIdx.x % parts * AT_ONCE, local = (warp & 1) * HPW + group;
        const uint32_t head = first + local, j0 = warp / 2 * EACH;
        RowGroup g(a.pos, a.rows, blockIdx.x / parts);
        Lanes x[EACH];
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i)
            x[i].load(a.qkv + (uint64_t)(g.first + j0 + i) * a.stride + (uint64_t)(a.n_q + head) * HD, head < heads && g.has(j0 + i));
        g.look(a.pos, a.seq);
        uint8_t* run = nullptr;  // the page of a whole run of 16 that has its places; the same in the CTA
        if (g.runs && g.rows == 16 && a.page((uint32_t)g.first + 15, HEAD)) run = a.page((uint32_t)g.first, HEAD);
#pragma unroll
        for (uint32_t i = 0; i < EACH; ++i) {
            if (!g.has(j0 + i)) continue;
            const uint32_t row = (uint32_t)(g.first + j0 + i);
            if (run) append_head<KIND, HD>(a, x[i], row, run, (uint32_t)g.p0 + j0 + i, head, s_head[warp * HPW + group], s_run[local]);
            else append_head<KIND, HD>(a, x[i], row, a.page(row, HEAD), (uint32_t)a.pos[row], head, s_head[warp * HPW + group]);
        }
        if (run == nullptr) return;
        __syncthreads();
        const uint32_t at = (uint32_t)g.p0 % KV_PAGE / 16 * RUN;
        for (uint32_t i = threadIdx.x; i < AT_ONCE * (RUN / 16); i += 256) {
            const uint32_t h = first + i / (RUN / 16), o = i % (RUN / 16) * 16;
            if (h < heads) *reinterpret_cast<uint4*>(a.part(run, h, HEAD) + at + o) = *reinterpret_cast<const uint4*>(s_run[i / (RUN / 16)] + o);
        }
    }
}

// A warp a row and kv head, keys and values.
template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(256) kv_read_kernel(KvPages c, const int32_t* pos, const int32_t* seq, float* k, float* v, uint64_t row_stride,
                                                      uint64_t head_stride, int32_t* bad_pos) {
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

// Sixteen positions of a head's keys or values from the run of memory that holds them: f(position, dimension, four values) for
// each four that a lane has.
template <uint32_t KIND, uint32_t HD, bool VALUES, class F>
__device__ __forceinline__ void read_run(const uint8_t* part, uint32_t in_page, F f) {
    constexpr uint32_t NB = HD / 32, BITS = KIND == KV_F16 ? 16 : KIND == KV_Q8_0 ? 8 : 4, VECS = 16 * HD * BITS / 8 / 512;
    const uint32_t lane = threadIdx.x & 31, r = lane / 4, c = lane % 4;
    const uint4* codes = reinterpret_cast<const uint4*>(part + in_page / 16 * (VECS * 512)) + lane;
    const uint8_t* scales = part + kv_code_bytes(KIND, HD);
    auto both = [&](uint32_t pos, uint32_t b) {  // scales of positions pos and pos + 8 of the run
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(scales + kv_scale_at<HD>(in_page + pos, b)));
        return __half22float2(*reinterpret_cast<const __half2*>(&w));
    };
    auto half_of = [](uint32_t w, uint32_t i) { return __half2float(__ushort_as_half((unsigned short)(i ? w >> 16 : w & 0xFFFF))); };
    if constexpr (KIND == KV_F16 && VALUES) {  // two vectors hold four dimensions
#pragma unroll
        for (uint32_t b = 0; b < NB; ++b) {
            const uint4 x = __ldg(codes + 2 * b * 32), y = __ldg(codes + (2 * b + 1) * 32);
            const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e)
                    f(8 * h + 2 * c + e, 32 * b + 4 * r,
                      make_float4(half_of(u[2 * h], e), half_of(u[2 * h + 1], e), half_of(v[2 * h], e), half_of(v[2 * h + 1], e)));
        }
        return;
    }
#pragma unroll
    for (uint32_t v = 0; v < VECS; ++v) {
        const uint4 x = __ldg(codes + v * 32);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
        if constexpr (KIND == KV_F16) {
            const uint32_t d = 32 * (v / 2) + 8 * c + 4 * (v % 2);
            f(r, d, make_float4(half_of(w[0], 0), half_of(w[0], 1), half_of(w[1], 0), half_of(w[1], 1)));
            f(r + 8, d, make_float4(half_of(w[2], 0), half_of(w[2], 1), half_of(w[3], 0), half_of(w[3], 1)));
        } else if constexpr (KIND == KV_Q8_0) {
            auto at = [&](uint32_t i) { return (float)((int)(w[i / 4] >> (8 * (i % 4)) & 0xFF) - 128); };
            if constexpr (VALUES) {
#pragma unroll
                for (uint32_t e = 0; e < 2; ++e) {
                    const float2 s = both(2 * c + e, v);
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h) {
                        const float g = h ? s.y : s.x;
                        f(8 * h + 2 * c + e, 32 * v + 4 * r, make_float4(at(4 * h + e) * g, at(4 * h + 2 + e) * g, at(8 + 4 * h + e) * g, at(10 + 4 * h + e) * g));
                    }
                }
            } else {
                const float2 s = both(r, v);
#pragma unroll
                for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                    for (uint32_t q = 0; q < 2; ++q) {
                        const float g = h ? s.y : s.x;
                        const uint32_t i = 8 * h + 4 * q;
                        f(r + 8 * h, 32 * v + 8 * c + 4 * q, make_float4(at(i) * g, at(i + 1) * g, at(i + 2) * g, at(i + 3) * g));
                    }
            }
        } else {
#pragma unroll
            for (uint32_t o = 0; o < 2; ++o) {  // the two blocks of the vector
                const uint32_t b = 2 * v + o;
                auto at = [&](uint32_t i, uint32_t byte, uint32_t high) { return (float)((int)(w[2 * o + i] >> (8 * byte + 4 * high) & 15) - 8); };
                if constexpr (VALUES) {
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        const float2 s = both(2 * c + e, b);
#pragma unroll
                        for (uint32_t h = 0; h < 2; ++h) {
                            const float g = h ? s.y : s.x;
                            const uint32_t y = 2 * e + h;
                            f(8 * h + 2 * c + e, 32 * b + 4 * r, make_float4(at(0, y, 0) * g, at(0, y, 1) * g, at(1, y, 0) * g, at(1, y, 1) * g));
                        }
                    }
                } else {
                    const float2 s = both(r, b);
#pragma unroll
                    for (uint32_t h = 0; h < 2; ++h)
#pragma unroll
                        for (uint32_t q = 0; q < 2; ++q) {
                            const float g = h ? s.y : s.x;
                            f(r + 8 * h, 32 * b + 8 * c + 4 * q, make_float4(at(q, h, 0) * g, at(q, 2 + h, 0) * g, at(q, h, 1) * g, at(q, 2 + h, 1) * g));
                        }
                }
            }
        }
    }
}

// Many rows: a warp has the keys or values of a head of 16 rows; where they are consecutive positions, from one run of memory.
template <uint32_t KIND, uint32_t HD, bool VALUES>
__device__ __forceinline__ void read_rows(const KvPages& c, const int32_t* pos, const int32_t* seq, uint32_t rows, const RowGroup& g,
                                          uint32_t head, float* out, uint64_t row_stride, int32_t* bad_pos) {
    constexpr uint32_t HEAD = kv_head_bytes(KIND, HD);
    const uint32_t lane = threadIdx.x & 31;
    float* to = out + g.first * (int64_t)row_stride;
    if (g.runs) {
        const uint32_t row = (uint32_t)(g.first + g.first_j);
        const int32_t p = pos[row];
        const uint8_t* page = page_of(c, seq ? seq[row] : (int32_t)row, p, HEAD);
        if (page != nullptr) {
            const uint8_t* part = page + (uint64_t)head * HEAD + (VALUES ? HEAD / 2 : 0);
            const uint32_t end = g.first_j + g.rows;
            read_run<KIND, HD, VALUES>(part, (uint32_t)p % KV_PAGE & ~15u, [&](uint32_t j, uint32_t d, float4 x) {
                if (j >= g.first_j && j < end) *reinterpret_cast<float4*>(to + j * row_stride + d) = x;
            });
            return;
        }
    }
    for (uint32_t j = g.first_j; j < g.first_j + g.rows; ++j) {
        const uint32_t row = (uint32_t)(g.first + j);
        const int32_t p = pos[row];
        const uint8_t* page = page_of(c, seq ? seq[row] : (int32_t)row, p, HEAD);
        if (page == nullptr && lane == 0 && bad_pos) atomicExch(bad_pos, 1);
        const uint8_t* part = page + (uint64_t)head * HEAD + (VALUES ? HEAD / 2 : 0);
        for (uint32_t d = 4 * lane; d < HD; d += 128)
            *reinterpret_cast<float4*>(to + j * row_stride + d) =
                page ? kv_load<KIND, HD, VALUES>(part, (uint32_t)p % KV_PAGE, d) : make_float4(NAN, NAN, NAN, NAN);
    }
}
template <uint32_t KIND, uint32_t HD>
__global__ void __launch_bounds__(256) kv_read_rows_kernel(KvPages c, const int32_t* pos, const int32_t* seq, uint32_t rows, float* k, float* v,
                                                           uint64_t row_stride, uint64_t head_stride, int32_t* bad_pos) {
    pdl_trigger_all();
    const uint32_t task = blockIdx.y * 8 + (threadIdx.x >> 5), head = task / 2;
    if (head >= c.n_kv) return;
    RowGroup g(pos, rows, blockIdx.x);
    if (g.rows == 0) return;
    g.look(pos, seq);
    if (task % 2)
        read_rows<KIND, HD, true>(c, pos, seq, rows, g, head, v + head * head_stride, row_stride, bad_pos);
    else
        read_rows<KIND, HD, false>(c, pos, seq, rows, g, head, k + head * head_stride, row_stride, bad_pos);
}

// From so many rows on, runs of 16 positions are put together, where rows may stand in runs (each row another sequence's: never).
// 1000 rows of a prompt, 32 query heads on 8 of 128, eight bits: 10.8 us, a warp a row 15.3; 4096 rows 46 and 67 (44 now); 512 rows 9.3 and
// 9.3; 24 heads on 8 of 64 in halves, 1000 rows 8.3 and 7.8, 4096 rows 16.3 and 24.6.  Reading back, 8 heads of 128: 1000 rows 4.8
// and 5.3, 512 rows 4.7 and 4.4.  Heads of 256 always a warp a row: a run's registers leave too few warps a SM (4096 rows read
// 14.1 and 8.6).
constexpr uint32_t MANY_ROWS = 768;
// Queries: warps a SM, with one head's worth each, from which on a warp takes more heads of its row (1000 rows, 16 heads of 256:
// 16 warps 10.4 us, 32 9.4, 64 9.7, 128 11.1).
constexpr uint32_t QUERY_WARPS = 32;

struct LaunchAppend {
    const AppendArgs& a;
    cudaStream_t s;
    template <uint32_t KIND, uint32_t HD>
    cudaError_t operator()() const {
        constexpr uint32_t HPW = HeadLanes<HD>::PER_WARP;
        const uint32_t per_warp = 256 / HD, most = (a.n_q + per_warp - 1) / per_warp;
        uint32_t turns = 1;
        while (turns < most && (uint64_t)a.rows * ((most + turns - 1) / turns) > QUERY_WARPS * num_sms()) turns *= 2;
        const uint32_t q_blocks = (uint32_t)(((uint64_t)a.rows * ((most + turns - 1) / turns) + 7) / 8), heads = 2 * a.c.n_kv;
        if constexpr (HD < 256) {
            if (a.seq != nullptr && a.rows >= MANY_ROWS) {
                const uint32_t kv_blocks = (a.rows + 30) / 16 * ((heads + 2 * HPW - 1) / (2 * HPW));
                return launch_pdl(kv_append_kernel<KIND, HD, true>, dim3(kv_blocks + q_blocks), 256, 0, s, a, kv_blocks, turns);
            }
        }
        const uint32_t kv_blocks = (uint32_t)(((uint64_t)a.rows * ((heads + HPW - 1) / HPW) + 7) / 8);
        return launch_pdl(kv_append_kernel<KIND, HD, false>, dim3(kv_blocks + q_blocks), 256, 0, s, a, kv_blocks, turns);
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
        if constexpr (HD < 256) {
            if (seq != nullptr && rows >= MANY_ROWS)
                return launch_pdl(kv_read_rows_kernel<KIND, HD>, dim3((rows + 30) / 16, (2 * c.n_kv + 7) / 8), 256, 0, s, c, pos, seq, rows,
                                  k, v, row_stride, head_stride, bad_pos);
        }
        return launch_pdl(kv_read_kernel<KIND, HD>, dim3(rows, (c.n_kv + 7) / 8), 256, 0, s, c, pos, seq, k, v, row_stride, head_stride,
                          bad_pos);
    }
};

}  // namespace

cudaError_t launch_kv_append(const KvPages& c, const RopeArgs& r, const float* qkv, uint64_t stride, const int32_t* pos,
                             const int32_t* seq, uint32_t rows, uint32_t n_q, const float* q_norm, const float* k_norm, float eps,
                             float* q_out, int32_t* bad_pos, cudaStream_t s) {
    cudaError_t e = for_kind(c.kind, c.hd, LaunchAppend{AppendArgs{c, r, qkv, stride, pos, seq, rows, n_q, q_norm, k_norm, eps, q_out, bad_pos}, s});
    return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_kv_read(const KvPages& c, const int32_t* pos, const int32_t* seq, uint32_t rows, float* k, float* v,
                           uint64_t row_stride, uint64_t head_stride, int32_t* bad_pos, cudaStream_t s) {
    cudaError_t e = for_kind(c.kind, c.hd, LaunchRead{c, pos, seq, rows, k, v, row_stride, head_stride, bad_pos, s});
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
