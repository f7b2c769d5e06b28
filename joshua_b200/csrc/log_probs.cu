// Log probabilities of rows of logits: of a given token, the row's entropy, the likeliest tokens.
//
// With M the row's largest logit, S = sum e, e = exp(l - M), and T = sum e (l - M):
//   log p(t) = (l_t - M) - log S,   entropy = log S - T / S.
// One pass over the row, a running maximum m a thread, sums brought to a new one as it comes: with d = m - m' and w = exp(d), T becomes
// w (T + d S) and S w S.  S is held without the 1 of the largest logit itself, so that log1p(S - 1) and T / S keep their relative
// accuracy where one token has nearly all of the weight (1 - p = 1e-9 is nothing beside 1 in f32).
//
// The likeliest n: keys of (logit, lower id first) as 64-bit numbers.  Keys above the n-th largest one found so far are put on a
// list, which is cut back to its n largest when it grows; the first border is the n-th largest of 32 groups' maxima of the first tile.
//
// A cluster of CTAs takes a row where rows are few, each a slice of it; rank 0 joins their sums and lists in order.
#include <cooperative_groups.h>

#include "serving.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;

using u64 = unsigned long long;

constexpr uint32_t LP_THREADS = 512, LP_WARPS = LP_THREADS / 32, LP_VECS = 2, LP_TILE = LP_THREADS * 4 * LP_VECS, LP_MOST_CTAS = 8;
constexpr uint32_t LP_CUT = 192;                   // a list of more is cut back behind the tile
constexpr uint32_t LP_CAP = LP_TILE + LP_CUT;      // so a tile's keys always fit
constexpr float LOG2E = 1.44269504f, LEAST = -1000.0f;

struct LogProbShared {
    float part[LP_WARPS][4];            // of the warps: maximum, S without the largest ones' 1, T, number of largest ones
    float all[4];                       // of the CTA
    u64 group[2 * LP_WARPS];
    u64 best[LOG_PROBS_MOST];           // in order
    uint32_t count;
    u64 list[LP_CAP];
};

__device__ __forceinline__ float ex2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// NaN weighs nothing, as -inf; an infinity counts as the largest number
__device__ __forceinline__ float logit_of(float l) { return l > -INFINITY ? fminf(l, 3.402823466e38f) : -INFINITY; }
// (logit, lower id first) as a number; -0 and 0 are one.  Never 0.
__device__ __forceinline__ u64 key_of(float l, uint32_t id) {
    const uint32_t u = __float_as_uint(l + 0.0f);
    return (u64)(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_logit(u64 k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}
__device__ __forceinline__ u64 max64(u64 a, u64 b) { return a > b ? a : b; }

// A thread's sums under its maximum m: S = held + s, T.
struct Sums {
    float m, s, t, held;
    __device__ __forceinline__ void rebase(float to) {
        const float d = fmaxf(m - to, LEAST), w = m > -INFINITY ? ex2_of(d * LOG2E) : 0.0f;
        const float all = held + s;
        t = w * fmaf(d, all, t), s = w * all, m = to;
    }
    // values of a tile; the first that is larger than all before is held apart
    __device__ __forceinline__ void add(const float (&x)[4 * LP_VECS], float top) {
        if (top > m) {
            rebase(top);
            held = 1.0f;
            bool skipped = false;
#pragma unroll
            for (uint32_t i = 0; i < 4 * LP_VECS; ++i) {
                const float d = fmaxf(x[i] - m, LEAST), e = ex2_of(d * LOG2E);
                const bool skip = !skipped && x[i] == m;
                skipped |= skip;
                s += skip ? 0.0f : e, t = fmaf(e, d, t);
            }
        } else if (m > -INFINITY) {
#pragma unroll
            for (uint32_t i = 0; i < 4 * LP_VECS; ++i) {
                const float d = fmaxf(x[i] - m, LEAST), e = ex2_of(d * LOG2E);
                s += e, t = fmaf(e, d, t);
            }
        }
    }
};

// The n largest of the list's keys, in order, into sh.best and at the list's beginning.  All threads.
__device__ __forceinline__ void cut_back(LogProbShared& sh, uint32_t n) {
    const uint32_t tid = threadIdx.x, count = sh.count;
    if (tid < n) sh.best[tid] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < count; i += LP_THREADS) {
        const u64 mine = sh.list[i];
        uint32_t above = 0;
        for (uint32_t j = 0; j < count && above < n; ++j) above += sh.list[j] > mine;
        if (above < n) sh.best[above] = mine;
    }
    __syncthreads();
    if (tid < n) sh.list[tid] = sh.best[tid];
    if (tid == 0) sh.count = min(count, n);
    __syncthreads();
}

__global__ void __launch_bounds__(LP_THREADS, 2) log_probs_kernel(LogProbArgs a, uint32_t ctas) {
    extern __shared__ __align__(16) uint8_t s_mem[];
    LogProbShared& sh = *reinterpret_cast<LogProbShared*>(s_mem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = blockIdx.x / ctas, rank = blockIdx.x % ctas, n = a.top;
    if (tid == 0) sh.count = 0;
    __syncthreads();
    pdl_trigger_all();
    const float* l = a.logits + row * a.stride;
    // vectors stand on 16-byte boundaries: position 0 is up to three floats in front of the row
    const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(l) / 4 % 4), end = a.vocab + shift;
    const uint32_t share = ((end + ctas - 1) / ctas + 3) / 4 * 4, x0 = min(end, rank * share), x1 = min(end, x0 + share);
    auto load = [&](uint32_t at, float (&x)[4 * LP_VECS]) {
#pragma unroll
        for (uint32_t v = 0; v < LP_VECS; ++v) {
            const uint32_t p = at + (v * LP_THREADS + tid) * 4;
            if (p >= shift && p + 4 <= x1) {
                const float* from = l + (p - shift);
                asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(x[4 * v]), "=f"(x[4 * v + 1]), "=f"(x[4 * v + 2]), "=f"(x[4 * v + 3])
                             : "l"(from));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) x[4 * v + i] = p + i >= shift && p + i < x1 ? l[p + i - shift] : -INFINITY;
            }
        }
    };
    Sums w{-INFINITY, 0.0f, 0.0f, 0.0f};
    u64 border = 0;  // of the list: keys above it
    float x[4 * LP_VECS];
    load(x0, x);
    for (uint32_t at = x0; at < x1; at += LP_TILE) {
        float y[4 * LP_VECS], top = -INFINITY;
#pragma unroll
        for (uint32_t i = 0; i < 4 * LP_VECS; ++i) y[i] = logit_of(x[i]), top = fmaxf(top, y[i]);
        if (at + LP_TILE < x1) load(at + LP_TILE, x);
        auto id = [&](uint32_t i) { return at + (i / 4 * LP_THREADS + tid) * 4 + i % 4 - shift; };
        if (at == x0) {
            u64 mine = 0;
#pragma unroll
            for (uint32_t i = 0; i < 4 * LP_VECS; ++i) mine = max64(mine, y[i] > -INFINITY ? key_of(y[i], id(i)) : 0);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mine = max64(mine, __shfl_xor_sync(0xFFFFFFFFu, mine, o));
            if (lane % 16 == 0) sh.group[tid / 16] = mine;
            __syncthreads();
            static_assert(2 * LP_WARPS == 32 && LOG_PROBS_MOST <= 32, "a lane a group");
            const u64 g = sh.group[lane];
            uint32_t above = 0;
#pragma unroll
            for (uint32_t j = 0; j < 32; ++j) above += __shfl_sync(0xFFFFFFFFu, g, j) > g;
            // a maximum for all threads to begin with: later ones seldom pass it
            const uint32_t first = __ffs(__ballot_sync(0xFFFFFFFFu, above == 0)) - 1;
            const u64 best = __shfl_sync(0xFFFFFFFFu, g, first);
            if (best) {
                w.m = key_logit(best);
                const uint32_t of = ~(uint32_t)best + shift - at;  // its place in the tile: its thread holds it apart
                if (of / 4 % LP_THREADS == tid) w.m = -INFINITY;
            }
            const uint32_t nth = __ballot_sync(0xFFFFFFFFu, n && g && above == n - 1);
            if (nth) border = __shfl_sync(0xFFFFFFFFu, g, __ffs(nth) - 1) - 1;
        }
        w.add(y, top);
        if (n) {
            const float least = border ? key_logit(border) : -INFINITY;
            if (top >= least) {
#pragma unroll
                for (uint32_t i = 0; i < 4 * LP_VECS; ++i)
                    if (y[i] >= least && y[i] > -INFINITY) {
                        const u64 k = key_of(y[i], id(i));
                        if (k > border) sh.list[atomicAdd(&sh.count, 1)] = k;
                    }
            }
            __syncthreads();
            if (sh.count > LP_CUT) {
                cut_back(sh, n);
                border = sh.best[n - 1];
            }
            __syncthreads();  // before keys are added again
        }
    }
    if (n) cut_back(sh, n);
    // the CTA's sums, in order
    auto join = [&](float m, float s, float t, float held, float (&r)[4]) {  // of the lanes of a warp; held: largest ones
        float top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
        const float d = m > -INFINITY ? fmaxf(m - top, LEAST) : LEAST, f = ex2_of(d * LOG2E);
        const float all = held + s;
        r[0] = top, r[1] = m == top ? s : f * all, r[2] = m > -INFINITY ? f * fmaf(d, all, t) : 0.0f, r[3] = m == top ? held : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 1; i < 4; ++i) r[i] += __shfl_xor_sync(0xFFFFFFFFu, r[i], o);
    };
    float r[4];
    join(w.m, w.s, w.t, w.held, r);
    if (lane == 0) sh.part[warp][0] = r[0], sh.part[warp][1] = r[1], sh.part[warp][2] = r[2], sh.part[warp][3] = r[3];
    __syncthreads();
    auto nothing = [](uint32_t i) { return i == 0 ? -INFINITY : 0.0f; };
    if (warp == 0) {
        float v[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) v[i] = lane < LP_WARPS ? sh.part[lane][i] : nothing(i);
        join(v[0], v[1], v[2], v[3], r);
        if (lane < 4) sh.all[lane] = lane == 0 ? r[0] : lane == 1 ? r[1] : lane == 2 ? r[2] : r[3];
    }
    if (ctas > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (rank == 0) {
            if (warp == 0) {
                float v[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) v[i] = lane < ctas ? cluster.map_shared_rank(&sh, lane)->all[i] : nothing(i);
                join(v[0], v[1], v[2], v[3], r);
            }
            for (uint32_t i = tid; i < ctas * n; i += LP_THREADS) sh.list[i] = cluster.map_shared_rank(&sh, i / n)->best[i % n];
            if (tid == 0) sh.count = ctas * n;
            __syncthreads();
            if (n) cut_back(sh, n);
        }
        cluster.sync();  // the others' shared memory has been read
        if (rank != 0) return;
    }
    if (warp != 0) return;
    // r[3] largest ones: the first is the 1 that log1p adds
    const float top = r[0], rest = r[1] + (r[3] - 1.0f), log_s = log1pf(rest);
    const bool none = !(top > -INFINITY);
    auto log_p = [&](float x) { return none ? -INFINITY : (x - top) - log_s; };
    if (lane == 0) {
        const int32_t t = a.token[row];
        a.log_prob[row] = t < 0 || (uint32_t)t >= a.vocab ? NAN : log_p(logit_of(l[t]));
        if (a.entropy) a.entropy[row] = none ? 0.0f : fmaxf(log_s - r[2] / (1.0f + rest), 0.0f);
    }
    if (lane < n) {
        const u64 k = sh.best[lane];
        a.top_token[(uint64_t)row * n + lane] = k ? (int32_t)~(uint32_t)k : -1;
        a.top_log_prob[(uint64_t)row * n + lane] = k ? log_p(key_logit(k)) : -INFINITY;
    }
}

}  // namespace

cudaError_t launch_log_probs(const LogProbArgs& a, uint32_t rows, cudaStream_t s) {
    static bool configured[MAX_DEVICES] = {};
    if (cudaError_t e = set_max_smem_once(log_probs_kernel, sizeof(LogProbShared), configured); e != cudaSuccess) return e;
    // as many CTAs a row as there is room for, two an SM, with two tiles each at least
    uint32_t ctas = 1;
    while (ctas < LP_MOST_CTAS && (uint64_t)rows * ctas * 2 <= 2 * (uint64_t)num_sms() && a.vocab / (2 * ctas) >= 2 * LP_TILE) ctas *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(rows * ctas);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.dynamicSmemBytes = sizeof(LogProbShared);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ctas, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctas > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, log_probs_kernel, a, ctas);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
