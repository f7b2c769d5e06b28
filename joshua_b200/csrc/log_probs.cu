// Log probabilities of rows of logits: of a given token, the row's entropy, the likeliest tokens.
//
// With M the row's largest logit, S = sum e, e = exp(l - M), and T = sum e (l - M):
//   log p(t) = (l_t - M) - log S,   entropy = log S - T / S.
// One pass over the row, a running maximum m a thread, sums brought to a new one as it comes: with d = m - m' and w = exp(d), T becomes
// w (T + d S) and S w S.  S is held without the 1 of the largest logit itself, so that log1p(S - 1) and T / S keep their relative
// accuracy where one token has nearly all of the weight (1 - p = 1e-9 is nothing beside 1 in f32).
//
// The likeliest n: keys of (logit, lower id first) as 64-bit numbers.  Keys above a border go on a list of their warp; the border is the
// n-th largest of the maxima of groups of threads, of the first tile to begin with and of all that came since a few times later, so a
// list seldom holds more than a few keys.  One that grows all the same is cut back to its n largest.
//
// CTAs go from row to row; a cluster of them takes one where rows are few or do not go round evenly, each a slice of it, and rank 0 joins
// their sums and lists in order.  A thread copies the values that it will read itself, some tiles ahead and into the next row: no
// barrier stands between tiles, and the memory works while a row's ends are joined.  What several threads learn of each other's values
// in between, they learn at barriers: results do not depend on who comes first.
//
// Many rows are bounded by the one read of the logits (1000 rows of 128256: 84 us, 6.1 TB/s; blocks of 512 threads, two an SM, 99 us:
// their barriers stop more of an SM at a time; four blocks an SM leave 64 registers a thread, with which 8 bytes spill), few rows by the
// steps from the launch to the end of a row (1 of 128256, 5 likeliest: 9.8 us, of which the tiles take half; 64 of 151936: 11.5 us, with
// the 20 likeliest 20.8 us).
#include <cooperative_groups.h>

#include <algorithm>

#include "f32x2.cuh"
#include "serving.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;

using u64 = unsigned long long;

constexpr uint32_t LP_THREADS = 256, LP_WARPS = LP_THREADS / 32, LP_VECS = 2, LP_VALUES = 4 * LP_VECS, LP_TILE = LP_THREADS * LP_VALUES;
constexpr uint32_t LP_STAGES = 4, LP_MOST_CTAS = 8;  // tiles on their way; CTAs a row
constexpr uint32_t LP_CUT = 48;                      // a warp's list of more is cut back
constexpr uint32_t LP_CAP = 32 * LP_VALUES + LP_CUT;  // so a tile's keys always fit
constexpr float LOG2E = 1.44269504f, LEAST = -1000.0f, LARGEST = 3.402823466e38f;
constexpr uint32_t LP_KEYS = LP_WARPS * LP_CUT;
static_assert(LOG_PROBS_MOST == 32 && LP_CUT >= LOG_PROBS_MOST && LP_CUT <= 64 && LP_MOST_CTAS * LOG_PROBS_MOST <= LP_KEYS, "lists");

struct Tops {
    float of32[32], of64[64];
};
struct LogProbShared {
    float4 ring[LP_STAGES][LP_VECS][LP_THREADS];
    u64 list[LP_WARPS][LP_CAP];
    alignas(16) u64 keys[LP_KEYS];        // of all lists, those above the border
    u64 best[2][LOG_PROBS_MOST];          // the CTA's, in order, of rows in turn
    u64 joined[LOG_PROBS_MOST];           // the cluster's
    alignas(16) Tops tops[2];             // largest ones of groups of threads, in turn
    float4 part[LP_WARPS];                // of the warps: maximum, S without the largest ones' 1, T, number of largest ones
    float4 all[2];                        // of the CTA, of rows in turn
    uint32_t total;                       // of sh.keys
};

__device__ __forceinline__ float ex2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// NaN weighs nothing, as -inf; an infinity counts as the largest number
__device__ __forceinline__ float logit_of(float l) { return fminf(fmaxf(l, -INFINITY), LARGEST); }
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
// of a warp
__device__ __forceinline__ float largest_of(float x) {
    float y;
    asm volatile("redux.sync.max.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float smallest_of(float x) {
    float y;
    asm volatile("redux.sync.min.f32 %0, %1, 0xFFFFFFFF;" : "=f"(y) : "f"(x));
    return y;
}

// A thread's sums under its maximum m: S = held + s, T = t, both halves of a pair.
struct Sums {
    float m, held;
    f32x2 s, t;
    __device__ __forceinline__ float s_of() const { return both(s).x + both(s).y; }
    __device__ __forceinline__ float t_of() const { return both(t).x + both(t).y; }
    // the same under a larger maximum
    __device__ __forceinline__ void rebase(float to) {
        const float d = fmaxf(m - to, LEAST), w = m > -INFINITY ? ex2_of(d * LOG2E) : 0.0f, all = held + s_of();
        s = pair(w * all, 0.0f), t = pair(w * fmaf(d, all, t_of()), 0.0f), held = 0.0f, m = to;
    }
    // Values of a tile, NaN and infinities among them, and their largest; the first that is larger than all before is held apart.
    __device__ __forceinline__ void add(const float (&x)[LP_VALUES], float top) {
        if (top > m) {
            top = fminf(top, LARGEST);
            bool skipped = top == m;  // m was the largest number already, and an infinity came
            if (!skipped) rebase(top), held = 1.0f;
            float st = s_of(), tt = t_of();
#pragma unroll
            for (uint32_t i = 0; i < LP_VALUES; ++i) {
                const float y = logit_of(x[i]), d = fmaxf(y - m, LEAST), e = ex2_of(d * LOG2E);
                const bool skip = !skipped && y == m;
                skipped |= skip;
                st += skip ? 0.0f : e, tt = fmaf(e, d, tt);
            }
            s = pair(st, 0.0f), t = pair(tt, 0.0f);
        } else if (m > -INFINITY) {
            const f32x2 less = pair(-m, -m), scale = pair(LOG2E, LOG2E);
#pragma unroll
            for (uint32_t i = 0; i < LP_VALUES; i += 2) {
                const float2 d = both(add2(pair(x[i], x[i + 1]), less));
                const f32x2 dd = pair(fmaxf(d.x, LEAST), fmaxf(d.y, LEAST));
                const float2 y = both(mul2(dd, scale));
                const f32x2 e = pair(ex2_of(y.x), ex2_of(y.y));
                s = add2(s, e), t = fma2(e, dd, t);
            }
        }
    }
};

// The n largest of some keys, in order, into best, which holds zeros.  All threads, behind a barrier.  (It and the next ones are there
// once: where a row is all that a CTA has, its time is that of code that comes for the first time.)
__device__ __noinline__ void rank(const u64* keys, uint32_t count, uint32_t n, u64* best) {
    for (uint32_t i = threadIdx.x; i < count; i += LP_THREADS) {
        const u64 mine = keys[i];
        uint32_t above = 0, j = 0;
        for (; j + 8 <= count && above < n; j += 8) {
#pragma unroll
            for (uint32_t k = 0; k < 8; k += 2) {
                const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + j + k);
                above += two.x > mine, above += two.y > mine;
            }
        }
        if (above < n)
            for (; j < count; ++j) above += keys[j] > mine;
        if (above < n) best[above] = mine;
    }
}
// The same for `lists` lists that are in order, n keys each, zeros at an end.
__device__ __noinline__ void merge(const u64* keys, uint32_t lists, uint32_t n, u64* best) {
    for (uint32_t i = threadIdx.x; i < lists * n; i += LP_THREADS) {
        const u64 mine = keys[i];
        uint32_t above = 0;
        for (uint32_t r = 0; r < lists; ++r) {
            uint32_t first = 0;  // keys of the list that are larger
#pragma unroll
            for (uint32_t by = LOG_PROBS_MOST; by > 0; by /= 2)
                if (first + by <= n && keys[r * n + first + by - 1] > mine) first += by;
            above += first;
        }
        if (mine && above < n) best[above] = mine;
    }
}
// The sums of the lanes of a warp: maximum, S without the largest ones' 1, T, number of largest ones.
__device__ __noinline__ float4 join(float4 x) {
    const float m = x.x, top = largest_of(m);
    const float d = m > -INFINITY ? fmaxf(m - top, LEAST) : LEAST, f = ex2_of(d * LOG2E);
    float r[3] = {m == top ? x.y : f * (x.w + x.y), m > -INFINITY ? f * fmaf(d, x.w + x.y, x.z) : 0.0f, m == top ? x.w : 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 3; ++i) r[i] += __shfl_xor_sync(0xFFFFFFFFu, r[i], o);
    return {top, r[0], r[1], r[2]};
}
// What groups of threads have seen until now, `most` of a thread: the largest of all, and the n-th largest of the groups' for the border.
// About G log(G / (G - n)) values of the first tile are above that of G groups: 32 groups for up to 24 of them, else 64 (with 32 for all,
// lists of 32 were cut back again and again: 4 rows of 151818 46 us).  All threads.
struct Look {
    float best, nth;
};
template <uint32_t PER>  // groups a lane
__device__ __forceinline__ float nth_of(const float* tops, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31;
    float g[PER];
    uint32_t above[PER] = {};
#pragma unroll
    for (uint32_t k = 0; k < PER; ++k) g[k] = tops[32 * k + lane];
#pragma unroll 8
    for (uint32_t j = 0; j < 32 * PER; j += 4) {
        const float4 x = *reinterpret_cast<const float4*>(tops + j);
#pragma unroll
        for (uint32_t k = 0; k < PER; ++k) above[k] += x.x > g[k], above[k] += x.y > g[k], above[k] += x.z > g[k], above[k] += x.w > g[k];
    }
    float least = INFINITY;
#pragma unroll
    for (uint32_t k = 0; k < PER; ++k) least = fminf(least, above[k] < n ? g[k] : INFINITY);
    return smallest_of(least);
}
__device__ __noinline__ Look look(Tops& tops, float most, uint32_t n) {
    static_assert(LP_THREADS == 256, "8 and 4 threads a group");
    const uint32_t tid = threadIdx.x, lane = tid & 31;
    float g = fminf(most, LARGEST);
    g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, 1));
    g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, 2));
    if (lane % 4 == 0) tops.of64[tid / 4] = g;
    g = fmaxf(g, __shfl_xor_sync(0xFFFFFFFFu, g, 4));
    if (lane % 8 == 0) tops.of32[tid / 8] = g;
    __syncthreads();
    return {largest_of(tops.of32[lane]), n == 0 ? -INFINITY : n <= 24 ? nth_of<1>(tops.of32, n) : nth_of<2>(tops.of64, n)};
}
// A warp's list of more than n keys cut back to its n largest; the smallest of them.  The warp.
__device__ __noinline__ u64 cut_back(u64* list, uint32_t count, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31;
    u64 last = ~0ull, mine = 0;
    for (uint32_t r = 0; r < n; ++r) {
        u64 k = 0;
        for (uint32_t i = lane; i < count; i += 32) {
            const u64 x = list[i];
            if (x < last && x > k) k = x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) k = max64(k, __shfl_xor_sync(0xFFFFFFFFu, k, o));
        last = k;
        if (lane == r) mine = k;
    }
    __syncwarp();
    if (lane < n) list[lane] = mine;
    __syncwarp();
    return last;
}

__device__ __forceinline__ void copy_ahead(float4* to, const float* from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}

__global__ void __launch_bounds__(LP_THREADS, 4) log_probs_kernel(LogProbArgs a, uint32_t rows, uint32_t ctas) {
    extern __shared__ __align__(16) uint8_t s_mem[];
    LogProbShared& sh = *reinterpret_cast<LogProbShared*>(s_mem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, slice = blockIdx.x % ctas, step = gridDim.x / ctas, n = a.top;
    pdl_trigger_all();
    // Vectors stand on 16-byte boundaries: a row's position 0 is `shift`, up to three, floats in front of it.  A CTA's slice: x0 .. x1.
    const uint32_t share = ((a.vocab + 3 + ctas - 1) / ctas + 3) / 4 * 4, tiles = (share + LP_TILE - 1) / LP_TILE;
    struct Slice {
        const float* from;
        uint32_t shift, x0, x1;
        __device__ __forceinline__ Slice(const LogProbArgs& a, uint32_t row, uint32_t rank, uint32_t share) {
            const float* l = a.logits + row * a.stride;
            shift = (uint32_t)(reinterpret_cast<uintptr_t>(l) / 4 % 4), from = l - shift;
            x0 = min(a.vocab + shift, rank * share), x1 = min(a.vocab + shift, x0 + share);
        }
        // whether the values from p to q are there, all of them
        __device__ __forceinline__ bool whole(uint32_t p, uint32_t q) const { return p >= shift && q <= x1; }
    };
    uint32_t row = blockIdx.x / ctas, ahead_row = row, ahead_tile = 0, slot = 0, turn = 0;
    Slice ahead(a, row, slice, share);
    auto copy = [&](uint32_t slot) {  // the next tile ahead
        const uint32_t at = ahead.x0 + ahead_tile * LP_TILE, p = at + tid * 4;
        if (ahead.whole(at, at + LP_TILE)) {
            const float* from = ahead.from + p;
#pragma unroll
            for (uint32_t v = 0; v < LP_VECS; ++v) copy_ahead(&sh.ring[slot][v][tid], from + v * LP_THREADS * 4);
        } else if (ahead_row < rows) {
#pragma unroll 1
            for (uint32_t v = 0; v < LP_VECS; ++v) {
                const uint32_t q = p + v * LP_THREADS * 4;
                if (ahead.whole(q, q + 4)) {
                    copy_ahead(&sh.ring[slot][v][tid], ahead.from + q);
                } else {
                    float x[4];
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) x[i] = q + i >= ahead.shift && q + i < ahead.x1 ? ahead.from[q + i] : -INFINITY;
                    sh.ring[slot][v][tid] = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        if (++ahead_tile == tiles) {
            ahead_tile = 0, ahead_row += step;
            if (ahead_row < rows) ahead = Slice(a, ahead_row, slice, share);
            else ahead.x0 = ahead.x1 = 0;  // nothing is left
        }
    };
#pragma unroll
    for (uint32_t i = 0; i < LP_STAGES; ++i) copy(i);
    uint32_t odd = 0;  // rows in turn
    for (; row < rows; row += step, odd ^= 1) {
        const Slice sl(a, row, slice, share);
        float given = NAN;
        if (slice == 0 && tid == 0) {
            const int32_t t = a.token[row];
            if (t >= 0 && (uint32_t)t < a.vocab) given = logit_of(sl.from[sl.shift + t]);
        }
        Sums w{-INFINITY, 0.0f, 0, 0};
        u64 border = 0;                             // of the lists: keys above it
        float least = -INFINITY, most = -INFINITY;  // its logit; the thread's largest one
        uint32_t count = 0, next_look = 0;          // of the warp's list; a tile
        auto look_again = [&] {
            const Look seen = look(sh.tops[turn ^= 1], most, n);
            if (seen.nth > least) border = key_of(seen.nth, 0xFFFFFFFFu), least = seen.nth;
            return seen.best;
        };
        for (uint32_t tile = 0; tile < tiles; ++tile) {
            const uint32_t at = sl.x0 + tile * LP_TILE;
            asm volatile("cp.async.wait_group %0;" ::"n"(LP_STAGES - 1) : "memory");
            float y[LP_VALUES], top = -INFINITY;
#pragma unroll
            for (uint32_t v = 0; v < LP_VECS; ++v) {
                const float4 x = sh.ring[slot][v][tid];
                y[4 * v] = x.x, y[4 * v + 1] = x.y, y[4 * v + 2] = x.z, y[4 * v + 3] = x.w;
            }
#pragma unroll
            for (uint32_t i = 0; i < LP_VALUES; i += 2) top = max3(top, y[i], y[i + 1]);
            most = fmaxf(most, top);
            if (tile == next_look) {  // the 1st, 4th, 16th, .. tile
                next_look = 4 * tile + 3;
                // a maximum for all threads that have no larger one: later values seldom pass it
                const float best = look_again();
                if (best > fmaxf(w.m, fminf(top, LARGEST))) w.rebase(best);
            }
            w.add(y, top);
            if (n && __any_sync(0xFFFFFFFFu, top >= least && top > -INFINITY)) {
                uint32_t mask = 0;
#pragma unroll
                for (uint32_t i = 0; i < LP_VALUES; ++i) mask |= y[i] >= least && y[i] > -INFINITY ? 1u << i : 0;
                while (__any_sync(0xFFFFFFFFu, mask != 0)) {
                    u64 k = 0;
                    if (mask) {
                        const uint32_t i = __ffs(mask) - 1;
                        mask &= mask - 1;
                        const float x = reinterpret_cast<const float*>(&sh.ring[slot][i / 4][tid])[i % 4];
                        k = key_of(logit_of(x), at + (i / 4 * LP_THREADS + tid) * 4 + i % 4 - sl.shift);
                    }
                    const uint32_t in = __ballot_sync(0xFFFFFFFFu, k > border);
                    if (k > border) sh.list[warp][count + __popc(in & ((1u << lane) - 1))] = k;
                    count += __popc(in);
                }
                __syncwarp();
                if (count > LP_CUT) {
                    const u64 last = cut_back(sh.list[warp], count, n);
                    count = n;
                    if (last - 1 > border) border = last - 1, least = key_logit(border);
                }
            }
            copy(slot);
            slot = slot + 1 == LP_STAGES ? 0 : slot + 1;
        }
        // the CTA's sums, in order
        float4 r = join({w.m, w.s_of(), w.t_of(), w.held});
        if (lane == 0) sh.part[warp] = r;
        if (n) {
            if (tid == 0) sh.total = 0;
            if (tid < n) sh.best[odd][tid] = 0;
            look_again();
            const u64 k0 = lane < count ? sh.list[warp][lane] : 0, k1 = lane + 32 < count ? sh.list[warp][lane + 32] : 0;
            const uint32_t in0 = __ballot_sync(0xFFFFFFFFu, k0 > border), in1 = __ballot_sync(0xFFFFFFFFu, k1 > border), below = (1u << lane) - 1;
            uint32_t to = 0;
            if (lane == 0 && (in0 | in1)) to = atomicAdd(&sh.total, __popc(in0) + __popc(in1));
            to = __shfl_sync(0xFFFFFFFFu, to, 0);
            if (k0 > border) sh.keys[to + __popc(in0 & below)] = k0;
            if (k1 > border) sh.keys[to + __popc(in0) + __popc(in1 & below)] = k1;
        }
        __syncthreads();
        const float4 none = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        if (warp == 0) {
            r = join(lane < LP_WARPS ? sh.part[lane] : none);
            if (lane == 0) sh.all[odd] = r;
        }
        const u64* best = sh.best[odd];
        if (n) {
            rank(sh.keys, sh.total, n, sh.best[odd]);
            __syncthreads();
        }
        if (ctas > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            cluster.sync();  // the next row's are others: what rank 0 reads here is still there
            if (slice == 0) {
                if (warp == 0) r = join(lane < ctas ? cluster.map_shared_rank(&sh, lane)->all[odd] : none);
                if (n) {
                    for (uint32_t i = tid; i < ctas * n; i += LP_THREADS) sh.keys[i] = cluster.map_shared_rank(&sh, i / n)->best[odd][i % n];
                    if (tid < n) sh.joined[tid] = 0;
                    __syncthreads();
                    merge(sh.keys, ctas, n, sh.joined);
                    __syncthreads();
                    best = sh.joined;
                }
            }
        }
        if (slice == 0 && warp == 0) {
            // r.w largest ones: the first is the 1 that log1p adds
            const float top = r.x, rest = r.y + (r.w - 1.0f), log_s = log1pf(rest);
            const bool nothing = !(top > -INFINITY);
            auto log_p = [&](float x) { return nothing ? -INFINITY : (x - top) - log_s; };
            if (lane == 0) {
                a.log_prob[row] = isnan(given) ? NAN : log_p(given);
                if (a.entropy) a.entropy[row] = nothing ? 0.0f : fmaxf(log_s - r.z / (1.0f + rest), 0.0f);
            }
            if (lane < n) {
                const u64 k = best[lane];
                a.top_token[(uint64_t)row * n + lane] = k ? (int32_t)~(uint32_t)k : -1;
                a.top_log_prob[(uint64_t)row * n + lane] = k ? log_p(key_logit(k)) : -INFINITY;
            }
        }
    }
    if (ctas > 1) cg::this_cluster().sync();  // rank 0 has read the others' shared memory
}

}  // namespace

cudaError_t launch_log_probs(const LogProbArgs& a, uint32_t rows, cudaStream_t s) {
    static bool configured[MAX_DEVICES] = {};
    static int room[MAX_DEVICES][LP_MOST_CTAS + 1] = {};  // clusters of so many CTAs at a time
    constexpr uint32_t LP_ENDS = 8;
    if (cudaError_t e = set_max_smem_once(log_probs_kernel, sizeof(LogProbShared), configured); e != cudaSuccess) return e;
    const int device = current_device();
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(LP_THREADS);
    cfg.dynamicSmemBytes = sizeof(LogProbShared);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    // CTAs a row: what takes the fewest tiles one after the other, each row's ends counted as LP_ENDS of them (300 rows of 128256 with the 5
    // likeliest, logits not in L2: 55 us with 4 of them, 45 us with 8)
    uint32_t ctas = 1;
    uint64_t least = UINT64_MAX;
    for (uint32_t c = 1; c <= LP_MOST_CTAS; c *= 2) {
        int& fit = room[device][c];
        if (fit == 0) {
            cfg.gridDim = dim3(c), cfg.numAttrs = 1, attr[0].val.clusterDim.x = c;
            int n = 0;
            if (cudaError_t e = cudaOccupancyMaxActiveClusters(&n, log_probs_kernel, &cfg); e != cudaSuccess) return e;
            if (n < 1) return cudaErrorInvalidConfiguration;
            fit = n;
        }
        const uint64_t turns = (rows + fit - 1) / fit, time = turns * ((a.vocab + c * LP_TILE - 1) / (c * LP_TILE) + LP_ENDS);
        if (time < least) least = time, ctas = c;
    }
    const uint32_t clusters = (uint32_t)std::min<uint64_t>(rows, room[device][ctas]);
    cfg.gridDim = dim3(clusters * ctas), cfg.numAttrs = 2, attr[0].val.clusterDim.x = ctas;
    cudaError_t e = cudaLaunchKernelEx(&cfg, log_probs_kernel, a, rows, ctas);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
