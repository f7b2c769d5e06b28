// One token of every row of logits: temperature, top-k, top-p, min-p, then a draw from a given random number.
//
// A token's weight is rint(2^32 exp((l - max) / T)), a whole number: sums of weights are exact in 64 bits, so no order of
// summation, no number of CTAs and no atomic changes which token comes out, and top-p and the draw have no rounding of their
// own.  A token below 2^-33 of the likeliest weighs nothing and is never drawn.  Tokens stand in order of (logit, lower id
// first); each rule keeps a leading run of that order, so together they keep the shortest:
//   top-k  the first k;   top-p  those with less than trunc(p W) in front of them, W the weight of the top-k run;
//   min-p  those with exp((l - max) / T) >= min_p.
// The token is the first id, in order of ids, at which the kept weights' running sum passes trunc(u W'), W' their sum.
//
// A cluster of CTAs takes a row, each a slice of it in shared memory: the logits are read once.  The border of top-k or top-p is
// found from a histogram of the distance to the maximum (numbers or weights of tokens in 2048 equal bins), and within the bin
// that holds it by comparing its tokens with one another; a bin with too many of them (equal logits) is halved by place instead.
// Where a top-k and the rest of its bin are 2048 tokens at most, they go to one CTA, which does the rest.
//
// Bound by the barriers of the cluster and the shared-memory passes between them, not by memory (64 rows of 151936 are 39 MB, 6 us
// of a copy): one row 17 us with a top-k of 40 (27 with top-p alone, whose histogram holds weights of all tokens), 64 rows 50 us
// and 84 us (vocabulary 128256).
#include <cooperative_groups.h>

#include "serving.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t SM_THREADS = 512, SM_WARPS = SM_THREADS / 32, SM_CTAS = 8, SM_MOST_CTAS = 16, SM_WINDOW = 64, SM_BINS = 2048, SM_FEW = 2048;

using u64 = unsigned long long;

// Logits as whole numbers of the same order, -0 and 0 as one; NaN and -inf come last, as 0.
__device__ __forceinline__ uint32_t logit_key(float l) {
    const uint32_t u = __float_as_uint(l + 0.0f);
    return l > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}

// Four logits, each read once: not kept in L1, and not moved above the wait for the kernel in front (64 rows of 151936 59.6 us, by
// plain loads, which the compiler orders worse, 61.2).
__device__ __forceinline__ float4 ld_once(const float* p) {
    float4 v;
    asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
    return v;
}

struct Token {
    u64 weight;
    uint32_t id;
};
struct SampleShared {
    union {
        struct {
            uint32_t number[SM_BINS], low[SM_BINS], high[SM_BINS];  // tokens, low and high halves of their weights
        } bins;
        u64 few[SM_FEW];  // places of a few tokens; bins.high then is where a bin's tokens go in their order (CTA 0)
    };
    // written by every CTA of the cluster, into all: a write in front of a barrier costs less than a read behind it
    float best[SM_MOST_CTAS], least[SM_MOST_CTAS];
    u64 part[SM_MOST_CTAS];
    uint32_t few_of[SM_MOST_CTAS];
    float red[2][SM_WARPS];
    uint32_t n_few, bin, number;
    static_assert(SM_FEW * 8 <= SM_BINS * 8, "bins.high lies behind the few");
    u64 border, before, sum, scan[SM_WARPS], scan2[SM_WARPS];
    int32_t window[SM_WINDOW];
};

template <class V>
__device__ __forceinline__ V warp_sum(V v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    return v;
}
template <class V>
__device__ __forceinline__ V warp_scan(V v, uint32_t lane) {  // sum of this lane's and those in front of it
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V up = __shfl_up_sync(0xFFFFFFFFu, v, o);
        v += lane >= o ? up : V(0);
    }
    return v;
}

// trunc(u total), below total
__device__ __forceinline__ u64 draw_of(float u, u64 total) {
    const double at = (double)u * (double)total;
    const u64 r = at >= 1.0 ? (u64)at : 0ull;
    return total != 0 && r >= total ? total - 1 : r;
}
// the weight that top-p keeps of `total`
__device__ __forceinline__ u64 most_of(float top_p, u64 total) {
    const double p = (double)top_p * (double)total;
    return p >= 1.0 ? (u64)p : 1ull;
}

// A row of logits spread over the cluster, and its rules.
struct Row {
    cg::cluster_group cluster;
    SampleShared& sh;
    float* l;         // this CTA's slice, padded with NaN to whole vectors on both sides
    int32_t lo;       // id of its first place
    uint32_t n;       // places, a multiple of 4
    uint32_t ctas, rank, tid, warp, lane;
    float best, temp, cutoff, to_bin;
    bool greedy;

    __device__ __forceinline__ float likeness(float x) const {  // exp((l - max) / T)
        if (!(x > -INFINITY)) return 0.0f;
        if (x == best) return 1.0f;
        const float d = __fsub_rn(x, best);
        return !greedy ? expf(temp == 1.0f ? d : __fdiv_rn(d, temp)) : 0.0f;
    }
    __device__ __forceinline__ static float weight_float(float e) { return rintf(e * 4294967296.0f); }
    __device__ __forceinline__ static u64 weight(float e) { return (u64)weight_float(e); }
    __device__ __forceinline__ u64 place(uint32_t i) const { return (u64)logit_key(l[i]) << 32 | (0xFFFFFFFFu - (uint32_t)(lo + (int32_t)i)); }
    __device__ __forceinline__ static float logit(u64 place) {
        const uint32_t key = (uint32_t)(place >> 32);
        return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
    }
    // f(logit, place) of the whole slice, in no order
    template <class F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
        for (uint32_t v = tid; v < n / 4; v += SM_THREADS) {
            const float4 x = reinterpret_cast<const float4*>(l)[v];
            f(x.x, 4 * v), f(x.y, 4 * v + 1), f(x.z, 4 * v + 2), f(x.w, 4 * v + 3);
        }
    }
    // the bin of a logit, SM_BINS for those that weigh nothing: beyond 23 T from the maximum (exp(-23) < 2^-33)
    __device__ __forceinline__ uint32_t bin(float x) const {
        if (x == best) return 0;
        const float d = best - x;
        return d <= cutoff ? min(SM_BINS - 1, (uint32_t)(d * to_bin)) : SM_BINS;
    }
    template <class V>
    __device__ __forceinline__ V& at(V& v, uint32_t r) const { return *cluster.map_shared_rank(&v, r); }

    // sum over the block, to all of its threads
    __device__ __forceinline__ u64 block_sum(u64 v) const {
        v = warp_sum(v);
        __syncthreads();
        if (lane == 0) sh.scan[warp] = v;
        __syncthreads();
        u64 t = 0;
#pragma unroll
        for (uint32_t w = 0; w < SM_WARPS; ++w) t += sh.scan[w];
        return t;
    }
    // sum of this thread's and those in front of it
    __device__ __forceinline__ u64 block_scan(u64 v) const {
        v = warp_scan(v, lane);
        __syncthreads();
        if (lane == 31) sh.scan[warp] = v;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < SM_WARPS; ++w) v += w < warp ? sh.scan[w] : 0;
        return v;
    }
    // number and weight of the tokens at places >= t, over the cluster
    __device__ void count(u64 t, uint32_t* number, u64* sum) const {
        uint32_t c = 0;
        u64 w = 0;
        each([&](float x, uint32_t i) {
            if (bin(x) < SM_BINS && place(i) >= t) ++c, w += weight(likeness(x));
        });
        const u64 c64 = block_sum(c), w64 = block_sum(w);
        cluster.sync();  // what was there has been read
        if (tid == 0) sh.number = (uint32_t)c64, sh.sum = w64;
        cluster.sync();
        *number = warp_sum(lane < ctas ? at(sh.number, lane) : 0u), *sum = warp_sum(lane < ctas ? at(sh.sum, lane) : 0ull);
    }

    // The bin in which the running number of the tokens at places >= from reaches k, or (top_p < 1) their running weight what
    // top-p keeps; what stands in front of the bin.  target: that number or weight.  in_bin: by number, how many tokens the bin
    // holds, and what stands in front of every bin is in CTA 0's bins.high.  False where there are fewer than k tokens; in_bin:
    // how many.
    // first: no call before, bins.high is zero everywhere.
    __device__ bool border_bin(bool first, uint32_t k, float top_p, u64 from, uint32_t* border, u64* before, uint32_t* in_bin, u64* target_out) const {
        const bool by_weight = top_p < 1.0f;
        for (uint32_t i = tid; i < SM_BINS; i += SM_THREADS) {
            if (by_weight) sh.bins.low[i] = sh.bins.high[i] = 0; else sh.bins.number[i] = 0;
        }
        if (tid == 0) sh.n_few = 0;
        __syncthreads();
        each([&](float x, uint32_t i) {
            const uint32_t b = bin(x);
            if (b >= SM_BINS || (from != 0 && place(i) < from)) return;
            if (by_weight) {  // at most 49152 tokens: both halves' sums stay below 2^32
                const u64 w = weight(likeness(x));
                atomicAdd(&sh.bins.low[b], (uint32_t)(w & 0xFFFF)), atomicAdd(&sh.bins.high[b], (uint32_t)(w >> 16));
            } else {
                atomicAdd(&sh.bins.number[b], 1);
            }
        });
        // a run of bins a CTA, a bin (of few CTAs: two, or four) a thread
        const uint32_t run = SM_BINS / ctas, b0 = rank * run;
        constexpr uint32_t MOST = SM_BINS / SM_THREADS;
        const uint32_t per = run >= SM_THREADS ? run / SM_THREADS : 1;
        const bool sent = first && !by_weight && ctas > 1;
        if (sent) {  // numbers to the CTAs that have the bins
            __syncthreads();
#pragma unroll
            for (uint32_t j = 0; j < MOST; ++j) {
                const uint32_t b = tid + j * SM_THREADS, n_bin = sh.bins.number[b];
                if (n_bin) atomicAdd(&at(sh.bins.high[b % run], b / run), n_bin);
            }
        }
        cluster.sync();
        u64 value[MOST], mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < MOST; ++j) {
            const uint32_t b = tid * per + j;
            value[j] = 0;
            if (j < per && b < run) {
                if (sent) {
                    value[j] = sh.bins.high[b];
                } else {
#pragma unroll 8
                    for (uint32_t r = 0; r < ctas; ++r)
                        value[j] += by_weight ? at(sh.bins.low[b0 + b], r) + ((u64)at(sh.bins.high[b0 + b], r) << 16) : at(sh.bins.number[b0 + b], r);
                }
            }
            mine += value[j];
        }
        u64 sum = warp_scan(mine, lane);
        __syncthreads();
        if (lane == 31) sh.scan[warp] = sum;
        __syncthreads();
        u64 all = 0, front = 0;
#pragma unroll
        for (uint32_t w = 0; w < SM_WARPS; ++w) front += w < warp ? sh.scan[w] : 0, all += sh.scan[w];
        sum += front;
        if (tid < ctas) at(sh.part[rank], tid) = all;
        cluster.sync();
        const u64 part = lane < ctas ? sh.part[lane] : 0;
        const u64 ahead = warp_sum(lane < rank ? part : 0), whole = warp_sum(part);
        const u64 target = by_weight ? most_of(top_p, whole) : k;
        *target_out = target;
        u64 upto = ahead + sum - mine;
        const bool fewer = whole < target;  // the same everywhere
#pragma unroll
        for (uint32_t j = 0; j < MOST; ++j) {
            const uint32_t b = tid * per + j;
            if (upto < target && upto + value[j] >= target) {  // one thread of one CTA
                for (uint32_t r = 0; r < ctas; ++r) at(sh.bin, r) = b0 + b, at(sh.before, r) = upto, at(sh.number, r) = (uint32_t)value[j];
            }
            if (!by_weight && j < per && b < run) at(sh.bins.high[b0 + b], 0) = (uint32_t)upto;
            upto += value[j];
        }
        cluster.sync();
        *border = fewer ? SM_BINS - 1 : sh.bin, *before = fewer ? 0 : sh.before, *in_bin = fewer ? (uint32_t)whole : sh.number;
        return !fewer;
    }
    // Behind border_bin: the places >= from of bins first .. last in CTA 0's list, and their number in all CTAs; of more than
    // SM_FEW, nothing else.  Every CTA has a share of the list; where one has more than that, the lists are fetched instead and
    // follow one another (few_of[0]: all of them, the others: 0).
    __device__ uint32_t gather(uint32_t first, uint32_t last, u64 from) const {
        const uint32_t share = SM_FEW / ctas;
        auto collect = [&] {  // (the histograms have been read in front of the last barrier)
            each([&](float x, uint32_t i) {
                const uint32_t b = bin(x);
                if (b < first || b > last) return;
                const u64 p = place(i);
                if (p < from) return;
                const uint32_t to = atomicAdd(&sh.n_few, 1);
                if (to < SM_FEW) sh.few[to] = p;
            });
            __syncthreads();
            return sh.n_few;
        };
        const uint32_t mine = collect();
        if (tid < ctas) at(sh.few_of[rank], tid) = mine;
        if (rank != 0 && mine <= share)
            for (uint32_t i = tid; i < mine; i += SM_THREADS) at(sh.few[rank * share + i], 0) = sh.few[i];
        cluster.sync();
        const uint32_t n_of = lane < ctas ? sh.few_of[lane] : 0, upto = warp_scan(n_of, lane), m = __shfl_sync(0xFFFFFFFFu, upto, 31);
        if (m > SM_FEW || __all_sync(0xFFFFFFFFu, n_of <= share)) return m;  // the same everywhere
        if (rank == 0) {
            __syncthreads();
            if (tid == 0) sh.n_few = 0;
            __syncthreads();
            collect();  // others have written over the end of its list
            for (uint32_t r = 1 + warp; r < ctas; r += SM_WARPS) {  // a warp a list
                const uint32_t more = __shfl_sync(0xFFFFFFFFu, n_of, r), to = __shfl_sync(0xFFFFFFFFu, upto, r) - more;
                const u64* list = cluster.map_shared_rank(sh.few, r);
                for (uint32_t i = lane; i < more; i += 32) sh.few[to + i] = list[i];
            }
            __syncthreads();
            if (tid < ctas) sh.few_of[tid] = tid == 0 ? m : 0;
        }
        cluster.sync();
        return m;
    }
    static constexpr uint32_t PER = SM_FEW / SM_THREADS, RUN = 256;
    // The m places of this CTA's list, the largest first.  In bins: each goes behind what bins.high says stands in front of its
    // bin, then behind the larger ones of the bin.  All of one bin: behind the larger ones.  Where more than RUN have to be
    // compared with one another: a bitonic sort.
    __device__ void order(uint32_t m, bool in_bins) const {
        u64 p[PER];  // 0: none
        uint32_t b[PER];
        bool long_run = false;
        __syncthreads();
        const bool dense = sh.few_of[0] == m;
        const uint32_t share = SM_FEW / ctas;
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t i = tid + j * SM_THREADS;
            const bool is = dense ? i < m : i % share < sh.few_of[i / share];
            p[j] = is ? sh.few[i] : 0, b[j] = is ? bin(logit(p[j])) : 0;
        }
        if (tid == 0) sh.n_few = 0;
        __syncthreads();
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j)
            if (p[j]) sh.few[atomicAdd(in_bins ? &sh.bins.high[b[j]] : &sh.n_few, 1)] = p[j];
        __syncthreads();
        uint32_t to[PER];
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j) {
            const uint32_t first = in_bins && b[j] ? sh.bins.high[b[j] - 1] : 0, last = in_bins ? sh.bins.high[b[j]] : m;
            to[j] = first;
            if (!p[j]) continue;
            long_run |= last - first > RUN;
            if (last - first <= RUN)
                for (uint32_t x = first; x < last; ++x) to[j] += sh.few[x] > p[j];
        }
        if (__syncthreads_or(long_run)) {
            sort(m);
            return;
        }
#pragma unroll
        for (uint32_t j = 0; j < PER; ++j)
            if (p[j]) sh.few[to[j]] = p[j];
        __syncthreads();
    }
    // The same by a bitonic sort; the steps up to 32 apart stay within a warp's 64 places.
    __device__ void sort(uint32_t m) const {
        uint32_t size = 64;
        while (size < m) size *= 2;
        for (uint32_t i = m + tid; i < size; i += SM_THREADS) sh.few[i] = 0;
        for (uint32_t run = 2; run <= size; run *= 2)
            for (uint32_t gap = run / 2; gap > 0; gap /= 2) {
                if (gap >= 32 || run == 2) __syncthreads(); else __syncwarp();
                for (uint32_t t = tid; t < size / 2; t += SM_THREADS) {
                    const uint32_t i = 2 * t - (t & (gap - 1)), j = i + gap;
                    const u64 x = sh.few[i], y = sh.few[j];
                    if ((x < y) == ((i & run) == 0)) sh.few[i] = y, sh.few[j] = x;
                }
            }
        __syncthreads();
    }
    // The place of the last token that a rule keeps of those at places >= from: the first k, or (top_p < 1) top-p's.
    __device__ u64 border_place(bool first, uint32_t k, float top_p, u64 from) const {
        const bool by_weight = top_p < 1.0f;
        uint32_t b, in_bin;
        u64 before, target;
        if (!border_bin(first, k, top_p, from, &b, &before, &in_bin, &target)) return from;
        const uint32_t m = gather(b, b, from);
        if (m <= SM_FEW) {
            if (rank == 0) {
                order(m, false);
                u64 w[PER], mine = 0;
#pragma unroll
                for (uint32_t j = 0; j < PER; ++j) {
                    const uint32_t i = tid * PER + j;
                    w[j] = i >= m ? 0 : by_weight ? weight(likeness(logit(sh.few[i]))) : 1;
                    mine += w[j];
                }
                u64 ahead = before + block_scan(mine) - mine;
#pragma unroll
                for (uint32_t j = 0; j < PER; ++j) {
                    if (ahead < target && ahead + w[j] >= target)
                        for (uint32_t r = 0; r < ctas; ++r) at(sh.border, r) = sh.few[tid * PER + j];
                    ahead += w[j];
                }
            }
            cluster.sync();
            return sh.border;
        }
        u64 t = 0;
        for (int bit = 63; bit >= 0; --bit) {
            uint32_t c;
            u64 w;
            count(max(from, t | 1ull << bit), &c, &w);
            if ((by_weight ? w : c) >= target) t |= 1ull << bit;
        }
        return max(from, t);
    }
};

__device__ __forceinline__ void give(const SampleArgs& a, uint32_t row, int32_t token, float prob) {
    a.token[row] = token;
    if (a.prob) a.prob[row] = prob;
    if (a.pos) a.pos[row] += 1;
    if (token < 0 || !a.window) return;
    // the sampled id takes the oldest one's place
    const int32_t have = a.window_state[2 * row], raw = a.window_state[2 * row + 1];
    const int32_t next = raw < 0 || raw >= (int32_t)SM_WINDOW ? 0 : raw;
    a.window[(uint64_t)row * SM_WINDOW + next] = token;
    a.window_state[2 * row] = min(max(have, 0) + 1, (int32_t)SM_WINDOW);
    a.window_state[2 * row + 1] = (next + 1) % (int32_t)SM_WINDOW;
}

__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(SampleArgs a) {
    extern __shared__ __align__(16) float s_l[];  // this CTA's logits
    __shared__ SampleShared sh;
    pdl_trigger_all();
    cg::cluster_group cluster = cg::this_cluster();
    cluster.barrier_arrive();  // others' shared memory may be written once they have begun
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.y;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    for (uint32_t i = tid; i < SM_BINS; i += SM_THREADS) sh.bins.high[i] = 0;
    // the row's rules, on their way with its logits
    const float given = a.temperature ? a.temperature[row] : 1.0f, temp = given > 3e38f ? 3e38f : given;  // NaN stays
    const float top_p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f, u = a.uniform[row];
    const int32_t wanted_k = a.top_k ? a.top_k[row] : 0;
    // slices end where the row's 16-byte vectors do; a vector that is not the row's throughout is read by its own logits
    const float* src = a.logits + row * a.stride;
    const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(src) / 4 % 4), vecs = (shift + a.vocab + 3) / 4;
    const uint32_t per = (vecs + ctas - 1) / ctas, v0 = min(vecs, rank * per), n = 4 * (min(vecs, v0 + per) - v0);
    const int32_t lo = (int32_t)(4 * v0) - (int32_t)shift;
    src += lo;
    float best = -INFINITY, least = INFINITY;
    auto see = [&](float v) {  // NaN is passed over
        best = fmaxf(best, v);
        if (v > -INFINITY) least = fminf(least, v);
    };
    constexpr uint32_t AHEAD = 4;
    for (uint32_t v = tid; v < n / 4; v += AHEAD * SM_THREADS) {
        float4 x[AHEAD];
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) {
            const uint32_t at = v + j * SM_THREADS;
            const int32_t id = lo + 4 * (int32_t)at;
            if (at < n / 4 && id >= 0 && id + 4 <= (int32_t)a.vocab) {
                x[j] = ld_once(src + 4 * (uint64_t)at);
            } else {
                float* e = &x[j].x;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    e[k] = at < n / 4 && id + k >= 0 && id + k < (int32_t)a.vocab ? src[4 * (int32_t)at + k] : NAN;
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < AHEAD; ++j) {
            if (v + j * SM_THREADS < n / 4) reinterpret_cast<float4*>(s_l)[v + j * SM_THREADS] = x[j];
            see(x[j].x), see(x[j].y), see(x[j].z), see(x[j].w);
        }
    }
    // the repetition penalty, on the copy: once for every occurrence in the recent window, by the thread of the first one
    const uint32_t held = a.window && a.penalty != 1.0f ? min((uint32_t)max(a.window_state[2 * row], 0), SM_WINDOW) : 0;
    if (held) {
        if (tid < held) sh.window[tid] = a.window[(uint64_t)row * SM_WINDOW + tid];
        __syncthreads();
        if (tid < held) {
            const int32_t tok = sh.window[tid];
            bool first = tok >= max(lo, 0) && tok < min(lo + (int32_t)n, (int32_t)a.vocab);
            uint32_t times = 0;
            for (uint32_t j = 0; j < held; ++j)
                if (sh.window[j] == tok) first &= j >= tid, ++times;
            if (first) {
                float v = s_l[tok - lo];
                for (uint32_t j = 0; j < times; ++j) v = v > 0.0f ? v / a.penalty : v * a.penalty;
                s_l[tok - lo] = v;
            }
        }
        __syncthreads();
        best = -INFINITY, least = INFINITY;
        for (uint32_t j = tid; j < n; j += SM_THREADS) see(s_l[j]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
        least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, o));
    }
    if (lane == 0) sh.red[0][warp] = best, sh.red[1][warp] = least;
    __syncthreads();
    auto reduce = [&](float x, float y) {
        best = x, least = y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
            least = fminf(least, __shfl_xor_sync(0xFFFFFFFFu, least, o));
        }
    };
    cluster.barrier_wait();
    if (warp == 0) {
        reduce(lane < SM_WARPS ? sh.red[0][lane] : -INFINITY, lane < SM_WARPS ? sh.red[1][lane] : INFINITY);
        if (lane < ctas) *cluster.map_shared_rank(&sh.best[rank], lane) = best, *cluster.map_shared_rank(&sh.least[rank], lane) = least;
    }
    cluster.sync();
    reduce(lane < ctas ? sh.best[lane] : -INFINITY, lane < ctas ? sh.least[lane] : INFINITY);
    if (!(best > -INFINITY)) {  // nothing to draw: the same in the whole cluster
        if (rank == 0 && tid == 0) give(a, row, -1, 0.0f);
        cluster.sync();
        return;
    }
    const bool greedy = !(temp > 0.0f);
    const uint32_t top_k = greedy ? 1u : (uint32_t)max(wanted_k, 0);
    const float cutoff = greedy ? 0.0f : 23.0f * temp;
    Row r{cluster, sh, s_l, lo, n, ctas, rank, tid, warp, lane, best, temp, cutoff, (float)SM_BINS / fminf(best - least, cutoff), greedy};

    u64 from = 0, total = 0;
    uint32_t border, in_bin;
    u64 before, target;
    if (top_k != 0 && top_k <= SM_FEW) {
        const bool cut = r.border_bin(true, top_k, 1.0f, 0, &border, &before, &in_bin, &target);
        // all tokens down to the bin of the last one kept (or all there are)
        if (before + in_bin <= SM_FEW) {
            const uint32_t m = r.gather(0, border, 0);
            if (rank == 0) {
                r.order(m, true);
                constexpr uint32_t PER = Row::PER;  // tokens PER tid .. of the order
                u64 w[PER], sum = 0;
                uint32_t id[PER];
#pragma unroll
                for (uint32_t j = 0; j < PER; ++j) {
                    const uint32_t at = tid * PER + j;
                    const u64 place = at < min(m, top_k) ? sh.few[at] : 0;
                    const float e = place ? r.likeness(Row::logit(place)) : 0.0f;
                    w[j] = Row::weight(e), id[j] = 0xFFFFFFFFu - (uint32_t)place;
                    sum += w[j];
                }
                u64 ahead = r.block_scan(sum) - sum;
                total = r.block_sum(sum);
                const u64 most = top_p < 1.0f ? most_of(top_p, total) : total;
                sum = 0;
#pragma unroll
                for (uint32_t j = 0; j < PER; ++j) {
                    const u64 mine = w[j];
                    if (ahead >= most || (min_p > 0.0f && mine && !(r.likeness(Row::logit(sh.few[tid * PER + j])) >= min_p))) w[j] = 0;
                    ahead += mine, sum += w[j];
                }
                total = r.block_sum(sum);
                const u64 draw = draw_of(u, total);
                // The first id at which the kept weights, in order of ids, pass the draw: among runs of ids (a thread a run), then
                // among the tokens of the run that it falls into.
                u64* weight_of = reinterpret_cast<u64*>(sh.bins.high);  // of a run; behind them, a run's tokens
                Token* tokens = reinterpret_cast<Token*>(weight_of + SM_THREADS);
                constexpr uint32_t MOST = (sizeof(sh.bins.high) - SM_THREADS * 8) / sizeof(Token);
                const uint32_t width = (a.vocab + SM_THREADS - 1) / SM_THREADS;
                weight_of[tid] = 0;
                if (tid == 0) sh.n_few = 0;
                __syncthreads();
#pragma unroll
                for (uint32_t j = 0; j < PER; ++j)
                    if (w[j]) atomicAdd(&weight_of[id[j] / width], w[j]);
                __syncthreads();
                const u64 upto = r.block_scan(weight_of[tid]);
                if (upto > draw && upto - weight_of[tid] <= draw) sh.bin = tid, sh.before = upto - weight_of[tid];
                __syncthreads();
#pragma unroll
                for (uint32_t j = 0; j < PER; ++j)
                    if (w[j] && id[j] / width == sh.bin) {
                        const uint32_t to = atomicAdd(&sh.n_few, 1);
                        if (to < MOST) tokens[to] = Token{w[j], id[j]};
                    }
                __syncthreads();
                const uint32_t n_run = sh.n_few;
                if (n_run <= MOST) {
                    for (uint32_t i = tid; i < n_run; i += SM_THREADS) {
                        const Token me = tokens[i];
                        u64 below = sh.before;
                        for (uint32_t x = 0; x < n_run; ++x) below += tokens[x].id < me.id ? tokens[x].weight : 0;
                        if (below <= draw && draw < below + me.weight) give(a, row, (int32_t)me.id, (float)((double)me.weight / (double)total));
                    }
                } else {  // bit by bit: the ids below it weigh at most the draw
                    uint32_t below = 0;
                    for (uint32_t bit = 1u << (31 - __clz(a.vocab)); bit != 0; bit >>= 1) {
                        sum = 0;
#pragma unroll
                        for (uint32_t j = 0; j < PER; ++j) sum += id[j] < (below | bit) ? w[j] : 0;
                        if (r.block_sum(sum) <= draw) below |= bit;
                    }
#pragma unroll
                    for (uint32_t j = 0; j < PER; ++j)
                        if (w[j] && id[j] == below) give(a, row, (int32_t)below, (float)((double)w[j] / (double)total));
                }
            }
            return;  // the others' memory was last touched in front of the last barrier
        }
    }
    if (top_k != 0) from = r.border_place(top_k > SM_FEW, top_k, 1.0f, 0);
    if (top_p < 1.0f) from = r.border_place(top_k == 0, 0, top_p, from);
    // the kept weights of this CTA, run by run of ids, a run a warp; as whole numbers in 64-bit floats, exact below 2^53
    const uint32_t seg = (n + SM_WARPS - 1) / SM_WARPS, s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
    auto kept = [&](uint32_t x) -> float {
        if (r.bin(s_l[x]) >= SM_BINS || (from != 0 && r.place(x) < from)) return 0.0f;
        const float e = r.likeness(s_l[x]);
        return e >= min_p ? Row::weight_float(e) : 0.0f;
    };
    double mine = 0.0;
#pragma unroll 2
    for (uint32_t x = s0 + lane; x < s1; x += 32) mine += (double)kept(x);
    const u64 w = (u64)warp_sum(mine);
    __syncthreads();
    if (lane == 0) sh.scan2[warp] = w;
    __syncthreads();
    u64 all = 0;
#pragma unroll
    for (uint32_t x = 0; x < SM_WARPS; ++x) all += sh.scan2[x];
    if (tid < ctas) r.at(sh.part[rank], tid) = all;
    cluster.sync();
    const u64 part = lane < ctas ? sh.part[lane] : 0;
    u64 ahead = warp_sum(lane < rank ? part : 0);
    total = warp_sum(part);
    const u64 draw = draw_of(u, total);
    if (ahead <= draw && draw < ahead + all) {  // one CTA: the run that the draw falls into, then its token by all threads
        uint32_t hit = 0;
        while (ahead + sh.scan2[hit] <= draw) ahead += sh.scan2[hit++];
        const uint32_t t0 = min(n, hit * seg), t1 = min(n, t0 + seg);
        for (uint32_t x = t0; x < t1; x += SM_THREADS) {
            const u64 me = x + tid < t1 ? (u64)kept(x + tid) : 0ull;
            const u64 upto = ahead + r.block_scan(me);
            if (upto > draw && upto - me <= draw) give(a, row, lo + (int32_t)(x + tid), (float)((double)me / (double)total));
            ahead += r.block_sum(me);
        }
    }
    cluster.sync();  // shared memory is read from the others until here
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, uint32_t rows, cudaStream_t s) {
    // 2048 logits a CTA or more (one row of 32000, top-p: 16.5 us, with 4096 18.5), eight CTAs a row; sixteen (beyond what every
    // device promises) while the rows are few: one row of 128256 27 us (eight: 36), 64 rows 84 with eight and 139 with sixteen
    uint32_t ctas = 1;
    while (ctas < (rows * SM_MOST_CTAS <= (uint32_t)num_sms() ? SM_MOST_CTAS : SM_CTAS) && a.vocab > ctas * 2048) ctas *= 2;
    const size_t smem = ((a.vocab + 3 + 3) / 4 + ctas - 1) / ctas * 16;  // of a row that begins inside a vector
    static bool configured[MAX_DEVICES] = {};
    if (cudaError_t e = set_max_smem_once(sample_kernel, SAMPLE_MAX_VOCAB / SM_CTAS * 4 + 16, configured); e != cudaSuccess) return e;
    static bool wide[MAX_DEVICES] = {};
    if (!wide[current_device()]) {
        if (cudaError_t e = cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); e != cudaSuccess) return e;
        wide[current_device()] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, rows);
    cfg.blockDim = dim3(SM_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, a);
    return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace jq
