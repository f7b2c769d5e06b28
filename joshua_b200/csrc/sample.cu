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
// A cluster of CTAs takes a row, each a slice of it in shared memory: the logits are read once.
#include <cooperative_groups.h>

#include "serving.cuh"

namespace jq {

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t SM_THREADS = 512, SM_CTAS = 8, SM_WINDOW = 64;

// Logits as whole numbers of the same order; NaN and -inf come last, as 0.
__device__ __forceinline__ uint32_t logit_key(float l) {
    const uint32_t u = __float_as_uint(l);
    return l > -INFINITY ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}

struct SampleShared {
    float best;
    unsigned long long sum[2], scan[SM_THREADS / 32];
    uint32_t cnt[2], red_cnt[SM_THREADS / 32];
    float red[SM_THREADS / 32];
    int32_t window[SM_WINDOW];
};

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(SampleArgs a) {
    extern __shared__ float s_l[];  // this CTA's logits
    __shared__ SampleShared sh;
    pdl_trigger_all();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t ctas = cluster.num_blocks(), rank = cluster.block_rank(), row = blockIdx.y;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t per = (a.vocab + ctas - 1) / ctas, lo = min(a.vocab, rank * per), n = min(a.vocab, lo + per) - lo;
    const float* src = a.logits + row * a.stride + lo;
    for (uint32_t i = tid; i < n; i += SM_THREADS) s_l[i] = src[i];
    // the repetition penalty, on the copy: once for every occurrence in the recent window, by the thread of the first one
    const uint32_t held = a.window ? min((uint32_t)max(a.window_state[2 * row], 0), SM_WINDOW) : 0;
    if (tid < held) sh.window[tid] = a.window[(uint64_t)row * SM_WINDOW + tid];
    __syncthreads();
    if (tid < held && a.penalty != 1.0f) {
        const int32_t tok = sh.window[tid];
        bool first = tok >= (int32_t)lo && tok < (int32_t)(lo + n);
        uint32_t times = 0;
        for (uint32_t i = 0; i < held; ++i)
            if (sh.window[i] == tok) first &= i >= tid, ++times;
        if (first) {
            float v = s_l[tok - lo];
            for (uint32_t i = 0; i < times; ++i) v = v > 0.0f ? v / a.penalty : v * a.penalty;
            s_l[tok - lo] = v;
        }
    }
    __syncthreads();
    float best = -INFINITY;
    for (uint32_t i = tid; i < n; i += SM_THREADS) best = fmaxf(best, s_l[i]);  // NaN is passed over
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xFFFFFFFFu, best, o));
    if (lane == 0) sh.red[warp] = best;
    __syncthreads();
    if (tid == 0) {
        for (uint32_t w = 1; w < SM_THREADS / 32; ++w) best = fmaxf(best, sh.red[w]);
        sh.best = best;
    }
    cluster.sync();
    best = -INFINITY;
    for (uint32_t r = 0; r < ctas; ++r) best = fmaxf(best, *cluster.map_shared_rank(&sh.best, r));

    const float temp = a.temperature ? a.temperature[row] : 1.0f, top_p = a.top_p ? a.top_p[row] : 1.0f;
    const float min_p = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
    const bool greedy = !(temp > 0.0f);
    const uint32_t top_k = greedy ? 1u : a.top_k ? (uint32_t)max(a.top_k[row], 0) : 0u;
    auto likeness = [&](float l) {  // exp((l - max) / T)
        if (!(l > -INFINITY)) return 0.0f;
        if (l == best) return 1.0f;
        return !greedy ? expf(__fdiv_rn(__fsub_rn(l, best), temp)) : 0.0f;
    };
    auto weight = [&](float e) { return (unsigned long long)__float2ull_rn(e * 4294967296.0f); };
    auto place = [&](uint32_t i) { return (unsigned long long)logit_key(s_l[i]) << 32 | (0xFFFFFFFFu - (lo + i)); };

    // number and weight of the tokens at places >= t, over the cluster
    uint32_t turn = 0;
    auto count = [&](unsigned long long t, uint32_t* number, unsigned long long* sum) {
        uint32_t c = 0;
        unsigned long long w = 0;
        for (uint32_t i = tid; i < n; i += SM_THREADS) {
            const float l = s_l[i], e = likeness(l);
            if (place(i) >= t && e > 0.0f) ++c, w += weight(e);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) c += __shfl_xor_sync(0xFFFFFFFFu, c, o), w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
        if (lane == 0) sh.red_cnt[warp] = c, sh.scan[warp] = w;
        __syncthreads();
        if (tid == 0) {
            for (uint32_t i = 1; i < SM_THREADS / 32; ++i) c += sh.red_cnt[i], w += sh.scan[i];
            sh.cnt[turn & 1] = c, sh.sum[turn & 1] = w;
        }
        cluster.sync();
        *number = 0, *sum = 0;
        for (uint32_t r = 0; r < ctas; ++r) {
            *number += *cluster.map_shared_rank(&sh.cnt[turn & 1], r);
            *sum += *cluster.map_shared_rank(&sh.sum[turn & 1], r);
        }
        ++turn;  // the other pair next: this one may still be read
    };
    uint32_t number;
    unsigned long long total, from = 0;
    count(from, &number, &total);
    if (top_k != 0 && number > top_k) {
        unsigned long long t = 0;
        for (int bit = 63; bit >= 0; --bit) {  // the largest place with top_k tokens from it on
            uint32_t c;
            unsigned long long w;
            count(t | 1ull << bit, &c, &w);
            if (c >= top_k) t |= 1ull << bit;
        }
        from = t;
        count(from, &number, &total);
    }
    if (top_p < 1.0f && total != 0) {
        const double p = (double)top_p * (double)total;
        const unsigned long long most = p >= 1.0 ? (unsigned long long)p : 1ull;
        unsigned long long t = 0;
        for (int bit = 63; bit >= 0; --bit) {  // the largest place with at least `most` from it on
            uint32_t c;
            unsigned long long w;
            count(t | 1ull << bit, &c, &w);
            if (w >= most) t |= 1ull << bit;
        }
        from = max(from, t);
    }
    // the kept weights of this CTA, warp by warp in order of ids
    const uint32_t seg = (n + SM_THREADS / 32 - 1) / (SM_THREADS / 32), s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
    auto kept = [&](uint32_t i) -> unsigned long long {
        const float e = likeness(s_l[i]);
        return place(i) >= from && e >= min_p ? weight(e) : 0ull;
    };
    unsigned long long w = 0;
    for (uint32_t i = s0 + lane; i < s1; i += 32) w += kept(i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xFFFFFFFFu, w, o);
    __syncthreads();
    if (lane == 0) sh.scan[warp] = w;
    __syncthreads();
    if (tid == 0) {
        unsigned long long all = 0;
        for (uint32_t i = 0; i < SM_THREADS / 32; ++i) all += sh.scan[i];
        sh.sum[turn & 1] = all;
    }
    cluster.sync();
    unsigned long long before = 0, all = 0;
    for (uint32_t r = 0; r < ctas; ++r) {
        const unsigned long long x = *cluster.map_shared_rank(&sh.sum[turn & 1], r);
        before += r < rank ? x : 0, all += x;
    }
    const double at = (double)a.uniform[row] * (double)all;
    unsigned long long r = at >= 1.0 ? (unsigned long long)at : 0ull;
    r = all != 0 && r >= all ? all - 1 : r;
    int32_t token = -1;
    if (all == 0) {
        if (rank == 0 && tid == 0) {
            a.token[row] = -1;
            if (a.prob) a.prob[row] = 0.0f;
        }
    } else {
        for (uint32_t i = 0; i < warp; ++i) before += sh.scan[i];
        if (before <= r && r < before + w) {  // one warp of one CTA
            for (uint32_t i = s0; i < s1; i += 32) {
                const unsigned long long mine = i + lane < s1 ? kept(i + lane) : 0ull;
                unsigned long long run = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long up = __shfl_up_sync(0xFFFFFFFFu, run, o);
                    run += lane >= o ? up : 0;
                }
                const uint32_t past = __ballot_sync(0xFFFFFFFFu, before + run > r);
                if (past) {
                    if (lane == __ffs(past) - 1) {
                        token = (int32_t)(lo + i + lane);
                        a.token[row] = token;
                        if (a.prob) a.prob[row] = (float)((double)mine / (double)all);
                    }
                    break;
                }
                before += __shfl_sync(0xFFFFFFFFu, run, 31);
            }
        }
    }
    if (token >= 0 && a.window) {  // the sampled id takes the oldest one's place
        const int32_t have = a.window_state[2 * row], raw = a.window_state[2 * row + 1];
        const int32_t next = raw < 0 || raw >= (int32_t)SM_WINDOW ? 0 : raw;
        a.window[(uint64_t)row * SM_WINDOW + next] = token;
        a.window_state[2 * row] = min(max(have, 0) + 1, (int32_t)SM_WINDOW);
        a.window_state[2 * row + 1] = (next + 1) % (int32_t)SM_WINDOW;
    }
    if (a.pos && rank == 0 && tid == 0) a.pos[row] += 1;
    cluster.sync();  // shared memory is read from the others until here
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, uint32_t rows, cudaStream_t s) {
    uint32_t ctas = 1;
    while (ctas < SM_CTAS && a.vocab > ctas * 4096) ctas *= 2;
    const size_t smem = (size_t)((a.vocab + ctas - 1) / ctas) * 4;
    static bool configured[MAX_DEVICES] = {};
    if (cudaError_t e = set_max_smem_once(sample_kernel, SAMPLE_MAX_VOCAB / SM_CTAS * 4, configured); e != cudaSuccess) return e;
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
