// sepia_b200/csrc/sample.cu -- one token per row of logits by temperature,
// top-k, top-p and min-p from one given uniform number (sepia_cuda_sample;
// definition in include/sepia_cuda.h).
//
// Each filter keeps a prefix of one order (greater logit first, then lower
// index), so a row's set is described by a cut: the last token in. Weights
// are integers: counts and masses are sums that no order of summation changes.
//
// The logits cross HBM once: a cluster of up to 8 CTAs holds a row in shared
// memory, and all passes run there. A cut is found by a histogram over
// (max - l)/T with linear bins (logits spread over them, so that few lanes
// meet in one counter), whose threshold bin is gathered and sorted by the
// cluster's first CTA. A bin that is too full for that (runs of equal logits)
// is cut by halving the range of keys, 32 passes.
#include "../../include/sepia_cuda.h"
#include "common.cuh"
#include "runtime.h"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace sepia {

constexpr int kSmThreads = 512;
constexpr int kSmBins = 1024;                // two per thread
constexpr int kSmList = 1024;                // tokens of a threshold bin that are sorted
constexpr int kSmMaxCluster = 8;
constexpr float kSmRange = 22.25f;           // beyond exp(-this) a weight rounds to 0
constexpr float kSmOne = 2147483648.0f;      // weight of the best token: 2^31
// 65536 logits a CTA: a bin's sums of 16-bit halves fit 32 bits, the row's mass is exact in fp64
constexpr int32_t kSmMaxVocab = 1 << 19;

typedef unsigned long long u64;

struct SmParams {
    const void *logits;
    int64_t stride;
    int32_t vocab, slice;                    // slice: logits of a CTA, a multiple of 16
    int32_t held;                            // the slice fits in shared memory
    const float *u, *temperature, *top_p, *min_p;
    const int32_t *top_k;
    int32_t *ids;
    float *prob;
};

// Order-preserving key of a logit; NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t sm_key(float v) {
    if (v != v) v = -INFINITY;
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float sm_unkey(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// e = exp((l - max)/T); the best token's is 1 also where max is infinite
__device__ __forceinline__ float sm_exp(float l, float best, float inv_t) {
    return l == best ? 1.0f : expf((l - best) * inv_t);
}
__device__ __forceinline__ u64 sm_weight(float e) { return (u64)__float2uint_rn(e * kSmOne); }

// The last token in
struct SmCut {
    float l;
    int idx;
};

struct SmShared {
    union {                                  // the list is filled when the bins have been read
        uint32_t hist[2][kSmBins];           // counts, or masses as sums of low and high 16 bits
        u64 list[kSmList];                   // key, complement of the index
    };
    float best[kSmMaxCluster];
    int best_idx[kSmMaxCluster];
    u64 sums[2][kSmMaxCluster], warp[kSmThreads / 32];
    int first_idx;
    u64 found_before;                        // count or mass of the bins above the threshold bin
    double thr;
    int bin, n_list;                         // bin: -1 no cut; n_list may pass kSmList
    SmCut cut;
};

__device__ u64 sm_block_sum(u64 v, u64 *sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    v = lane < kSmThreads / 32 ? sh[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// Sum over the threads before this one.
__device__ u64 sm_block_before(u64 v, u64 *sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += t;
    }
    __syncthreads();
    if (lane == 31) sh[warp] = x;
    __syncthreads();
    u64 w = lane < warp && lane < kSmThreads / 32 ? sh[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    return w + x - v;
}

// f(logit, index in the row) for every logit of the slice, 16 bytes a load
// where the pointer allows. x: first logit of the slice, n of them from i0.
template <typename T, typename F>
__device__ __forceinline__ void sm_each(const T *x, int n, int i0, F f) {
    constexpr int E = 16 / (int)sizeof(T);
    const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    const int body = (n - head) / E;
    for (int i = threadIdx.x; i < body; i += kSmThreads) {
        const uint4 raw = *reinterpret_cast<const uint4 *>(x + head + i * E);
        const T *v = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int e = 0; e < E; e++) f((float)v[e], i0 + head + i * E + e);
    }
    const int rest = head + n - (head + body * E);     // before and after the aligned part
    if ((int)threadIdx.x < rest) {
        const int i = (int)threadIdx.x < head ? (int)threadIdx.x : body * E + (int)threadIdx.x;
        f((float)x[i], i0 + i);
    }
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads, 2) k_sample(const SmParams P) {
    extern __shared__ __align__(16) uint8_t sm_raw[];
    __shared__ SmShared S;
    cg::cluster_group cl = cg::this_cluster();
    const int C = cl.num_blocks(), rank = cl.block_rank();
    const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, V = P.vocab;
    SmShared *first = cl.map_shared_rank(&S, 0);
    griddep_wait();
    griddep_launch();
    const int i0 = min(V, rank * P.slice), n = min(V, i0 + P.slice) - i0;
    const T *gx = (const T *)P.logits + (int64_t)row * P.stride + i0;
    // the slice in shared memory keeps the row's place between 16-byte boundaries
    T *hx = reinterpret_cast<T *>(sm_raw + (reinterpret_cast<uintptr_t>(gx) & 15));
    const T *x = P.held ? hx : gx;
    const float t = P.temperature ? P.temperature[row] : 1.0f;
    const int k = P.top_k ? P.top_k[row] : 0;
    const float p = P.top_p ? P.top_p[row] : 1.0f;
    const float mp = P.min_p && P.min_p[row] > 0.0f ? fminf(P.min_p[row], 1.0f) : 0.0f, u = P.u[row];

    // ---- the row into shared memory; its greatest logit ----
    float top = -INFINITY;                             // NaN loses every fmaxf
    {
        constexpr int E = 16 / (int)sizeof(T), kAhead = 8;
        const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(gx) & 15)) & 15) / (int)sizeof(T));
        const int body = (n - head) / E;
        for (int i = tid; i < body; i += kAhead * kSmThreads) {
            uint4 raw[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; a++)
                raw[a] = __ldg(reinterpret_cast<const uint4 *>(gx + head + min(i + a * kSmThreads, body - 1) * E));
#pragma unroll
            for (int a = 0; a < kAhead; a++) {
                const int j = min(i + a * kSmThreads, body - 1);
                if (P.held) *reinterpret_cast<uint4 *>(hx + head + j * E) = raw[a];
                const T *v = reinterpret_cast<const T *>(&raw[a]);
#pragma unroll
                for (int e = 0; e < E; e++) top = fmaxf(top, (float)v[e]);
            }
        }
        const int rest = n - body * E;
        if (tid < rest) {
            const int i = tid < head ? tid : body * E + tid;
            const T v = gx[i];
            if (P.held) hx[i] = v;
            top = fmaxf(top, (float)v);
        }
    }
    top = warp_max(top);
    if (lane == 0) reinterpret_cast<float *>(S.warp)[tid >> 5] = top;
    if (tid == 0) S.first_idx = INT32_MAX;
    __syncthreads();
    if (tid < C) {
        for (int w = 0; w < kSmThreads / 32; w++) top = fmaxf(top, reinterpret_cast<float *>(S.warp)[w]);
        cl.map_shared_rank(&S, tid)->best[rank] = top;
    }
    cl.sync();
    top = S.best[0];
    for (int r = 1; r < C; r++) top = fmaxf(top, S.best[r]);
    if (top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            P.ids[row] = -1;
            if (P.prob) P.prob[row] = 0.0f;
        }
        return;
    }
    auto first_best = [&]() {                          // the lowest index of the greatest logit
        sm_each(x, n, i0, [&](float l, int i) {
            if (l == top) atomicMin(&S.first_idx, i);
        });
        __syncthreads();
        if (tid < C) cl.map_shared_rank(&S, tid)->best_idx[rank] = S.first_idx;
        cl.sync();
        int i = S.best_idx[0];
        for (int r = 1; r < C; r++) i = min(i, S.best_idx[r]);
        return i;
    };
    if (!(t > 0.0f)) {
        const int i = first_best();
        if (rank == 0 && tid == 0) {
            P.ids[row] = i;
            if (P.prob) P.prob[row] = 1.0f;
        }
        return;
    }
    const float inv_t = __fdiv_rn(1.0f, t);

    // ---- sums over the whole row: every CTA tells all ----
    int turn = 0;
    auto cluster_sum = [&](u64 v, u64 *mine_before) {
        const u64 s = sm_block_sum(v, S.warp);
        if (tid < C) cl.map_shared_rank(&S, tid)->sums[turn][rank] = s;
        cl.sync();
        u64 all = 0, before = 0;
        for (int r = 0; r < C; r++) {
            before += r < rank ? S.sums[turn][r] : 0;
            all += S.sums[turn][r];
        }
        turn ^= 1;                                     // the next sum must not overwrite what is still read
        if (mine_before) *mine_before = before;
        return all;
    };
    // Below this a weight rounds to 0: rounding of the bound itself cannot
    // pass a logit at less than the range (both are fp32 numbers).
    const float floor_l = top - kSmRange * t;
    SmCut cut = {floor_l, INT32_MAX};                  // tokens in: l > cut.l, or l == cut.l up to an index
    // The cut at the token where the running count (of the order) reaches
    // `want`, or the running mass reaches `want` times the mass of the tokens
    // that are in. range: tokens with (max - l)/T beyond it cannot be the
    // cut; their mass still counts.
    auto find_cut = [&](bool mass, double want, float range) {
        const float per = kSmBins / range, near = range < kSmRange ? fmaxf(cut.l, top - range * t) : cut.l;
        for (int i = tid; i < 2 * kSmBins; i += kSmThreads) (&S.hist[0][0])[i] = 0;
        if (tid == 0) S.n_list = 0;
        __syncthreads();
        u64 beyond = 0;
        auto bin_of = [&](float l) { return min(kSmBins - 1, (int)((top - l) * inv_t * per)); };   // inf - inf: 0
        sm_each(x, n, i0, [&](float l, int i) {
            if (!(l >= cut.l) || (l == cut.l && i > cut.idx)) return;
            if (!mass) {
                atomicAdd(&S.hist[0][bin_of(l)], 1u);
                return;
            }
            const uint32_t w = (uint32_t)sm_weight(sm_exp(l, top, inv_t));
            if (l >= near) {
                const int b = bin_of(l);
                atomicAdd(&S.hist[0][b], w & 0xffffu);
                atomicAdd(&S.hist[1][b], w >> 16);
            } else {
                beyond += w;
            }
        });
        const u64 far_mass = mass ? cluster_sum(beyond, nullptr) : 0;
        if (!mass) cl.sync();
        if (rank == 0) {                               // the threshold bin
            u64 v[2] = {0, 0};
            for (int r = 0; r < C; r++) {
                const SmShared *q = cl.map_shared_rank(&S, r);
#pragma unroll
                for (int e = 0; e < 2; e++)
                    v[e] += (u64)q->hist[0][2 * tid + e] + (mass ? (u64)q->hist[1][2 * tid + e] << 16 : 0);
            }
            const u64 before = sm_block_before(v[0] + v[1], S.warp);
            const u64 all = sm_block_sum(v[0] + v[1], S.warp);
            const double thr = mass ? want * (double)(all + far_mass) : want;
            if (tid == 0) S.bin = -1, S.thr = thr;
            __syncthreads();
            u64 b = before;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if ((double)b < thr && (double)(b + v[e]) >= thr) S.bin = 2 * tid + e, S.found_before = b;
                b += v[e];
            }
            __syncthreads();
            if (tid > 0 && tid < C) {
                SmShared *q = cl.map_shared_rank(&S, tid);
                q->bin = S.bin;
                q->thr = S.thr;
                q->found_before = S.found_before;
            }
        }
        cl.sync();
        const int bin = S.bin;
        if (bin < 0) return;                           // a count past all tokens of any weight: nothing to cut
        // its tokens to the first CTA; a bound of half a bin more spares most of them the bin's arithmetic
        const float bin_lo = fmaxf(near, top - ((float)bin + 1.5f) / per * t), bin_hi = top - ((float)bin - 0.5f) / per * t;
        sm_each(x, n, i0, [&](float l, int i) {
            if (!(l >= bin_lo && (l <= bin_hi || bin == 0)) || bin_of(l) != bin || (l == cut.l && i > cut.idx)) return;
            const int at = atomicAdd(&first->n_list, 1);
            if (at < kSmList) first->list[at] = ((u64)sm_key(l) << 32) | (0xffffffffu - (uint32_t)i);
        });
        cl.sync();
        const int have = first->n_list;
        const double thr = S.thr;
        const u64 above = S.found_before;
        if (have <= kSmList) {
            if (rank == 0) {                           // sorted by the order, then summed
                int m = 2;
                while (m < have) m <<= 1;
                for (int i = have + tid; i < m; i += kSmThreads) S.list[i] = 0;
                __syncthreads();
                for (int size = 2; size <= m; size <<= 1)
                    for (int step = size >> 1; step > 0; step >>= 1) {
                        for (int i = tid; i < m / 2; i += kSmThreads) {
                            const int a = 2 * i - (i & (step - 1)), b = a + step;
                            const u64 va = S.list[a], vb = S.list[b];
                            if ((va < vb) == ((a & size) == 0)) S.list[a] = vb, S.list[b] = va;
                        }
                        __syncthreads();
                    }
                u64 v[2] = {0, 0};
#pragma unroll
                for (int e = 0; e < 2; e++)
                    if (2 * tid + e < have)
                        v[e] = mass ? sm_weight(sm_exp(sm_unkey((uint32_t)(S.list[2 * tid + e] >> 32)), top, inv_t)) : 1;
                u64 b = above + sm_block_before(v[0] + v[1], S.warp);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    if ((double)b < thr && (double)(b + v[e]) >= thr) {
                        const u64 y = S.list[2 * tid + e];
                        S.cut.l = sm_unkey((uint32_t)(y >> 32));
                        S.cut.idx = (int)(0xffffffffu - (uint32_t)y);
                    }
                    b += v[e];
                }
                __syncthreads();
                if (tid > 0 && tid < C) cl.map_shared_rank(&S, tid)->cut = S.cut;
            }
            cl.sync();
            cut = S.cut;
            return;
        }
        // Too many for the list: the greatest key whose tokens and those above
        // reach the threshold, bit by bit; then how many tokens of that very
        // key are in, and the index of the last of them.
        auto sum_ge = [&](uint32_t key, bool indexes, uint32_t upto) {
            u64 s = 0;
            sm_each(x, n, i0, [&](float l, int i) {
                if (!(l >= cut.l) || (l == cut.l && i > cut.idx)) return;
                const uint32_t y = sm_key(l);
                if (indexes ? y == key && (uint32_t)i <= upto : y >= key)
                    s += mass && !indexes ? sm_weight(sm_exp(l, top, inv_t)) : 1;
            });
            return cluster_sum(s, nullptr);
        };
        uint32_t key = 0;
        for (int b = 31; b >= 0; b--)
            if ((double)sum_ge(key | (1u << b), false, 0) >= thr) key |= 1u << b;
        const u64 over = sum_ge(key + 1, false, 0), w = mass ? sm_weight(sm_exp(sm_unkey(key), top, inv_t)) : 1;
        u64 r = (u64)((thr - (double)over) / (double)w);
        while (r > 0 && (double)(over + (r - 1) * w) >= thr) r--;
        while ((double)(over + r * w) < thr) r++;
        uint32_t lo = 0, hi = (uint32_t)V - 1;         // the smallest index that has r of them up to it
        while (lo < hi) {
            const uint32_t mid = lo + (hi - lo) / 2;
            if (sum_ge(key, true, mid) >= r) hi = mid;
            else lo = mid + 1;
        }
        cl.sync();
        cut.l = sm_unkey(key);
        cut.idx = (int)lo;
    };
    if (k > 0 && k < V) find_cut(false, (double)k, kSmRange);
    if (!(p >= 1.0f)) {
        if (p > 0.0f) {
            // Without top-k, tokens below (1 - p)/(2 V) of the best together weigh
            // less than half of what lies behind the cut (the other half is room
            // for rounded weights), so the bins need not reach that far.
            const float q = 1.0f - p;
            const bool narrow = !(k > 0 && k < V) && q >= 0.00390625f;
            find_cut(true, (double)p, narrow ? fminf(kSmRange, logf(2.0f * (float)V / q)) : kSmRange);
        } else {
            cut.l = top;
            cut.idx = first_best();
        }
    }

    // ---- the draw: the CTA, then the run of tokens, then the token ----
    auto weight = [&](float l, int i) -> u64 {
        if (!(l >= cut.l) || (l == cut.l && i > cut.idx)) return 0;
        const float e = sm_exp(l, top, inv_t);
        return mp > 0.0f && !(e >= mp) ? 0 : sm_weight(e);
    };
    u64 sum = 0, before;
    sm_each(x, n, i0, [&](float l, int i) { sum += weight(l, i); });
    const u64 total = cluster_sum(sum, &before);
    const double at = floor((double)u * (double)total);
    u64 target = at > 0.0 ? (u64)at : 0;
    target = target < total ? target : total - 1;
    const u64 here = S.sums[turn ^ 1][rank];
    if (target < before || target >= before + here) return;
    const int len = ((n + kSmThreads - 1) / kSmThreads) | 1;      // odd: a run a thread, no bank met twice
    const int a = min(n, tid * len), b = min(n, a + len);
    sum = 0;
    for (int i = a; i < b; i++) sum += weight((float)x[i], i0 + i);
    before += sm_block_before(sum, S.warp);
    if (before <= target && target < before + sum) {
        u64 run = before;
        for (int i = a; i < b; i++) {
            const u64 w = weight((float)x[i], i0 + i);
            run += w;
            if (run > target) {
                P.ids[row] = i0 + i;
                if (P.prob) P.prob[row] = (float)((double)w / (double)total);
                break;
            }
        }
    }
}

// A cluster of C CTAs for each row: as few as hold the row with two CTAs an
// SM, more while SMs would stand idle and a CTA keeps a few thousand logits.
template <typename T>
static int sm_launch(SmParams &P, int rows, cudaStream_t st) {
    const int sms = dev_info().sm_count > 0 ? dev_info().sm_count : 148;
    constexpr int kRoom = 115712 - (int)sizeof(SmShared) - 16;    // of half an SM
    auto slice = [&](int c) { return (P.vocab + c - 1) / c + 15 & ~15; };
    int C = 1;
    while (C < kSmMaxCluster && ((int64_t)slice(C) * (int)sizeof(T) > kRoom || (rows * C < sms && slice(C) > 4096))) C *= 2;
    P.slice = slice(C);
    const int64_t bytes = (int64_t)P.slice * (int)sizeof(T) + 16;
    P.held = bytes + (int)sizeof(SmShared) + 1024 <= dev_info().smem_optin;
    const int smem = P.held ? (int)bytes : 0;
    if (smem && !ensure_smem((const void *)k_sample<T>, smem)) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(rows * C));
    cfg.blockDim = dim3(kSmThreads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return check(cudaLaunchKernelEx(&cfg, k_sample<T>, P), "sample launch");
}

}  // namespace sepia

using namespace sepia;

extern "C" int sepia_cuda_sample(int x_f16, const void *logits, int64_t stride, int32_t rows, int32_t vocab,
                                 const float *u, const float *temperature, const int32_t *top_k, const float *top_p,
                                 const float *min_p, int32_t *ids, float *prob, void *stream) {
    const char *what = "sample";
    if (rows < 0 || vocab <= 0 || vocab > kSmMaxVocab)
        return fail("%s: %d rows of %d logits (1 to %d)", what, rows, vocab, kSmMaxVocab);
    if (rows == 0) return 1;
    if (!logits || !u || !ids) return fail("%s: null pointer", what);
    if (rows > INT32_MAX / kSmMaxCluster) return fail("%s: %d rows are too many", what, rows);
    if (reinterpret_cast<uintptr_t>(logits) % (x_f16 ? 2 : 4)) return fail("%s: logits are not aligned", what);
    if (stride < vocab) return fail("%s: row stride %lld is shorter than %d", what, (long long)stride, vocab);
    SmParams P;
    P.logits = logits;
    P.stride = stride;
    P.vocab = vocab;
    P.u = u;
    P.temperature = temperature;
    P.top_p = top_p;
    P.min_p = min_p;
    P.top_k = top_k;
    P.ids = ids;
    P.prob = prob;
    return x_f16 ? sm_launch<__half>(P, rows, as_stream(stream)) : sm_launch<float>(P, rows, as_stream(stream));
}
