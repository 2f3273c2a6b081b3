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
// meet in one counter). Where the tokens down to the threshold bin are few,
// the usual case, the cluster's first CTA takes them all and does the rest
// (further cuts, the draw) in a sorted list. Otherwise it takes the threshold
// bin alone, splits it by a second histogram, and the draw is one more pass of
// the cluster. A bin that is too full for the list is first split by the
// cluster; what even that leaves too full (runs of equal logits) is cut by
// halving the range of keys, 32 passes. Time goes into instructions, some 35
// for each logit that has a weight, most of them the exponential and its place
// in the histogram, and into the cluster's barriers.
#include "../../include/sepia_cuda.h"
#include "common.cuh"
#include "runtime.h"

#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace sepia {

constexpr int kSmThreads = 512;              // 256 save a fifth of the instructions but wait longer: 228 us for 192 x 200058, 512 take 201
constexpr int kSmBins = 1024;
constexpr int kSmPer = kSmBins / kSmThreads; // bins (and list entries) of a thread
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
// (l - max)/T, at most 0, and e = exp of it; the best token's is 1 also where
// max is infinite, or 1/T is (the least of NaN and 0 is 0)
__device__ __forceinline__ float sm_exponent(float l, float best, float inv_t) {
    return fminf(__fmul_rn(__fsub_rn(l, best), inv_t), 0.0f);
}
__device__ __forceinline__ float sm_exp(float l, float best, float inv_t) { return expf(sm_exponent(l, best, inv_t)); }
__device__ __forceinline__ u64 sm_weight(float e) { return (u64)__float2uint_rn(__fmul_rn(e, kSmOne)); }
// A token's place among the bins, from its exponent, and among the parts of
// a bin, from its place. The histogram, the gather and the sums have to put a
// token into the same bin wherever they work it out, so every step is rounded
// by itself here: the compiler must not join two of them at one site and not
// at another. Each step keeps the order of places.
__device__ __forceinline__ float sm_place(float exponent, float per) { return __fmul_rn(exponent, per); }
__device__ __forceinline__ float sm_part_place(float place, int bin) {
    return __fmul_rn(__fadd_rn(__fsub_rn(place, (float)bin), 0.5f), (float)kSmBins);
}
// The nearest whole number, by adding 2^23 (a conversion would hold up the
// exponentials' unit); places may lie past the last bin by their rounding.
__device__ __forceinline__ int sm_nearest(float place) {
    return (int)min(kSmBins - 1u, __float_as_uint(__fadd_rn(place, 8388608.0f)) - 0x4b000000u);
}
__device__ __forceinline__ int sm_part(float part_place) { return sm_nearest(fmaxf(__fsub_rn(part_place, 0.5f), 0.0f)); }

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
    u64 sums[2][kSmMaxCluster][2], warp[kSmThreads / 32];
    int first_idx, n_short;
    u64 short_list[32];                      // tokens of the threshold's part of the bin
    u64 found_before, found_here;            // count or mass of the bins above the threshold bin, and of it
    int counts[kSmMaxCluster];               // tokens that each CTA gathered
    int bin, n_list;                         // bin: -1 no cut; n_list may pass kSmList
    SmCut cut;
};

// Sum over the warp, below 2^54: two sums of 27-bit halves, each by one instruction
__device__ __forceinline__ u64 sm_warp_sum(u64 v) {
    return (u64)__reduce_add_sync(0xffffffffu, (uint32_t)v & 0x7ffffffu) +
           ((u64)__reduce_add_sync(0xffffffffu, (uint32_t)(v >> 27)) << 27);
}
__device__ u64 sm_block_sum(u64 v, u64 *sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    v = sm_warp_sum(v);
    __syncthreads();
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    return sm_warp_sum(lane < kSmThreads / 32 ? sh[lane] : 0);
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
    return sm_warp_sum(lane < warp && lane < kSmThreads / 32 ? sh[lane] : 0) + x - v;
}

// A slice in index order: logits before the first 16-byte boundary (warp 0
// takes them), whole vectors (a run for each warp), the rest (the last warp).
template <typename T>
struct SmSlice {
    static constexpr int E = 16 / (int)sizeof(T);
    const T *x;
    int n, i0, head, body, lo, hi;           // i0: the slice's first index in the row; lo, hi: this warp's vectors
    __device__ __forceinline__ SmSlice(const T *x_, int n_, int i0_) : x(x_), n(n_), i0(i0_) {
        const int warp = threadIdx.x >> 5;
        head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
        body = (n - head) / E;
        const int run = (body + kSmThreads / 32 - 1) / (kSmThreads / 32);
        lo = min(body, warp * run);
        hi = min(body, lo + run);
    }
    __device__ __forceinline__ void load(int j, float (&v)[E]) const {
        const uint4 raw = *reinterpret_cast<const uint4 *>(x + head + j * E);
        const T *y = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = (float)y[e];
    }
    __device__ __forceinline__ int index(int j) const { return i0 + head + j * E; }
    // The lane's logit (the others NaN) of the part before (0) or after (1) the vectors; its index, or -1
    __device__ __forceinline__ int ragged(int part, float (&v)[E]) const {
        const int lane = threadIdx.x & 31, at = part ? head + body * E + lane : lane;
        const bool on = part ? (threadIdx.x >> 5) == kSmThreads / 32 - 1 && at < n : (threadIdx.x >> 5) == 0 && lane < head;
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = __int_as_float(0x7fffffff);
        if (on) v[0] = (float)x[at];
        return on ? i0 + at : -1;
    }
    // f(vector, index of its first logit) over the slice; NaN where there is none
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        float v[E];
        for (int j = lo + (threadIdx.x & 31); j < hi; j += 32) {
            load(j, v);
            f(v, index(j));
        }
        if (head + body * E == n && head == 0) return;
#pragma unroll 1
        for (int part = 0; part < 2; part++) {
            const int i = ragged(part, v);
            if (i >= 0) f(v, i);
        }
    }
};

// list[0, m) in descending order; m a power of two
__device__ void sm_sort(u64 *list, int m) {
    for (int size = 2; size <= m; size <<= 1)
        for (int step = size >> 1; step > 0; step >>= 1) {
            for (int i = threadIdx.x; i < m / 2; i += kSmThreads) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const u64 va = list[a], vb = list[b];
                if ((va < vb) == ((a & size) == 0)) list[a] = vb, list[b] = va;
            }
            __syncthreads();
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
    // A CTA's shared memory may be written by the others once it is known to
    // have started: it arrives here, and they wait before their first store.
    cl.barrier_arrive();
    griddep_wait();
    griddep_launch();
    const int i0 = min(V, rank * P.slice), n = min(V, i0 + P.slice) - i0;
    const T *gx = (const T *)P.logits + (int64_t)row * P.stride + i0;
    // the slice in shared memory keeps the row's place between 16-byte boundaries
    T *hx = reinterpret_cast<T *>(sm_raw + (reinterpret_cast<uintptr_t>(gx) & 15));
    constexpr int E = SmSlice<T>::E;
    const SmSlice<T> X(P.held ? hx : gx, n, i0);
    const float t = P.temperature ? P.temperature[row] : 1.0f;
    const int k = P.top_k ? P.top_k[row] : 0;
    const float p = P.top_p ? P.top_p[row] : 1.0f;
    const float mp = P.min_p && P.min_p[row] > 0.0f ? fminf(P.min_p[row], 1.0f) : 0.0f, u = P.u[row];

    // ---- the row into shared memory; its greatest logit ----
    float top = -INFINITY;                             // NaN loses every fmaxf
    {
        constexpr int kAhead = 8;
        const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(gx) & 15)) & 15) / (int)sizeof(T));
        const int body = (n - head) / E;
        const uint4 *from = reinterpret_cast<const uint4 *>(gx + head) + tid;
        uint4 *to = reinterpret_cast<uint4 *>(hx + head) + tid;
        auto take = [&](int j, const uint4 &raw) {
            if (P.held) to[j] = raw;
            const T *v = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (int e = 0; e < E; e++) top = fmaxf(top, (float)v[e]);
        };
        int j = 0;
        for (; j + tid + (kAhead - 1) * kSmThreads < body; j += kAhead * kSmThreads) {
            uint4 raw[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; a++) raw[a] = __ldg(from + j + a * kSmThreads);
#pragma unroll
            for (int a = 0; a < kAhead; a++) take(j + a * kSmThreads, raw[a]);
        }
        {
            uint4 raw[kAhead - 1];                     // fewer than kAhead are left
#pragma unroll
            for (int a = 0; a < kAhead - 1; a++)
                if (j + tid + a * kSmThreads < body) raw[a] = __ldg(from + j + a * kSmThreads);
#pragma unroll
            for (int a = 0; a < kAhead - 1; a++)
                if (j + tid + a * kSmThreads < body) take(j + a * kSmThreads, raw[a]);
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
    cl.barrier_wait();                                 // every CTA has started; hidden behind the load
    if (tid < C) {
#pragma unroll
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
        X.each([&](const float (&v)[E], int i) {
#pragma unroll
            for (int e = 0; e < E; e++)
                if (v[e] == top) atomicMin(&S.first_idx, i + e);
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
    auto cluster_sum = [&](u64 v, u64 other, u64 *before, u64 *other_all) {
        const u64 s = sm_block_sum(v, S.warp), o = other_all ? sm_block_sum(other, S.warp) : 0;
        if (tid < C) {
            SmShared *q = cl.map_shared_rank(&S, tid);
            q->sums[turn][rank][0] = s;
            q->sums[turn][rank][1] = o;
        }
        cl.sync();
        u64 all = 0, less = 0, others = 0;
        for (int r = 0; r < C; r++) {
            less += r < rank ? S.sums[turn][r][0] : 0;
            all += S.sums[turn][r][0];
            others += S.sums[turn][r][1];
        }
        turn ^= 1;                                     // the next sum must not overwrite what is still read
        if (before) *before = less;
        if (other_all) *other_all = others;
        return all;
    };
    // Below this a weight rounds to 0: rounding of the bound itself cannot
    // pass a logit at less than the range (both are fp32 numbers).
    // Never as low as -infinity, whatever T: such a logit is out.
    const float floor_l = fmaxf(top - kSmRange * t, -3.402823466e38f);
    SmCut cut = {floor_l, INT32_MAX};                  // tokens in: l > cut.l, or l == cut.l up to an index
    auto in = [&](float l, int i) { return l >= cut.l && !(l == cut.l && i > cut.idx); };
    // Weights of a vector's tokens that are in, 0 for the others; false: all 0
    auto weigh = [&](const float (&v)[E], int i, uint32_t (&w)[E], float (&x)[E]) {
        float most = v[0];
#pragma unroll
        for (int e = 1; e < E; e++) most = fmaxf(most, v[e]);
        if (!(most >= cut.l)) return false;
#pragma unroll
        for (int e = 0; e < E; e++) {
            x[e] = sm_exponent(v[e], top, inv_t);
            const uint32_t y = (uint32_t)sm_weight(expf(x[e]));
            w[e] = v[e] >= cut.l ? y : 0u;
        }
        if (cut.idx != INT32_MAX) {                    // the whole cluster
#pragma unroll
            for (int e = 0; e < E; e++)
                if (v[e] == cut.l && i + e > cut.idx) w[e] = 0u;
        }
        return true;
    };
    // The rest of a row whose first `have` tokens are in the list: all cuts and
    // the draw, by one CTA. by_mass: they end at mass thr, else at k tokens.
    auto finish = [&](int have, bool by_mass, double thr) {
        int m = 2;
        while (m < have) m <<= 1;
        if (have <= kSmThreads / 2) {
            // Few tokens: each one's sums over those before it, by pairs, the
            // others of a token spread over kSmThreads / m neighbouring lanes
            // (two sorts of 155 tokens took 11 us, this takes 3).
            m = max(m, kSmThreads / 32);
            uint32_t *weight_of = reinterpret_cast<uint32_t *>(S.list + kSmList / 2);
            const int lanes = kSmThreads / m, me = tid / lanes, part = tid % lanes;
            const u64 y = me < have ? S.list[me] : 0;
            const float e = sm_exp(sm_unkey((uint32_t)(y >> 32)), top, inv_t);
            uint32_t w = me < have ? (uint32_t)sm_weight(e) : 0u;
            if (part == 0 && me < have) weight_of[me] = w;
            __syncthreads();
            u64 mass_before = 0;
            int rank_of = 0;
            for (int j = part; j < have; j += lanes)
                if (S.list[j] > y) rank_of++, mass_before += weight_of[j];
            for (int o = 1; o < lanes; o <<= 1) {
                rank_of += __shfl_xor_sync(0xffffffffu, rank_of, o);
                mass_before += __shfl_xor_sync(0xffffffffu, mass_before, o);
            }
            bool is_in = me < have && (by_mass || rank_of < k);
            if (!by_mass) thr = p >= 1.0f ? 1e300 : (double)p * (double)sm_block_sum(is_in && part == 0 ? w : 0, S.warp);
            is_in = is_in && ((double)mass_before < thr || rank_of == 0) && !(mp > 0.0f && !(e >= mp));
            if (!is_in) w = 0;
            __syncthreads();
            if (part == 0 && me < have) weight_of[me] = w;
            const u64 total = sm_block_sum(part == 0 ? w : 0, S.warp);
            u64 run = 0;                               // of the tokens of lower index
            for (int j = part; j < have; j += lanes)
                if ((uint32_t)S.list[j] > (uint32_t)y) run += weight_of[j];
            for (int o = 1; o < lanes; o <<= 1) run += __shfl_xor_sync(0xffffffffu, run, o);
            const double at_u = floor((double)u * (double)total);
            u64 target = at_u > 0.0 ? (u64)at_u : 0;
            target = target < total ? target : total - 1;
            if (part == 0 && run <= target && target < run + w) {
                P.ids[row] = (int32_t)(0xffffffffu - (uint32_t)y);
                if (P.prob) P.prob[row] = (float)((double)w / (double)total);
            }
            return;
        }
        for (int i = have + tid; i < m; i += kSmThreads) S.list[i] = 0;
        __syncthreads();
        sm_sort(S.list, m);
        u64 y[kSmPer], w[kSmPer], sum = 0;
#pragma unroll
        for (int e = 0; e < kSmPer; e++) {
            const int at = kSmPer * tid + e;
            y[e] = at < have ? S.list[at] : 0;
            w[e] = at < have && (by_mass || at < k) ? sm_weight(sm_exp(sm_unkey((uint32_t)(y[e] >> 32)), top, inv_t)) : 0;
            sum += w[e];
        }
        u64 run = sm_block_before(sum, S.warp);
        if (!by_mass) thr = p >= 1.0f ? 1e300 : (double)p * (double)sm_block_sum(sum, S.warp);
        __syncthreads();
        sum = 0;
#pragma unroll
        for (int e = 0; e < kSmPer; e++) {
            const int at = kSmPer * tid + e;
            const bool is_in = (double)run < thr || at == 0;
            run += w[e];
            if (!is_in || (mp > 0.0f && !(sm_exp(sm_unkey((uint32_t)(y[e] >> 32)), top, inv_t) >= mp))) w[e] = 0;
            sum += w[e];
            if (at < m) S.list[at] = w[e] ? (y[e] << 32) | w[e] : 0;      // now by the index, which rises
        }
        const u64 total = sm_block_sum(sum, S.warp);
        sm_sort(S.list, m);
        const double at_u = floor((double)u * (double)total);
        u64 target = at_u > 0.0 ? (u64)at_u : 0;
        target = target < total ? target : total - 1;
        sum = 0;
#pragma unroll
        for (int e = 0; e < kSmPer; e++) {
            y[e] = kSmPer * tid + e < m ? S.list[kSmPer * tid + e] : 0;
            sum += y[e] & 0xffffffffu;
        }
        run = sm_block_before(sum, S.warp);
#pragma unroll
        for (int e = 0; e < kSmPer; e++) {
            const u64 v = y[e] & 0xffffffffu;
            if (run <= target && target < run + v) {
                P.ids[row] = (int32_t)(0xffffffffu - (uint32_t)(y[e] >> 32));
                if (P.prob) P.prob[row] = (float)((double)v / (double)total);
            }
            run += v;
        }
    };
    // The cut at the token where the running count (of the order) reaches
    // `want`, or the running mass reaches `want` times the mass of the tokens
    // that are in. range: tokens with (max - l)/T beyond it cannot be the
    // cut; their mass still counts.
    // True: the first CTA has drawn the token, nothing is left to do.
    auto find_cut = [&](bool mass, double want, float range) {
        const float per = -(float)kSmBins / range, near = range < kSmRange ? fmaxf(cut.l, top - range * t) : cut.l;
        for (int i = tid; i < 2 * kSmBins; i += kSmThreads) (&S.hist[0][0])[i] = 0;
        if (tid == 0) S.bin = -1;
        __syncthreads();
        u64 beyond = 0;
        auto place_of = [&](float l) { return sm_place(sm_exponent(l, top, inv_t), per); };
        auto bin_of = [&](float l) { return sm_nearest(place_of(l)); };
        X.each([&](const float (&v)[E], int i) {
            if (!mass) {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (in(v[e], i + e)) atomicAdd(&S.hist[0][bin_of(v[e])], 1u);
                return;
            }
            uint32_t w[E];
            float x[E];
            if (!weigh(v, i, w, x)) return;
            if (range < kSmRange) {                    // such weights are below 2^31 (1 - p)/(2 V): E of them fit 32 bits
                uint32_t far = 0;
#pragma unroll
                for (int e = 0; e < E; e++) far += v[e] < near ? w[e] : 0u;
                beyond += far;
            }
#pragma unroll
            for (int e = 0; e < E; e++)
                if (v[e] >= near) {                    // some have weight 0: not in after all
                    const int b = sm_nearest(sm_place(x[e], per));   // bin_of
                    atomicAdd(&S.hist[0][b], w[e] & 0xffffu);
                    atomicAdd(&S.hist[1][b], w[e] >> 16);
                }
        });
        // The threshold bin, of counters that start at running sum `from`: each
        // CTA adds its share of the bins over the cluster, a run of `each`
        // neighbours a thread. S.bin stays -1 where the threshold is not met.
        double thr = want;
        auto add_bins = [&](u64 from, bool know_thr) {
            cl.sync();
            const int share = kSmBins / C, each = max(1, share / kSmThreads), first_bin = rank * share + tid * each;
            u64 v[kSmPer] = {}, mine = 0;
#pragma unroll
            for (int e = 0; e < kSmPer; e++)
                if (e < each && tid * each < share) {
                    uint32_t x[kSmMaxCluster][2];
#pragma unroll
                    for (int r = 0; r < kSmMaxCluster; r++) {
                        const SmShared *q = cl.map_shared_rank(&S, r < C ? r : 0);
                        x[r][0] = r < C ? q->hist[0][first_bin + e] : 0;
                        x[r][1] = r < C && mass ? q->hist[1][first_bin + e] : 0;
                    }
#pragma unroll
                    for (int r = 0; r < kSmMaxCluster; r++) v[e] += (u64)x[r][0] + ((u64)x[r][1] << 16);
                    mine += v[e];
                }
            u64 b = 0, far_mass = 0;
            const u64 all = cluster_sum(mine, beyond, &b, &far_mass);
            if (mass && !know_thr) thr = want * (double)(all + far_mass);
            b += from + sm_block_before(mine, S.warp);
#pragma unroll
            for (int e = 0; e < kSmPer; e++) {
                if ((double)b < thr && (double)(b + v[e]) >= thr)
                    for (int r = 0; r < C; r++) {
                        SmShared *q = cl.map_shared_rank(&S, r);
                        q->bin = first_bin + e;
                        q->found_before = b;
                        q->found_here = v[e];
                    }
                b += v[e];
            }
            cl.sync();
        };
        add_bins(0, false);
        const int bin = S.bin;
        if (bin < 0) return false;                     // a count past all tokens of any weight: nothing to cut
        u64 above = S.found_before;
        // A token's part of the bin (of part `sub` of it, where that is in question)
        int sub = -1;
        auto part_of = [&](float l) { return sm_part(sm_part_place(place_of(l), bin)); };
        auto part_of_sub = [&](float l) {
            return sm_part(__fmul_rn(__fsub_rn(sm_part_place(place_of(l), bin), (float)sub), (float)kSmBins));
        };
        // Tokens of bins from .. bin (of part `sub` of the bin) into the lists of their CTAs, then
        // (if they fit) into the first CTA's; how many there are. Bounds a
        // little past the bins (half a bin to either side of whole numbers)
        // spare most tokens the bin's arithmetic.
        auto gather = [&](int from) {
            const float bin_lo = bin == kSmBins - 1 ? near : fmaxf(near, top + ((float)bin + 0.6f) / per * t);
            const float bin_hi = from ? top + ((float)from - 0.6f) / per * t : top;
            const float mid = from ? 0.5f * (bin_lo + bin_hi) : top, half = from ? fmaxf(bin_hi - mid, mid - bin_lo) : top - bin_lo;
            __syncthreads();
            if (tid == 0) S.n_list = 0;
            __syncthreads();
            X.each([&](const float (&v)[E], int i) {
                float d = fabsf(v[0] - mid);           // NaN at an infinite maximum: passes
#pragma unroll
                for (int e = 1; e < E; e++) d = fminf(d, fabsf(v[e] - mid));
                if (d > half) return;
#pragma unroll
                for (int e = 0; e < E; e++) {
                    if (fabsf(v[e] - mid) > half || !(v[e] >= near)) continue;
                    const int b = bin_of(v[e]);
                    if (b >= from && b <= bin && in(v[e], i + e) &&
                        (sub < 0 || part_of(v[e]) == sub)) {
                        const int at = atomicAdd(&S.n_list, 1);
                        if (at < kSmList) S.list[at] = ((u64)sm_key(v[e]) << 32) | (0xffffffffu - (uint32_t)(i + e));
                    }
                }
            });
            __syncthreads();
            const int n_here = S.n_list;
            if (tid < C) cl.map_shared_rank(&S, tid)->counts[rank] = n_here;
            cl.sync();
            int all_n = 0, before_n = 0;
            for (int r = 0; r < C; r++) {
                before_n += r < rank ? S.counts[r] : 0;
                all_n += S.counts[r];
            }
            if (all_n <= kSmList && rank > 0)
                for (int i = tid; i < n_here; i += kSmThreads) first->list[before_n + i] = S.list[i];
            cl.sync();
            return all_n;
        };
        // All tokens down to the threshold: as many as the count says, or at
        // most their mass over the least weight among them. Where that bound is
        // high the attempt is spared (192 rows of 200058, nucleus sampling: 185
        // us, always trying 212, never 201).
        const u64 down = above + S.found_here;
        const double least = mass ? exp(((double)bin + 0.5) / (double)per) * (double)kSmOne : 1.0;
        if ((double)down <= least * (mass ? 65536.0 : (double)kSmList)) {
            const int have = gather(0);
            if (have <= kSmList) {
                if (rank == 0) finish(have, mass, thr);
                return true;
            }
        }
        int have = gather(bin);
        if (have > kSmList) {
            // Too many: a second histogram over the bin alone, in as many parts
            for (int i = tid; i < 2 * kSmBins; i += kSmThreads) (&S.hist[0][0])[i] = 0;
            if (tid == 0) S.bin = -1;
            __syncthreads();
            beyond = 0;
            X.each([&](const float (&v)[E], int i) {
#pragma unroll
                for (int e = 0; e < E; e++)
                    if (v[e] >= near && bin_of(v[e]) == bin && in(v[e], i + e)) {
                        const uint32_t w = mass ? sm_weight(sm_exp(v[e], top, inv_t)) : 1u;
                        const int b = part_of(v[e]);   // sub is not set yet
                        atomicAdd(&S.hist[0][b], w & 0xffffu);
                        if (mass) atomicAdd(&S.hist[1][b], w >> 16);
                    }
            });
            add_bins(above, true);
            sub = S.bin;
            above = S.found_before;
            have = gather(bin);
        }
        if (have <= kSmList) {
            if (rank == 0) {
                auto value = [&](u64 y) -> u64 {
                    return !mass ? 1 : sm_weight(sm_exp(sm_unkey((uint32_t)(y >> 32)), top, inv_t));
                };
                // this thread's tokens of the list, and their part of the bin
                u64 y[kSmPer], val[kSmPer], z[kSmPer], over, q = 0;
                int part[kSmPer];
#pragma unroll
                for (int e = 0; e < kSmPer; e++) {
                    const bool on = tid + e * kSmThreads < have;
                    y[e] = on ? S.list[tid + e * kSmThreads] : 0;
                    val[e] = on ? value(y[e]) : 0;
                    const float l = sm_unkey((uint32_t)(y[e] >> 32));
                    part[e] = !on ? -1 : sub < 0 ? part_of(l) : part_of_sub(l);
                }
                __syncthreads();                       // the list is read: its room becomes counters again
                for (int i = tid; i < 2 * kSmBins; i += kSmThreads) (&S.hist[0][0])[i] = 0;
                if (tid == 0) S.n_short = 0;
                __syncthreads();
#pragma unroll
                for (int e = 0; e < kSmPer; e++)
                    if (part[e] >= 0) {
                        atomicAdd(&S.hist[0][part[e]], (uint32_t)val[e] & 0xffffu);
                        atomicAdd(&S.hist[1][part[e]], (uint32_t)val[e] >> 16);
                    }
                __syncthreads();
#pragma unroll
                for (int e = 0; e < kSmPer; e++) {
                    z[e] = (u64)S.hist[0][kSmPer * tid + e] + ((u64)S.hist[1][kSmPer * tid + e] << 16);
                    q += z[e];
                }
                q = above + sm_block_before(q, S.warp);
#pragma unroll
                for (int e = 0; e < kSmPer; e++) {
                    if ((double)q < thr && (double)(q + z[e]) >= thr) S.bin = kSmPer * tid + e, S.found_before = q;
                    q += z[e];
                }
                __syncthreads();
                over = S.found_before;
#pragma unroll
                for (int e = 0; e < kSmPer; e++)
                    if (part[e] == S.bin) {
                        const int at = atomicAdd(&S.n_short, 1);
                        if (at < 32) S.short_list[at] = y[e];
                    }
                __syncthreads();
                if (S.n_short <= 32) {                 // one warp: each token's sum of those before it
                    if (tid < 32) {
                        const u64 mine = tid < S.n_short ? S.short_list[tid] : 0, w = tid < S.n_short ? value(mine) : 0;
                        u64 c = over;
                        for (int i = 0; i < S.n_short; i++) {
                            const u64 other = __shfl_sync(0xffffffffu, mine, i), ow = __shfl_sync(0xffffffffu, w, i);
                            c += other > mine ? ow : 0;
                        }
                        if (tid < S.n_short && (double)c < thr && (double)(c + w) >= thr) {
                            S.cut.l = sm_unkey((uint32_t)(mine >> 32));
                            S.cut.idx = (int)(0xffffffffu - (uint32_t)mine);
                        }
                    }
                } else {                               // the list once more, sorted by the order, then summed
                    int m = 2;
                    while (m < have) m <<= 1;
#pragma unroll
                    for (int e = 0; e < kSmPer; e++) S.list[tid + e * kSmThreads] = y[e];
                    __syncthreads();
                    sm_sort(S.list, m);
                    q = 0;
#pragma unroll
                    for (int e = 0; e < kSmPer; e++) {
                        z[e] = kSmPer * tid + e < have ? value(S.list[kSmPer * tid + e]) : 0;
                        q += z[e];
                    }
                    q = above + sm_block_before(q, S.warp);
#pragma unroll
                    for (int e = 0; e < kSmPer; e++) {
                        if ((double)q < thr && (double)(q + z[e]) >= thr) {
                            S.cut.l = sm_unkey((uint32_t)(S.list[kSmPer * tid + e] >> 32));
                            S.cut.idx = (int)(0xffffffffu - (uint32_t)S.list[kSmPer * tid + e]);
                        }
                        q += z[e];
                    }
                }
                __syncthreads();
                if (tid > 0 && tid < C) cl.map_shared_rank(&S, tid)->cut = S.cut;
            }
            cl.sync();
            cut = S.cut;
            return false;
        }
        // Too many for the list: the greatest key whose tokens and those above
        // reach the threshold, bit by bit; then how many tokens of that very
        // key are in, and the index of the last of them.
        auto sum_ge = [&](uint32_t key, bool indexes, uint32_t upto) {
            u64 s = 0;
            X.each([&](const float (&v)[E], int i) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const uint32_t y = sm_key(v[e]);
                    if (in(v[e], i + e) && (indexes ? y == key && (uint32_t)(i + e) <= upto : y >= key))
                        s += mass && !indexes ? sm_weight(sm_exp(v[e], top, inv_t)) : 1;
                }
            });
            return cluster_sum(s, 0, nullptr, nullptr);
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
        return false;
    };
    if (k > 0 && k < V && find_cut(false, (double)k, kSmRange)) return;
    if (!(p >= 1.0f)) {
        if (p > 0.0f) {
            // Without top-k, tokens below (1 - p)/(2 V) of the best together weigh
            // less than half of what lies behind the cut (the other half is room
            // for rounded weights), so the bins need not reach that far.
            const float q = 1.0f - p;
            const bool narrow = !(k > 0 && k < V) && q >= 0.00390625f;
            if (find_cut(true, (double)p, narrow ? fminf(kSmRange, logf(2.0f * (float)V / q)) : kSmRange)) return;
        } else {
            cut.l = top;
            cut.idx = first_best();
        }
    }

    // ---- the draw: the CTA, then the warp's run, then the token ----
    auto weigh_min_p = [&](const float (&v)[E], int i, uint32_t (&w)[E]) {
        u64 s = 0;
        float x[E];
        if (!weigh(v, i, w, x)) {
#pragma unroll
            for (int e = 0; e < E; e++) w[e] = 0u;
            return s;
        }
        if (mp > 0.0f) {                               // the whole cluster
#pragma unroll
            for (int e = 0; e < E; e++)
                if (!(expf(x[e]) >= mp)) w[e] = 0u;
        }
#pragma unroll
        for (int e = 0; e < E; e++) s += w[e];
        return s;
    };
    u64 sum = 0, before;
    X.each([&](const float (&v)[E], int i) {
        uint32_t w[E];
        sum += weigh_min_p(v, i, w);
    });
    const u64 total = cluster_sum(sum, 0, &before, nullptr);
    const double at = floor((double)u * (double)total);
    u64 target = at > 0.0 ? (u64)at : 0;
    target = target < total ? target : total - 1;
    const u64 here = S.sums[turn ^ 1][rank][0];
    if (target < before || target >= before + here) return;
    sum = sm_warp_sum(sum);
    before += sm_block_before(lane == 0 ? sum : 0, S.warp);
    before = __shfl_sync(0xffffffffu, before, 0);      // of the warps before this one
    if (target < before || target >= before + sum) return;
    // steps of the warp's run, in index order; true when the token was in this one
    auto step = [&](const float (&v)[E], int i, bool on) {
        uint32_t w[E];
        const u64 mine = on ? weigh_min_p(v, i, w) : 0;    // below 2^35
        const u64 all = sm_warp_sum(mine);
        if (target >= before + all) {
            before += all;
            return false;
        }
        u64 up = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 y = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += y;
        }
        u64 run = before + up - mine;
        if (on && run <= target && target < run + mine) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                if (run <= target && target < run + w[e]) {
                    P.ids[row] = i + e;
                    if (P.prob) P.prob[row] = (float)((double)w[e] / (double)total);
                }
                run += w[e];
            }
        }
        return true;
    };
    float v[E];
    int i = X.ragged(0, v);
    if (step(v, i, i >= 0)) return;
    for (int j = X.lo; j < X.hi; j += 32) {
        const bool on = j + lane < X.hi;
        if (on) X.load(j + lane, v);
        if (step(v, X.index(j + lane), on)) return;
    }
    i = X.ragged(1, v);
    step(v, i, i >= 0);
}

// A cluster of C CTAs for each row: as few as hold the row with two CTAs an
// SM, more while SMs would stand idle and a CTA keeps a few thousand logits (33
// rows of 50021 fp16 logits: 20 us with 8 CTAs a row, 31 with the one that holds it).
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
