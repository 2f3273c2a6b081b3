// sepia_b200/csrc/sample.cu -- one token per row of logits by temperature,
// top-k, top-p and min-p from one given uniform number (sepia_cuda_sample;
// definition in include/sepia_cuda.h).
//
// Each filter keeps a prefix of one order (greater logit first, then lower
// index), so a row's set is described by a cut: the logit of the last token
// in, and how many of the tokens with that very logit are in. Weights are
// integers: counts and masses are sums that no order of summation changes.
#include "../../include/sepia_cuda.h"
#include "common.cuh"
#include "runtime.h"

namespace sepia {

constexpr int kSmThreads = 1024;
constexpr float kSmOne = 2147483648.0f;      // weight of the best token: 2^31
constexpr int32_t kSmMaxVocab = 1 << 22;     // sums stay below 2^53: exact in fp64 too

typedef unsigned long long u64;

struct SmParams {
    const void *logits;
    int64_t stride;
    int32_t vocab;
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

__device__ u64 sm_block_sum(u64 v, u64 *sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if (lane == 0) sh[warp] = v;
    __syncthreads();
    v = sh[lane];
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
    u64 w = lane < warp ? sh[lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    return w + x - v;
}

// One CTA per row; every cut is found bit by bit over the key.
template <typename T>
__global__ void __launch_bounds__(kSmThreads) k_sample(const SmParams P) {
    __shared__ u64 sh[32];
    const int row = blockIdx.x, tid = threadIdx.x, V = P.vocab;
    griddep_wait();
    griddep_launch();
    const T *x = (const T *)P.logits + (int64_t)row * P.stride;
    if (tid == 0) {
        P.ids[row] = -1;
        if (P.prob) P.prob[row] = 0.0f;
    }
    u64 best = 0;
    for (int i = tid; i < V; i += kSmThreads) {
        const u64 k = ((u64)sm_key((float)x[i]) << 32) | (0xffffffffu - (uint32_t)i);
        best = k > best ? k : best;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 t = __shfl_xor_sync(0xffffffffu, best, o);
        best = t > best ? t : best;
    }
    if ((tid & 31) == 0) sh[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < 32; w++) best = sh[w] > best ? sh[w] : best;
    __syncthreads();
    const float top = sm_unkey((uint32_t)(best >> 32));
    if (top == -INFINITY) return;
    const float t = P.temperature ? P.temperature[row] : 1.0f;
    if (!(t > 0.0f)) {
        if (tid == 0) {
            P.ids[row] = (int32_t)(0xffffffffu - (uint32_t)best);
            if (P.prob) P.prob[row] = 1.0f;
        }
        return;
    }
    const float inv_t = __fdiv_rn(1.0f, t);
    const int k = P.top_k ? P.top_k[row] : 0;
    const float p = P.top_p ? P.top_p[row] : 1.0f;
    const float mp = P.min_p ? fminf(P.min_p[row], 1.0f) : 0.0f;
    uint32_t cut = 0;                 // kept: key > cut, and the first `ties` tokens of key == cut
    u64 ties = (u64)V;
    auto sum_ge = [&](uint32_t key, bool mass) {
        u64 s = 0;
        for (int i = tid; i < V; i += kSmThreads) {
            const float l = (float)x[i];
            if (sm_key(l) >= key) s += mass ? sm_weight(sm_exp(l, top, inv_t)) : 1;
        }
        return sm_block_sum(s, sh);
    };
    u64 mass = 0;
    if (k > 0 && k < V) {
        for (int b = 31; b >= 0; b--) {
            const uint32_t c = cut | (1u << b);
            if (sum_ge(c, false) >= (u64)k) cut = c;
        }
        ties = (u64)k - (cut == 0xffffffffu ? 0 : sum_ge(cut + 1, false));
    }
    if (!(p >= 1.0f)) {
        const u64 w0 = sm_weight(sm_exp(sm_unkey(cut), top, inv_t));
        mass = cut ? sum_ge(cut + 1, true) + ties * w0 : sum_ge(0, true);
        const double thr = (double)p * (double)mass;
        uint32_t c2 = 0;
        for (int b = 31; b >= 0; b--) {
            const uint32_t c = c2 | (1u << b);
            if (c <= cut || (double)sum_ge(c, true) >= thr) c2 = c;
        }
        if (!(thr > 0.0)) c2 = (uint32_t)(best >> 32);
        const u64 above = sum_ge(c2 + 1, true), w = sm_weight(sm_exp(sm_unkey(c2), top, inv_t));
        u64 r = w && thr > (double)above ? (u64)((thr - (double)above) / (double)w) : 0;
        while (r > 0 && (double)(above + (r - 1) * w) >= thr) r--;
        while (w && (double)(above + r * w) < thr) r++;
        if (r == 0) r = 1;
        ties = c2 == cut && ties < r ? ties : r;
        cut = c2;
    }
    // the draw: threads own runs of the row in index order
    const int len = (V + kSmThreads - 1) / kSmThreads;
    const int i0 = min(V, tid * len), i1 = min(V, i0 + len);
    u64 eq = 0;
    for (int i = i0; i < i1; i++) eq += sm_key((float)x[i]) == cut;
    const u64 eq0 = sm_block_before(eq, sh);
    auto weight = [&](int i, u64 &seen) -> u64 {
        const float l = (float)x[i];
        const uint32_t key = sm_key(l);
        const float e = sm_exp(l, top, inv_t);
        bool in = key > cut;
        if (key == cut) in = seen++ < ties;
        if (mp > 0.0f) in = in && e >= mp;
        return in ? sm_weight(e) : 0;
    };
    u64 sum = 0, seen = eq0;
    for (int i = i0; i < i1; i++) sum += weight(i, seen);
    const u64 before = sm_block_before(sum, sh);
    const u64 total = sm_block_sum(sum, sh);
    const float u = P.u[row];
    const double at = floor((double)u * (double)total);
    u64 target = at > 0.0 ? (u64)at : 0;
    target = target < total ? target : total - 1;
    if (before <= target && target < before + sum) {
        u64 run = before;
        seen = eq0;
        for (int i = i0; i < i1; i++) {
            const u64 w = weight(i, seen);
            run += w;
            if (run > target) {
                P.ids[row] = i;
                if (P.prob) P.prob[row] = (float)((double)w / (double)total);
                break;
            }
        }
    }
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
    const cudaError_t e = x_f16 ? launch_pdl(k_sample<__half>, (unsigned)rows, kSmThreads, 0, as_stream(stream), P)
                                : launch_pdl(k_sample<float>, (unsigned)rows, kSmThreads, 0, as_stream(stream), P);
    return check(e, "sample launch");
}
