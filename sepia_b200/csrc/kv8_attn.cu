// sepia_b200/csrc/kv8_attn.cu -- attention of new tokens over the paged
// 8-bit cache (sepia_cuda_kv8_attn; rules in include/sepia_cuda.h).
#include "kv8.cuh"
#include "runtime.h"

#include <cuda_fp8.h>

namespace sepia {

struct K8Params {
    SepiaKv8Cache c;
    SepiaKv8Step b;
    SepiaKv8Attn a;
    int *err;
};

// One warp per (token, head); a lane owns 4 dims; one key at a time, with
// the running maximum and sum of the softmax.
template <typename T>
__global__ void __launch_bounds__(32) k_kv8_attn(const K8Params P) {
    const int lane = threadIdx.x, d = 4 * lane, h = blockIdx.x, i = blockIdx.y, s = blockIdx.z;
    const int Dh = P.c.head_dim, B = P.c.block, H = P.a.n_heads, Hkv = P.c.n_kv_heads, hk = h / (H / Hkv);
    griddep_wait();
    griddep_launch();
    const Kv8Seq sq = kv8_seq(P.c, P.b, s, P.err);
    if (i >= sq.rows) return;
    const int n = sq.n0 + i, pos = sq.held + i;
    float q[4] = {}, o[4] = {}, m = -INFINITY, l = 0.0f;
    if (sq.add >= 0) {
        if (d < Dh)
            for (int e = 0; e < 4; e++)
                q[e] = (float)((const T *)P.a.q)[(int64_t)n * P.a.q_stride + (int64_t)h * Dh + d + e];
        const int tail0 = (sq.held + sq.add) / B * B;
        for (int j = P.a.window ? max(0, pos - P.a.window + 1) : 0; j <= pos; j++) {
            float k[4] = {}, v[4] = {}, ks = 1.0f, vs = 1.0f;
            if (j >= tail0) {
                const int64_t at = (((int64_t)sq.slot * Hkv + hk) * B + (j - tail0)) * Dh + d;
                if (d < Dh)
                    for (int e = 0; e < 4; e++) {
                        k[e] = __half2float(((const __half *)P.c.k_tail)[at + e]);
                        v[e] = __half2float(((const __half *)P.c.v_tail)[at + e]);
                    }
            } else {
                const int id = kv8_block(P.c, P.b, s, j / B, P.err);
                if (id < 0) continue;
                const int64_t at = (((int64_t)id * Hkv + hk) * B + j % B) * Dh + d;
                ks = P.c.k_scale[(int64_t)id * Hkv + hk];
                vs = P.c.v_scale[(int64_t)id * Hkv + hk];
                if (d < Dh)
                    for (int e = 0; e < 4; e++) {
                        k[e] = (float)((const __nv_fp8_e4m3 *)P.c.k)[at + e];
                        v[e] = (float)((const __nv_fp8_e4m3 *)P.c.v)[at + e];
                    }
            }
            float x = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
            x = warp_sum(x) * (ks * P.a.scale);
            if (pos - j < P.a.rel_extent)
                x += P.a.rel_logits[((int64_t)n * H + h) * P.a.rel_extent + pos - j] * (P.a.tau ? P.a.tau[n] : 1.0f);
            const float mn = fmaxf(m, x);
            if (mn == -INFINITY) continue;
            const float f = expf(m - mn), p = expf(x - mn);
            m = mn;
            l = l * f + p;
            for (int e = 0; e < 4; e++) o[e] = o[e] * f + p * vs * v[e];
        }
    }
    if (d < Dh)
        for (int e = 0; e < 4; e++) ((T *)P.a.out)[((int64_t)n * H + h) * Dh + d + e] = (T)(l > 0.0f ? o[e] / l : 0.0f);
}

}  // namespace sepia

using namespace sepia;

static int k8_check(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a) {
    const char *what = "kv8_attn";
    if (!kv8_check(c, b, what)) return 0;
    if (!a) return fail("%s: null argument", what);
    if (a->n_heads <= 0 || a->n_heads % c->n_kv_heads)
        return fail("%s: %d query heads over %d KV heads", what, a->n_heads, c->n_kv_heads);
    if (a->window < 0 || a->rel_extent < 0) return fail("%s: negative window or rel_extent", what);
    return 1;
}

extern "C" size_t sepia_cuda_kv8_attn_ws_bytes(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a) {
    return k8_check(c, b, a) ? 16 : 0;
}

extern "C" int sepia_cuda_kv8_attn(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a, void *ws,
                                   size_t ws_bytes, void *stream) {
    const char *what = "kv8_attn";
    if (!k8_check(c, b, a)) return 0;
    if (b->n_seqs == 0 || b->n_tokens == 0 || b->max_new == 0) return 1;
    if (!a->q || !a->out) return fail("%s: null q or out", what);
    if (a->q_stride < (int64_t)a->n_heads * c->head_dim) return fail("%s: q_stride is shorter than a token", what);
    if (a->rel_extent && !a->rel_logits) return fail("%s: rel_extent without rel_logits", what);
    const size_t need = sepia_cuda_kv8_attn_ws_bytes(c, b, a);
    if (!ws || ws_bytes < need) return fail("%s: workspace of %zu bytes < %zu needed", what, ws_bytes, need);
    K8Params P;
    P.c = *c;
    P.b = *b;
    P.a = *a;
    P.err = dev_info().err;
    const dim3 grid((unsigned)a->n_heads, (unsigned)b->max_new, (unsigned)b->n_seqs);
    const cudaError_t e = a->x_f16 ? launch_pdl(k_kv8_attn<__half>, grid, 32, 0, as_stream(stream), P)
                                   : launch_pdl(k_kv8_attn<float>, grid, 32, 0, as_stream(stream), P);
    return check(e, "kv8_attn launch");
}
