// sepia_b200/csrc/kv8_append.cu -- new keys and values into the paged 8-bit
// cache, with the norms of queries and keys and the position rotation on
// the way (sepia_cuda_kv8_append; layout and rules in include/sepia_cuda.h).
//
// A block is rounded to 8 bits when it is full, so a CTA owns one block of
// one KV head of K or of V: it takes the rows that the step brings and those
// that wait in the tail, and either writes e4m3 codes with the block's scale
// or puts the new rows into the tail. A warp owns whole rows (4 dims a
// lane), so a norm is one warp reduction, and a rotation partner is in the
// same lane or one shuffle away. Further CTAs norm, rotate and scale the
// queries.
//
// A prompt is bound by HBM and, close behind, by instructions (a norm is a
// warp reduction for 4 values a lane): 8192 tokens, 64 heads over 8, fp32, 120
// us, 5.2 TB/s with 69 % of the issue slots busy. One token is latency, 4.0 us:
// launch, lengths, rows (one round of loads for a whole block), norm, store.
// 128-thread CTAs lost on every size (one token 7.8 us, 8192 tokens 144).
#include "kv8.cuh"
#include "runtime.h"

#include <cuda_fp8.h>

namespace sepia {

constexpr int kApThreads = 256;
constexpr int kApWarps = kApThreads / 32;
constexpr int kApQRows = 4;                 // query rows per warp

struct ApParams {
    SepiaKv8Cache c;
    SepiaKv8Step b;
    SepiaKv8Append a;
    int touched;             // blocks that a sequence's new tokens may touch
    int q_items;             // query CTAs per sequence
    int kv_ctas;             // CTAs of keys and values, before those of queries
    int vec_k, vec_v, vec_q; // the tensor's rows allow one vector load per lane
    double inv_dh;           // 1 / head_dim
    int *err;
};

template <typename T>
struct Vec4;
template <>
struct Vec4<float> { using type = float4; };
template <>
struct Vec4<__half> { using type = uint2; };

// 4 consecutive elements as fp32
template <typename T>
__device__ __forceinline__ void load4(const T *p, int vec, float (&x)[4]) {
    if (vec) {
        typename Vec4<T>::type raw = *reinterpret_cast<const typename Vec4<T>::type *>(p);
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (float)e[i];
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (float)p[i];
    }
}

// fp16 with magnitudes above the largest finite value saturated; NaN stays NaN
__device__ __forceinline__ __half sat_half(__half h) {
    const unsigned short u = __half_as_ushort(h);
    return (u & 0x7fffu) == 0x7c00u ? __ushort_as_half((unsigned short)(u - 1u)) : h;
}
__device__ __forceinline__ __half to_half(float x) { return sat_half(__float2half_rn(x)); }
__device__ __forceinline__ __half to_half(double x) { return sat_half(__float2half_rn((float)x)); }

// The smallest power of two s with amax / s <= 448 = 1.75 * 2^8. amax is the
// magnitude of an fp16 number, so it is a normal fp32 number or zero.
__device__ __forceinline__ float block_scale(float amax) {
    if (!(amax > 0.0f)) return 1.0f;
    const uint32_t u = __float_as_uint(amax);
    return __uint_as_float((((u >> 23) - 8u) + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u)) << 23);
}

// 1/sqrt(mean square + eps) of a warp's row from its lanes' sums of squares
__device__ __forceinline__ float inv_rms(float s, double inv_dh, float eps) {
    return rsqrtf(fmaf(warp_sum(s), (float)inv_dh, eps));
}
__device__ __forceinline__ double inv_rms(double s, double inv_dh, float eps) {
    return rsqrt(fma(warp_sum_d(s), inv_dh, (double)eps));
}

// RMS norm of the warp's row (w: the lane's weights), then the rotation; a
// lane owns dims 4*lane ..+3. Queries are worked out in fp32, keys in fp64:
// a key is rounded to fp16 and then to 8 bits, and with fp32 noise before
// them some of these roundings would go the other way.
template <typename R>
__device__ __forceinline__ void norm_rotate(R (&x)[4], const float *w, const SepiaKv8Append &a, double inv_dh, const float2 *cs) {
    const int lane = threadIdx.x & 31, d = 4 * lane;
    if (w) {
        R s = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) s += x[i] * x[i];
        s = inv_rms(s, inv_dh, a.eps);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = (R)w[i] * (x[i] * s);
    }
    if (cs) {                                          // the position's cosines and sines; the whole warp
        if (a.rot_adjacent) {
            if (d < a.rot_dim) {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float2 t = cs[(d + i) / 2];
                    const R u = x[i], v = x[i + 1];
                    x[i] = u * (R)t.x - v * (R)t.y;
                    x[i + 1] = v * (R)t.x + u * (R)t.y;
                }
            }
        } else {
            const int half = a.rot_dim / 2, hl = half / 4;   // the partner sits hl lanes away
            const bool low = d < half;
            const int from = low ? lane + hl : lane - hl;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const R y = __shfl_sync(0xffffffffu, x[i], from & 31);
                if (d < a.rot_dim) {
                    const float2 t = cs[low ? d + i : d - half + i];
                    x[i] = low ? x[i] * (R)t.x - y * (R)t.y : x[i] * (R)t.x + y * (R)t.y;
                }
            }
        }
    }
}

// The position's row of the rotation table; NULL (and the error word) past its end
__device__ __forceinline__ const float2 *rotation_row(const SepiaKv8Append &a, int pos, int *err) {
    if (!a.rot_dim) return nullptr;
    if (pos < a.rot_positions) return reinterpret_cast<const float2 *>(a.rotation) + (int64_t)pos * (a.rot_dim / 2);
    set_error(err, kErrBadArgs);
    return nullptr;
}

// MR: rows of a block per warp. A kernel for each block size: with one for
// blocks of 64 the shorter ones ran through rows that they do not have (48
// tokens, blocks of 32: 10.0 us, 7.8 now; ragged pieces, blocks of 16: 21.5, 16.2).
// Blocks of 64 keep 8 rows in flight at 64 registers a thread and spill 16 to 23 words.
template <typename T, int MR>
__global__ void __launch_bounds__(kApThreads, MR == 2 ? 5 : 4) k_kv8_append(const ApParams P) {
    __shared__ float s_amax[kApWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, d = 4 * lane;
    constexpr int B = MR * kApWarps;
    const int Dh = P.c.head_dim, Hkv = P.c.n_kv_heads;
    griddep_wait();
    griddep_launch();
    if ((int)blockIdx.x >= P.kv_ctas) {
        // ---- queries: rows (token, head) of one sequence ----
        const int item = blockIdx.x - P.kv_ctas;
        const int s = item / P.q_items, H = P.a.n_heads;
        const Kv8Seq sq = kv8_seq(P.c, P.b, s, P.err);
        const int first = ((item - s * P.q_items) * kApWarps + warp) * kApQRows;
        if (sq.add < 0) {                              // idle or out of bounds: zeros, of more than max_new rows too
            kv8_zero_rows((T *)P.a.q_out, sq.n0, sq.rows, H * Dh, (unsigned)(item - s * P.q_items) * kApThreads + tid,
                          (unsigned)P.q_items * kApThreads);
            return;
        }
        const int rows = sq.rows * H;
        if (first >= rows) return;                     // the whole warp
        const int i0 = first / H, h0 = first - i0 * H; // rows are (token, head); the next row's by counting on
        float x[kApQRows][4], w[4] = {}, f[kApQRows];
        if (P.a.q_norm && d < Dh)
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = P.a.q_norm[d + e];
        int i = i0, h = h0;
#pragma unroll
        for (int j = 0; j < kApQRows; j++) {
#pragma unroll
            for (int e = 0; e < 4; e++) x[j][e] = 0.0f;
            f[j] = 1.0f;
            if (first + j < rows) {
                if (d < Dh) load4((const T *)P.a.q + (int64_t)(sq.n0 + i) * P.a.q_stride + h * Dh + d, P.vec_q, x[j]);
                if (P.a.q_scale) f[j] = P.a.q_scale[sq.n0 + i];
            }
            if (++h == H) h = 0, i++;
        }
        i = i0, h = h0;
#pragma unroll
        for (int j = 0; j < kApQRows; j++) {
            if (first + j < rows) {                    // the whole warp
                norm_rotate(x[j], P.a.q_norm ? w : nullptr, P.a, P.inv_dh, rotation_row(P.a, sq.held + i, P.err));
                if (d < Dh) {
                    T y[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) y[e] = (T)(x[j][e] * f[j]);
                    *reinterpret_cast<typename Vec4<T>::type *>((T *)P.a.q_out + ((int64_t)(sq.n0 + i) * H + h) * Dh + d) =
                        *reinterpret_cast<const typename Vec4<T>::type *>(y);
                }
            }
            if (++h == H) h = 0, i++;
        }
        return;
    }
    // ---- keys (even) or values (odd) of one block of one head ----
    int item = blockIdx.x;
    const bool is_v = item & 1;
    item >>= 1;
    const int hk = item % Hkv;
    item /= Hkv;
    const int t = item % P.touched, s = item / P.touched;
    const Kv8Seq sq = kv8_seq(P.c, P.b, s, P.err);
    if (sq.add <= 0) return;
    const int total = sq.held + sq.add;
    const int b0 = sq.held / B, r0 = sq.held - b0 * B, last = total / B, tail_rows = total - last * B;
    const T *x_in = (const T *)(is_v ? P.a.v : P.a.k);
    const int64_t stride = is_v ? P.a.v_stride : P.a.k_stride;
    const int vec = is_v ? P.vec_v : P.vec_k;
    const bool exact = !is_v && (P.a.k_norm || P.a.rot_dim);   // else the row is rounded as it is
    float w[4] = {};
    if (!is_v && P.a.k_norm && d < Dh)
#pragma unroll
        for (int e = 0; e < 4; e++) w[e] = P.a.k_norm[d + e];
    __half *tail = (__half *)(is_v ? P.c.v_tail : P.c.k_tail) + ((int64_t)sq.slot * Hkv + hk) * B * Dh;
    uint8_t *codes = (uint8_t *)(is_v ? P.c.v : P.c.k);
    float *scales = is_v ? P.c.v_scale : P.c.k_scale;

    for (int blk = b0 + t;;) {
        const bool full = blk < last;
        if (!full && (blk > last || tail_rows == 0)) return;
        // With tail rows in its first block, the first block's CTA also
        // writes the last block's tail, after it has read the old rows.
        if (!full && blk != b0 && r0 && t) return;
        const int lo = blk == b0 ? r0 : 0;             // rows below wait in the tail
        const int hi = full ? B : tail_rows;
        const int base = blk * B - sq.held;            // row r of the block is new token base + r
        // a tail's warps without a new row are done
        if (!full && (hi - 1 - warp < 0 || (hi - 1 - warp) / kApWarps * kApWarps + warp < lo)) return;
        // every row first, new ones and (where the block ends) those of the tail: one round of loads
        float x[MR][4];
#pragma unroll
        for (int j = 0; j < MR; j++) {
            const int r = warp + kApWarps * j;
            x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.0f;
            if (r >= hi || d >= Dh) continue;
            if (r >= lo) {
                load4(x_in + (int64_t)(sq.n0 + base + r) * stride + hk * Dh + d, vec, x[j]);
            } else if (full) {
                load4(tail + r * Dh + d, 1, x[j]);
            }
        }
        __half2 y[MR][2];
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < MR; j++) {
            const int r = warp + kApWarps * j;
            if (exact && r >= lo && r < hi) {          // the whole warp
                double z[4] = {x[j][0], x[j][1], x[j][2], x[j][3]};
                norm_rotate(z, P.a.k_norm ? w : nullptr, P.a, P.inv_dh, rotation_row(P.a, sq.held + base + r, P.err));
                y[j][0] = __halves2half2(to_half(z[0]), to_half(z[1]));
                y[j][1] = __halves2half2(to_half(z[2]), to_half(z[3]));
            } else {
                y[j][0] = __halves2half2(to_half(x[j][0]), to_half(x[j][1]));
                y[j][1] = __halves2half2(to_half(x[j][2]), to_half(x[j][3]));
            }
            if (!full && r >= lo && r < hi && d < Dh) {
                uint2 raw;
                raw.x = *reinterpret_cast<const uint32_t *>(&y[j][0]);
                raw.y = *reinterpret_cast<const uint32_t *>(&y[j][1]);
                *reinterpret_cast<uint2 *>(tail + r * Dh + d) = raw;
            }
            const float2 f0 = __half22float2(y[j][0]), f1 = __half22float2(y[j][1]);
            amax = fmaxf(amax, fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y))));
        }
        if (!full) return;
        amax = warp_max(amax);
        if (lane == 0) s_amax[warp] = amax;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kApWarps; w++) amax = fmaxf(amax, s_amax[w]);
        const float scale = block_scale(amax), inv = 1.0f / scale;
        const int id = kv8_block(P.c, P.b, s, blk, P.err);
        if (id >= 0) {
            uint8_t *o = codes + ((int64_t)id * Hkv + hk) * B * Dh;
#pragma unroll
            for (int j = 0; j < MR; j++) {
                const int r = warp + kApWarps * j;
                if (r < B && d < Dh) {
                    float2 f0 = __half22float2(y[j][0]), f1 = __half22float2(y[j][1]);
                    f0.x *= inv; f0.y *= inv; f1.x *= inv; f1.y *= inv;
                    const uint32_t lo8 = __nv_cvt_float2_to_fp8x2(f0, __NV_SATFINITE, __NV_E4M3);
                    const uint32_t hi8 = __nv_cvt_float2_to_fp8x2(f1, __NV_SATFINITE, __NV_E4M3);
                    *reinterpret_cast<uint32_t *>(o + r * Dh + d) = lo8 | (hi8 << 16);
                }
            }
            if (tid == 0) scales[(int64_t)id * Hkv + hk] = scale;
        }
        if (t || !r0 || blk == last) return;
        __syncthreads();                               // s_amax is free again, every old tail row is read
        blk = last;
    }
}

int kv8_check(const SepiaKv8Cache *c, const SepiaKv8Step *b, const char *what) {
    if (!c || !b) return fail("%s: null argument", what);
    if (c->block != 16 && c->block != 32 && c->block != 64)
        return fail("%s: block of %d tokens (16, 32 or 64)", what, c->block);
    if (c->head_dim <= 0 || c->head_dim > kKv8MaxDh || c->head_dim % 16)
        return fail("%s: head_dim %d (a multiple of 16 up to %d)", what, c->head_dim, kKv8MaxDh);
    if (c->n_blocks <= 0 || c->n_slots <= 0 || c->n_kv_heads <= 0)
        return fail("%s: bad cache sizes: %d blocks, %d slots, %d KV heads", what, c->n_blocks, c->n_slots,
                    c->n_kv_heads);
    if (!c->k || !c->v || !c->k_scale || !c->v_scale || !c->k_tail || !c->v_tail)
        return fail("%s: null cache pointer", what);
    if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) |
         reinterpret_cast<uintptr_t>(c->k_tail) | reinterpret_cast<uintptr_t>(c->v_tail)) & 15)
        return fail("%s: cache arrays must be 16-byte aligned", what);
    if (b->n_seqs < 0 || b->n_tokens < 0 || b->max_new < 0 || b->max_kv < 0 || b->table_cols < 0)
        return fail("%s: negative step size", what);
    if (!b->start && b->n_tokens != b->n_seqs)
        return fail("%s: %d tokens of %d sequences need `start`", what, b->n_tokens, b->n_seqs);
    if (b->n_seqs && (!b->table || !b->kv_len)) return fail("%s: null step pointer", what);
    if ((int64_t)b->max_kv + c->block > INT32_MAX) return fail("%s: max_kv %d too large", what, b->max_kv);
    return 1;
}

// One vector load per lane: the row's first element and every row start on the vector's boundary.
static int rows_vec(const void *p, int64_t stride, int x_f16) {
    const int64_t b = x_f16 ? 8 : 16, sz = x_f16 ? 2 : 4;
    return reinterpret_cast<uintptr_t>(p) % b == 0 && (stride * sz) % b == 0;
}

template <typename T>
static int ap_launch(const ApParams &P, unsigned ctas, cudaStream_t st) {
    const int rows = P.c.block / kApWarps;
    const cudaError_t e = rows == 2   ? launch_pdl(k_kv8_append<T, 2>, ctas, kApThreads, 0, st, P)
                          : rows == 4 ? launch_pdl(k_kv8_append<T, 4>, ctas, kApThreads, 0, st, P)
                                      : launch_pdl(k_kv8_append<T, 8>, ctas, kApThreads, 0, st, P);
    return check(e, "kv8_append launch");
}

}  // namespace sepia

using namespace sepia;

extern "C" int sepia_cuda_kv8_append(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Append *a,
                                     void *stream) {
    const char *what = "kv8_append";
    if (!kv8_check(c, b, what)) return 0;
    if (!a) return fail("%s: null argument", what);
    if (b->n_seqs == 0 || b->n_tokens == 0 || b->max_new == 0) return 1;
    const int64_t kv_row = (int64_t)c->n_kv_heads * c->head_dim;
    if (!a->k || !a->v) return fail("%s: null k or v", what);
    if (a->k_stride < kv_row || a->v_stride < kv_row)
        return fail("%s: a token stride is shorter than %lld elements", what, (long long)kv_row);
    if (a->q) {
        if (a->n_heads <= 0 || !a->q_out) return fail("%s: q needs n_heads and q_out", what);
        if (a->q_stride < (int64_t)a->n_heads * c->head_dim) return fail("%s: q_stride is shorter than a token", what);
        if (!rows_vec(a->q_out, 0, a->x_f16)) return fail("%s: q_out must be aligned to 4 elements", what);
    }
    if (a->rot_dim) {
        if (a->rot_dim < 0 || a->rot_dim % 8 || a->rot_dim > c->head_dim)
            return fail("%s: rot_dim %d (a multiple of 8 up to head_dim)", what, a->rot_dim);
        if (!a->rotation || a->rot_positions <= 0) return fail("%s: rotation without a table", what);
        if (reinterpret_cast<uintptr_t>(a->rotation) & 7) return fail("%s: rotation must be 8-byte aligned", what);
    }
    ApParams P;
    P.c = *c;
    P.b = *b;
    P.a = *a;
    P.err = dev_info().err;
    P.inv_dh = 1.0 / (double)c->head_dim;
    P.touched = (c->block - 1 + b->max_new - 1) / c->block + 1;
    const int64_t rows = a->q ? (int64_t)b->max_new * a->n_heads : 0;
    const int64_t per = kApWarps * kApQRows;
    const int64_t kv_ctas = (int64_t)b->n_seqs * P.touched * c->n_kv_heads * 2;
    const int64_t q_items = (rows + per - 1) / per, all = kv_ctas + b->n_seqs * q_items;
    if (all > INT32_MAX || rows > INT32_MAX - per) return fail("%s: step too large", what);
    P.kv_ctas = (int)kv_ctas;
    P.q_items = (int)(q_items ? q_items : 1);
    P.vec_k = rows_vec(a->k, a->k_stride, a->x_f16);
    P.vec_v = rows_vec(a->v, a->v_stride, a->x_f16);
    P.vec_q = a->q ? rows_vec(a->q, a->q_stride, a->x_f16) : 0;
    return a->x_f16 ? ap_launch<__half>(P, (unsigned)all, as_stream(stream)) : ap_launch<float>(P, (unsigned)all, as_stream(stream));
}
