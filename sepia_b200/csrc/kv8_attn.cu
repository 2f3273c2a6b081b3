// sepia_b200/csrc/kv8_attn.cu -- attention of new tokens over the paged
// 8-bit cache (sepia_cuda_kv8_attn; rules in include/sepia_cuda.h).
//
// One pass over the visible keys with the running maximum and sum of the
// softmax. The heads of a KV head's group, and the new tokens, are the rows
// of one matrix product, so every code crosses HBM once for all of them.
//
//   Work      grid (split, KV head x row tile, sequence); a CTA owns a chunk
//             of positions, its warps take 16-key tiles of it in turn, each
//             with its own maximum, sum and output, merged at the end. A
//             second kernel merges the chunks of a long context, many rows
//             at once (as the last step of the last CTA of each KV head the
//             same sum took 65 us of 95 at 1 x 32768: 8 CTAs at work).
//   Operands  mma m16n8k16 in fp16 with fp32 sums. e4m3 codes are fp16
//             numbers exactly; block scales multiply the score and the
//             weight. fp32 rows: q and the weight are split into two fp16
//             terms (22 bits) that sit in the two halves of the 16-row
//             operand, 8 rows a tile; fp16 rows: 16 rows a tile.
//   Layout    the dims of a k step and of an output column are permuted so
//             that a lane's codes are 16 consecutive bytes of a key row (K)
//             or of four key rows (V). Each lane copies just the bytes that it
//             will use into a ring of its own in shared memory (cp.async), so
//             no lane waits for another and nothing conflicts.
#include "kv8.cuh"
#include "runtime.h"

#include <cuda_fp16.h>
#include <algorithm>

namespace sepia {

constexpr int kK8Warps = 4;
constexpr int kK8Threads = 32 * kK8Warps;
constexpr int kK8Tile = 16;              // keys per warp step
constexpr int kK8CtasPerSm = 3;
constexpr float kLog2e = 1.4426950408889634f;
// A weight's exponent may pass the running maximum by this before the
// maximum is moved (and the output rescaled): weights reach e^5.5 = 245,
// times kPOne below 65504, the largest fp16.
constexpr float kSlack = 5.5f;
// Weights are handed to the tensor core times 2^7: with the slack that keeps
// 22 bits of a weight down to 2^-20 of the largest.
constexpr float kPOne = 128.0f;

struct K8Params {
    SepiaKv8Cache c;
    SepiaKv8Step b;
    SepiaKv8Attn a;
    int G, row_tiles, splits, chunk;     // chunk: positions per split, a multiple of kK8Tile * kK8Warps
    float *part;                         // [n_seqs, n_kv_heads * row_tiles, splits, rows of a tile, Dh + 2]
    int *err;
};

__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_half2_hi(uint32_t two) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(two));
    return r;
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// cp.async of `bytes` (16 or 8 or 4) or of zeros
template <int N>
__device__ __forceinline__ void cp_async_or_zero(uint32_t dst, const void *src, bool on) {
    const int n = on ? N : 0;
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(N), "r"(n) : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

template <typename T, int DP>
struct K8Cfg {
    static constexpr bool kTwo = sizeof(T) == 4;      // two fp16 terms per row
    static constexpr int RT = kTwo ? 8 : 16;          // rows of a tile
    static constexpr int RL = kTwo ? 1 : 2;           // rows of a lane
    static constexpr int KW = DP / 64;                // 16-byte pieces of a key row per lane
    static constexpr int VB = DP / 8;                 // bytes of a value row per lane
    static constexpr int NT = DP / 8, KS = DP / 16;   // output columns of 8, k steps of 16
    static constexpr int kStages = kTwo ? 4 : 3;
    static constexpr int kKeyB = 2 * KW * 512, kValB = 4 * VB * 32, kBiasB = 4 * RL * 128;
    static constexpr int kStageB = kKeyB + kValB + kBiasB + 16;   // the last 16: the block's scales
    static constexpr int kMergeB = kK8Warps * RT * (DP + 2) * 4;
    static constexpr int kSmem = kStages * kStageB * kK8Warps > kMergeB ? kStages * kStageB * kK8Warps : kMergeB;
};

template <typename T, int DP>
__global__ void __launch_bounds__(kK8Threads, kK8CtasPerSm) k_kv8_attn(const K8Params P) {
    using F = K8Cfg<T, DP>;
    constexpr int RL = F::RL, RT = F::RT;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int split = blockIdx.x, s = blockIdx.z;
    const int hk = blockIdx.y / P.row_tiles, rt = blockIdx.y - hk * P.row_tiles;
    const int Dh = P.c.head_dim, B = P.c.block, H = P.a.n_heads, Hkv = P.c.n_kv_heads, G = P.G;
    griddep_wait();
    griddep_launch();
    const Kv8Seq sq = kv8_seq(P.c, P.b, s, P.err);
    const int rows = sq.rows * G - rt * RT;            // rows of this tile that exist (may exceed RT)
    if (rows <= 0) return;
    if (sq.add < 0) {                                  // idle or out of bounds: zeros
        if (split == 0)
            for (int i = tid; i < min(rows, RT) * Dh; i += kK8Threads) {
                const int R = rt * RT + i / Dh, t = R / G;
                ((T *)P.a.out)[((int64_t)(sq.n0 + t) * H + hk * G + (R - t * G)) * Dh + i % Dh] = (T)0.0f;
            }
        return;
    }
    // tokens of the tile, the positions that any of them sees, this CTA's chunk
    const int ta = rt * RT / G, tb = min(sq.add - 1, (rt * RT + RT - 1) / G);
    const int pa = sq.held + ta, pb = sq.held + tb;
    const int window = P.a.window, E = P.a.rel_extent;
    const int tail0 = (sq.held + sq.add) / B * B;
    const int lo = window ? max(0, pa - window + 1) / kK8Tile * kK8Tile : 0;
    const int n_act = (pb + 1 - lo + P.chunk - 1) / P.chunk;
    if (split >= n_act) return;
    const int c0 = lo + split * P.chunk, c1 = min(pb + 1, c0 + P.chunk);

    // ---- this lane's rows and their q operand ----
    int pos[RL], n_row[RL], h_row[RL];
    float qmul[RL], tau[RL];
    uint32_t qa[F::KS][4];
#pragma unroll
    for (int j = 0; j < RL; j++) {
        const int r = gid + 8 * j, R = min(rt * RT + r, sq.add * G - 1), t = R / G;
        const bool on = r < rows;
        n_row[j] = sq.n0 + t;
        pos[j] = sq.held + t;
        h_row[j] = hk * G + R - t * G;
        tau[j] = P.a.tau && on ? P.a.tau[n_row[j]] : 1.0f;
        const T *q = (const T *)P.a.q + (int64_t)n_row[j] * P.a.q_stride + (int64_t)h_row[j] * Dh;
        float x[F::KS][4], amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++) {
            const int d = 64 * (ks / 4) + 16 * tig + 4 * (ks % 4);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[ks][e] = on && d < Dh ? (float)q[d + e] : 0.0f;
                amax = fmaxf(amax, fabsf(x[ks][e]));
            }
        }
        if constexpr (F::kTwo) {
            // the row times a power of two that puts its largest in [2^13, 2^14): both terms stay normal fp16
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = amax > 0.0f ? max((int)(__float_as_uint(amax) >> 23) - 127, -100) : 13;
            const float f = __uint_as_float((uint32_t)(127 + 13 - ex) << 23);
            qmul[j] = P.a.scale * __uint_as_float((uint32_t)(127 - 13 + ex) << 23);
#pragma unroll
            for (int ks = 0; ks < F::KS; ks++) {
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const float u = x[ks][e] * f, v = x[ks][e + 1] * f;
                    const __half2 hi = __floats2half2_rn(u, v);
                    const float2 b = __half22float2(hi);
                    qa[ks][e] = *reinterpret_cast<const uint32_t *>(&hi);        // a0 / a2: rows 0-7
                    qa[ks][e + 1] = pack_half2(u - b.x, v - b.y);                // a1 / a3: rows 8-15
                }
            }
        } else {
            qmul[j] = P.a.scale;
#pragma unroll
            for (int ks = 0; ks < F::KS; ks++) {
                qa[ks][j] = pack_half2(x[ks][0], x[ks][1]);
                qa[ks][2 + j] = pack_half2(x[ks][2], x[ks][3]);
            }
        }
    }

    float O[F::NT][4], m[RL], l[RL], vref = 0.0f;
#pragma unroll
    for (int nt = 0; nt < F::NT; nt++) O[nt][0] = O[nt][1] = O[nt][2] = O[nt][3] = 0.0f;
#pragma unroll
    for (int j = 0; j < RL; j++) m[j] = -INFINITY, l[j] = 0.0f;

    // One 16-key tile at position t0. kf(n, ks, b0, b1): key fragment of keys
    // t0 + 8n + gid; vf(nt, b0, b1): value fragment; bias(j, i): term i of
    // this lane's row j, keys t0 + 2 tig + {0, 1, 8, 9}; clean(): values that
    // are not numbers to 0, and which of those keys had any.
    auto tile = [&](int t0, float ks_, float vs, auto kf, auto vf, auto bias, auto clean) {
        float S[2][4];
#pragma unroll
        for (int n = 0; n < 2; n++) {
            S[n][0] = S[n][1] = S[n][2] = S[n][3] = 0.0f;
#pragma unroll
            for (int ks = 0; ks < F::KS; ks++) {
                uint32_t b0, b1;
                kf(n, ks, b0, b1);
                mma16(S[n], qa[ks], b0, b1);
            }
        }
        const bool biased = E && pa - (t0 + kK8Tile - 1) < E;
        const bool masked = t0 + kK8Tile - 1 > pa || (window && t0 <= pb - window) || ks_ < 0.0f;
        float p[RL][4];
        bool grow = false;
        uint32_t seen = 0;                             // bit 4j + i: row j sees key i
#pragma unroll
        for (int j = 0; j < RL; j++) {
            const float f = ks_ * qmul[j];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int n = i >> 1, e = i & 1;
                const float x = F::kTwo ? S[n][e] + S[n][e + 2] : S[n][e + 2 * j];
                p[j][i] = x * f;
            }
            if (biased) {
#pragma unroll
                for (int i = 0; i < 4; i++) p[j][i] += bias(j, i) * tau[j];
            }
            if (masked) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int at = t0 + 2 * tig + (i & 1) + 8 * (i >> 1);
                    if (at > pos[j] || (window && at <= pos[j] - window) || ks_ < 0.0f) p[j][i] = -INFINITY;
                }
            }
            const float top = fmaxf(fmaxf(p[j][0], p[j][1]), fmaxf(p[j][2], p[j][3]));
#pragma unroll
            for (int i = 0; i < 4; i++) seen |= p[j][i] == -INFINITY ? 0u : 1u << (4 * j + i);
            grow |= top > m[j] + kSlack || (top > m[j] && m[j] < -1e30f);
        }
        float vmul = kPOne;
        if (vs > vref) {                               // the whole warp: scales are powers of two
            const float f = vref / vs;
#pragma unroll
            for (int nt = 0; nt < F::NT; nt++) O[nt][0] *= f, O[nt][1] *= f, O[nt][2] *= f, O[nt][3] *= f;
            vref = vs;
        } else {
            vmul = kPOne * (vs / vref);
        }
        if (__any_sync(0xffffffffu, grow)) {
            float f[RL];
#pragma unroll
            for (int j = 0; j < RL; j++) {
                float top = fmaxf(fmaxf(p[j][0], p[j][1]), fmaxf(p[j][2], p[j][3]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                top = fmaxf(top, m[j]);
                f[j] = top == -INFINITY ? 1.0f : exp2_fast((m[j] - top) * kLog2e);
                m[j] = top;
                l[j] *= f[j];
            }
#pragma unroll
            for (int nt = 0; nt < F::NT; nt++) {
                O[nt][0] *= f[0], O[nt][1] *= f[0];
                O[nt][2] *= f[RL - 1], O[nt][3] *= f[RL - 1];
            }
        }
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < RL; j++) {
            const float mj = m[j] == -INFINITY ? 0.0f : m[j];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                p[j][i] = exp2_fast((p[j][i] - mj) * kLog2e);
                l[j] += p[j][i];
                p[j][i] *= vmul;
            }
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const __half2 hi = __floats2half2_rn(p[j][2 * n], p[j][2 * n + 1]);
                w[2 * n + j] = *reinterpret_cast<const uint32_t *>(&hi);
                if constexpr (F::kTwo) {
                    const float2 b = __half22float2(hi);
                    w[2 * n + 1] = pack_half2(p[j][2 * n] - b.x, p[j][2 * n + 1] - b.y);
                }
            }
        }
        if (biased || masked) {
            // A value that is not a number must not reach a row that does not
            // see its key (0 * NaN): in a tile with hidden keys such values
            // count as 0, and a row that does see one gets a sum of NaN.
            if (__any_sync(0xffffffffu, seen != (1u << (4 * RL)) - 1u)) {
                uint32_t nan = clean();                // bit i: key i, among this lane's dims
                nan |= __shfl_xor_sync(0xffffffffu, nan, 4);
                nan |= __shfl_xor_sync(0xffffffffu, nan, 8);
                nan |= __shfl_xor_sync(0xffffffffu, nan, 16);
#pragma unroll
                for (int j = 0; j < RL; j++)
                    if (seen >> (4 * j) & nan) l[j] = __int_as_float(0x7fffffff);
            }
        }
#pragma unroll
        for (int nt = 0; nt < F::NT; nt++) {
            uint32_t b0, b1;
            vf(nt, b0, b1);
            mma16(O[nt], w, b0, b1);
        }
    };

    // ---- coded tiles: this warp's share of [c0, min(c1, tail0)), through its ring ----
    const int ce = min(c1, tail0);
    const int n_tiles = ce > c0 ? (ce - c0 + kK8Tile - 1) / kK8Tile : 0;
    const int mine = n_tiles > warp ? (n_tiles - warp + kK8Warps - 1) / kK8Warps : 0;
    uint8_t *ring = smem + warp * F::kStages * F::kStageB;
    const uint32_t ring_u = smem_u32(ring);
    int id_l = -1;
    float ks_l = -1.0f, vs_l = 1.0f;
    auto issue = [&](int i) {
        if (i < mine) {
            if ((i & 31) == 0) {                       // this lane's block of the next 32 tiles
                const int k = i + lane;
                if (k < mine) {
                    id_l = kv8_block(P.c, P.b, s, (c0 + (warp + kK8Warps * k) * kK8Tile) / B, P.err);
                    ks_l = id_l >= 0 ? P.c.k_scale[(int64_t)id_l * Hkv + hk] : -1.0f;
                    vs_l = id_l >= 0 ? P.c.v_scale[(int64_t)id_l * Hkv + hk] : 1.0f;
                }
            }
            const int id = __shfl_sync(0xffffffffu, id_l, i & 31);
            const float ks = __shfl_sync(0xffffffffu, ks_l, i & 31), vs = __shfl_sync(0xffffffffu, vs_l, i & 31);
            const int t0 = c0 + (warp + kK8Warps * i) * kK8Tile;
            const uint32_t st = ring_u + (i % F::kStages) * F::kStageB;
            const int64_t row0 = ((int64_t)max(id, 0) * Hkv + hk) * B + (t0 & (B - 1));
            const uint8_t *K = (const uint8_t *)P.c.k + row0 * Dh, *V = (const uint8_t *)P.c.v + row0 * Dh;
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int j = 0; j < F::KW; j++) {
                    const int d = 64 * j + 16 * tig;
                    cp_async_or_zero<16>(st + (n * F::KW + j) * 512 + lane * 16, d < Dh ? K + (gid + 8 * n) * Dh + d : K,
                                         d < Dh && id >= 0);
                }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int r = 2 * tig + (k & 1) + 8 * (k >> 1), d = gid * F::VB;
                cp_async_or_zero<F::VB>(st + F::kKeyB + k * (32 * F::VB) + lane * F::VB, d < Dh ? V + r * Dh + d : V,
                                        d < Dh && id >= 0);
            }
            if (E && pa - (t0 + kK8Tile - 1) < E) {
#pragma unroll
                for (int j = 0; j < RL; j++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int far = pos[j] - (t0 + 2 * tig + (k & 1) + 8 * (k >> 1));
                        const bool on = far >= 0 && far < E;
                        const float *src = P.a.rel_logits + ((int64_t)n_row[j] * H + h_row[j]) * E;
                        cp_async_or_zero<4>(st + F::kKeyB + F::kValB + (4 * j + k) * 128 + lane * 4, on ? src + far : src, on);
                    }
            }
            if (lane == 0)
                *reinterpret_cast<float2 *>(ring + (i % F::kStages) * F::kStageB + F::kKeyB + F::kValB + F::kBiasB) =
                    make_float2(ks, vs);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < F::kStages - 1; i++) issue(i);

    // ---- the tail's fp16 tiles, one a warp, while the ring fills ----
    {
        const int t0 = tail0 + kK8Tile * warp;
        if (t0 >= c0 && t0 < c1) {
            const int64_t at = (((int64_t)sq.slot * Hkv + hk) * B + (t0 - tail0)) * Dh;
            const __half *K = (const __half *)P.c.k_tail + at, *V = (const __half *)P.c.v_tail + at;
            const int held = sq.held + sq.add - t0;    // keys of the tile that exist
            uint4 v[4][F::VB / 8];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int r = 2 * tig + (k & 1) + 8 * (k >> 1), d = gid * F::VB;
#pragma unroll
                for (int j = 0; j < F::VB / 8; j++)
                    v[k][j] = r < held && d + 8 * j < Dh ? *reinterpret_cast<const uint4 *>(V + r * Dh + d + 8 * j)
                                                         : make_uint4(0, 0, 0, 0);
            }
            tile(
                t0, 1.0f, 1.0f,
                [&](int n, int ks, uint32_t &b0, uint32_t &b1) {
                    const int d = 64 * (ks / 4) + 16 * tig + 4 * (ks % 4), r = gid + 8 * n;
                    const uint2 x = r < held && d < Dh ? *reinterpret_cast<const uint2 *>(K + r * Dh + d) : make_uint2(0, 0);
                    b0 = x.x;
                    b1 = x.y;
                },
                [&](int nt, uint32_t &b0, uint32_t &b1) {
                    const uint32_t *a = reinterpret_cast<const uint32_t *>(v[0]), *b = reinterpret_cast<const uint32_t *>(v[1]);
                    const uint32_t *c = reinterpret_cast<const uint32_t *>(v[2]), *d = reinterpret_cast<const uint32_t *>(v[3]);
                    const uint32_t sel = nt & 1 ? 0x7632 : 0x5410;
                    b0 = __byte_perm(a[nt / 2], b[nt / 2], sel);
                    b1 = __byte_perm(c[nt / 2], d[nt / 2], sel);
                },
                [&](int j, int i) {
                    const int far = pos[j] - (t0 + 2 * tig + (i & 1) + 8 * (i >> 1));
                    return far >= 0 && far < E ? P.a.rel_logits[((int64_t)n_row[j] * H + h_row[j]) * E + far] : 0.0f;
                },
                [&]() {
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        uint32_t *x = reinterpret_cast<uint32_t *>(v[k]);
#pragma unroll
                        for (int e = 0; e < F::VB / 2; e++) {
                            const uint32_t at = __vcmpgtu2(x[e] & 0x7fff7fffu, 0x7c007c00u);
                            x[e] &= ~at;
                            nan |= at ? 1u << k : 0u;
                        }
                    }
                    return nan;
                });
        }
    }

    for (int i = 0; i < mine; i++) {
        __syncwarp();                                  // every lane is done with the stage that is filled next
        issue(i + F::kStages - 1);
        cp_async_wait<F::kStages - 1>();
        __syncwarp();
        const uint8_t *st = ring + (i % F::kStages) * F::kStageB;
        const float2 sc = *reinterpret_cast<const float2 *>(st + F::kKeyB + F::kValB + F::kBiasB);
        uint32_t kw[2][F::KW * 4], vw[4][F::VB / 4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int j = 0; j < F::KW; j++)
                *reinterpret_cast<uint4 *>(&kw[n][4 * j]) = *reinterpret_cast<const uint4 *>(st + (n * F::KW + j) * 512 + lane * 16);
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint8_t *src = st + F::kKeyB + k * (32 * F::VB) + lane * F::VB;
            if constexpr (F::VB == 16) *reinterpret_cast<uint4 *>(vw[k]) = *reinterpret_cast<const uint4 *>(src);
            else *reinterpret_cast<uint2 *>(vw[k]) = *reinterpret_cast<const uint2 *>(src);
        }
        tile(
            c0 + (warp + kK8Warps * i) * kK8Tile, sc.x, sc.y,
            [&](int n, int ks, uint32_t &b0, uint32_t &b1) {
                b0 = e4m3x2_to_half2(kw[n][ks]);
                b1 = e4m3x2_to_half2_hi(kw[n][ks]);
            },
            [&](int nt, uint32_t &b0, uint32_t &b1) {
                const uint32_t sel = nt & 2 ? 0x7362 : 0x5140;
                const uint32_t x = __byte_perm(vw[0][nt / 4], vw[1][nt / 4], sel);
                const uint32_t y = __byte_perm(vw[2][nt / 4], vw[3][nt / 4], sel);
                b0 = nt & 1 ? e4m3x2_to_half2_hi(x) : e4m3x2_to_half2(x);
                b1 = nt & 1 ? e4m3x2_to_half2_hi(y) : e4m3x2_to_half2(y);
            },
            [&](int j, int k) {
                return *reinterpret_cast<const float *>(st + F::kKeyB + F::kValB + (4 * j + k) * 128 + lane * 4);
            },
            [&]() {
                uint32_t nan = 0;
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int e = 0; e < F::VB / 4; e++) {
                        const uint32_t at = __vcmpeq4(vw[k][e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        vw[k][e] &= ~at;
                        nan |= at ? 1u << k : 0u;
                    }
                return nan;
            });
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- merge the warps: rows of m, l and the output, in warp order ----
    float *mg = reinterpret_cast<float *>(smem) + warp * RT * (DP + 2);
#pragma unroll
    for (int j = 0; j < RL; j++) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
        float *o = mg + (gid + 8 * j) * (DP + 2);
        if (tig == 0) o[0] = m[j], o[1] = l[j];
        const float f = vref / kPOne;
#pragma unroll
        for (int nt = 0; nt < F::NT; nt++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                o[2 + (2 * tig + e) * F::VB + nt] = f * (F::kTwo ? O[nt][e] + O[nt][e + 2] : O[nt][e + 2 * j]);
    }
    __syncthreads();
    const int live = min(rows, RT), group = blockIdx.z * gridDim.y + blockIdx.y;
    const int64_t stride = (int64_t)RT * (Dh + 2);
    float *part = P.part + (int64_t)group * P.splits * stride;
    auto put = [&](int r, int d, float o, float sum) {
        const int R = rt * RT + r, t = R / G;
        ((T *)P.a.out)[((int64_t)(sq.n0 + t) * H + hk * G + (R - t * G)) * Dh + d] = (T)(sum == 0.0f ? 0.0f : o / sum);
    };
    for (int i = tid; i < live * Dh; i += kK8Threads) {
        const int r = i / Dh, d = i - r * Dh;
        const float *o = reinterpret_cast<const float *>(smem) + r * (DP + 2);
        float M = -INFINITY, L = 0.0f, A = 0.0f;
#pragma unroll
        for (int w = 0; w < kK8Warps; w++) M = fmaxf(M, o[w * RT * (DP + 2)]);
#pragma unroll
        for (int w = 0; w < kK8Warps; w++) {
            const float *ow = o + w * RT * (DP + 2);
            const float f = ow[0] == -INFINITY ? 0.0f : exp2_fast((ow[0] - M) * kLog2e);
            L += f * ow[1];
            A += f * ow[2 + d];
        }
        if (n_act == 1) {
            put(r, d, A, L);
        } else {
            float *to = part + split * stride + r * (Dh + 2);
            if (d == 0) to[0] = M, to[1] = L;
            to[2 + d] = A;
        }
    }
}

// Merges the chunks of a row, in chunk order within each of the W warps that
// share the row, then across the warps. One CTA does kK8Warps / W rows.
template <typename T, int W>
__global__ void __launch_bounds__(kK8Threads) k_kv8_merge(const K8Params P) {
    constexpr int RT = sizeof(T) == 4 ? 8 : 16;
    __shared__ float s_part[W > 1 ? kK8Warps : 1][kKv8MaxDh + 2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, d = 4 * lane;
    const int Dh = P.c.head_dim, H = P.a.n_heads, G = P.G, s = blockIdx.y;
    griddep_wait();
    griddep_launch();
    const int at = blockIdx.x * (kK8Warps / W) + warp / W, h = at % H, t = at / H;
    const Kv8Seq sq = kv8_seq(P.c, P.b, s, nullptr);
    if (sq.add < 0 || t >= sq.add) return;             // with W > 1 the whole CTA
    // the row's tile, and the chunks that k_kv8_attn cut for it
    const int hk = h / G, R = t * G + h - hk * G, rt = R / RT, r = R - rt * RT;
    const int ta = rt * RT / G, tb = min(sq.add - 1, (rt * RT + RT - 1) / G);
    const int lo = P.a.window ? max(0, sq.held + ta - P.a.window + 1) / kK8Tile * kK8Tile : 0;
    const int n_act = (sq.held + tb + 1 - lo + P.chunk - 1) / P.chunk;
    if (n_act <= 1) return;
    const int group = s * P.c.n_kv_heads * P.row_tiles + hk * P.row_tiles + rt;
    const int64_t stride = (int64_t)RT * (Dh + 2);
    const float *part = P.part + (int64_t)group * P.splits * stride + (int64_t)r * (Dh + 2);
    float M = -INFINITY, L = 0.0f, A[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = lane; k < n_act; k += 32) M = fmaxf(M, part[k * stride]);
    M = warp_max(M);
    const int per = (n_act + W - 1) / W, k0 = (warp % W) * per, k1 = min(n_act, k0 + per);
    constexpr int kAhead = 8;                          // chunks in flight per warp
    for (int k = k0; k < k1; k += kAhead) {
        float2 x[kAhead][2], ml[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float2 *p = reinterpret_cast<const float2 *>(part + min(k + i, k1 - 1) * stride);
            ml[i] = p[0];
            x[i][0] = d < Dh ? p[1 + d / 2] : make_float2(0.0f, 0.0f);
            x[i][1] = d < Dh ? p[2 + d / 2] : make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            if (k + i >= k1) break;
            const float f = ml[i].x == -INFINITY ? 0.0f : exp2_fast((ml[i].x - M) * kLog2e);
            L += f * ml[i].y;
            A[0] += f * x[i][0].x, A[1] += f * x[i][0].y, A[2] += f * x[i][1].x, A[3] += f * x[i][1].y;
        }
    }
    if constexpr (W > 1) {
        if (d < Dh)
            for (int e = 0; e < 4; e++) s_part[warp][2 + d + e] = A[e];
        if (lane == 0) s_part[warp][0] = L;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int w = 1; w < W; w++) {
            L += s_part[w][0];
            if (d < Dh)
                for (int e = 0; e < 4; e++) A[e] += s_part[w][2 + d + e];
        }
    }
    if (d < Dh) {
        T *o = (T *)P.a.out + ((int64_t)(sq.n0 + t) * H + h) * Dh + d;
        for (int e = 0; e < 4; e++) o[e] = (T)(L == 0.0f ? 0.0f : A[e] / L);
    }
}

struct K8Plan {
    int G, row_tiles, splits, chunk;
    size_t bytes;
};

// Chunks: one wave of equal chunks over all CTA slots while that leaves a
// chunk at most kMaxChunk positions; longer work runs in several waves of
// kMaxChunk, so that ragged sequences even out.
static K8Plan k8_plan(const SepiaKv8Cache &c, const SepiaKv8Step &b, const SepiaKv8Attn &a) {
    constexpr int64_t kUnit = kK8Tile * kK8Warps, kMaxChunk = 1024;
    K8Plan p;
    const int rt = a.x_f16 ? 16 : 8;
    p.G = a.n_heads / c.n_kv_heads;
    p.row_tiles = (int)(((int64_t)b.max_new * p.G + rt - 1) / rt);
    const int64_t span = a.window ? std::min<int64_t>(b.max_kv, (int64_t)a.window + b.max_new + kK8Tile) : b.max_kv;
    const int64_t groups = (int64_t)b.n_seqs * c.n_kv_heads * p.row_tiles;
    const int64_t slots = (int64_t)(dev_info().sm_count > 0 ? dev_info().sm_count : 148) * kK8CtasPerSm;
    const int64_t one = (groups * span + slots - 1) / slots;
    p.chunk = (int)(std::min(kMaxChunk, std::max<int64_t>(one, 1)) + kUnit - 1) / kUnit * kUnit;
    p.splits = (int)std::max<int64_t>(1, (span + p.chunk - 1) / p.chunk);
    p.bytes = p.splits > 1 ? (size_t)groups * p.splits * rt * (c.head_dim + 2) * 4 : 0;
    return p;
}

template <typename T, int DP>
static int k8_launch(const K8Params &P, cudaStream_t st) {
    constexpr int smem = K8Cfg<T, DP>::kSmem;
    if (!ensure_smem((const void *)k_kv8_attn<T, DP>, smem)) return 0;
    const dim3 grid((unsigned)P.splits, (unsigned)(P.c.n_kv_heads * P.row_tiles), (unsigned)P.b.n_seqs);
    if (!check(launch_pdl(k_kv8_attn<T, DP>, grid, dim3(kK8Threads), smem, st, P), "kv8_attn launch")) return 0;
    if (P.splits == 1) return 1;
    // one warp per row while a row has few chunks, four beyond
    const int64_t rows = (int64_t)P.b.max_new * P.a.n_heads;
    const dim3 g1((unsigned)((rows + kK8Warps - 1) / kK8Warps), (unsigned)P.b.n_seqs), g4((unsigned)rows, (unsigned)P.b.n_seqs);
    const cudaError_t e = P.splits <= 8 ? launch_pdl(k_kv8_merge<T, 1>, g1, dim3(kK8Threads), 0, st, P)
                                        : launch_pdl(k_kv8_merge<T, 4>, g4, dim3(kK8Threads), 0, st, P);
    return check(e, "kv8_attn merge launch");
}

static int k8_check(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a) {
    const char *what = "kv8_attn";
    if (!kv8_check(c, b, what)) return 0;
    if (!a) return fail("%s: null argument", what);
    if (a->n_heads <= 0 || a->n_heads % c->n_kv_heads)
        return fail("%s: %d query heads over %d KV heads", what, a->n_heads, c->n_kv_heads);
    if (a->window < 0 || a->rel_extent < 0) return fail("%s: negative window or rel_extent", what);
    if ((int64_t)b->max_new * a->n_heads > INT32_MAX / 2) return fail("%s: step too large", what);
    if (b->n_seqs > 65535) return fail("%s: %d sequences (at most 65535)", what, b->n_seqs);
    return 1;
}

}  // namespace sepia

using namespace sepia;

extern "C" size_t sepia_cuda_kv8_attn_ws_bytes(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a) {
    if (!k8_check(c, b, a)) return 0;
    return std::max<size_t>(16, k8_plan(*c, *b, *a).bytes);
}

extern "C" int sepia_cuda_kv8_attn(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a, void *ws,
                                   size_t ws_bytes, void *stream) {
    const char *what = "kv8_attn";
    if (!k8_check(c, b, a)) return 0;
    if (b->n_seqs == 0 || b->n_tokens == 0 || b->max_new == 0) return 1;
    if (!a->q || !a->out) return fail("%s: null q or out", what);
    if (a->q_stride < (int64_t)a->n_heads * c->head_dim) return fail("%s: q_stride is shorter than a token", what);
    if (a->rel_extent && !a->rel_logits) return fail("%s: rel_extent without rel_logits", what);
    const K8Plan p = k8_plan(*c, *b, *a);
    if ((int64_t)c->n_kv_heads * p.row_tiles > 65535) return fail("%s: step too large", what);
    if (!ws || ws_bytes < std::max<size_t>(16, p.bytes)) return fail("%s: workspace of %zu bytes < %zu needed", what, ws_bytes, p.bytes);
    if (reinterpret_cast<uintptr_t>(ws) & 15) return fail("%s: workspace must be 16-byte aligned", what);
    K8Params P;
    P.c = *c;
    P.b = *b;
    P.a = *a;
    P.G = p.G;
    P.row_tiles = p.row_tiles;
    P.splits = p.splits;
    P.chunk = p.chunk;
    P.part = (float *)ws;
    P.err = dev_info().err;
    cudaStream_t st = as_stream(stream);
    if (c->head_dim <= 64) return a->x_f16 ? k8_launch<__half, 64>(P, st) : k8_launch<float, 64>(P, st);
    return a->x_f16 ? k8_launch<__half, 128>(P, st) : k8_launch<float, 128>(P, st);
}
