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
#include <type_traits>

namespace sepia {

constexpr int kK8Warps = 4;
constexpr int kK8Threads = 32 * kK8Warps;
constexpr int kK8Tile = 16;              // keys of one scale: a block is a multiple of it
constexpr int kK8Unit = 2 * kK8Tile;     // keys per warp step
constexpr int kK8Stages = 2;             // steps in a warp's ring
constexpr int kK8CtasPerSm = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
// Weights reach the tensor core as 2^(score - maximum + kPBits), in base 2.
// The maximum is only moved (and the output rescaled) when a weight would
// pass 2^15, so it may lag; kPBits leaves it 8 binary places to do so and
// keeps 22 bits of a weight down to 2^-20 of the largest.
constexpr float kPBits = 7.0f, kPMax = 15.0f;

struct K8Params {
    SepiaKv8Cache c;
    SepiaKv8Step b;
    SepiaKv8Attn a;
    int G, row_tiles, splits, chunk;     // chunk: positions per split, a multiple of kK8Unit * kK8Warps
    int bias_rows;                       // rows of a lane that have a band: 0, 1 or 2
    uint32_t two16;
    float *part;                         // [n_seqs, n_kv_heads * row_tiles, splits, rows of a tile, Dh + 2]
    int *err;
};

// The low two e4m3 codes of a word as fp16: one conversion. The high two
// are first moved down by a multiplication (high half of x * 2^16), which
// runs beside the conversions: shifts, permutes and conversions share one
// pipe of half the rate (measured 64 lanes a clock and SM each).
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t x, uint32_t two16) {
    uint32_t y;
    asm("mul.hi.u32 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(two16));
    return e4m3_lo(y);
}
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// cp.async of N (16, 8 or 4) bytes; of zeros where `on` is false
template <int N>
__device__ __forceinline__ void cp_async_bytes(uint32_t dst, const void *src) {
    if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(N) : "memory");
}
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
    static constexpr int kKeyB = 2 * KW * 512, kValB = 4 * VB * 32, kTileB = kKeyB + kValB;
    static constexpr int kHeadB = 16;                 // a step's scales
    static constexpr int kPitch = DP + 8;             // of a merge row: 8 rows of 8-byte stores meet no bank twice
    static constexpr int kMergeB = kK8Warps * RT * kPitch * 4;
    // bytes of a ring stage with the bias of `rows` rows a lane
    static constexpr int stage(int rows) { return 2 * kTileB + kHeadB + rows * 8 * 128; }
};

// FULL: head_dim is DP (64 or 128), every offset a constant; otherwise the
// dims past head_dim are read as zeros.
template <typename T, int DP, bool FULL>
__global__ void __launch_bounds__(kK8Threads, kK8CtasPerSm) k_kv8_attn(const K8Params P) {
    using F = K8Cfg<T, DP>;
    constexpr int RL = F::RL, RT = F::RT;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int split = blockIdx.x, s = blockIdx.z;
    const int hk = blockIdx.y / P.row_tiles, rt = blockIdx.y - hk * P.row_tiles;
    const int Dh = FULL ? DP : P.c.head_dim, B = P.c.block, H = P.a.n_heads, Hkv = P.c.n_kv_heads, G = P.G;
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

    // ---- coded steps: this warp's share of [c0, min(c1, tail0)), through its ring ----
    const int ce = min(c1, tail0);
    const int n_units = ce > c0 ? (ce - c0 + kK8Unit - 1) / kK8Unit : 0;
    const int mine = n_units > warp ? (n_units - warp + kK8Warps - 1) / kK8Warps : 0;
    const int stage_b = F::stage(P.bias_rows);
    uint8_t *ring = smem + warp * kK8Stages * stage_b;
    const uint32_t ring_u = smem_u32(ring);
    int pos[RL];
    const float *rel[RL];
#pragma unroll
    for (int j = 0; j < RL; j++) {
        const int R = min(rt * RT + gid + 8 * j, sq.add * G - 1), t = R / G;
        pos[j] = sq.held + t;
        rel[j] = P.a.rel_logits + ((int64_t)(sq.n0 + t) * H + hk * G + R - t * G) * E;
    }
    int id_l = 0;
    float ks_l = -1.0f, ev_l = 0.0f;
    auto issue = [&](int i) {
        if (i < mine) {
            if ((i & 15) == 0) {                       // lane: tile lane % 2 of step i + lane / 2
                const int at = c0 + (warp + kK8Warps * (i + (lane >> 1))) * kK8Unit + (lane & 1) * kK8Tile;
                ks_l = -1.0f;                          // a tile that is not there: all its keys hidden
                ev_l = 0.0f;
                id_l = 0;
                if (at < ce) {
                    const int id = kv8_block(P.c, P.b, s, at / B, P.err);
                    if (id >= 0) {
                        id_l = id;
                        ks_l = P.c.k_scale[(int64_t)id * Hkv + hk];
                        ev_l = (float)((int)(__float_as_uint(P.c.v_scale[(int64_t)id * Hkv + hk]) >> 23 & 255) - 127);
                    }
                }
            }
            const int t0 = c0 + (warp + kK8Warps * i) * kK8Unit;
            const uint32_t st = ring_u + (i & (kK8Stages - 1)) * stage_b;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int id = __shfl_sync(0xffffffffu, id_l, (2 * i + u) & 31);
                const int64_t row0 = ((int64_t)id * Hkv + hk) * B + ((t0 + u * kK8Tile) & (B - 1));
                const uint8_t *K = (const uint8_t *)P.c.k + row0 * Dh + gid * Dh + 16 * tig;
                const uint8_t *V = (const uint8_t *)P.c.v + row0 * Dh + 2 * tig * Dh + gid * F::VB;
                const uint32_t at = st + u * F::kTileB + lane * 16;
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int j = 0; j < F::KW; j++) {
                        if constexpr (FULL) cp_async_bytes<16>(at + (n * F::KW + j) * 512, K + n * 8 * Dh + j * 64);
                        else cp_async_or_zero<16>(at + (n * F::KW + j) * 512, K + n * 8 * Dh + j * 64, 64 * j + 16 * tig < Dh);
                    }
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t to = st + u * F::kTileB + F::kKeyB + k * (32 * F::VB) + lane * F::VB;
                    const uint8_t *src = V + ((k & 1) + 8 * (k >> 1)) * Dh;
                    if constexpr (FULL) cp_async_bytes<F::VB>(to, src);
                    else cp_async_or_zero<F::VB>(to, src, gid * F::VB < Dh);
                }
            }
            if (E && pa - (t0 + kK8Unit - 1) < E) {
#pragma unroll
                for (int j = 0; j < RL; j++) {
                    if (j >= P.bias_rows) break;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const int far = pos[j] - (t0 + 2 * tig + (k & 1) + 8 * (k >> 1));
                        const bool on = far >= 0 && far < E;
                        cp_async_or_zero<4>(st + 2 * F::kTileB + F::kHeadB + (8 * j + k) * 128 + lane * 4,
                                            rel[j] + (on ? far : 0), on);
                    }
                }
            }
            if ((lane >> 1) == (i & 15))
                *reinterpret_cast<float2 *>(ring + (i & (kK8Stages - 1)) * stage_b + 2 * F::kTileB + 8 * (lane & 1)) =
                    make_float2(ks_l, ev_l);
        }
        cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kK8Stages - 1; i++) issue(i);

    // ---- this lane's rows and their q operand ----
    float qmul[RL], tau[RL];
    uint32_t qa[F::KS][4];
#pragma unroll
    for (int j = 0; j < RL; j++) {
        const int r = gid + 8 * j, R = min(rt * RT + r, sq.add * G - 1), t = R / G;
        const bool on = r < rows;
        tau[j] = P.a.tau && on ? P.a.tau[sq.n0 + t] : 1.0f;
        const T *q = (const T *)P.a.q + (int64_t)(sq.n0 + t) * P.a.q_stride + (int64_t)(hk * G + R - t * G) * Dh;
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
            qmul[j] = P.a.scale * kLog2e * __uint_as_float((uint32_t)(127 - 13 + ex) << 23);
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
            qmul[j] = P.a.scale * kLog2e;
#pragma unroll
            for (int ks = 0; ks < F::KS; ks++) {
                qa[ks][j] = pack_half2(x[ks][0], x[ks][1]);
                qa[ks][2 + j] = pack_half2(x[ks][2], x[ks][3]);
            }
        }
    }

    // Running maximum in base 2 (a lag is allowed), sum, and output / 2^eref.
    float O[F::NT][4], m2[RL], l[RL], eref = -1000.0f;
#pragma unroll
    for (int nt = 0; nt < F::NT; nt++) O[nt][0] = O[nt][1] = O[nt][2] = O[nt][3] = 0.0f;
#pragma unroll
    for (int j = 0; j < RL; j++) m2[j] = kLowest, l[j] = 0.0f;

    // One step of U 16-key tiles from position t0; ksc, ev: each tile's key
    // scale (negative: hidden) and the exponent of its value scale.
    // kf(S): the key products, S[2 u + n] for keys 8 n .. of tile u; pv(u, w): the weights'
    // products with tile u's values into O; bias(j, i): term i of this lane's
    // row j, keys t0 + 2 tig + {0, 1, 8, 9, 16, ...}; clean(u): values that
    // are not numbers to 0, and which of the lane's four keys had any.
    auto step = [&](auto units, int t0, const float *ksc, const float *ev, auto kf, auto pv, auto bias, auto clean) {
        constexpr int U = decltype(units)::value;
        float x[RL][4 * U], f2[RL][U], lv[U], S[2 * U][4];
#pragma unroll
        for (int n = 0; n < 2 * U; n++) S[n][0] = S[n][1] = S[n][2] = S[n][3] = 0.0f;
        kf(S);
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int j = 0; j < RL; j++) {
                f2[j][u] = ksc[u] * qmul[j];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float *y = S[2 * u + (i >> 1)];
                    x[j][4 * u + i] = F::kTwo ? y[i & 1] + y[(i & 1) + 2] : y[(i & 1) + 2 * j];
                }
            }
        const float top_ev = U == 2 ? fmaxf(ev[0], ev[U - 1]) : ev[0];
        if (top_ev > eref) {                           // the whole warp
            const float f = exp2_fast(eref - top_ev);
#pragma unroll
            for (int nt = 0; nt < F::NT; nt++) O[nt][0] *= f, O[nt][1] *= f, O[nt][2] *= f, O[nt][3] *= f;
            eref = top_ev;
        }
        const bool biased = E && pa - (t0 + U * kK8Tile - 1) < E;
        bool masked = t0 + U * kK8Tile - 1 > pa || (window && t0 <= pb - window) || ksc[0] < 0.0f || ksc[U - 1] < 0.0f;
        if (biased || masked) {
            uint32_t seen = 0;                         // bit 4 U j + i: row j sees key i
#pragma unroll
            for (int j = 0; j < RL; j++)
#pragma unroll
                for (int i = 0; i < 4 * U; i++) {
                    const int at = t0 + 2 * tig + (i & 1) + 8 * (i >> 1);
                    float y = x[j][i] * f2[j][i / 4];
                    if (biased) {
                        // a score of the type's lowest stays a number in base 2
                        const float b = bias(j, i) * tau[j] * kLog2e;
                        y = y + b;
                        if (y < kLowest && bias(j, i) * tau[j] > -INFINITY) y = kLowest;
                    }
                    if (at > pos[j] || (window && at <= pos[j] - window) || ksc[i / 4] < 0.0f) y = -INFINITY;
                    x[j][i] = y;
                    seen |= y == -INFINITY ? 0u : 1u << (4 * U * j + i);
                }
#pragma unroll
            for (int j = 0; j < RL; j++)
#pragma unroll
                for (int u = 0; u < U; u++) f2[j][u] = 1.0f;
            // A value that is not a number must not reach a row that does not
            // see its key (0 * NaN): in a step with hidden keys such values
            // count as 0, and a row that does see one gets a sum of NaN.
            if (__any_sync(0xffffffffu, seen != (1u << (4 * U * RL)) - 1u)) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    uint32_t nan = clean(u);
                    nan |= __shfl_xor_sync(0xffffffffu, nan, 4);
                    nan |= __shfl_xor_sync(0xffffffffu, nan, 8);
                    nan |= __shfl_xor_sync(0xffffffffu, nan, 16);
#pragma unroll
                    for (int j = 0; j < RL; j++)
                        if (seen >> (4 * U * j + 4 * u) & nan) l[j] = __int_as_float(0x7fffffff);
                }
            }
        }
        float p[RL][4 * U], top = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; u++) lv[u] = ev[u] - eref + kPBits;
#pragma unroll
        for (int j = 0; j < RL; j++)
#pragma unroll
            for (int i = 0; i < 4 * U; i++) {
                p[j][i] = fmaf(x[j][i], f2[j][i / 4], -m2[j]) + lv[i / 4];   // exact where both are the lowest
                top = fmaxf(top, p[j][i]);
            }
        if (__any_sync(0xffffffffu, top > kPMax)) {
            float f[RL];
#pragma unroll
            for (int j = 0; j < RL; j++) {
                float t = kLowest;
#pragma unroll
                for (int i = 0; i < 4 * U; i++) t = fmaxf(t, x[j][i] * f2[j][i / 4]);
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 1));
                t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 2));
                t = fmaxf(t, m2[j]);
                f[j] = exp2_fast(m2[j] - t);
                m2[j] = t;
                l[j] *= f[j];
#pragma unroll
                for (int i = 0; i < 4 * U; i++) p[j][i] = fmaf(x[j][i], f2[j][i / 4], -t) + lv[i / 4];
            }
#pragma unroll
            for (int nt = 0; nt < F::NT; nt++) {
                O[nt][0] *= f[0], O[nt][1] *= f[0];
                O[nt][2] *= f[RL - 1], O[nt][3] *= f[RL - 1];
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            uint32_t w[4];
            const float il = exp2_fast(-lv[u]);
#pragma unroll
            for (int j = 0; j < RL; j++) {
                float *q = &p[j][4 * u];
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = exp2_fast(q[i]);
                l[j] = fmaf((q[0] + q[1]) + (q[2] + q[3]), il, l[j]);
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const __half2 hi = __floats2half2_rn(q[2 * n], q[2 * n + 1]);
                    w[2 * n + j] = *reinterpret_cast<const uint32_t *>(&hi);
                    if constexpr (F::kTwo) {
                        const float2 b = __half22float2(hi);
                        w[2 * n + 1] = pack_half2(q[2 * n] - b.x, q[2 * n + 1] - b.y);
                    }
                }
            }
            pv(u, w);
        }
    };
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;

    // ---- the tail's fp16 tiles, one a warp, while the ring fills ----
    {
        const int t0 = tail0 + kK8Tile * warp;
        if (t0 >= c0 && t0 < c1) {
            const int64_t at = (((int64_t)sq.slot * Hkv + hk) * B + (t0 - tail0)) * Dh;
            const __half *K = (const __half *)P.c.k_tail + at, *V = (const __half *)P.c.v_tail + at;
            const int held = sq.held + sq.add - t0;    // keys of the tile that exist
            const float one = 1.0f, zero = 0.0f;
            uint32_t v[4][F::VB / 2];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int r = 2 * tig + (k & 1) + 8 * (k >> 1), d = gid * F::VB;
#pragma unroll
                for (int j = 0; j < F::VB / 8; j++)
                    *reinterpret_cast<uint4 *>(&v[k][4 * j]) =
                        r < held && d + 8 * j < Dh ? *reinterpret_cast<const uint4 *>(V + r * Dh + d + 8 * j)
                                                   : make_uint4(0, 0, 0, 0);
            }
            step(
                One(), t0, &one, &zero,
                [&](float (&S)[2][4]) {
#pragma unroll
                    for (int ks = 0; ks < F::KS; ks++) {
                        const int d = 64 * (ks / 4) + 16 * tig + 4 * (ks % 4);
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            const int r = gid + 8 * n;
                            const uint2 x = r < held && d < Dh ? *reinterpret_cast<const uint2 *>(K + r * Dh + d)
                                                               : make_uint2(0, 0);
                            mma16(S[n], qa[ks], x.x, x.y);
                        }
                    }
                },
                [&](int, const uint32_t (&w)[4]) {
#pragma unroll
                    for (int nt = 0; nt < F::NT; nt++) {
                        const uint32_t sel = nt & 1 ? 0x7632 : 0x5410;
                        mma16(O[nt], w, __byte_perm(v[0][nt / 2], v[1][nt / 2], sel),
                              __byte_perm(v[2][nt / 2], v[3][nt / 2], sel));
                    }
                },
                [&](int j, int i) {
                    const int far = pos[j] - (t0 + 2 * tig + (i & 1) + 8 * (i >> 1));
                    return far >= 0 && far < E ? rel[j][far] : 0.0f;
                },
                [&](int) {
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int e = 0; e < F::VB / 2; e++) {
                            const uint32_t at = __vcmpgtu2(v[k][e] & 0x7fff7fffu, 0x7c007c00u);
                            v[k][e] &= ~at;
                            nan |= at ? 1u << k : 0u;
                        }
                    return nan;
                });
        }
    }

    const uint32_t two16 = P.two16;                    // 2^16, unknown to the compiler (see e4m3_hi)
    for (int i = 0; i < mine; i++) {
        __syncwarp();                                  // every lane is done with the stage that is filled next
        issue(i + kK8Stages - 1);
        cp_async_wait<kK8Stages - 1>();
        __syncwarp();
        uint8_t *st = ring + (i & (kK8Stages - 1)) * stage_b;
        const float4 sc = *reinterpret_cast<const float4 *>(st + 2 * F::kTileB);
        const float ksc[2] = {sc.x, sc.z}, ev[2] = {sc.y, sc.w};
        step(
            Two(), c0 + (warp + kK8Warps * i) * kK8Unit, ksc, ev,
            [&](float (&S)[4][4]) {
#pragma unroll
                for (int j = 0; j < F::KW; j++) {
                    uint4 k[4];
#pragma unroll
                    for (int n = 0; n < 4; n++)
                        k[n] = *reinterpret_cast<const uint4 *>(st + (n >> 1) * F::kTileB + ((n & 1) * F::KW + j) * 512 + lane * 16);
#pragma unroll
                    for (int e = 0; e < 4; e++)
#pragma unroll
                        for (int n = 0; n < 4; n++) {  // four independent chains
                            const uint32_t kw = e == 0 ? k[n].x : e == 1 ? k[n].y : e == 2 ? k[n].z : k[n].w;
                            mma16(S[n], qa[4 * j + e], e4m3_lo(kw), e4m3_hi(kw, two16));
                        }
                }
            },
            [&](int u, const uint32_t (&w)[4]) {
                uint32_t v[4][F::VB / 4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint8_t *src = st + u * F::kTileB + F::kKeyB + k * (32 * F::VB) + lane * F::VB;
                    if constexpr (F::VB == 16) *reinterpret_cast<uint4 *>(v[k]) = *reinterpret_cast<const uint4 *>(src);
                    else *reinterpret_cast<uint2 *>(v[k]) = *reinterpret_cast<const uint2 *>(src);
                }
#pragma unroll
                for (int nt = 0; nt < F::NT; nt += 2) {
                    const uint32_t sel = nt & 2 ? 0x7362 : 0x5140;
                    const uint32_t x = __byte_perm(v[0][nt / 4], v[1][nt / 4], sel);
                    const uint32_t y = __byte_perm(v[2][nt / 4], v[3][nt / 4], sel);
                    mma16(O[nt], w, e4m3_lo(x), e4m3_lo(y));
                    mma16(O[nt + 1], w, e4m3_hi(x, two16), e4m3_hi(y, two16));
                }
            },
            [&](int j, int k) {
                if (j >= P.bias_rows) return 0.0f;     // rows that do not exist have no room in the ring
                return *reinterpret_cast<const float *>(st + 2 * F::kTileB + F::kHeadB + (8 * j + k) * 128 + lane * 4);
            },
            [&](int u) {                               // the lane's own copies, in its ring
                uint32_t nan = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t *v = reinterpret_cast<uint32_t *>(st + u * F::kTileB + F::kKeyB + k * (32 * F::VB) + lane * F::VB);
#pragma unroll
                    for (int e = 0; e < F::VB / 4; e++) {
                        const uint32_t at = __vcmpeq4(v[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        if (at) v[e] &= ~at;
                        nan |= at ? 1u << k : 0u;
                    }
                }
                return nan;
            });
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- merge the warps, in warp order. A row's output lies in the order
    // of the lanes' columns: entry 8 nt + c is dim c * VB + nt ----
    float *mg = reinterpret_cast<float *>(smem) + warp * RT * F::kPitch;
#pragma unroll
    for (int j = 0; j < RL; j++) {
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 1);
        l[j] += __shfl_xor_sync(0xffffffffu, l[j], 2);
        float *o = mg + (gid + 8 * j) * F::kPitch;
        if (tig == 0) *reinterpret_cast<float2 *>(o + DP) = make_float2(m2[j], l[j]);
        const float f = exp2_fast(eref - kPBits);
#pragma unroll
        for (int nt = 0; nt < F::NT; nt++)
            *reinterpret_cast<float2 *>(o + 8 * nt + 2 * tig) =
                make_float2(f * (F::kTwo ? O[nt][0] + O[nt][2] : O[nt][2 * j]),
                            f * (F::kTwo ? O[nt][1] + O[nt][3] : O[nt][1 + 2 * j]));
    }
    __syncthreads();
    const int live = min(rows, RT), group = blockIdx.z * gridDim.y + blockIdx.y;
    float *part = P.part + ((int64_t)group * P.splits + split) * RT * (DP + 2);
    for (int i = tid; i < live * DP; i += kK8Threads) {
        const int r = i / DP, c = i - r * DP, d = (c & 7) * F::VB + (c >> 3);
        const float *o = reinterpret_cast<const float *>(smem) + r * F::kPitch;
        float M = kLowest, L = 0.0f, A = 0.0f;
#pragma unroll
        for (int w = 0; w < kK8Warps; w++) M = fmaxf(M, o[w * RT * F::kPitch + DP]);
#pragma unroll
        for (int w = 0; w < kK8Warps; w++) {
            const float *ow = o + w * RT * F::kPitch;
            const float f = exp2_fast(ow[DP] - M);
            L += f * ow[DP + 1];
            A += f * ow[c];
        }
        if (n_act == 1) {
            const int R = rt * RT + r, t = R / G;
            if (d < Dh)
                ((T *)P.a.out)[((int64_t)(sq.n0 + t) * H + hk * G + (R - t * G)) * Dh + d] = (T)(L == 0.0f ? 0.0f : A / L);
        } else {
            float *to = part + r * (DP + 2);
            if (c == 0) *reinterpret_cast<float2 *>(to) = make_float2(M, L);
            to[2 + c] = A;
        }
    }
}

// Merges the chunks of a row, in chunk order within each of the W warps that
// share the row, then across the warps. One CTA does kK8Warps / W rows.
template <typename T, int DP, int W>
__global__ void __launch_bounds__(kK8Threads) k_kv8_merge(const K8Params P) {
    constexpr int RT = K8Cfg<T, DP>::RT;
    __shared__ float s_part[W > 1 ? kK8Warps : 1][DP + 2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = 4 * lane;
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
    constexpr int64_t stride = (int64_t)RT * (DP + 2);
    const float *part = P.part + (int64_t)group * P.splits * stride + r * (DP + 2);
    float M = kLowest, L = 0.0f, A[4] = {0.0f, 0.0f, 0.0f, 0.0f};
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
            x[i][0] = c < DP ? p[1 + c / 2] : make_float2(0.0f, 0.0f);
            x[i][1] = c < DP ? p[2 + c / 2] : make_float2(0.0f, 0.0f);
        }
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const float f = k + i < k1 ? exp2_fast(ml[i].x - M) : 0.0f;
            L += f * ml[i].y;
            A[0] += f * x[i][0].x, A[1] += f * x[i][0].y, A[2] += f * x[i][1].x, A[3] += f * x[i][1].y;
        }
    }
    if constexpr (W > 1) {
        if (c < DP)
            for (int e = 0; e < 4; e++) s_part[warp][2 + c + e] = A[e];
        if (lane == 0) s_part[warp][0] = L;
        __syncthreads();
        if (warp) return;
#pragma unroll
        for (int w = 1; w < W; w++) {
            L += s_part[w][0];
            if (c < DP)
                for (int e = 0; e < 4; e++) A[e] += s_part[w][2 + c + e];
        }
    }
    T *o = (T *)P.a.out + ((int64_t)(sq.n0 + t) * H + h) * Dh;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const int d = ((c + e) & 7) * (DP / 8) + ((c + e) >> 3);
        if (c < DP && d < Dh) o[d] = (T)(L == 0.0f ? 0.0f : A[e] / L);
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
    constexpr int64_t kUnit = kK8Unit * kK8Warps, kMaxChunk = 1024;
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
    p.bytes = p.splits > 1 ? (size_t)groups * p.splits * rt * ((c.head_dim <= 64 ? 64 : 128) + 2) * 4 : 0;
    return p;
}

template <typename T, int DP, bool FULL>
static int k8_launch(K8Params &P, cudaStream_t st) {
    using F = K8Cfg<T, DP>;
    const int64_t rows = (int64_t)P.b.max_new * P.a.n_heads;
    P.bias_rows = P.a.rel_extent == 0 ? 0 : (int64_t)P.b.max_new * P.G <= 8 ? 1 : F::RL;
    const int smem = std::max(kK8Warps * kK8Stages * F::stage(P.bias_rows), F::kMergeB);
    if (!ensure_smem((const void *)k_kv8_attn<T, DP, FULL>, smem)) return 0;
    const dim3 grid((unsigned)P.splits, (unsigned)(P.c.n_kv_heads * P.row_tiles), (unsigned)P.b.n_seqs);
    if (!check(launch_pdl(k_kv8_attn<T, DP, FULL>, grid, dim3(kK8Threads), smem, st, P), "kv8_attn launch")) return 0;
    if (P.splits == 1) return 1;
    // one warp per row while a row has few chunks, four beyond
    const dim3 g1((unsigned)((rows + kK8Warps - 1) / kK8Warps), (unsigned)P.b.n_seqs), g4((unsigned)rows, (unsigned)P.b.n_seqs);
    const cudaError_t e = P.splits <= 8 ? launch_pdl(k_kv8_merge<T, DP, 1>, g1, dim3(kK8Threads), 0, st, P)
                                        : launch_pdl(k_kv8_merge<T, DP, 4>, g4, dim3(kK8Threads), 0, st, P);
    return check(e, "kv8_attn merge launch");
}

template <typename T>
static int k8_launch_dim(K8Params &P, cudaStream_t st) {
    const int Dh = P.c.head_dim;
    if (Dh <= 64) return Dh == 64 ? k8_launch<T, 64, true>(P, st) : k8_launch<T, 64, false>(P, st);
    return Dh == 128 ? k8_launch<T, 128, true>(P, st) : k8_launch<T, 128, false>(P, st);
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
    P.two16 = 65536u;
    P.part = (float *)ws;
    P.err = dev_info().err;
    cudaStream_t st = as_stream(stream);
    return a->x_f16 ? k8_launch_dim<__half>(P, st) : k8_launch_dim<float>(P, st);
}
