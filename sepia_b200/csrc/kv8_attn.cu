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
//   Operands  mma m16n8k16 in fp16 with fp32 sums, the codes as the 16-row
//             operand (scores: 16 keys x 8 rows; output: 16 dims x 8 rows),
//             so that 8 rows fill it. e4m3 codes are fp16 numbers exactly;
//             block scales multiply the score and the weight. The weight is
//             two fp16 terms (22 bits), summed in one result; so is an fp32 q.
//   Layout    the dims of a k step and of an output tile are permuted so that
//             a lane's codes are 16 consecutive bytes of a key row (K) or of
//             four key rows (V). A warp copies its tiles as they lie (cp.async,
//             512 bytes in a row an instruction; copying each lane's own bytes
//             instead needed no exchange between lanes but reached 4.1 TB/s
//             where this reaches 5.8) into shared memory of its own, 16-byte
//             pieces swizzled so that neither side meets a bank twice. The
//             slots hold one step: keys are fetched again as soon as their
//             scores are done, values when their output is, each behind the
//             other half of the step and three more warps of the scheduler.
//   Measured  1 x 32768, 64 heads over 8, fp32: 20.5 us, of which 12 (5.6 TB/s)
//             are key steps and the rest start and merge; 64 ragged sequences
//             of 2048 to 4096, fp16: 89 us, 4.6 TB/s; a window of 4096: 9.7 us.
//             With more rows (12 x 6001, 4 new tokens: 79 us) the chains of
//             conversions and products bind, 25 us at the product's full rate.
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
// CTAs an SM holds: by registers (128 a thread)
constexpr int k8_ctas(int nb) { return nb == 1 ? 4 : 3; }
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;
// Weights reach the tensor core as 2^(score - maximum + kPBits), in base 2,
// and as 2^(the value scale's exponent less the greatest one met) of that.
// The maximum is only moved (and the output rescaled) when a weight would
// pass 2^15, so it may lag by two places. The smallest fp16 step, 2^-24, is
// then 2^-37 of the greatest weight, and 2^-37 + the spread of the scales.
// Tiles without any value (hidden ones, zeros) count as of the exponent
// kNoValue, below those of all scales (2^-32 for the least fp16 number): with
// the scale of 1 that stands beside a block of zeros they would cost the others'
// weights as many places as their values are small.
constexpr float kPBits = 13.0f, kPMax = 15.0f, kNoValue = -60.0f;

struct K8Params {
    SepiaKv8Cache c;
    SepiaKv8Step b;
    SepiaKv8Attn a;
    int G, row_tiles, splits, chunk;     // chunk: positions per split, a multiple of kK8Unit * kK8Warps
    int tile0;                           // the launch's first row tile (0 where tiles are cut into chunks)
    int q_vec;                           // four elements of q in one load
    float *part;                         // [n_seqs, n_kv_heads * row_tiles, splits, rows of a tile, Dh]
    float2 *part_ml;                     // [n_seqs, n_kv_heads * row_tiles, splits, rows of a tile]: maximum, sum
    int *err;
};

// The low and the high two e4m3 codes of a word as fp16
__device__ __forceinline__ uint32_t e4m3_lo(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\t}" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ uint32_t e4m3_hi(uint32_t x) {
    uint32_t r;
    asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(x));
    return r;
}
// The warp's 8 x 8 matrix of halves (row: lane / 4, columns 2 (lane % 4) and the next) transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
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

// NB groups of 8 rows share a warp's converted codes.
template <typename T, int DP, int NB>
struct K8Cfg {
    static constexpr int UNITS = NB == 1 ? 2 : 1;     // 16-key tiles whose scores are in registers at once
    static constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;   // fp16 terms of a row of q
    static constexpr int RT = 8 * NB;                 // rows of a tile
    static constexpr int KW = DP / 64;                // 16-byte pieces of a key row per lane
    static constexpr int VB = DP / 8;                 // bytes of a value row per lane
    static constexpr int MT = DP / 16, KS = DP / 16;  // output tiles of 16 dims, k steps of 16
    static constexpr int kKeyB = kK8Tile * DP, kValB = kKeyB, kTileB = 2 * kKeyB;
    static constexpr int kHeadB = 16;                 // a step's scales
    static constexpr int kPitch = DP + 4;             // of a merge row: the lanes' stores meet no bank twice
    static constexpr int kMergeB = kK8Warps * RT * (kPitch + 2) * 4;
    static constexpr bool kQRegs = NB == 1 && TERMS == 1;   // q operands in registers, else in shared memory
    static constexpr int kQB = kQRegs ? 0 : NB * KS * 32 * 8 * TERMS;
    // bytes of a warp's slots, with room for a band where there is one
    static constexpr int stage(bool band) { return 2 * kTileB + kHeadB + (band ? NB * 8 * 128 : 0); }
};

// Four dims of a row: sums over the weights' total; zeros where nothing was seen
template <typename T>
__device__ __forceinline__ void put_row(T *to, const float (&A)[4], float L) {
    T y[4];
#pragma unroll
    for (int e = 0; e < 4; e++) y[e] = (T)(L == 0.0f ? 0.0f : A[e] / L);
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(to) = *reinterpret_cast<const uint4 *>(y);
    else *reinterpret_cast<uint2 *>(to) = *reinterpret_cast<const uint2 *>(y);
}

// FULL: head_dim is DP (64 or 128), every offset a constant; otherwise the
// dims past head_dim are read as zeros (128 dims that way: 1 x 32768 22.0 us,
// constant 20.5; 64 sequences 93.5 and 89). Four CTAs an SM leave 128 registers,
// and the forms for 128 dims spill 8 to 40 bytes (those with FULL 8 and 12).
template <typename T, int DP, int NB, bool FULL>
__global__ void __launch_bounds__(kK8Threads, k8_ctas(NB)) k_kv8_attn(const K8Params P) {
    using F = K8Cfg<T, DP, NB>;
    constexpr int RT = F::RT, TERMS = F::TERMS;
    extern __shared__ __align__(16) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
    const int split = blockIdx.x, s = blockIdx.z;
    const int tile = P.tile0 + blockIdx.y, hk = tile / P.row_tiles, rt = tile - hk * P.row_tiles;
    const int Dh = FULL ? DP : P.c.head_dim, B = P.c.block, H = P.a.n_heads, Hkv = P.c.n_kv_heads, G = P.G;
    griddep_wait();
    griddep_launch();
    const Kv8Seq sq = kv8_seq(P.c, P.b, s, P.err);
    const int64_t cell = ((int64_t)(s * gridDim.y + blockIdx.y) * P.splits + split) * RT;   // of this chunk's rows
    if (P.splits > 1 && tid < RT) P.part_ml[cell + tid] = make_float2(kLowest, 0.0f);       // empty until it is not
    if (sq.add < 0) {                                  // idle or out of bounds: zeros, of more than max_new rows too
        if (split == 0)
            kv8_zero_rows((T *)P.a.out, sq.n0, sq.rows, H * Dh, blockIdx.y * kK8Threads + tid, gridDim.y * kK8Threads);
        return;
    }
    const int rows = sq.rows * G - rt * RT;            // rows of this tile that exist (may exceed RT)
    if (rows <= 0) return;
    // tokens of the tile, the positions that any of them sees, this CTA's chunk
    const int ta = rt * RT / G, tb = min(sq.add - 1, (rt * RT + RT - 1) / G);
    const int pa = sq.held + ta, pb = sq.held + tb;
    const int window = P.a.window, E = P.a.rel_extent;
    const int tail0 = (sq.held + sq.add) / B * B;
    const int lo = window ? max(0, pa - window + 1) / kK8Tile * kK8Tile : 0;
    const int n_act = (pb + 1 - lo + P.chunk - 1) / P.chunk;
    if (split >= n_act) return;
    const int c0 = lo + split * P.chunk, c1 = min(pb + 1, c0 + P.chunk);

    // ---- coded steps: this warp's share of [c0, min(c1, tail0)), through its slots ----
    const int ce = min(c1, tail0);
    const int n_units = ce > c0 ? (ce - c0 + kK8Unit - 1) / kK8Unit : 0;
    const int mine = n_units > warp ? (n_units - warp + kK8Warps - 1) / kK8Warps : 0;
    const int stage_b = F::stage(E > 0);
    uint8_t *st = smem + F::kQB + warp * stage_b;
    const uint32_t st_u = smem_u32(st);
    // the pool's block of this lane's tile: tile lane % 2 of step i + lane / 2
    int id_l = -1;
    auto look_up = [&](int i) {
        const int at = c0 + (warp + kK8Warps * (i + (lane >> 1))) * kK8Unit + (lane & 1) * kK8Tile;
        id_l = at < ce ? kv8_block(P.c, P.b, s, at / B, P.err) : -1;
    };
    look_up(0);

    // ---- q: lane (gid, tig) holds 16 dims of row gid of each group ----
    auto row_of = [&](int r, int &t, int &h) {         // of a row of the tile, or of the last one that exists
        const int R = min(rt * RT + r, sq.add * G - 1);
        t = R / G;
        h = hk * G + R - t * G;
    };
    T q_raw[F::KS][4];                                 // of group `warp` (or the only one), fetched before all else
    const int q_group = F::kQRegs ? 0 : warp;
    if (q_group < NB) {
        int t, h;
        row_of(8 * q_group + gid, t, h);
        const T *q = (const T *)P.a.q + (int64_t)(sq.n0 + t) * P.a.q_stride + (int64_t)h * Dh;
        const bool on = 8 * q_group + gid < rows;
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++) {
            const int d = 64 * (ks / 4) + 16 * tig + 4 * (ks % 4);
            if (on && d < Dh) {
                if (P.q_vec) {
                    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(q_raw[ks]) = *reinterpret_cast<const uint4 *>(q + d);
                    else *reinterpret_cast<uint2 *>(q_raw[ks]) = *reinterpret_cast<const uint2 *>(q + d);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) q_raw[ks][e] = q[d + e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) q_raw[ks][e] = (T)0.0f;
            }
        }
    }
    // this lane's rows of each group as columns of a product: 2 tig and 2 tig + 1
    int pos[NB][2];
    int rel_at[NB][2];                                 // their bands, from the first token's
    const float *rel = P.a.rel_logits + (int64_t)(sq.n0 + ta) * H * E;
#pragma unroll
    for (int g = 0; g < NB; g++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            int t, h;
            row_of(8 * g + 2 * tig + e, t, h);
            pos[g][e] = sq.held + t;
            rel_at[g][e] = ((t - ta) * H + h) * E;
        }

    // Copies: piece q (16 bytes) of a tile to its place in shared memory. In
    // lines of 128 bytes, pieces 0-7: keys swap the halves of every second
    // line of whole rows; values move by twice the row pair.
    auto place = [&](int q, bool values) {
        const int row = FULL ? q / (DP / 16) : q / (Dh / 16), c = FULL ? q % (DP / 16) : q - row * (Dh / 16);
        const int piece = row * (DP / 16) + c, f = values ? ((row >> 1) & 3) * 2 : DP == 128 ? (row & 1) * 4 : 0;
        return ((piece & ~7) | ((piece & 7) ^ f)) * 16;
    };
    constexpr int NC = DP / 32;                        // copies of a lane per tile
    int to_k[NC], to_v[NC];
#pragma unroll
    for (int k = 0; k < NC; k++) to_k[k] = place(lane + 32 * k, false), to_v[k] = place(lane + 32 * k, true);
    if constexpr (!FULL) {                             // dims past head_dim: zeros, once
        for (int k = lane; k < 2 * F::kTileB / 16; k += 32) reinterpret_cast<uint4 *>(st)[k] = make_uint4(0, 0, 0, 0);
        __syncwarp();
    }
    auto copy = [&](int i, const uint8_t *from, int offset, const int (&to)[NC]) {
#pragma unroll
        for (int u = 0; u < 2; u++) {
            const int id = max(0, __shfl_sync(0xffffffffu, id_l, (2 * i + u) & 31));
            const int at = c0 + (warp + kK8Warps * i) * kK8Unit + u * kK8Tile;
            const uint8_t *src = from + (((int64_t)id * Hkv + hk) * B + (at & (B - 1))) * Dh + lane * 16;
#pragma unroll
            for (int k = 0; k < NC; k++)
                if (FULL || lane + 32 * k < Dh) cp_async_bytes<16>(st_u + u * F::kTileB + offset + to[k], src + k * 512);
        }
    };
    // ... and where the lane's operands lie: keys gid + 8 n, piece 4 j + tig; values of keys 2 tig + {0, 1, 8, 9}
    int from_k[F::KW], from_v[2];
#pragma unroll
    for (int j = 0; j < F::KW; j++) from_k[j] = DP == 128 ? gid * 128 + (4 * (j ^ (gid & 1)) + tig) * 16 : gid * 64 + tig * 16;
#pragma unroll
    for (int k = 0; k < 2; k++)
        from_v[k] = DP == 128 ? (2 * tig + k) * 128 + (gid ^ (2 * tig)) * 16
                              : tig * 128 + (((4 * k + (gid >> 1)) ^ (2 * tig)) * 16) + (gid & 1) * 8;
    auto fetch_keys = [&](int i) {                     // and the scales
        if (i < mine) {
            if (i && (i & 15) == 0) look_up(i);
            if ((lane >> 1) == (i & 15)) {             // a tile that is not there: hidden
                const int to = 2 * F::kTileB + 8 * (lane & 1);
                if (id_l >= 0) {
                    cp_async_bytes<4>(st_u + to, P.c.k_scale + (int64_t)id_l * Hkv + hk);
                    cp_async_bytes<4>(st_u + to + 4, P.c.v_scale + (int64_t)id_l * Hkv + hk);
                } else {
                    *reinterpret_cast<float2 *>(st + to) = make_float2(-1.0f, __uint_as_float((uint32_t)(127 + (int)kNoValue) << 23));
                }
            }
            copy(i, (const uint8_t *)P.c.k, 0, to_k);
        }
        cp_async_commit();
    };
    auto fetch_values = [&](int i) {                   // and the band
        if (i < mine) {
            const int t0 = c0 + (warp + kK8Warps * i) * kK8Unit;
            copy(i, (const uint8_t *)P.c.v, F::kKeyB, to_v);
            if (E && pa - (t0 + kK8Unit - 1) < E) {
#pragma unroll
                for (int g = 0; g < NB; g++)
#pragma unroll
                    for (int k = 0; k < 8; k++) {      // key gid + 8 (k / 2), row 2 tig + k % 2
                        const int far = pos[g][k & 1] - (t0 + gid + 8 * (k >> 1));
                        const bool on = far >= 0 && far < E;
                        cp_async_or_zero<4>(st_u + 2 * F::kTileB + F::kHeadB + (8 * g + k) * 128 + lane * 4,
                                            rel + rel_at[g][k & 1] + (on ? far : 0), on);
                    }
            }
        }
        cp_async_commit();
    };
    fetch_keys(0);
    fetch_values(0);

    // ---- q as operands ----
    static_assert(NB <= kK8Warps, "a warp per group writes its operands");
    constexpr int NQ = F::kQRegs ? F::KS : 1;
    uint32_t qb[NQ][2 * TERMS];                        // [k step][term][half]
    float qx = 1.0f;                                   // row gid's factor on its products
    if (q_group < NB) {
        float x[F::KS][4], amax = 0.0f;
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[ks][e] = (float)q_raw[ks][e];
                amax = fmaxf(amax, fabsf(x[ks][e]));
            }
        float f = 1.0f;
        if constexpr (TERMS == 2) {
            // the row times a power of two that puts its largest in [2^13, 2^14): both terms stay normal fp16
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            const int ex = amax > 0.0f ? max((int)(__float_as_uint(amax) >> 23) - 127, -100) : 13;
            f = __uint_as_float((uint32_t)(127 + 13 - ex) << 23);
            qx = __uint_as_float((uint32_t)(127 - 13 + ex) << 23);
        }
#pragma unroll
        for (int ks = 0; ks < F::KS; ks++) {
            uint32_t w[2 * TERMS];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float u = x[ks][2 * e] * f, v = x[ks][2 * e + 1] * f;
                const __half2 hi = __floats2half2_rn(u, v);
                w[e] = *reinterpret_cast<const uint32_t *>(&hi);
                if constexpr (TERMS == 2) {
                    const float2 b = __half22float2(hi);
                    w[2 + e] = pack_half2(u - b.x, v - b.y);
                }
            }
            if constexpr (F::kQRegs) {
#pragma unroll
                for (int e = 0; e < 2 * TERMS; e++) qb[ks][e] = w[e];
            } else {
                uint32_t *to = reinterpret_cast<uint32_t *>(smem) + ((q_group * F::KS + ks) * 32 + lane) * (2 * TERMS);
#pragma unroll
                for (int e = 0; e < 2 * TERMS; e++) to[e] = w[e];
            }
        }
    }
    auto q_op = [&](int g, int ks, uint32_t (&w)[2 * TERMS]) {
        if constexpr (F::kQRegs) {
#pragma unroll
            for (int e = 0; e < 2 * TERMS; e++) w[e] = qb[ks][e];
        } else {
            const uint32_t *from = reinterpret_cast<const uint32_t *>(smem) + ((g * F::KS + ks) * 32 + lane) * (2 * TERMS);
            if constexpr (TERMS == 2) *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(from);
            else *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(from);
        }
    };

    float qmul[NB][2], tau[NB][2];                     // of the lane's rows as columns
#pragma unroll
    for (int g = 0; g < NB; g++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            int t, h;
            row_of(8 * g + 2 * tig + e, t, h);
            tau[g][e] = P.a.tau ? P.a.tau[sq.n0 + t] : 1.0f;
            qmul[g][e] = P.a.scale * kLog2e;
        }
    if constexpr (!F::kQRegs) {
        __shared__ float s_qx[RT];
        if (q_group < NB && tig == 0) s_qx[8 * q_group + gid] = qx;
        __syncthreads();
#pragma unroll
        for (int g = 0; g < NB; g++)
#pragma unroll
            for (int e = 0; e < 2; e++) qmul[g][e] *= s_qx[8 * g + 2 * tig + e];
    }

    // Running maximum in base 2 (a lag is allowed), sum, and output / 2^eref;
    // O[g][mt]: dims gid * VB + 2 mt (+ 1 in entries 2, 3), rows 2 tig (+ 1 in entries 1, 3).
    float O[NB][F::MT][4], m2[NB][2], l[NB][2], eref = -1000.0f;
#pragma unroll
    for (int g = 0; g < NB; g++) {
        m2[g][0] = m2[g][1] = kLowest;
        l[g][0] = l[g][1] = 0.0f;
#pragma unroll
        for (int mt = 0; mt < F::MT; mt++) O[g][mt][0] = O[g][mt][1] = O[g][mt][2] = O[g][mt][3] = 0.0f;
    }

    // One step of U 16-key tiles from position t0; ksc, ev: each tile's key
    // scale (negative: hidden) and the exponent of its value scale. kf(S):
    // the key products; entry i of S[g][u]: key gid + 8 (i / 2), row
    // 2 tig + i % 2. vf(u, mt, a): the values' operand. bias(g, i): the band's
    // entry for key gid + 8 (i / 2), row i % 2. some(u): whether any of this
    // lane's values is not 0 (called after kf). clean(u): values that are not
    // numbers to 0, and which of the tile's 16 keys had any among this lane's.
    auto step = [&](auto units, int t0, const float *ksc, float *ev, auto kf, auto vf, auto bias, auto some, auto clean) {
        constexpr int U = decltype(units)::value;
        float S[NB][U][4], f2[U], lv[U];
        kf(S);
        float top_ev = U == 2 ? fmaxf(ev[0], ev[U - 1]) : ev[0];
        if (top_ev > eref) {                           // the whole warp; seldom
#pragma unroll
            for (int u = 0; u < U; u++)
                if (!__any_sync(0xffffffffu, some(u))) ev[u] = kNoValue;
            top_ev = fmaxf(eref, U == 2 ? fmaxf(ev[0], ev[U - 1]) : ev[0]);
            const float f = exp2_fast(eref - top_ev);
#pragma unroll
            for (int g = 0; g < NB; g++)
#pragma unroll
                for (int mt = 0; mt < F::MT; mt++)
                    O[g][mt][0] *= f, O[g][mt][1] *= f, O[g][mt][2] *= f, O[g][mt][3] *= f;
            eref = top_ev;
        }
#pragma unroll
        for (int u = 0; u < U; u++) f2[u] = ksc[u], lv[u] = ev[u] - eref + kPBits;
        const bool biased = E && pa - (t0 + U * kK8Tile - 1) < E;
        const bool masked =
            t0 + U * kK8Tile - 1 > pa || (window && t0 <= pb - window) || ksc[0] < 0.0f || ksc[U - 1] < 0.0f;
        // Scores, in base 2: S * (f2 * qmul). In a step with a band or hidden keys
        // they are worked out here and the factor left is 1.
        bool scored = false;
        if (biased || masked) {
            scored = true;
            bool all = true;
            uint32_t nan[U];
#pragma unroll
            for (int g = 0; g < NB; g++)
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int at = t0 + u * kK8Tile + gid + 8 * (i >> 1), e = i & 1;
                        float y = S[g][u][i] * (f2[u] * qmul[g][e]);
                        if (biased) {
                            // a score of the type's lowest stays a number in base 2
                            const float b = bias(g, 4 * u + i) * tau[g][e];
                            y = fmaf(b, kLog2e, y);
                            if (y < kLowest && b > -INFINITY) y = kLowest;
                        }
                        if (at > pos[g][e] || (window && at <= pos[g][e] - window) || ksc[u] < 0.0f) y = -INFINITY;
                        S[g][u][i] = y;
                        all = all && y != -INFINITY;
                    }
            // A value that is not a number must not reach a row that does not
            // see its key (0 * NaN): in a step with hidden keys such values
            // count as 0, and a row that does see one gets a sum of NaN.
            if (__any_sync(0xffffffffu, !all)) {
#pragma unroll
                for (int u = 0; u < U; u++) {
                    nan[u] = __reduce_or_sync(0xffffffffu, clean(u));
#pragma unroll
                    for (int g = 0; g < NB; g++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (S[g][u][i] != -INFINITY && (nan[u] >> (gid + 8 * (i >> 1)) & 1))
                                l[g][i & 1] = __int_as_float(0x7fffffff);
                }
            }
        }
        float p[NB][U][4], top = -INFINITY;
        auto weigh = [&]() {
#pragma unroll
            for (int g = 0; g < NB; g++)
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int i = 0; i < 4; i++)        // exact where score and maximum are both the lowest
                        p[g][u][i] = fmaf(S[g][u][i], scored ? 1.0f : f2[u] * qmul[g][i & 1], -m2[g][i & 1]) + lv[u];
        };
        weigh();
#pragma unroll
        for (int g = 0; g < NB; g++)
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, p[g][u][i]);
        if (__any_sync(0xffffffffu, top > kPMax)) {
#pragma unroll
            for (int g = 0; g < NB; g++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float t = m2[g][e];
#pragma unroll
                    for (int u = 0; u < U; u++) {
                        const float f = scored ? 1.0f : f2[u] * qmul[g][e];
                        t = fmaxf(t, fmaxf(S[g][u][e] * f, S[g][u][2 + e] * f));
                    }
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 4));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 8));
                    t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, 16));
                    const float f = exp2_fast(m2[g][e] - t);
                    m2[g][e] = t;
                    l[g][e] *= f;
#pragma unroll
                    for (int mt = 0; mt < F::MT; mt++) O[g][mt][e] *= f, O[g][mt][2 + e] *= f;
                }
            weigh();
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const float il = exp2_fast(-lv[u]);
            // weights as two fp16 terms, for fp16 rows too: with one (11 bits) 41 % of the
            // results of 64 fp16 sequences were not the exact ones' fp16 values (86 us), with two 0.2 % (88.5)
            uint32_t w[NB][2][2];
#pragma unroll
            for (int g = 0; g < NB; g++) {
                float *q = p[g][u];
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = exp2_fast(q[i]);
#pragma unroll
                for (int e = 0; e < 2; e++) l[g][e] = fmaf(q[e] + q[2 + e], il, l[g][e]);
#pragma unroll
                for (int n = 0; n < 2; n++) {          // keys gid + 8 n: 8 x 8 weights, turned
                    const __half2 hi = __floats2half2_rn(q[2 * n], q[2 * n + 1]);
                    w[g][0][n] = transpose8(*reinterpret_cast<const uint32_t *>(&hi));
                    const float2 b = __half22float2(hi);
                    w[g][1][n] = transpose8(pack_half2(q[2 * n] - b.x, q[2 * n + 1] - b.y));
                }
            }
#pragma unroll
            for (int mt = 0; mt < F::MT; mt++) {
                uint32_t a[4];
                vf(u, mt, a);
#pragma unroll
                for (int g = 0; g < NB; g++)
#pragma unroll
                    for (int k = 0; k < 2; k++) mma16(O[g][mt], a, w[g][k][0], w[g][k][1]);
            }
        }
    };
    using One = std::integral_constant<int, 1>;

    // ---- the tail's fp16 tiles, one a warp, while the slots fill ----
    {
        const int t0 = tail0 + kK8Tile * warp;
        if (t0 >= c0 && t0 < c1) {
            const int64_t at = (((int64_t)sq.slot * Hkv + hk) * B + (t0 - tail0)) * Dh;
            const __half *K = (const __half *)P.c.k_tail + at, *V = (const __half *)P.c.v_tail + at;
            const int held = sq.held + sq.add - t0;    // keys of the tile that exist
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
            // Values as codes are: times the power of two that puts the tile's
            // largest in [2^8, 2^9), so that its weights are of the codes'
            // size (a scale of 1 would leave those of coded blocks few bits)
            __half2 most = __half2half2(__ushort_as_half(0));
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < F::VB / 2; e++) most = __hmax2(most, __habs2(*reinterpret_cast<const __half2 *>(&v[k][e])));
            const float amax = warp_max(fmaxf(__low2float(most), __high2float(most)));
            const int ex = amax > 0.0f ? (int)(__float_as_uint(amax) >> 23) - 127 - 8 : (int)kNoValue;
            const float f = __uint_as_float((uint32_t)(127 - ex) << 23), one = 1.0f;
            float ev_tail = (float)ex;
#pragma unroll
            for (int k = 0; k < 4; k++)
#pragma unroll
                for (int e = 0; e < F::VB / 2; e++) {
                    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&v[k][e]));
                    v[k][e] = pack_half2(x.x * f, x.y * f);
                }
            step(
                One(), t0, &one, &ev_tail,
                [&](float (&S)[NB][1][4]) {
#pragma unroll
                    for (int g = 0; g < NB; g++) S[g][0][0] = S[g][0][1] = S[g][0][2] = S[g][0][3] = 0.0f;
#pragma unroll
                    for (int ks = 0; ks < F::KS; ks++) {
                        const int d = 64 * (ks / 4) + 16 * tig + 4 * (ks % 4);
                        uint2 x[2];
#pragma unroll
                        for (int n = 0; n < 2; n++)
                            x[n] = gid + 8 * n < held && d < Dh ? *reinterpret_cast<const uint2 *>(K + (gid + 8 * n) * Dh + d)
                                                               : make_uint2(0, 0);
                        const uint32_t a[4] = {x[0].x, x[1].x, x[0].y, x[1].y};
#pragma unroll
                        for (int g = 0; g < NB; g++) {
                            uint32_t w[2 * TERMS];
                            q_op(g, ks, w);
#pragma unroll
                            for (int k = 0; k < TERMS; k++) mma16(S[g][0], a, w[2 * k], w[2 * k + 1]);
                        }
                    }
                },
                [&](int, int mt, uint32_t (&a)[4]) {   // dims 2 mt and 2 mt + 1 of the lane's: the two halves of word mt
                    a[0] = __byte_perm(v[0][mt], v[1][mt], 0x5410);
                    a[1] = __byte_perm(v[0][mt], v[1][mt], 0x7632);
                    a[2] = __byte_perm(v[2][mt], v[3][mt], 0x5410);
                    a[3] = __byte_perm(v[2][mt], v[3][mt], 0x7632);
                },
                [&](int g, int i) {
                    const int far = pos[g][i & 1] - (t0 + gid + 8 * (i >> 1));
                    return far >= 0 && far < E ? rel[rel_at[g][i & 1] + far] : 0.0f;
                },
                [&](int) { return true; },             // ev_tail is of the values themselves
                [&](int) {
                    uint32_t nan = 0;
#pragma unroll
                    for (int k = 0; k < 4; k++)
#pragma unroll
                        for (int e = 0; e < F::VB / 2; e++) {
                            const uint32_t at = __vcmpgtu2(v[k][e] & 0x7fff7fffu, 0x7c007c00u);
                            v[k][e] &= ~at;
                            nan |= at ? 1u << (2 * tig + (k & 1) + 8 * (k >> 1)) : 0u;
                        }
                    return nan;
                });
        }
    }

    for (int i = 0; i < mine; i++) {
        cp_async_wait<1>();                            // the keys
        __syncwarp();
        const float4 sc = *reinterpret_cast<const float4 *>(st + 2 * F::kTileB);
        float ksc[2] = {sc.x, sc.z};
        float ev[2] = {(float)((int)(__float_as_uint(sc.y) >> 23 & 255) - 127),
                             (float)((int)(__float_as_uint(sc.w) >> 23 & 255) - 127)};
        uint32_t v[4][F::VB / 4];
#pragma unroll 1
        for (int u0 = 0; u0 < 2; u0 += F::UNITS) {
        uint8_t *at = st + u0 * F::kTileB;
        step(
            std::integral_constant<int, F::UNITS>(), c0 + (warp + kK8Warps * i) * kK8Unit + u0 * kK8Tile, ksc + u0, ev + u0,
            [&](float (&S)[NB][F::UNITS][4]) {
                float R[NB][F::UNITS][4];              // the second term's sums, or the odd k steps'
#pragma unroll
                for (int g = 0; g < NB; g++)
#pragma unroll
                    for (int u = 0; u < F::UNITS; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) S[g][u][e] = R[g][u][e] = 0.0f;
#pragma unroll
                for (int j = 0; j < F::KW; j++) {
                    uint4 k[F::UNITS][2];
#pragma unroll
                    for (int u = 0; u < F::UNITS; u++)
#pragma unroll
                        for (int n = 0; n < 2; n++)
                            k[u][n] = *reinterpret_cast<const uint4 *>(at + u * F::kTileB + n * 8 * DP + from_k[j]);
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        uint32_t a[F::UNITS][4];
#pragma unroll
                        for (int u = 0; u < F::UNITS; u++) {
                            const uint32_t x = e == 0 ? k[u][0].x : e == 1 ? k[u][0].y : e == 2 ? k[u][0].z : k[u][0].w;
                            const uint32_t y = e == 0 ? k[u][1].x : e == 1 ? k[u][1].y : e == 2 ? k[u][1].z : k[u][1].w;
                            a[u][0] = e4m3_lo(x), a[u][1] = e4m3_lo(y), a[u][2] = e4m3_hi(x), a[u][3] = e4m3_hi(y);
                        }
#pragma unroll
                        for (int g = 0; g < NB; g++) {
                            uint32_t w[2 * TERMS];
                            q_op(g, 4 * j + e, w);
#pragma unroll
                            for (int u = 0; u < F::UNITS; u++) {
                                if constexpr (TERMS == 2) {
                                    mma16(S[g][u], a[u], w[0], w[1]);
                                    mma16(R[g][u], a[u], w[2 * TERMS - 2], w[2 * TERMS - 1]);
                                } else {
                                    mma16(e & 1 ? R[g][u] : S[g][u], a[u], w[0], w[1]);
                                }
                            }
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < NB; g++)
#pragma unroll
                    for (int u = 0; u < F::UNITS; u++)
#pragma unroll
                        for (int e = 0; e < 4; e++) S[g][u][e] += R[g][u][e];
                __syncwarp();                          // every lane has read the keys and the scales
                if (u0 + F::UNITS == 2) fetch_keys(i + 1);
                if (u0 == 0) {                         // the values
                    if constexpr (F::UNITS == 2) cp_async_wait<1>();
                    else cp_async_wait<0>();
                    __syncwarp();
                }
            },
            [&](int u, int mt, uint32_t (&a)[4]) {
                if (mt == 0) {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint8_t *src = at + u * F::kTileB + F::kKeyB + (k >> 1) * 8 * DP + from_v[k & 1];
                        if constexpr (F::VB == 16) *reinterpret_cast<uint4 *>(v[k]) = *reinterpret_cast<const uint4 *>(src);
                        else *reinterpret_cast<uint2 *>(v[k]) = *reinterpret_cast<const uint2 *>(src);
                    }
                }
                const uint32_t sel = mt & 1 ? 0x7362 : 0x5140;   // two dims of two keys
                const uint32_t x = __byte_perm(v[0][mt / 2], v[1][mt / 2], sel);
                const uint32_t y = __byte_perm(v[2][mt / 2], v[3][mt / 2], sel);
                a[0] = e4m3_lo(x), a[1] = e4m3_hi(x), a[2] = e4m3_lo(y), a[3] = e4m3_hi(y);
            },
            [&](int g, int k) {
                return *reinterpret_cast<const float *>(st + 2 * F::kTileB + F::kHeadB + (8 * g + 4 * u0 + k) * 128 + lane * 4);
            },
            [&](int u) {
                uint32_t any = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t *x = reinterpret_cast<const uint32_t *>(at + u * F::kTileB + F::kKeyB + (k >> 1) * 8 * DP + from_v[k & 1]);
#pragma unroll
                    for (int e = 0; e < F::VB / 4; e++) any |= x[e];
                }
                return (any & 0x7f7f7f7fu) != 0;
            },
            [&](int u) {                               // in the slots: no other lane reads these bytes
                uint32_t nan = 0;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint32_t *x = reinterpret_cast<uint32_t *>(at + u * F::kTileB + F::kKeyB + (k >> 1) * 8 * DP + from_v[k & 1]);
#pragma unroll
                    for (int e = 0; e < F::VB / 4; e++) {
                        const uint32_t y = __vcmpeq4(x[e] & 0x7f7f7f7fu, 0x7f7f7f7fu);
                        if (y) x[e] &= ~y;
                        nan |= y ? 1u << (2 * tig + (k & 1) + 8 * (k >> 1)) : 0u;
                    }
                }
                return nan;
            });
        }
        __syncwarp();                                  // every lane has read the values
        fetch_values(i + 1);
    }
    cp_async_wait<0>();
    __syncthreads();

    // ---- merge the warps, in warp order. A row's output lies in the order
    // of the lanes: entry 8 x + c is dim c * VB + x ----
    float *mg = reinterpret_cast<float *>(smem) + warp * RT * F::kPitch;
    float2 *ml = reinterpret_cast<float2 *>(reinterpret_cast<float *>(smem) + kK8Warps * RT * F::kPitch);
    const float unit = exp2_fast(eref - kPBits);
#pragma unroll
    for (int g = 0; g < NB; g++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = 8 * g + 2 * tig + e;
            l[g][e] += __shfl_xor_sync(0xffffffffu, l[g][e], 4);
            l[g][e] += __shfl_xor_sync(0xffffffffu, l[g][e], 8);
            l[g][e] += __shfl_xor_sync(0xffffffffu, l[g][e], 16);
            if (gid == 0) ml[warp * RT + r] = make_float2(m2[g][e], l[g][e]);
#pragma unroll
            for (int mt = 0; mt < F::MT; mt++) {
                mg[r * F::kPitch + 16 * mt + gid] = unit * O[g][mt][e];
                mg[r * F::kPitch + 16 * mt + 8 + gid] = unit * O[g][mt][2 + e];
            }
        }
    __syncthreads();
    // a warp merges whole rows, 4 dims a lane
    for (int r = warp; r < min(rows, RT); r += kK8Warps) {
        float M = kLowest, L = 0.0f, A[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        float2 x[kK8Warps];
#pragma unroll
        for (int w = 0; w < kK8Warps; w++) x[w] = ml[w * RT + r], M = fmaxf(M, x[w].x);
        const int d = 4 * lane, c = d / F::VB + 8 * (d % F::VB);
        const float *o = reinterpret_cast<const float *>(smem) + r * F::kPitch + c;
#pragma unroll
        for (int w = 0; w < kK8Warps; w++) {
            const float f = exp2_fast(x[w].x - M);
            L += f * x[w].y;
            if (d < DP)
#pragma unroll
                for (int e = 0; e < 4; e++) A[e] += f * o[w * RT * F::kPitch + 8 * e];
        }
        if (P.splits == 1) {
            int t, h;
            row_of(r, t, h);
            if (d < Dh) put_row((T *)P.a.out + ((int64_t)(sq.n0 + t) * H + h) * Dh + d, A, L);
        } else {
            if (d < Dh) *reinterpret_cast<float4 *>(P.part + (cell + r) * Dh + d) = make_float4(A[0], A[1], A[2], A[3]);
            if (lane == 0) P.part_ml[cell + r] = make_float2(M, L);
        }
    }
}

// Merges the chunks of a row, W warps to a row: each takes a run of them in
// order, then their results are added in order. One CTA does kK8Warps / W
// rows. Chunks that no key fell into hold a sum of 0.
template <typename T, int NB, int W>
__global__ void __launch_bounds__(kK8Threads) k_kv8_merge(const K8Params P) {
    constexpr int RT = 8 * NB;
    __shared__ float s_part[W > 1 ? kK8Warps : 1][kKv8MaxDh];
    __shared__ float2 s_ml[kK8Warps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, d = 4 * lane;
    const int Dh = P.c.head_dim, H = P.a.n_heads, G = P.G, s = blockIdx.y;
    const int at = blockIdx.x * (kK8Warps / W) + warp / W, h = at % H, t = at / H;
    const int hk = h / G, R = t * G + h - hk * G, rt = R / RT, r = R - rt * RT;
    if (t >= P.b.max_new) return;                      // with W > 1 the whole CTA
    const int64_t cell = ((int64_t)(s * P.c.n_kv_heads + hk) * P.row_tiles + rt) * P.splits * RT + r;
    const int per = (P.splits + W - 1) / W, k0 = (warp % W) * per, k1 = min(P.splits, k0 + per);
    griddep_wait();
    griddep_launch();
    const int n0 = P.b.start ? P.b.start[s] : s, n1 = P.b.start ? P.b.start[s + 1] : s + 1;
    float M = kLowest, L = 0.0f, A[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    constexpr int kAhead = 16;                         // chunks in flight per warp
    for (int k = k0; k < k1; k += kAhead) {
        float4 x[kAhead];
        float2 y[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; i++) {
            const int64_t c = cell + (int64_t)min(k + i, k1 - 1) * RT;
            y[i] = __ldcg(P.part_ml + c);
            x[i] = d < Dh ? __ldcg(reinterpret_cast<const float4 *>(P.part + c * Dh + d)) : make_float4(0, 0, 0, 0);
        }
        float top = M;
#pragma unroll
        for (int i = 0; i < kAhead; i++) top = fmaxf(top, y[i].x);
        const float g = exp2_fast(M - top);
        M = top;
        L *= g, A[0] *= g, A[1] *= g, A[2] *= g, A[3] *= g;
#pragma unroll
        for (int i = 0; i < kAhead; i++)
            if (k + i < k1 && y[i].y != 0.0f) {        // an empty chunk's row was not written
                const float f = exp2_fast(y[i].x - M);
                L += f * y[i].y;
                A[0] += f * x[i].x, A[1] += f * x[i].y, A[2] += f * x[i].z, A[3] += f * x[i].w;
            }
    }
    if constexpr (W > 1) {
        if (d < Dh) *reinterpret_cast<float4 *>(&s_part[warp][d]) = make_float4(A[0], A[1], A[2], A[3]);
        if (lane == 0) s_ml[warp] = make_float2(M, L);
        __syncthreads();
        if (warp) return;
        M = kLowest;
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, s_ml[w].x);
        L = A[0] = A[1] = A[2] = A[3] = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = exp2_fast(s_ml[w].x - M);
            L += f * s_ml[w].y;
            if (d < Dh)
#pragma unroll
                for (int e = 0; e < 4; e++) A[e] += f * s_part[w][d + e];
        }
    }
    // a sequence whose rows break a bound has none here (k_kv8_attn zeroed what lies inside the step)
    if (d < Dh && kv8_rows_ok(P.b, n0, n1 - n0) && t < n1 - n0)
        put_row((T *)P.a.out + ((int64_t)(n0 + t) * H + h) * Dh + d, A, L);
}

struct K8Plan {
    int G, rt, row_tiles, splits, chunk;   // rt: rows of a tile
    size_t cells, bytes;
};

// Chunks: one wave of equal chunks over all CTA slots while that leaves a
// chunk at most kMaxChunk positions; longer work runs in several waves of
// kMaxChunk, so that ragged sequences even out (64 ragged sequences: 89 us
// with 1024, 95 with 512). Where rows alone make four waves (long pieces of
// prompts) nothing is cut: 512 new tokens on 4096 take 497 us, cut 582, and no
// workspace.
static K8Plan k8_plan(const SepiaKv8Cache &c, const SepiaKv8Step &b, const SepiaKv8Attn &a) {
    constexpr int64_t kUnit = kK8Unit * kK8Warps, kMaxChunk = 1024;
    K8Plan p;
    p.G = a.n_heads / c.n_kv_heads;
    // Two groups of 8 rows a tile convert half the codes, but take 168
    // registers a thread where one takes 128. Measured as one group / two (us,
    // fp32, 8 heads a KV head): 12 sequences of 6001 with 32 rows 79 / 86, 48
    // rows 115 / 115, 64 rows 151 / 147, 72 rows 169 / 164, 128 rows 295 / 274;
    // 1 x 32768 with 40 rows 62 / 69, 64 rows 90 / 85; 6 x 300 with 48 rows 18.1 /
    // 17.9, 64 rows 19.8 / 24.4. From 48 to 64 rows neither side wins; the rule
    // keeps the one that small calls need.
    const int rt = p.rt = (int64_t)b.max_new * p.G <= 64 ? 8 : 16;
    p.row_tiles = (int)(((int64_t)b.max_new * p.G + rt - 1) / rt);
    const int64_t span = a.window ? std::min<int64_t>(b.max_kv, (int64_t)a.window + b.max_new + kK8Tile) : b.max_kv;
    const int64_t groups = (int64_t)b.n_seqs * c.n_kv_heads * p.row_tiles;
    const int64_t slots = (int64_t)(dev_info().sm_count > 0 ? dev_info().sm_count : 148) * k8_ctas(rt / 8);
    const int64_t one = (groups * span + slots - 1) / slots;
    const int64_t want = groups >= 4 * slots ? span : std::min(kMaxChunk, one);
    p.chunk = (int)((std::max<int64_t>(want, 1) + kUnit - 1) / kUnit * kUnit);
    p.splits = (int)std::max<int64_t>(1, (span + p.chunk - 1) / p.chunk);
    p.cells = p.splits > 1 ? (size_t)groups * p.splits * rt : 0;
    p.bytes = p.cells * (c.head_dim * 4 + 8);
    return p;
}

template <typename T, int DP, int NB, bool FULL>
static int k8_launch(K8Params &P, cudaStream_t st) {
    using F = K8Cfg<T, DP, NB>;
    const int64_t rows = (int64_t)P.b.max_new * P.a.n_heads;
    const int smem = std::max(F::kQB + kK8Warps * F::stage(P.a.rel_extent > 0), F::kMergeB);
    if (!ensure_smem((const void *)k_kv8_attn<T, DP, NB, FULL>, smem)) return 0;
    // The tiles of a long piece of a prompt (16384 tokens of 64 heads) may be
    // more than a grid's y holds; k8_plan cuts tiles only where they are few.
    constexpr int kMaxY = 65535;
    const int tiles = P.c.n_kv_heads * P.row_tiles;
    for (P.tile0 = 0; P.tile0 < tiles; P.tile0 += kMaxY) {
        const dim3 grid((unsigned)P.splits, (unsigned)std::min(kMaxY, tiles - P.tile0), (unsigned)P.b.n_seqs);
        if (!check(launch_pdl(k_kv8_attn<T, DP, NB, FULL>, grid, dim3(kK8Threads), smem, st, P), "kv8_attn launch")) return 0;
    }
    if (P.splits == 1) return 1;
    // One warp per row while a row has few chunks, four beyond: 64 sequences of
    // 4 chunks 89 us (four warps: 101), one of 64 chunks 20.5 us (one warp: 25).
    const dim3 g1((unsigned)((rows + kK8Warps - 1) / kK8Warps), (unsigned)P.b.n_seqs), g4((unsigned)rows, (unsigned)P.b.n_seqs);
    const cudaError_t e = P.splits <= 8 ? launch_pdl(k_kv8_merge<T, NB, 1>, g1, dim3(kK8Threads), 0, st, P)
                                        : launch_pdl(k_kv8_merge<T, NB, 4>, g4, dim3(kK8Threads), 0, st, P);
    return check(e, "kv8_attn merge launch");
}

template <typename T, int DP, bool FULL>
static int k8_launch_rows(K8Params &P, int rt, cudaStream_t st) {
    return rt == 8 ? k8_launch<T, DP, 1, FULL>(P, st) : k8_launch<T, DP, 2, FULL>(P, st);
}

template <typename T>
static int k8_launch_dim(K8Params &P, int rt, cudaStream_t st) {
    const int Dh = P.c.head_dim;
    if (Dh <= 64) return Dh == 64 ? k8_launch_rows<T, 64, true>(P, rt, st) : k8_launch_rows<T, 64, false>(P, rt, st);
    return Dh == 128 ? k8_launch_rows<T, 128, true>(P, rt, st) : k8_launch_rows<T, 128, false>(P, rt, st);
}

static int k8_check(const SepiaKv8Cache *c, const SepiaKv8Step *b, const SepiaKv8Attn *a) {
    const char *what = "kv8_attn";
    if (!kv8_check(c, b, what)) return 0;
    if (!a) return fail("%s: null argument", what);
    if (a->n_heads <= 0 || a->n_heads % c->n_kv_heads)
        return fail("%s: %d query heads over %d KV heads", what, a->n_heads, c->n_kv_heads);
    if (a->window < 0 || a->rel_extent < 0) return fail("%s: negative window or rel_extent", what);
    // offsets inside a tile's bands are 32-bit: at most 17 tokens
    if ((int64_t)a->n_heads * a->rel_extent > INT32_MAX / 17) return fail("%s: rel_extent %d too large", what, a->rel_extent);
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
    if (reinterpret_cast<uintptr_t>(a->out) & (a->x_f16 ? 7 : 15)) return fail("%s: out must be aligned to 4 elements", what);
    if (a->q_stride < (int64_t)a->n_heads * c->head_dim) return fail("%s: q_stride is shorter than a token", what);
    if (a->rel_extent && !a->rel_logits) return fail("%s: rel_extent without rel_logits", what);
    const K8Plan p = k8_plan(*c, *b, *a);
    if (p.splits > 1 && (int64_t)c->n_kv_heads * p.row_tiles > 65535) return fail("%s: step too large", what);
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
    const int64_t q_b = a->x_f16 ? 8 : 16, q_sz = a->x_f16 ? 2 : 4;
    P.q_vec = reinterpret_cast<uintptr_t>(a->q) % q_b == 0 && a->q_stride * q_sz % q_b == 0;
    P.part = (float *)ws;
    P.part_ml = (float2 *)(P.part + p.cells * c->head_dim);
    P.err = dev_info().err;
    cudaStream_t st = as_stream(stream);
    return a->x_f16 ? k8_launch_dim<__half>(P, p.rt, st) : k8_launch_dim<float>(P, p.rt, st);
}
