// sepia_b200/csrc/kv8.cuh -- what the kernels of the paged 8-bit K/V cache
// share (layout and rules: include/sepia_cuda.h, SepiaKv8Cache): a
// sequence's part of a step, checked on the device, and the block lookup.
#pragma once
#include "../../include/sepia_cuda.h"
#include "common.cuh"

namespace sepia {

constexpr int kKv8MaxDh = 128;

// One sequence's part of a step. add < 0: idle or out of bounds; `rows` of
// its token rows, from n0, still lie inside the step's n_tokens, and may be
// more than max_new where that bound is the broken one.
struct Kv8Seq {
    int n0, rows;        // first new token, token rows inside the step
    int held, add;       // tokens held before the step, new tokens
    int slot;
};

// Whether a sequence's token rows are within the step's bounds
__device__ __forceinline__ bool kv8_rows_ok(const SepiaKv8Step &b, int n0, int add) {
    return n0 >= 0 && add >= 0 && (int64_t)n0 + add <= b.n_tokens && add <= b.max_new;
}

__device__ __forceinline__ Kv8Seq kv8_seq(const SepiaKv8Cache &c, const SepiaKv8Step &b, int s, int *err) {
    Kv8Seq q;
    q.held = b.kv_len[s];
    q.slot = b.slot ? b.slot[s] : s;
    q.n0 = b.start ? b.start[s] : s;
    q.add = b.start ? b.start[s + 1] - q.n0 : 1;
    const bool rows_ok = kv8_rows_ok(b, q.n0, q.add);
    q.rows = rows_ok ? q.add : q.n0 >= 0 ? max(0, min(q.add, b.n_tokens - q.n0)) : 0;
    const int64_t total = (int64_t)q.held + q.add;
    const bool fits = total <= b.max_kv && total <= (int64_t)b.table_cols * c.block && q.slot >= 0 && q.slot < c.n_slots;
    if (q.held < 0 || !rows_ok || !fits) {
        if (!rows_ok || q.held >= 0) set_error(err, kErrBadArgs);
        q.add = -1;
    }
    return q;
}

// Zeros for the step's rows of a sequence that is skipped, row elements `row`,
// by the threads first, first + all, ...; out of line, for it is rare and
// would cost the kernels around it registers.
template <typename T>
__device__ __noinline__ void kv8_zero_rows(T *out, int n0, int rows, int row, unsigned first, unsigned all) {
    const int64_t n = (int64_t)rows * row;
    for (int64_t e = first; e < n; e += all) out[(int64_t)n0 * row + e] = (T)0.0f;
}

// Pool block of column `col` of sequence s; -1 (and the error word) if the table's entry is out of range.
__device__ __forceinline__ int kv8_block(const SepiaKv8Cache &c, const SepiaKv8Step &b, int s, int col, int *err) {
    const int id = b.table[(int64_t)s * b.table_cols + col];
    if (id >= 0 && id < c.n_blocks) return id;
    set_error(err, kErrBadArgs);
    return -1;
}

// Host checks of a cache and a step; 1, or 0 with a message.
int kv8_check(const SepiaKv8Cache *c, const SepiaKv8Step *b, const char *what);

}  // namespace sepia
