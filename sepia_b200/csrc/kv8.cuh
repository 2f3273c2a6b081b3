// sepia_b200/csrc/kv8.cuh -- what the kernels of the paged 8-bit K/V cache
// share (layout and rules: include/sepia_cuda.h, SepiaKv8Cache): a
// sequence's part of a step, checked on the device, and the block lookup.
#pragma once
#include "../../include/sepia_cuda.h"
#include "common.cuh"

namespace sepia {

constexpr int kKv8MaxDh = 128;

// One sequence's part of a step. add < 0: idle or out of bounds (`rows` of
// its token rows, from n0, still lie inside the step's n_tokens).
struct Kv8Seq {
    int n0, rows;        // first new token, token rows inside the step
    int held, add;       // tokens held before the step, new tokens
    int slot;
};

__device__ __forceinline__ Kv8Seq kv8_seq(const SepiaKv8Cache &c, const SepiaKv8Step &b, int s, int *err) {
    Kv8Seq q;
    q.held = b.kv_len[s];
    q.slot = b.slot ? b.slot[s] : s;
    q.n0 = b.start ? b.start[s] : s;
    q.add = b.start ? b.start[s + 1] - q.n0 : 1;
    const bool rows_ok = q.n0 >= 0 && q.add >= 0 && (int64_t)q.n0 + q.add <= b.n_tokens && q.add <= b.max_new;
    q.rows = rows_ok ? q.add : 0;
    const int64_t total = (int64_t)q.held + q.add;
    const bool fits = total <= b.max_kv && total <= (int64_t)b.table_cols * c.block && q.slot >= 0 && q.slot < c.n_slots;
    if (q.held < 0 || !rows_ok || !fits) {
        if (!rows_ok || q.held >= 0) set_error(err, kErrBadArgs);
        q.add = -1;
    }
    return q;
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
