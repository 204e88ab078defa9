// pgc_ragged.cuh — a ragged batch as the kernels read it: per-sequence query rows and lengths from
// device memory, checked against the host bounds that sized the launch and the workspace.
#pragma once

#include "pgc_common.cuh"
#include "pgc_internal.h"

namespace pgc {

struct RaggedSeq {
    int row0;  // first query row; -1: q_starts is out of order here
    int n;     // query rows; 0: nothing to do
    int len;   // cached tokens, the queries included
};

// Sequence b. Query rows outside [0, total_q] or out of order: the sequence is skipped (n = 0), and so
// are all behind it, for which the caller looks out (row0 = -1): no row then belongs to two sequences,
// and a batch has at most total_q rows. More rows than max_q_len: the sequence is skipped. A length outside
// [0, max_seq_len]: its cache counts as empty, so its rows see nothing. All are recorded in *err
// (nullable: one thread of a launch records).
__device__ __forceinline__ RaggedSeq ragged_seq(const RaggedBatch &r, int b, DevError *err) {
    RaggedSeq s;
    const int end = r.q_starts[b + 1];
    s.row0 = r.q_starts[b];
    s.len = r.seq_lens[b];
    // 0 <= row0 <= end <= total_q is checked first, so the difference cannot overflow
    const bool in_order = s.row0 >= 0 && end >= s.row0 && end <= r.total_q;
    if (!in_order || end - s.row0 > r.max_q_len) {
        if (err != nullptr) record_error(err, kErrRowsOutOfRange, b);
        s.row0 = in_order ? 0 : -1;
        s.n = 0;
        return s;
    }
    s.n = end - s.row0;
    if (s.len < 0 || s.len > r.max_seq_len) {
        if (err != nullptr && s.n > 0) record_error(err, kErrLenOutOfRange, b);
        s.len = 0;
    }
    return s;
}

// The sum of the costs of the sequences before the first whose cost is -1 (rows out of order), and their
// number. Called by a whole warp.
__device__ __forceinline__ int64_t ragged_total(const int64_t *cost, int batch, int &live) {
    const int lane = threadIdx.x & 31;
    auto sum = [&](int end, int &first_bad) {
        int64_t total = 0;
        for (int b = lane; b < end; b += 32) {
            if (cost[b] < 0)
                first_bad = min(first_bad, b);
            else
                total += cost[b];
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        first_bad = __reduce_min_sync(0xffffffffu, first_bad);
        return total;
    };
    live = batch;
    int64_t total = sum(batch, live);
    if (live < batch) total = sum(live, live);
    return total;
}

// Slot of sequence b in a slot-indexed array, -1 when it may not be used: outside [0, num_slots),
// or named by an earlier sequence of the batch too (the slot belongs to the first). Called by a
// whole warp; slots == nullptr is the identity (the host checked batch <= num_slots).
__device__ __forceinline__ int64_t ragged_slot(const int32_t *slots, int64_t num_slots, int b, DevError *err) {
    if (slots == nullptr) return b;
    const int lane = threadIdx.x & 31;
    const int32_t slot = slots[b];
    bool bad = slot < 0 || slot >= num_slots;
    for (int i = lane; i < b; i += 32) bad |= slots[i] == slot;
    if (!__any_sync(0xffffffffu, bad)) return slot;
    if (err != nullptr && lane == 0) record_error(err, kErrSlotOutOfRange, b);
    return -1;
}

}  // namespace pgc
