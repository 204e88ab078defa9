// pgc_ragged.cuh — a ragged batch as the kernels read it: per-sequence query rows and lengths from
// device memory, checked against the host bounds that sized the launch and the workspace.
#pragma once

#include "pgc_common.cuh"
#include "pgc_internal.h"

namespace pgc {

struct RaggedSeq {
    int row0;  // first query row
    int n;     // query rows; 0: nothing to do
    int len;   // cached tokens, the queries included
};

// Sequence b. Query rows outside [0, total_q], out of order or more than max_q_len: the sequence is
// skipped (n = 0). A length outside [0, max_seq_len]: its cache counts as empty, so its rows see
// nothing. Both are recorded in *err (nullable: one thread of a launch records).
__device__ __forceinline__ RaggedSeq ragged_seq(const RaggedBatch &r, int b, DevError *err) {
    RaggedSeq s;
    const int end = r.q_starts[b + 1];
    s.row0 = r.q_starts[b];
    s.len = r.seq_lens[b];
    // 0 <= row0 <= end <= total_q is checked first, so the difference cannot overflow
    if (s.row0 < 0 || end < s.row0 || end > r.total_q || end - s.row0 > r.max_q_len) {
        if (err != nullptr) record_error(err, kErrRowsOutOfRange, b);
        s.row0 = s.n = 0;
        return s;
    }
    s.n = end - s.row0;
    if (s.len < 0 || s.len > r.max_seq_len) {
        if (err != nullptr && s.n > 0) record_error(err, kErrLenOutOfRange, b);
        s.len = 0;
    }
    return s;
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
