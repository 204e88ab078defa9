// chunk_attn.cu — causal GQA attention of a ragged batch of chunks over the paged cache, with the
// log-sum-exp of every row and, on request, each cached token's received attention (sm_100a).
//
// For sequence b with n query rows and L cached tokens (the rows included), row i sits at position
// p = L - n + i and sees tokens [0, p]:
//     s_t = scale q.k_t,  lse = log sum_{t <= p} exp(s_t),  o = sum_t exp(s_t - lse) v_t
// and, with weights, w[kv head][t] += sum over the kv head's 4 query heads and the rows of
// exp(s_t - lse). A row that sees nothing (p < 0) has o = 0 and lse = -inf.
//
// Forms, chosen by the host bounds:
//   * up to PGC_MAX_QUERIES rows a sequence: chunk_split_kernel (mma.sync), bound by the K/V bytes (64
//     sequences of 1024 to 32768 tokens, 2.1 GB: 333 us, 6.3 TB/s); with weights it leaves the scores in
//     the workspace, 16 B per row, kv head and token beside 1 KiB of K and V, so that K is read once.
//     Few short sequences take its cluster form, bound by latency (one row over 4097 tokens: 10.3 us,
//     over 500: 6.6);
//   * more rows: chunk_pair_kernel on the 5th-gen tensor cores (1600 tokens over 24576: 540 us, 1230
//     TFLOP/s), and chunk_weights.cu for the weights.
// These are medians of calls behind one another; the first ones, before the power cap lowers the clock, take
// 323 us and 464 (1430 TFLOP/s). Comparisons of large calls below were taken in such short bursts.
// But for the cluster form, the line of all the batch's tiles is cut into equal consecutive shares, one
// per CTA (or pair) of a fixed grid: lengths are on the device, and a grid by the host's bounds would be
// empty for the most part where they are ragged (387 us for the 64 sequences above). A unit of work cut by
// a share's border leaves fp32 partials, at most two units a share (its first and its last), which a
// second kernel joins; every other unit is written where it is computed.
#include <cuda.h>

#include <type_traits>

#include "pgc_common.cuh"
#include "pgc_internal.h"
#include "pgc_ragged.cuh"
#include "pgc_tcgen05.cuh"

namespace pgc {

PGC_DEFINE_ERROR_WORD(g_chunk_err);

namespace {

// v * sigmoid(gate) with the approximate exponential and reciprocal: off by (4 + 2 |gate|) ulp at most
// (2 of the exponential, 1 of the reciprocal, 1 of the product; the exponent's rounding is |gate| log2(e)
// half ulps), far inside the bf16 rounding behind it, down to gates of -87.3. Below, where the sigmoid is
// less than 2^-126, the reciprocal is flushed and the result is 0: off by 2^-126 |v| at most. The exact ones
// were 5 us of a 64-token unit's end.
__device__ __forceinline__ float sigmoid_gate(float v, uint32_t gate_bits) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp2(-kLog2e * bf16_bits_to_f32(gate_bits))));
    return v * r;
}

// A row's log-sum-exp as the weights take it: in log2 units, in which the scores are, since the way through
// natural units and back rounds three times where |m| is large; +inf for a row whose sum is 0, so that
// its -inf scores add nothing. Partials hold their maxima in log2 units too.
__device__ __forceinline__ float lse_log2(float m, float sum) { return sum == 0.f ? INFINITY : m + log2f(sum); }
// The same for the caller: natural units, -inf for such a row.
__device__ __forceinline__ float lse_natural(float m, float sum) { return sum == 0.f ? -INFINITY : m * kLn2 + logf(sum); }

// =============================================================================================
// The schedule. A unit is a (sequence, kv head, block of kTok query tokens); its tiles are blocks of
// kKeys keys. The line of work is the units' tiles, units in that order, each unit preceded by the
// kOver tiles' worth of time that its start and end cost (Q's load, the pipeline's drain and the
// epilogue), so that shares of many small units are not longer than shares of one large one.
// =============================================================================================
struct PairTiling {
    static constexpr int kTok = 64, kKeys = 128;
    static constexpr bool kWarpScan = false;
    static constexpr int kOver = 4;  // measured: 10 to 12 thousand cycles a unit, 2600 a tile
    // at least one tile behind a lead: 26.2 us against 32.6 with 8 for 3 chunks of up to 90 over 1500, 23.7
    // against 26.8 for 20 rows over 3000
    static constexpr int kMinShare = 5;
};
struct SplitTiling {
    static constexpr int kTok = PGC_MAX_QUERIES, kKeys = kPage;
    static constexpr bool kWarpScan = true;
    static constexpr int kOver = 1;
    static constexpr int kMinShare = 5;
};
static_assert(PairTiling::kMinShare > PairTiling::kOver && SplitTiling::kMinShare > SplitTiling::kOver,
              "a share that begins in a unit's lead must reach its first tile");

// Tiles of one unit: the keys that its last row sees, at least one tile (rows that see nothing still
// get their zeros).
template <class T>
__device__ __forceinline__ int unit_tiles(int n, int len, int qt) {
    const int keys = len - n + min((qt + 1) * T::kTok, n);
    return keys > T::kKeys ? (keys + T::kKeys - 1) / T::kKeys : 1;
}

// A share as a walk over (unit, tile range); every role steps its own copy.
struct Walk {
    int seq, kvh, qt;
    int row0, n, len;  // of the sequence
    int tiles;         // of the unit
    int t0, t1;        // the share's tiles of it
    int off;           // where the share enters the unit's kOver + tiles
    int left;          // of the share from there on
};

__device__ __forceinline__ void walk_seq(const RaggedBatch &rag, Walk &w) {
    const RaggedSeq s = ragged_seq(rag, w.seq, nullptr);
    w.row0 = s.row0;
    w.n = s.n;
    w.len = s.len;
}
template <class T>
__device__ __forceinline__ void walk_unit(Walk &w, int off) {
    w.tiles = unit_tiles<T>(w.n, w.len, w.qt);
    w.off = off;
    w.t0 = max(0, off - T::kOver);
    const int cost = w.tiles + T::kOver;
    w.t1 = w.left >= cost - off ? w.tiles : off + w.left - T::kOver;
}
// Next unit; false at the end of the share. A share that ends in a unit's lead leaves the unit to the
// next share.
template <class T>
__device__ __forceinline__ bool walk_next(const RaggedBatch &rag, Walk &w) {
    w.left -= w.tiles + T::kOver - w.off;
    if (w.left <= T::kOver) return false;
    if (++w.qt * T::kTok >= w.n) {
        w.qt = 0;
        if (++w.kvh == kNumKvHeads) {
            w.kvh = 0;
            do {
                if (++w.seq >= rag.batch) return false;
                walk_seq(rag, w);
            } while (w.n == 0);
        }
    }
    walk_unit<T>(w, 0);
    return true;
}
// Whether the unit is the share's last: what walk_next would say, without stepping.
template <class T>
__device__ __forceinline__ bool walk_last(const Walk &w) {
    return w.left - (w.tiles + T::kOver - w.off) <= T::kOver;
}

// The line's length and the shares it is cut into: the first `longer` ones take base + 1 tiles, the
// others base.
struct Line {
    int64_t total, base;
    int shares, longer;
};

// 64-bit quotients of non-negative numbers, in 32 bits where they fit (the 64-bit division is a few
// hundred cycles on the way to the first load).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
    return a / b;
}
template <class T>
__device__ __forceinline__ Line make_line(int64_t total, int grid) {
    Line l;
    const int64_t w = quotient(total, T::kMinShare);
    l.total = total;
    l.shares = w < 1 ? 1 : w > grid ? grid : (int)w;
    l.base = quotient(total, l.shares);
    l.longer = (int)(total - l.base * l.shares);
    return l;
}
__device__ __forceinline__ int64_t share_begin(const Line &l, int index) { return l.base * index + min(index, l.longer); }
__device__ __forceinline__ int share_of(const Line &l, int64_t tile) {
    const int64_t cut = (l.base + 1) * l.longer;
    return tile < cut ? (int)quotient(tile, l.base + 1) : l.longer + (int)quotient(tile - cut, l.base);
}

// Start of the walk: `off` into sequence wk.seq, whose kv heads take `per` of the line each.
template <class T>
__device__ __forceinline__ void walk_start(Walk &wk, int64_t off, int64_t per, int64_t left) {
    wk.kvh = (int)quotient(off, per);
    off -= wk.kvh * per;
    for (wk.qt = 0;; ++wk.qt) {
        const int c = unit_tiles<T>(wk.n, wk.len, wk.qt) + T::kOver;
        if (off < c) break;
        off -= c;
    }
    // Within int from 18 shares on: the sequences' rows are disjoint, so there are at most 2^22 / 64 + 4096
    // units a kv head, of at most 2^17 tiles and a lead.
    wk.left = (int)left;
    walk_unit<T>(wk, (int)off);
}
template <class T>
__device__ __forceinline__ int64_t seq_cost(const RaggedSeq &s) {  // of one kv head
    if (s.n <= T::kTok) return s.n == 0 ? 0 : unit_tiles<T>(s.n, s.len, 0) + T::kOver;
    int64_t c = 0;
    for (int qt = 0; qt * T::kTok < s.n; ++qt) c += unit_tiles<T>(s.n, s.len, qt) + T::kOver;
    return c;
}

// Share `index` of a grid of `grid`. Run by the whole CTA; `line` (shared memory) is written by thread
// 0, `out` is shared memory that the larger batches go through, `cost` their scratch (one int64 per
// sequence). Returns false when the share is empty. Sequences from the first with rows out of order on have
// no tiles; `live` (nullable) gets the number of those before it. With kWarpScan batches of up to 128 sequences are scanned by every warp for itself,
// which needs no barrier: 1.5 us off a single sequence's decode (in the pair kernel the registers that it
// takes cost 2 % of the main loop).
template <class T>
__device__ __forceinline__ bool find_share(const RaggedBatch &rag, int64_t *cost, int index, int grid, Walk *out,
                                           Line *line, DevError *err, Walk &wk, int *live_out = nullptr) {
    constexpr int kChunks = 4;
    const int lane = threadIdx.x & 31;
    wk.seq = -1;
    if (T::kWarpScan && rag.batch <= 32 * kChunks) {
        // a sequence has at most 2^22 tiles and leads (PGC_CHUNK_MAX_TOKENS): 32 bits hold the line
        RaggedSeq s[kChunks];
        int c[kChunks], incl[kChunks], total = 0, live = rag.batch;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            s[k] = RaggedSeq{0, 0, 0};
            if (k * 32 + lane < rag.batch) s[k] = ragged_seq(rag, k * 32 + lane, threadIdx.x < 32 ? err : nullptr);
            c[k] = incl[k] = 0;
        }
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            if (k * 32 >= rag.batch) break;
            const uint32_t bad = __ballot_sync(0xffffffffu, s[k].row0 < 0);
            if (bad != 0) live = min(live, k * 32 + __ffs(bad) - 1);
            c[k] = k * 32 + lane < live ? (int)seq_cost<T>(s[k]) * kNumKvHeads : 0;
            incl[k] = c[k];
#pragma unroll 1
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl[k], o);
                if (lane >= o) incl[k] += v;
            }
            incl[k] += total;
            total = __shfl_sync(0xffffffffu, incl[k], 31);
        }
        const Line ln = make_line<T>(total, grid);
        if (threadIdx.x == 0) {
            *line = ln;
            if (live_out != nullptr) *live_out = live;
        }
        const int begin = (int)share_begin(ln, index), end = (int)share_begin(ln, index + 1);
        if (index >= ln.shares || end <= begin) return false;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            const uint32_t hit = __ballot_sync(0xffffffffu, incl[k] > begin);
            if (hit == 0) continue;
            const int src = __ffs(hit) - 1;
            wk.seq = k * 32 + src;
            wk.row0 = __shfl_sync(0xffffffffu, s[k].row0, src);
            wk.n = __shfl_sync(0xffffffffu, s[k].n, src);
            wk.len = __shfl_sync(0xffffffffu, s[k].len, src);
            const int all = __shfl_sync(0xffffffffu, c[k], src);
            const int before = __shfl_sync(0xffffffffu, incl[k], src) - all;
            walk_start<T>(wk, begin - before, all / kNumKvHeads, end - begin);
            break;
        }
        return true;
    }
    for (int b = threadIdx.x; b < rag.batch; b += blockDim.x) {
        const RaggedSeq s = ragged_seq(rag, b, err);
        cost[b] = s.row0 < 0 ? -1 : seq_cost<T>(s) * kNumKvHeads;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int live;
        const int64_t total = ragged_total(cost, rag.batch, live);
        const Line ln = make_line<T>(total, grid);
        const int64_t begin = share_begin(ln, index), end = share_begin(ln, index + 1);
        if (index < ln.shares && end > begin) {
            int64_t before = 0;
            for (int b0 = 0; b0 < live; b0 += 32) {
                const int64_t c = b0 + lane < live ? cost[b0 + lane] : 0;
                int64_t incl = c;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
                    if (lane >= o) incl += v;
                }
                const uint32_t hit = __ballot_sync(0xffffffffu, before + incl > begin);
                if (hit != 0) {
                    const int src = __ffs(hit) - 1;
                    wk.seq = b0 + src;
                    before += __shfl_sync(0xffffffffu, incl - c, src);
                    break;
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
            walk_seq(rag, wk);
            walk_start<T>(wk, begin - before, cost[wk.seq] / kNumKvHeads, end - begin);
        }
        if (lane == 0) {
            *out = wk;
            *line = ln;
            if (live_out != nullptr) *live_out = live;
        }
    }
    __syncthreads();
    wk = *out;
    return wk.seq >= 0;
}

// Where a unit is cut: a share leaves the unit that its start cuts in its slot 0 of the partials and
// the unit that only its end cuts in its slot 1. The unit goes on in slot 0 of the shares behind. The
// share with its first tile writes the unit's record.
struct Fragment {
    int first, last;  // the shares with the unit's first and last tile; equal: not cut
    int row;          // the unit's first query row
    int rows_kvh;     // its query rows * 4 + kv head
};
template <class T>
__device__ __forceinline__ void write_record(Fragment *f, const Walk &w, const Line &l, int index) {
    const int behind = w.tiles + T::kOver - w.off - w.left;  // of the unit behind the share's end
    const int last = w.t1 < w.tiles ? share_of(l, share_begin(l, index + 1) + behind - 1) : index;
    *reinterpret_cast<int4 *>(f) = make_int4(index, last, w.row0 + w.qt * T::kTok,
                                             min(T::kTok, w.n - w.qt * T::kTok) * kNumKvHeads + w.kvh);
}

// =============================================================================================
// Up to 4 rows a sequence. One CTA per share of 16-token pages: a producer warp streams each page's K
// and V (8 KiB each) through a 4-stage ring by TMA, and consumer warp w takes every fourth page, with
// the 4 GQA heads x up to 4 rows as the M = 16 of mma.m16n8k16, the online softmax in registers. The
// tensor pipe is mostly idle (a kv head has 4 to 16 query rows): HBM bounds it. The producer and the
// ring run on from unit to unit, Q is double-buffered, so only the end of the share drains.
// Two CTAs an SM (register-bound) keep 128 KiB of pages in flight.
// In the cluster form (kCluster) a cluster of CTAs has one unit, its pages split evenly in order, and joins
// through distributed shared memory: no shares to find, no partials in memory, no second launch. A CTA has
// an SM to itself, and one issuing warp's TMA delivers only about 21 B a cycle to an SM: four producer
// warps (K or V, of every second page) took one row over 4097 tokens from 11.8 to 10.7 us, over 16000 from
// 26.1 to 21.5. Eight consumer warps instead of four made it slower (12.8).
// =============================================================================================
constexpr int kTileBytes = kPage * kHeadDim * 2;  // one (page, kv head) of K or V: 8 KiB
constexpr int kStageBytes = 2 * kTileBytes;
constexpr int kRows = PGC_MAX_QUERIES * kGroup;
constexpr int kQRowBytes = kHeadDim * 2 + 16;  // padded row: conflict-free ldmatrix
constexpr int kJoinPitch = kHeadDim + 8;       // floats of a joined row, padded: conflict-free float2 stores

struct SplitParams {
    RaggedBatch rag;
    const uint16_t *q;
    const int32_t *block_tables;
    int max_pages_per_seq;
    int64_t num_pages;
    const uint16_t *gate;
    uint16_t *out;
    float *lse;        // nullable
    float *lse2;       // nullable: as the weights take it (lse_log2)
    Fragment *frags;   // [batch][4]
    int *live;         // sequences that have one: those before the first with rows out of order
    float *parts;      // [shares][2][4 * max_q_len][258]
    float *scores;     // nullable: [total_q][4][score_stride][4], scaled by log2(e)
    int64_t score_stride;
    float scale_log2;
    int cluster;  // CTAs of a cluster, in the cluster form
    ChunkWeights w;
};

constexpr int kConsumers = 4;
template <int kStagesOf, int kProducersOf>
struct SplitSmem {
    static constexpr int kStages = kStagesOf, kProducers = kProducersOf;
    static constexpr int kThreads = (kConsumers + kProducers) * 32;
    static constexpr int kRing = 0;  // 1024-aligned
    static constexpr int kQ = kRing + kStages * kStageBytes;
    static constexpr int kJoin = kQ + 2 * kRows * kQRowBytes;
    static constexpr int kM = kJoin + kConsumers * 4 * kJoinPitch * 4;  // [4 warps][16 rows]
    static constexpr int kL = kM + kConsumers * kRows * 4;
    static constexpr int kBar = kL + kConsumers * kRows * 4;  // full[stages], empty[stages], q_full[2], q_empty[2]
    static constexpr int kWalk = kBar + (2 * kStages + 4) * 8;  // per consumer warp
    static constexpr int kLine = kWalk + kConsumers * sizeof(Walk);
    static constexpr int kAbort = kLine + 24;
    static constexpr int kBytes = kAbort + 8;
    static constexpr int kAlloc = kBytes + 1024;  // + alignment slack
    static_assert(kStages % kConsumers == 0, "each stage must belong to one consumer warp");
    static_assert(sizeof(Walk) <= 48 && sizeof(Line) <= 24 && kWalk % 8 == 0, "schedule slots");
    static_assert(PGC_CHUNK_MAX_BATCH * 8 <= kStages * kStageBytes, "the schedule's scratch is the ring");
    static_assert(kConsumers * kRows * kJoinPitch * 4 <= kJoin, "the last join's scratch is the ring and Q");
    static_assert(kRows * kHeadDim * 4 <= kM - kJoin, "the cluster's exchange is the join's scratch");
};
constexpr int kMaxCluster = 16;
using LineSmem = SplitSmem<4, 1>;     // two CTAs an SM
using ClusterSmem = SplitSmem<8, 4>;  // one CTA an SM
static_assert(2 * ClusterSmem::kAlloc > 227 * 1024, "a cluster's CTAs are to have an SM each");

// Untiled bulk copy global -> shared, completion bytes on `bar`; 16-byte aligned, a multiple of 16.
__device__ __forceinline__ void bulk_load(void *smem_dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(smem_dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

// One (page, kv head) of a pool, by its pool_page_map.
__device__ __forceinline__ void tma_load_page(void *smem_dst, const void *tmap, int32_t row, uint64_t *bar, uint64_t policy) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
        " [%0], [%1, {%2, %3, %2}], [%4], %5;" ::"r"(smem_u32(smem_dst)),
        "l"(reinterpret_cast<uint64_t>(tmap)), "r"(0), "r"(row), "r"(smem_u32(bar)), "l"(policy)
        : "memory");
}

// Two floats of another CTA's shared memory, at this CTA's address of them.
__device__ __forceinline__ float2 load_peer2(const void *at, uint32_t rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(cluster_map(smem_u32(at), rank)) : "memory");
    return v;
}

// The end of the cluster form's one unit. Every consumer warp has its part of O in `o` (on m_s, with
// c0 and c1 to the CTA's common maximum) and the parts of the sums in l_s. The CTA adds its warps' up into
// `part` ([16 rows][256] and the rows' maximum and sum), and CTA `rank` joins 256 / ctas dims of all rows
// from the cluster's parts, in the CTAs' order. With scores it then adds its own tokens' weights.
template <bool kScores, class Sync>
__device__ __forceinline__ void join_cluster(const SplitParams &p, uint8_t *ring, uint8_t *scratch, float *m_s, float *l_s,
                                             const Walk &w, const float (&o)[32][4], float c0, float c1, int ctas, int rank,
                                             const Sync &sync) {
    __shared__ float2 stat[kRows];                // m (log2 units) and l of this CTA, read by the cluster
    __shared__ float2 stats[kRows][kMaxCluster];  // of all
    __shared__ __align__(16) float lse2[kRows];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int r0 = lane >> 2, cpair = (lane & 3) * 2, nrows = w.n * kGroup;
    float *buf = reinterpret_cast<float *>(ring), *part = reinterpret_cast<float *>(scratch);
    constexpr int kThreads = kConsumers * 32;
    const int jrows = nrows <= 4 ? 4 : nrows <= 8 ? 8 : 16;
    float *to = buf + (warp * jrows + r0) * kJoinPitch + cpair;
    if (r0 < nrows) {
#pragma unroll
        for (int i = 0; i < 32; ++i) *reinterpret_cast<float2 *>(to + i * 8) = make_float2(o[i][0] * c0, o[i][1] * c0);
    }
    if (r0 + 8 < nrows) {
#pragma unroll
        for (int i = 0; i < 32; ++i) *reinterpret_cast<float2 *>(to + 8 * kJoinPitch + i * 8) = make_float2(o[i][2] * c1, o[i][3] * c1);
    }
    sync();
    const int dim = tid % (kHeadDim / 2) * 2;
    for (int r = tid / (kHeadDim / 2); r < nrows; r += kThreads / (kHeadDim / 2)) {
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < kConsumers; ++q)
            acc = __fadd2_rn(acc, *reinterpret_cast<const float2 *>(&buf[(q * jrows + r) * kJoinPitch + dim]));
        *reinterpret_cast<float2 *>(&part[r * kHeadDim + dim]) = acc;
    }
    if (tid < nrows) {
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int q = 0; q < kConsumers; ++q) {
            m = fmaxf(m, m_s[q * kRows + tid]);
            l += l_s[q * kRows + tid];
        }
        stat[tid] = make_float2(m, l);
    }
    const int pairs = kHeadDim / 2 / ctas;  // of dims, of every row: this CTA's part of the join
    auto out_row = [&](int r) { return (int64_t)(w.row0 + r / kGroup) * kNumQHeads + w.kvh * kGroup + r % kGroup; };
    auto load_gate = [&](int e) -> uint32_t {
        if (p.gate == nullptr || e >= nrows * pairs) return 0;
        return *reinterpret_cast<const uint32_t *>(p.gate + out_row(e / pairs) * kHeadDim + (rank * pairs + e % pairs) * 2);
    };
    uint32_t gv = load_gate(tid);  // ahead of the barriers
    cluster_sync_all();
    for (int i = tid; i < nrows * ctas; i += kThreads) stats[i / ctas][i % ctas] = load_peer2(&stat[i / ctas], i % ctas);
    sync();
    for (int e = tid; e < nrows * pairs; e += kThreads) {
        const int r = e / pairs, d = (rank * pairs + e % pairs) * 2;
        float2 v[kMaxCluster];
#pragma unroll
        for (int q = 0; q < kMaxCluster; ++q)
            if (q < ctas) v[q] = load_peer2(&part[r * kHeadDim + d], q);
        const uint32_t g = gv;
        gv = load_gate(e + kThreads);
        float mx = -INFINITY;
        for (int q = 0; q < ctas; ++q) mx = fmaxf(mx, stats[r][q].x);
        const float base = mx == -INFINITY ? 0.f : mx;
        float den = 0.f;
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < kMaxCluster; ++q) {
            if (q >= ctas) break;
            const float c = fast_exp2(stats[r][q].x - base);
            den += stats[r][q].y * c;
            acc.x += v[q].x * c;
            acc.y += v[q].y * c;
        }
        const float inv = den == 0.f ? 0.f : 1.f / den;
        acc.x *= inv;
        acc.y *= inv;
        if (p.gate != nullptr) {
            acc.x = sigmoid_gate(acc.x, g & 0xffffu);
            acc.y = sigmoid_gate(acc.y, g >> 16);
        }
        *reinterpret_cast<uint32_t *>(p.out + out_row(r) * kHeadDim + d) = pack_bf16x2(acc.x, acc.y);
        if (e % pairs == 0) {
            if (kScores) lse2[r] = lse_log2(mx, den);
            if (rank == 0 && p.lse != nullptr) p.lse[out_row(r)] = lse_natural(mx, den);
        }
    }
    if (kScores) {
        sync();  // also this CTA's scores are all written
        const int64_t slot = ragged_slot(p.w.slots, p.w.num_slots, w.seq, w.kvh == 0 && rank == 0 && warp == 0 ? &g_chunk_err : nullptr);
        if (slot >= 0) {
            float *wt = p.w.weights + (slot * kNumKvHeads + w.kvh) * p.w.stride;
            const float4 *s = reinterpret_cast<const float4 *>(p.scores) + ((int64_t)w.row0 * kNumKvHeads + w.kvh) * p.score_stride;
            const int end = min(w.len, w.t1 * kPage);
            for (int t = w.t0 * kPage + tid; t < end; t += kThreads) {
                float sum = wt[t];
                for (int j = max(0, t - (w.len - w.n)); j < w.n; ++j) {  // the rows that see it
                    const float4 x = s[(int64_t)j * kNumKvHeads * p.score_stride + t];
                    const float4 l = *reinterpret_cast<const float4 *>(&lse2[j * kGroup]);
                    sum += (fast_exp2(x.x - l.x) + fast_exp2(x.y - l.y)) + (fast_exp2(x.z - l.z) + fast_exp2(x.w - l.w));
                }
                wt[t] = sum;
            }
        }
    }
    cluster_sync_all();  // peers may still read this CTA's part
}

template <bool kScores, bool kCluster>
__global__ void __launch_bounds__(kCluster ? ClusterSmem::kThreads : LineSmem::kThreads, kCluster ? 1 : 2)
    chunk_split_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                       const SplitParams p) {
    using SplitSmem = std::conditional_t<kCluster, ClusterSmem, LineSmem>;
    constexpr int kStages = SplitSmem::kStages, kProducers = SplitSmem::kProducers;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *full = reinterpret_cast<uint64_t *>(smem + SplitSmem::kBar);
    uint64_t *empty = full + kStages;
    uint64_t *q_full = empty + kStages;
    uint64_t *q_empty = q_full + 2;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int index = blockIdx.x;
    Line *line = reinterpret_cast<Line *>(smem + SplitSmem::kLine);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + SplitSmem::kAbort);
    auto wait = [&](uint64_t *bar, uint32_t parity, int where) {
        return wait_or_abort(bar, parity, abort_flag, &g_chunk_err, where);
    };

    pdl_trigger();
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&full[s], kProducers == 1 ? 1 : 2);
            mbar_init(&empty[s], 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(&q_full[s], 1);
            mbar_init(&q_empty[s], kConsumers);
        }
        fence_mbar_init();
        tma_prefetch_desc(&tmk);
        tma_prefetch_desc(&tmv);
    }
    pdl_wait();
    Walk w;
    const int ctas = p.cluster, rank = kCluster ? index % ctas : 0;
    if constexpr (kCluster) {
        const int unit = index / ctas;
        w.seq = unit / kNumKvHeads;
        w.kvh = unit % kNumKvHeads;
        w.qt = 0;
        const RaggedSeq s = ragged_seq(p.rag, w.seq, unit % kNumKvHeads + rank + threadIdx.x == 0 ? &g_chunk_err : nullptr);
        bool bad = s.n == 0;
        for (int b = lane; b < w.seq; b += 32) bad |= p.rag.q_starts[b] < 0 || p.rag.q_starts[b + 1] < p.rag.q_starts[b];
        if (__any_sync(0xffffffffu, bad)) return;  // the whole cluster
        w.row0 = s.row0;
        w.n = s.n;
        w.len = s.len;
        w.tiles = unit_tiles<SplitTiling>(w.n, w.len, 0);
        w.t0 = (int)((int64_t)w.tiles * rank / ctas);
        w.t1 = (int)((int64_t)w.tiles * (rank + 1) / ctas);
        w.off = w.left = 0;  // nothing behind it
    } else {
        const bool busy = find_share<SplitTiling>(p.rag, reinterpret_cast<int64_t *>(smem + SplitSmem::kRing), index,
                                                  gridDim.x, reinterpret_cast<Walk *>(smem + SplitSmem::kWalk), line,
                                                  index == 0 ? &g_chunk_err : nullptr, w, index == 0 ? p.live : nullptr);
        if (!busy) return;
        fence_proxy_async_smem();  // the schedule's scratch becomes the ring
    }
    __syncthreads();

    if (warp >= kConsumers) {
        // ------------------------------------------------------------ producers
        // one for all, or of four: K or V (bit 0), of every second tile (bit 1)
        const int pw = warp - kConsumers;
        const uint64_t pol = l2_policy_evict_first();
        int g = 0;
        for (int unit = 0;; ++unit) {
            const int qb = unit & 1;
            bool ok = true;
            if (lane == 0 && pw == kProducers - 1) {
                ok = unit < 2 || wait(&q_empty[qb], ((unit >> 1) - 1) & 1, 21);
                if (ok) {
                    mbar_arrive_expect_tx(&q_full[qb], (uint32_t)w.n * kGroup * kHeadDim * 2);
                    for (int r = 0; r < w.n * kGroup; ++r)
                        bulk_load(smem + SplitSmem::kQ + (qb * kRows + r) * kQRowBytes,
                                  p.q + ((int64_t)(w.row0 + r / kGroup) * kNumQHeads + w.kvh * kGroup + r % kGroup) * kHeadDim,
                                  kHeadDim * 2, &q_full[qb]);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0);
            const int32_t *table = p.block_tables + (int64_t)w.seq * p.max_pages_per_seq;
            int ids = 0;
            for (int t = w.t0; ok && t < w.t1; ++t, ++g) {
                // a warp-wide look-up of the next 32 pages
                const int k = (t - w.t0) & 31;
                if (k == 0) {
                    __syncwarp();
                    const int i = t + lane;
                    ids = i < w.t1 && i * kPage < w.len ? table[i] : 0;
                    if (ids < 0 || ids >= p.num_pages) {
                        record_error(&g_chunk_err, kErrPageOutOfRange, ids);
                        ids = 0;
                    }
                }
                const int page = __shfl_sync(0xffffffffu, ids, k);
                if (lane == 0 && (kProducers == 1 || (g & 1) == pw >> 1)) {
                    const int s = g % kStages, round = g / kStages;
                    if (round > 0 && !wait(&empty[s], (round - 1) & 1, 22)) {
                        ok = false;
                    } else if (t * kPage < w.len) {
                        uint8_t *stage = smem + SplitSmem::kRing + s * kStageBytes;
                        mbar_arrive_expect_tx(&full[s], kProducers == 1 ? kStageBytes : kTileBytes);
                        const int row = (page * kNumKvHeads + w.kvh) * kPage;
                        if (kProducers == 1 || (pw & 1) == 0) tma_load_page(stage, &tmk, row, &full[s], pol);
                        if (kProducers == 1 || (pw & 1) == 1) tma_load_page(stage + kTileBytes, &tmv, row, &full[s], pol);
                    } else {
                        mbar_arrive(&full[s]);  // an empty cache: the tile is all masked
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0);
            }
            if (!ok || kCluster || !walk_next<SplitTiling>(p.rag, w)) break;
        }
        return;
    }

    // ---------------------------------------------------------------- consumers
    float *m_s = reinterpret_cast<float *>(smem + SplitSmem::kM);
    float *l_s = reinterpret_cast<float *>(smem + SplitSmem::kL);
    float *join = reinterpret_cast<float *>(smem + SplitSmem::kJoin);
    const int r0 = lane >> 2;          // C-fragment rows r0 and r0 + 8
    const int cpair = (lane & 3) * 2;  // C-fragment column pair
    // ldmatrix lane roles: matrix mi = lane / 8, row-in-matrix = lane % 8
    const int mi = lane >> 3;
    const int k_tok = (mi >> 1) * 8 + (lane & 7);  // K: matrices (tok 0-7|8-15) x (k lo|hi)
    const int k_dim_off = (mi & 1) * 8;
    const int v_tok = (mi & 1) * 8 + (lane & 7);   // V: matrices (tok lo|hi) x (dim lo|hi)
    const int v_dim_off = (mi >> 1) * 8;
    auto sync = [&]() { asm volatile("bar.sync 1, %0;" ::"r"(kConsumers * 32) : "memory"); };

    // The walk lives in shared memory, a copy per warp: the tile loop needs the registers.
    Walk *const ws = reinterpret_cast<Walk *>(smem + SplitSmem::kWalk) + warp;
    if (lane == 0) *ws = w;
    __syncwarp();
    int g0 = 0;  // the CTA's tiles before this unit
    for (int unit = 0;; ++unit) {
        const int n = ws->n, L = ws->len, nrows = n * kGroup, qb = unit & 1, t1 = ws->t1;
        g0 -= ws->t0;  // tile t is the CTA's g0 + t
        // visible token bound per C row: row j sees tokens < L - n + j + 1; rows of nobody see none
        const int vis0 = r0 < nrows ? L - n + r0 / kGroup + 1 : 0;
        const int vis1 = r0 + 8 < nrows ? L - n + (r0 + 8) / kGroup + 1 : 0;
        const uint32_t q_base = smem_u32(smem + SplitSmem::kQ) + (qb * kRows + (lane & 15)) * kQRowBytes + (lane >> 4) * 16;
        float o[32][4];
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
        // A wait that gives up is recorded and the warp runs on, every later wait returning at once, so
        // that the four warps stay in step at their barriers.
        wait(&q_full[qb], (unit >> 1) & 1, 23);
        for (int t = ws->t0 + ((warp - g0 - ws->t0) & (kConsumers - 1)); t < t1; t += kConsumers) {
            const int g = g0 + t;  // g % 4 == warp
            const int s = g % kStages;
            if (!wait(&full[s], (g / kStages) & 1, 24)) break;
            uint8_t *kt = smem + SplitSmem::kRing + s * kStageBytes;
            uint8_t *vt = kt + kTileBytes;
            const uint32_t k_base = smem_u32(kt);
            const uint32_t v_base = smem_u32(vt);
            const int tok0 = t * kPage;
            const int nvalid = min(kPage, L - tok0);

            // S[16 rows x 16 tokens] = Q K^T
            float sacc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int kk = 0; kk < kHeadDim / 16; ++kk) {
                uint32_t a0, a1, a2, a3, b0, b1, b2, b3;
                ldsm_x4(q_base + kk * 32, a0, a1, a2, a3);
                ldsm_x4(k_base + swz_page_offset(k_tok, kk * 16 + k_dim_off), b0, b1, b2, b3);
                mma_bf16_16816(sacc[0], a0, a1, a2, a3, b0, b1);
                mma_bf16_16816(sacc[1], a0, a1, a2, a3, b2, b3);
            }

            // masked, log2-scaled scores; online softmax in registers
            float sc[2][4];
            float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int tk = tok0 + i * 8 + cpair + e;
                    sc[i][e] = (tk < vis0) ? sacc[i][e] * p.scale_log2 : -INFINITY;
                    sc[i][2 + e] = (tk < vis1) ? sacc[i][2 + e] * p.scale_log2 : -INFINITY;
                    mx0 = fmaxf(mx0, sc[i][e]);
                    mx1 = fmaxf(mx1, sc[i][2 + e]);
                }
            }
            if (kScores) {
                // the rows and lanes of a tile fill whole 32-byte sectors of [token][head]
                float *s0 = p.scores + (((int64_t)(ws->row0 + r0 / kGroup) * kNumKvHeads + ws->kvh) * p.score_stride + tok0 + cpair) * kGroup + r0 % kGroup;
                float *s1 = s0 + 2 * kNumKvHeads * p.score_stride * kGroup;  // row r0 + 8: two query tokens on
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int tk = tok0 + i * 8 + cpair + e;
                        if (tk < vis0) s0[(i * 8 + e) * kGroup] = sc[i][e];
                        if (tk < vis1) s1[(i * 8 + e) * kGroup] = sc[i][2 + e];
                    }
                }
            }
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
            const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
            const float mu0 = (mn0 == -INFINITY) ? 0.f : mn0;
            const float mu1 = (mn1 == -INFINITY) ? 0.f : mn1;
            const bool grow = mn0 != m0 || mn1 != m1;
            const float corr0 = fast_exp2(m0 - mu0);  // m = -inf -> 0
            const float corr1 = fast_exp2(m1 - mu1);
            m0 = mn0;
            m1 = mn1;
            float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    sc[i][e] = fast_exp2(sc[i][e] - mu0);
                    sc[i][2 + e] = fast_exp2(sc[i][2 + e] - mu1);
                    ps0 += sc[i][e];
                    ps1 += sc[i][2 + e];
                }
            }
            l0 = l0 * corr0 + ps0;
            l1 = l1 * corr1 + ps1;
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    o[i][0] *= corr0;
                    o[i][1] *= corr0;
                    o[i][2] *= corr1;
                    o[i][3] *= corr1;
                }
            }
            const uint32_t pa0 = pack_bf16x2(sc[0][0], sc[0][1]);
            const uint32_t pa1 = pack_bf16x2(sc[0][2], sc[0][3]);
            const uint32_t pa2 = pack_bf16x2(sc[1][0], sc[1][1]);
            const uint32_t pa3 = pack_bf16x2(sc[1][2], sc[1][3]);

            if (nvalid < kPage) {
                // Slots past the sequence end hold stale bytes; zero their V rows so that a NaN
                // pattern cannot leak through a zero probability.
                for (int idx = lane; idx < (kPage - nvalid) * 4 * 8; idx += 32) {
                    const int row = nvalid + idx / 32;
                    const int u = idx % 32;  // 4 boxes x 8 units of 16 B
                    *reinterpret_cast<uint4 *>(vt + (u >> 3) * 2048 + row * 128 + (u & 7) * 16) = make_uint4(0, 0, 0, 0);
                }
                fence_proxy_async_smem();  // generic writes before any later async-proxy refill
                __syncwarp();
            }

            // O[16 x 256] += P[16 x 16] V[16 x 256]
            uint32_t b0, b1, b2, b3;
#pragma unroll
            for (int nd = 0; nd < 16; ++nd) {
                ldsm_x4_trans(v_base + swz_page_offset(v_tok, nd * 16 + v_dim_off), b0, b1, b2, b3);
                mma_bf16_16816(o[2 * nd], pa0, pa1, pa2, pa3, b0, b1);
                mma_bf16_16816(o[2 * nd + 1], pa0, pa1, pa2, pa3, b2, b3);
            }
            __syncwarp();
            if (lane == 0) release_stage(&empty[s], b3, blockIdx.z);  // a one-dimensional grid: 0
        }

        // ------------------------------------------------------------ join the 4 warp states
        if (lane == 0) mbar_arrive(&q_empty[qb]);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
        l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        if ((lane & 3) == 0) {
            m_s[warp * kRows + r0] = m0;
            m_s[warp * kRows + r0 + 8] = m1;
        }
        sync();
        float ma0 = -INFINITY, ma1 = -INFINITY;
#pragma unroll
        for (int q = 0; q < kConsumers; ++q) {
            ma0 = fmaxf(ma0, m_s[q * kRows + r0]);
            ma1 = fmaxf(ma1, m_s[q * kRows + r0 + 8]);
        }
        const float c0 = m0 == -INFINITY ? 0.f : fast_exp2(m0 - ma0);
        const float c1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - ma1);
        // the sums on the common maximum, read behind the next barrier
        if ((lane & 3) == 0) {
            l_s[warp * kRows + r0] = l0 * c0;
            l_s[warp * kRows + r0 + 8] = l1 * c1;
        }
        if constexpr (kCluster) {
            join_cluster<kScores>(p, smem, smem + SplitSmem::kJoin, m_s, l_s, *ws, o, c0, c1, ctas, rank, sync);
            return;
        }
        Walk w = *ws;
        const bool whole = w.t0 == 0 && w.t1 == w.tiles;
        float *part = p.parts + (int64_t)(index * 2 + (w.t0 > 0 ? 0 : 1)) * p.rag.max_q_len * kGroup * kPartial;
        auto out_row = [&](int r) { return (int64_t)(w.row0 + r / kGroup) * kNumQHeads + w.kvh * kGroup + r % kGroup; };
        // dims d, d + 1 of row r; loaded ahead of the barrier before their use
        auto load_gate = [&](int r, int d) -> uint32_t {
            return whole && p.gate != nullptr ? *reinterpret_cast<const uint32_t *>(p.gate + out_row(r) * kHeadDim + d) : 0;
        };
        auto emit = [&](int r, int d, float2 acc, uint32_t gv) {
            const float den = (l_s[r] + l_s[kRows + r]) + (l_s[2 * kRows + r] + l_s[3 * kRows + r]);
            const float ma = fmaxf(fmaxf(m_s[r], m_s[kRows + r]), fmaxf(m_s[2 * kRows + r], m_s[3 * kRows + r]));
            if (!whole) {
                float *dst = part + r * kPartial;
                *reinterpret_cast<float2 *>(dst + 2 + d) = acc;
                if (d == 0) *reinterpret_cast<float2 *>(dst) = make_float2(ma, den);
                return;
            }
            const int64_t row = out_row(r);
            const float inv = den == 0.f ? 0.f : 1.f / den;
            acc.x *= inv;
            acc.y *= inv;
            if (p.gate != nullptr) {
                acc.x = sigmoid_gate(acc.x, gv & 0xffffu);
                acc.y = sigmoid_gate(acc.y, gv >> 16);
            }
            *reinterpret_cast<uint32_t *>(p.out + row * kHeadDim + d) = pack_bf16x2(acc.x, acc.y);
            if (d == 0 && p.lse != nullptr) p.lse[row] = lse_natural(ma, den);
            if (kScores && d == 0) p.lse2[row] = lse_log2(ma, den);
        };
        // the share's last unit: the ring and Q are free, and hold all rows at once
        const bool last = walk_last<SplitTiling>(w);
        if (nrows <= 4 || last) {
            // one round: [4 warps][4, 8 or 16 rows][256 dims]
            float *buf = nrows <= 4 ? join : reinterpret_cast<float *>(smem);
            const int jrows = nrows <= 4 ? 4 : nrows <= 8 ? 8 : 16;
            float *to = buf + (warp * jrows + r0) * kJoinPitch + cpair;
            if (r0 < nrows) {
#pragma unroll
                for (int i = 0; i < 32; ++i) *reinterpret_cast<float2 *>(to + i * 8) = make_float2(o[i][0] * c0, o[i][1] * c0);
            }
            if (r0 + 8 < nrows) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    *reinterpret_cast<float2 *>(to + 8 * kJoinPitch + i * 8) = make_float2(o[i][2] * c1, o[i][3] * c1);
            }
            uint32_t gv[kGroup];
#pragma unroll
            for (int g = 0; g < kGroup; ++g) gv[g] = load_gate(g, 2 * threadIdx.x);
            sync();
            for (int rb = 0; rb < nrows; rb += kGroup) {
#pragma unroll
                for (int g = 0; g < kGroup; ++g) {
                    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                    for (int q = 0; q < kConsumers; ++q)
                        acc = __fadd2_rn(acc, *reinterpret_cast<const float2 *>(&buf[(q * jrows + rb + g) * kJoinPitch + 2 * threadIdx.x]));
                    emit(rb + g, 2 * threadIdx.x, acc, gv[g]);
                }
                if (rb + kGroup < nrows) {
#pragma unroll
                    for (int g = 0; g < kGroup; ++g) gv[g] = load_gate(rb + kGroup + g, 2 * threadIdx.x);
                }
            }
            if (last) {
                if (threadIdx.x == 0 && w.t0 == 0) write_record<SplitTiling>(&p.frags[w.seq * kNumKvHeads + w.kvh], w, *line, index);
                return;
            }
            sync();
        } else {
            // four rounds of 64 dims: [4 warps][16 rows][64 dims]
#pragma unroll
            for (int round = 0; round < 4; ++round) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float *to = &join[(warp * 16 + r0) * (kJoinPitch / 4) + i * 8 + cpair];
                    *reinterpret_cast<float2 *>(to) = make_float2(o[round * 8 + i][0] * c0, o[round * 8 + i][1] * c0);
                    *reinterpret_cast<float2 *>(to + 8 * (kJoinPitch / 4)) = make_float2(o[round * 8 + i][2] * c1, o[round * 8 + i][3] * c1);
                }
                sync();
                for (int i = threadIdx.x; i < nrows * 32; i += kConsumers * 32) {
                    const int r = i >> 5, d = (i & 31) * 2;
                    float2 acc = make_float2(0.f, 0.f);
#pragma unroll
                    for (int q = 0; q < kConsumers; ++q)
                        acc = __fadd2_rn(acc, *reinterpret_cast<const float2 *>(&join[(q * 16 + r) * (kJoinPitch / 4) + d]));
                    emit(r, round * 64 + d, acc, load_gate(r, round * 64 + d));
                }
                sync();
            }
        }
        if (threadIdx.x == 0 && w.t0 == 0) write_record<SplitTiling>(&p.frags[w.seq * kNumKvHeads + w.kvh], w, *line, index);
        g0 += t1;
        walk_next<SplitTiling>(p.rag, w);  // there is one: the last unit returned above
        __syncwarp();
        if (lane == 0) *ws = w;
        __syncwarp();
    }
}

// =============================================================================================
// More rows a sequence: two-SM tcgen05 kernel (cta_group::2). The tile of work and the roles are
// those of the single-sequence prefill kernel: a cluster of two CTAs runs one kv head for 64 query
// tokens (each CTA's 32 tokens x 4 GQA heads stacked into 128 rows, M = 256), each CTA stages its
// own Q, 64 of a 128-key tile's keys and 128 of its value dims, S (two tiles) and O live in TMEM and
// P is written over S. A share belongs to a pair, one pair per two SMs.
// Loads, MMAs and softmax run on across units: the next unit's K, V and Q loads and its first S
// products overlap this unit's last products and its epilogue.
// =============================================================================================
constexpr int kBM = 128;  // rows of a CTA: 32 tokens x 4 heads
constexpr int kTokTile = 32;
constexpr int kUnitTok = PairTiling::kTok;
constexpr uint32_t kTmemCols = 512;
constexpr float kLazyRescale = 8.0f;  // log2 units: rescale O only when the max grows by > 2^8
constexpr int kSoftmaxWarps = 16;
constexpr int kProducerWarps = 2;
constexpr int kPairThreads = 32 * (kSoftmaxWarps + 1 + 2 * kProducerWarps);
constexpr int kKeys = PairTiling::kKeys;      // keys per tile
constexpr int kQBytes = kBM * kHeadDim * 2;   // [4 dim blocks][128 rows][128 B]
constexpr int kKHalf = 64 * kHeadDim * 2;     // this CTA's 64 keys: [4][64][128 B]
constexpr int kVHalf = kKeys * 128 * 2;       // this CTA's 128 dims: [2][128][128 B]
constexpr int kKSlots = 3;
constexpr int kVSlots = 2;
constexpr uint32_t kTO = 0;    // O: 256 columns
constexpr uint32_t kTS = 256;  // S tiles: 2 x 128 columns; P(j) over the first 64 of S(j)
struct PairParams {
    RaggedBatch rag;
    const int32_t *block_tables;
    int max_pages_per_seq;
    int64_t num_pages;
    const uint16_t *v_pages;
    const uint16_t *gate;
    uint16_t *out;
    float *lse;
    float *lse2;      // nullable
    Fragment *frags;  // [pairs]
    float *parts;     // [pairs][2][kPairPart]
    float scale_log2;
};

// Floats of a pair's partial: O as [256 dims / 4][256 rows][4], then the rows' maxima and their sums, so
// that the epilogue's threads, one per row, store 16 bytes side by side (a row of its own a thread took
// 5 us a unit).
constexpr int kPairStat = 2 * kBM * kHeadDim;
constexpr int kPairPart = kPairStat + 2 * 2 * kBM;

struct PairSmem {
    static constexpr int kQ = 0;
    static constexpr int kK = kQ + kQBytes;
    static constexpr int kV = kK + kKSlots * kKHalf;
    static constexpr int kBar = kV + kVSlots * kVHalf;
    // leader-side: q_full, k_full[3], v_full[2], p_full[2], o_free; both sides: q_empty, k_empty[3],
    // v_empty[2], s_full[2], pv_done[2]
    static constexpr int kNumBars = 2 + kKSlots + kVSlots + 2 + 1 + kKSlots + kVSlots + 2 + 2;
    static constexpr int kRed = kBar + kNumBars * 8;
    static constexpr int kWalk = kRed + 4 * kBM * 4;  // red: [4 key quarters][128 rows] fp32
    static constexpr int kLine = kWalk + 48;
    static constexpr int kTmemSlot = kLine + 24;
    static constexpr int kAbort = kTmemSlot + 8;
    static constexpr int kBytes = kAbort + 8;
};
static_assert(PairSmem::kWalk % 8 == 0, "walk slot");
static_assert(PairSmem::kBytes <= 232448, "pair shared memory exceeds the sm_100 limit");
static_assert(PGC_CHUNK_MAX_BATCH * 8 <= kKSlots * kKHalf, "the schedule's scratch is the K ring");

// A pair's walk takes the unit that its share's start cuts last: every other unit it begins at its first
// key, and as the pairs run at one speed, those of one kv head then read the same keys at about the same
// time, from L2. A chunk of 1600 over 24576 reads 240 MB from HBM that way; in the line's order it read
// 940 MB, as many cycles but a lower clock under the power cap (496 us instead of 463).
// `first` is where the share starts, `later` whether that unit is still to come.
__device__ __forceinline__ bool pair_begin(const RaggedBatch &rag, Walk &w) {
    if (w.t0 == 0 || walk_last<PairTiling>(w)) return false;
    walk_next<PairTiling>(rag, w);
    return true;
}
__device__ __forceinline__ bool pair_next(const RaggedBatch &rag, Walk &w, bool &later, const Walk *first) {
    if (walk_next<PairTiling>(rag, w)) return true;
    if (!later) return false;
    later = false;
    w = *first;
    w.left = w.tiles + PairTiling::kOver - w.off;  // and no further
    return true;
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    chunk_pair_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                      const __grid_constant__ CUtensorMap tmv, const PairParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_trigger();
    pdl_wait();
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    // both CTAs of a pair see the same alignment, so both leave together
    if ((smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) record_error(&g_chunk_err, kErrSmemAlign, 0);
        return;
    }
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + PairSmem::kBar);
    uint64_t *q_full = bars;                // leader: both CTAs' Q bytes
    uint64_t *q_empty = q_full + 1;         // each: the unit's S products are done with Q
    uint64_t *k_full = q_empty + 1;         // leader [3]: both CTAs' K halves
    uint64_t *v_full = k_full + kKSlots;    // leader [2]: both CTAs' V halves
    uint64_t *p_full = v_full + kVSlots;    // leader [2]: both CTAs' softmax warps
    uint64_t *o_free = p_full + 2;          // leader: both CTAs' softmax warps have read O
    uint64_t *k_empty = o_free + 1;         // each [3]
    uint64_t *v_empty = k_empty + kKSlots;  // each [2]
    uint64_t *s_full = v_empty + kVSlots;   // each [2]
    uint64_t *pv_done = s_full + 2;         // each [2]
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + PairSmem::kTmemSlot);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + PairSmem::kAbort);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;
    Line *line = reinterpret_cast<Line *>(smem + PairSmem::kLine);

    Walk w;
    const bool busy = find_share<PairTiling>(p.rag, reinterpret_cast<int64_t *>(smem + PairSmem::kK), pair, gridDim.x >> 1,
                                             reinterpret_cast<Walk *>(smem + PairSmem::kWalk),
                                             line, blockIdx.x == 0 ? &g_chunk_err : nullptr, w);
    // the record of the share, that no unit is cut by its end until its walk has ended
    if (leader && threadIdx.x == 0) p.frags[pair].last = p.frags[pair].first = 0;
    if (!busy) return;  // both CTAs of the pair
    const Walk *first = reinterpret_cast<const Walk *>(smem + PairSmem::kWalk);
    bool later = pair_begin(p.rag, w);
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        mbar_init(q_full, 2);
        mbar_init(q_empty, 1);
        for (int s = 0; s < kKSlots; ++s) {
            mbar_init(&k_full[s], 2 * kProducerWarps);
            mbar_init(&k_empty[s], 1);
        }
        for (int s = 0; s < kVSlots; ++s) {
            mbar_init(&v_full[s], 2 * kProducerWarps);
            mbar_init(&v_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&p_full[b], 2 * kSoftmaxWarps);
            mbar_init(&s_full[b], 1);
            mbar_init(&pv_done[b], 1);
        }
        mbar_init(o_free, 2 * kSoftmaxWarps);
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_proxy_async_smem();  // the schedule's scratch becomes the K ring
    tc_fence_before();
    cluster_sync_all();  // both CTAs' barriers are initialised before anyone signals them
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    auto leader_addr = [&](uint64_t *bar) { return cluster_map(smem_u32(bar), 0); };
    auto wait = [&](uint64_t *bar, uint32_t parity, int where) {
        return wait_or_abort(bar, parity, abort_flag, &g_chunk_err, where);
    };
    auto page_at = [&](const Walk &w, int i) -> int {
        const int page = p.block_tables[(int64_t)w.seq * p.max_pages_per_seq + i];
        if (page >= 0 && page < p.num_pages) return page;
        record_error(&g_chunk_err, kErrPageOutOfRange, page);
        return 0;
    };

    if (warp >= kSoftmaxWarps + 1 && warp < kSoftmaxWarps + 1 + kProducerWarps) {
        // ------------------------------------------------------------ TMA: Q and this CTA's K half
        // producer kw loads pages {2kw, 2kw+1} of this CTA's 64 keys (4 boxes of 64 dims each)
        const int kw = warp - (kSoftmaxWarps + 1);
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_normal();
            if (kw == 0) {
                tma_prefetch_desc(&tmq);
                tma_prefetch_desc(&tmk);
            }
            int g = 0;  // tiles of this pair so far
            bool ok = true;
            for (int unit = 0; ok; ++unit) {
                if (kw == 0) {
                    if (unit > 0 && !wait(q_empty, (unit - 1) & 1, 1)) break;
                    // rows past the sequence's own are other sequences' (or zeros past total_q):
                    // their results are dropped
                    const uint32_t qbar = leader_addr(q_full);
                    mbar_arrive_expect_tx_cluster(qbar, kQBytes);
                    const int tok = w.row0 + w.qt * kUnitTok + (int)rank * kTokTile;
                    for (int c = 0; c < 4; ++c)
                        tma_load_3d_pair(smem + PairSmem::kQ + c * (kBM * 128), &tmq, c * 64, w.kvh * kGroup, tok, qbar);
                }
                for (int t = w.t0; t < w.t1; ++t, ++g) {
                    const int sl = g % kKSlots;
                    if (g >= kKSlots && !wait(&k_empty[sl], ((g / kKSlots) - 1) & 1, 2)) {
                        ok = false;
                        break;
                    }
                    const int key0 = t * kKeys + (int)rank * 64;  // this CTA's 64 keys
                    int npg = 0;
                    for (int pp = 2 * kw; pp < 2 * kw + 2; ++pp)
                        if (key0 + pp * kPage < w.len) ++npg;
                    const uint32_t kbar = leader_addr(&k_full[sl]);
                    mbar_arrive_expect_tx_cluster(kbar, (uint32_t)npg * 4 * 2048);
                    uint8_t *dst = smem + PairSmem::kK + sl * kKHalf;
                    for (int pp = 2 * kw; pp < 2 * kw + npg; ++pp) {
                        const int row = (page_at(w, (key0 >> 4) + pp) * kNumKvHeads + w.kvh) * kPage;
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            tma_load_2d_pair(dst + c * (64 * 128) + pp * 2048, &tmk, c * 64, row, kbar, pol);
                    }
                }
                if (!pair_next(p.rag, w, later, first)) break;
            }
        }
    } else if (warp >= kSoftmaxWarps + 1 + kProducerWarps) {
        // ------------------------------------------------------------ TMA: this CTA's V half
        // (value dims [128 * rank, +128) of all 128 keys). Producer vw owns keys [64 vw, +64). Rows
        // past the cache end are zeroed and a partial final page is copied row by row, so that no
        // stale slot (possibly a NaN pattern) meets a zero probability in P.V.
        const int vw = warp - (kSoftmaxWarps + 1 + kProducerWarps);
        const int r0 = vw * 64, r1 = r0 + 64;
        if (lane == 0 && vw == 0) tma_prefetch_desc(&tmv);
        const uint64_t pol = l2_policy_evict_normal();
        int g = 0;
        bool ok = true;
        while (ok) {
            for (int t = w.t0; t < w.t1; ++t, ++g) {
                const int sl = g % kVSlots;
                bool go = true;
                if (lane == 0 && g >= kVSlots) go = wait(&v_empty[sl], ((g / kVSlots) - 1) & 1, 3);
                if (!__shfl_sync(0xffffffffu, go ? 1 : 0, 0)) {
                    ok = false;
                    break;
                }
                const int key0 = t * kKeys;
                const int valid = min(kKeys, w.len - key0);  // keys of this tile in the cache
                const int full_pages = valid / kPage;        // loaded by TMA
                uint8_t *dst = smem + PairSmem::kV + sl * kVHalf;
                const int first = max(full_pages * kPage, r0);  // first row not loaded by TMA
                if (first < r1) {
                    for (int i = lane; i < (r1 - first) * 2 * 8; i += 32) {
                        const int row = first + i / 16;
                        const int u = i % 16;
                        *reinterpret_cast<uint4 *>(dst + (u >> 3) * (kKeys * 128) + row * 128 + (u & 7) * 16) =
                            make_uint4(0, 0, 0, 0);
                    }
                    __syncwarp();
                    const int tail = valid - full_pages * kPage;  // valid rows in the partial page
                    if (tail > 0 && full_pages * kPage >= r0 && full_pages * kPage < r1) {
                        const int page = page_at(w, (key0 >> 4) + full_pages);
                        const uint16_t *src = p.v_pages + ((int64_t)page * kNumKvHeads + w.kvh) * kPage * kHeadDim;
                        for (int i = lane; i < tail * 2 * 8; i += 32) {
                            const int rr = i / 16, u = i % 16;  // row in page, 16-B unit of 2 blocks
                            const int db = u >> 3, unit = u & 7;
                            const uint4 v = *reinterpret_cast<const uint4 *>(
                                src + (int64_t)rr * kHeadDim + ((int)rank * 2 + db) * 64 + unit * 8);
                            const int row = full_pages * kPage + rr;
                            *reinterpret_cast<uint4 *>(dst + db * (kKeys * 128) + row * 128 +
                                                       ((unit ^ (row & 7)) << 4)) = v;
                        }
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                if (lane == 0) {
                    const int pp0 = r0 / kPage, pp1 = min(full_pages, r1 / kPage);
                    const uint32_t vbar = leader_addr(&v_full[sl]);
                    mbar_arrive_expect_tx_cluster(vbar, (uint32_t)max(pp1 - pp0, 0) * 2 * 2048);
                    for (int pp = pp0; pp < pp1; ++pp) {
                        const int row = (page_at(w, (key0 >> 4) + pp) * kNumKvHeads + w.kvh) * kPage;
#pragma unroll
                        for (int db = 0; db < 2; ++db)
                            tma_load_2d_pair(dst + db * (kKeys * 128) + pp * 2048, &tmv,
                                             ((int)rank * 2 + db) * 64, row, vbar, pol);
                    }
                }
                __syncwarp();
            }
            if (!pair_next(p.rag, w, later, first)) break;
        }
    } else if (warp == kSoftmaxWarps) {
        // ------------------------------------------------------------ pair MMA issuer (leader)
        if (leader) {
            const uint32_t me = elect_one();
            constexpr uint32_t idesc_s = umma_idesc(2 * kBM, kKeys, false, false);
            constexpr uint32_t idesc_o = umma_idesc(2 * kBM, kHeadDim, false, true);
            // descriptors step in units of 16 bytes; 128 KiB and more never carry out of the address field
            const uint64_t q_desc = umma_desc(smem_u32(smem + PairSmem::kQ), 16, 1024);
            const uint64_t k_desc = umma_desc(smem_u32(smem + PairSmem::kK), 16, 1024);
            const uint64_t v_desc = umma_desc(smem_u32(smem + PairSmem::kV), kKeys * 128, 1024);
            // `ahead` is the next tile whose S is to be issued: S(g + 2) goes out behind PV(g), but
            // the first S of a unit only behind the last PV of the unit before it, because it waits
            // for that unit's Q to be replaced.
            Walk a = w;
            int at = a.t0, ag = 0, aunit = 0;
            bool more = true, ok = true, alater = later;
            auto issue_s = [&]() -> bool {
                const int b = ag & 1, sl = ag % kKSlots;
                if (at == a.t0 && !wait(q_full, aunit & 1, 4)) return false;
                if (!wait(&k_full[sl], (ag / kKSlots) & 1, 5)) return false;
                tc_fence_after();
                const uint64_t kd = k_desc + (uint32_t)(sl * (kKHalf >> 4));
#pragma unroll
                for (int kk = 0; kk < kHeadDim / 16; ++kk)
                    umma2_ss_elected(me, tmem + kTS + b * kKeys, q_desc + (((kk >> 2) * (kBM * 128) + (kk & 3) * 32) >> 4),
                                     kd + (((kk >> 2) * (64 * 128) + (kk & 3) * 32) >> 4), idesc_s, kk > 0 ? 1u : 0u);
                umma2_commit_pair_elected(me, &k_empty[sl]);
                umma2_commit_pair_elected(me, &s_full[b]);
                ++ag;
                if (++at == a.t1) {
                    umma2_commit_pair_elected(me, q_empty);
                    more = pair_next(p.rag, a, alater, first);
                    at = a.t0;
                    ++aunit;
                }
                return true;
            };
            int g = 0;
            for (int unit = 0; ok; ++unit) {
                for (int t = w.t0; ok && t < w.t1; ++t, ++g) {
                    // S(g) and, within the unit, S(g + 1) are out before PV(g) is waited for
                    while (ok && more && ag < g + 2 && (ag <= g || aunit == unit)) ok = issue_s();
                    if (!ok) break;
                    const int b = g & 1, sl = g % kVSlots;
                    if ((t == w.t0 && unit > 0 &&
                         !wait_or_abort_cluster(o_free, (unit - 1) & 1, abort_flag, &g_chunk_err, 6)) ||
                        !wait_or_abort_cluster(&p_full[b], (g >> 1) & 1, abort_flag, &g_chunk_err, 7) ||
                        !wait_or_abort_cluster(&v_full[sl], (g / kVSlots) & 1, abort_flag, &g_chunk_err, 8)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t vd = v_desc + (uint32_t)(sl * (kVHalf >> 4));
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        umma2_ts_elected(me, tmem + kTO, tmem + kTS + b * kKeys + kk * 8, vd + ((kk * 2048) >> 4), idesc_o,
                                         (t > w.t0 || kk > 0) ? 1u : 0u);
                    umma2_commit_pair_elected(me, &v_empty[sl]);
                    umma2_commit_pair_elected(me, &pv_done[b]);
                }
                if (!ok || !pair_next(p.rag, w, later, first)) break;
            }
        }
    } else {
        // ------------------------------------------------------------ softmax + epilogue
        // Warps w, w+4, w+8 and w+12 share TMEM lanes 32*(w%4)..+31 (one row per thread) and split
        // each 128-key S tile into key quarters [32*cg, +32) and O into dims [64*cg, +64). Warps
        // whose 8 tokens all lie past the sequence's rows only keep the barriers in step: their
        // rows of P and O hold whatever they held, and no other row reads them.
        const int qd = warp & 3;
        const int cg = warp >> 2;
        const int r = qd * 32 + lane;
        const uint32_t lane_addr = (uint32_t)(qd * 32) << 16;
        float *red = reinterpret_cast<float *>(smem + PairSmem::kRed);  // [4 key quarters][128 rows]
        const uint32_t pbar[2] = {leader_addr(&p_full[0]), leader_addr(&p_full[1])};
        const uint32_t obar = leader_addr(o_free);
        const float c = p.scale_log2;
        // A wait that gives up (another role has recorded why) does not take a warp out of step: it
        // runs on through its tiles, every later wait returning at once, so that the four warps
        // of a lane quarter always meet at their named barrier.
        int g = 0;
        for (;;) {
            const int tok = w.qt * kUnitTok + (int)rank * kTokTile + r / kGroup;  // of the sequence
            const bool row_ok = tok < w.n;
            const bool live = w.qt * kUnitTok + (int)rank * kTokTile + qd * 8 < w.n;
            const int vis = w.len - w.n + tok;
            float m = -INFINITY, l = 0.f;
            for (int t = w.t0; t < w.t1; ++t, ++g) {
                const int b = g & 1;
                wait(&s_full[b], (g >> 1) & 1, 9);
                tc_fence_after();
                if (live) {
                    float sv[32];
                    tmem_ld32(tmem + lane_addr + kTS + b * kKeys + cg * 32, sv);
                    tmem_wait_ld();
                    const int key0 = t * kKeys + cg * 32;
                    if (!(key0 + 31 <= vis && row_ok)) {
#pragma unroll
                        for (int i = 0; i < 32; ++i) sv[i] = (row_ok && key0 + i <= vis) ? sv[i] : -INFINITY;
                    }
                    float mx = max32(sv);
                    red[cg * kBM + r] = mx;
                    // all four quarters have read S tile b (so P may overwrite it) and posted their max
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + qd) : "memory");
                    mx = fmaxf(fmaxf(red[r], red[kBM + r]), fmaxf(red[2 * kBM + r], red[3 * kBM + r]));
                    // and have read the maxima before the next tile rewrites them
                    asm volatile("bar.sync %0, 128;" ::"r"(1 + qd) : "memory");
                    const float m_new = fmaxf(m, mx * c);
                    float corr = 1.f;
                    if (m_new > m + kLazyRescale) {
                        corr = (m == -INFINITY) ? 0.f : fast_exp2(m - m_new);
                        m = m_new;
                    }
                    const float m_use = (m == -INFINITY) ? 0.f : m;
                    const float2 c2 = make_float2(c, c), nm2 = make_float2(-m_use, -m_use);
                    float2 ps2 = make_float2(0.f, 0.f);
                    uint32_t pw[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float2 x = __ffma2_rn(make_float2(sv[i], sv[i + 1]), c2, nm2);
                        const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                        ps2 = __fadd2_rn(ps2, e);
                        pw[i >> 1] = pack_bf16x2(e.x, e.y);
                    }
                    l = l * corr + (ps2.x + ps2.y);
                    if (t > w.t0 && __any_sync(0xffffffffu, corr != 1.f)) {
                        wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, 10);
                        tc_fence_after();
#pragma unroll 1
                        for (int cc = 0; cc < 2; ++cc) {
                            float o[32];
                            const uint32_t col = kTO + cg * 64 + cc * 32;
                            tmem_ld32(tmem + lane_addr + col, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const float2 v = __fmul2_rn(make_float2(o[i], o[i + 1]), make_float2(corr, corr));
                                o[i] = v.x;
                                o[i + 1] = v.y;
                            }
                            tmem_st32(tmem + lane_addr + col, o);
                        }
                    }
                    tmem_st16u(tmem + lane_addr + kTS + b * kKeys + cg * 16, pw);
                    tmem_wait_st();
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(pbar[b]);
            }
            wait(&pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, 11);
            tc_fence_after();
            const bool whole = w.t0 == 0 && w.t1 == w.tiles;
            const int slot = w.t0 > 0 ? 0 : 1;
            const int64_t orow = (int64_t)(w.row0 + tok) * kNumQHeads + w.kvh * kGroup + r % kGroup;
            uint32_t ow[32];  // the thread's 64 dims of a whole unit's row, bf16
            if (live) {
                red[cg * kBM + r] = l;
                asm volatile("bar.sync %0, 128;" ::"r"(1 + qd) : "memory");
                const float l_row = (red[r] + red[kBM + r]) + (red[2 * kBM + r] + red[3 * kBM + r]);
                asm volatile("bar.sync %0, 128;" ::"r"(1 + qd) : "memory");  // before the next unit's maxima
                const float inv = l_row == 0.f ? 0.f : 1.f / l_row;
                float *part = p.parts + (int64_t)(pair * 2 + slot) * kPairPart + rank * kBM + r;
                if (cg == 0) {
                    if (!whole) {
                        part[kPairStat] = m;
                        part[kPairStat + 2 * kBM] = l_row;
                    } else if (row_ok) {
                        if (p.lse != nullptr) p.lse[orow] = lse_natural(m, l_row);
                        if (p.lse2 != nullptr) p.lse2[orow] = lse_log2(m, l_row);
                    }
                }
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    float o[32];
                    const int col = cg * 64 + cc * 32;
                    tmem_ld32(tmem + lane_addr + kTO + col, o);
                    tmem_wait_ld();
                    if (!whole) {
                        // [dim / 4][row][4]: a warp's rows lie side by side
                        float4 *dst = reinterpret_cast<float4 *>(p.parts + (int64_t)(pair * 2 + slot) * kPairPart) + rank * kBM + r;
#pragma unroll
                        for (int i = 0; i < 32; i += 4)
                            dst[((col + i) / 4) * 2 * kBM] = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                        continue;
                    }
                    // a row with nothing visible has P = 0 throughout: o = 0 and inv = 0
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= inv;
                    if (p.gate != nullptr && row_ok) {
                        const uint4 *gp = reinterpret_cast<const uint4 *>(p.gate + orow * kHeadDim + col);
#pragma unroll
                        for (int i = 0; i < 32; i += 8) {
                            const uint4 gv = gp[i / 8];
                            const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
                            for (int k = 0; k < 8; ++k)
                                o[i + k] = sigmoid_gate(o[i + k], (gw[k >> 1] >> ((k & 1) * 16)) & 0xffffu);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 32; i += 2) ow[cc * 16 + i / 2] = pack_bf16x2(o[i], o[i + 1]);
                }
            }
            // O is read: the next unit's products may go on while this one's rows are stored
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(obar);
            if (live && whole && row_ok) {
                uint16_t *dst = p.out + orow * kHeadDim + cg * 64;
#pragma unroll
                for (int i = 0; i < 32; i += 4)
                    *reinterpret_cast<uint4 *>(dst + 2 * i) = make_uint4(ow[i], ow[i + 1], ow[i + 2], ow[i + 3]);
            }
            if (leader && threadIdx.x == 0 && w.t0 == 0 && walk_last<PairTiling>(w))
                write_record<PairTiling>(&p.frags[pair], w, *line, pair);
            if (!pair_next(p.rag, w, later, first)) break;
        }
    }
    // neither CTA may leave (or free TMEM) while the pair MMA or the peer can still touch it
    tc_fence_before();
    cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

// =============================================================================================
// The end of a call: joins the fragments of the units that were cut and, behind the split kernel, adds
// the weights.
// =============================================================================================
constexpr int kFinishThreads = 512;
constexpr int kFinishWarps = kFinishThreads / 32;
constexpr int kAddTokens = 2048;

struct FinishParams {
    const Fragment *frags;
    const float *parts;  // [shares][2][rows][258], the pair form's [pairs][2][kPairPart]
    int records;
    int rows;          // of a fragment
    int merge_blocks;  // the blocks behind them add weights
    const uint16_t *gate;
    uint16_t *out;
    float *lse;
    float *lse2;  // nullable; written behind the pair kernel, read behind the split kernel
    RaggedBatch rag;  // the split form's: its records are by (sequence, kv head)
    const int *live;
    const float *scores;
    int64_t score_stride;
    ChunkWeights w;
    int add_chunks;  // blocks per (sequence, kv head)
};

__device__ __forceinline__ Fragment read_record(const FinishParams &p, int i) {
    const int4 f = *reinterpret_cast<const int4 *>(&p.frags[i]);
    return Fragment{f.x, f.y, f.z, f.w};
}
// Floats from a row's first fragment (slot 1 of the first share) to its fragment i (slot 0 of share
// first + i), over a base at slot 0 of the first share.
__device__ __forceinline__ int64_t fragment_at(const FinishParams &p, int i) {
    return (int64_t)(i == 0 ? 1 : 2 * i) * p.rows * kPartial;
}

// Behind the pair kernel: block (share, y, z) joins rows [32 y, +32) and dims [64 z, +64) of the unit that
// the share's end cuts. Lane = row and a warp per 8 dims, as the partials lie, four fragments' loads in
// flight; the joined rows go out through shared memory.
constexpr int kMergeThreads = 256;
constexpr int kMergeDims = 64;

__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(const FinishParams p) {
    __shared__ float rows_s[32][kMergeDims + 1];
    pdl_trigger();
    pdl_wait();
    const Fragment f = read_record(p, blockIdx.x);
    const int nrows = f.rows_kvh / kNumKvHeads * kGroup, kvh = f.rows_kvh % kNumKvHeads;
    if (f.first >= f.last || (int)blockIdx.y * 32 >= nrows) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int r = blockIdx.y * 32 + lane;
    const int np = f.last - f.first + 1;
    constexpr int kFrags = 4;
    const int quad = blockIdx.z * (kMergeDims / 4) + warp * 2;  // the warp's two groups of 4 dims
    float ma = -INFINITY, den = 0.f;
    float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
    for (int i0 = 0; i0 < np; i0 += kFrags) {
        float m[kFrags], l[kFrags];
        float4 v[kFrags][2];
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            // fragment i: slot 1 of the first share, then slot 0 of the next ones; past the last the
            // first of these again, with weight 0
            const int i = i0 + j < np ? i0 + j : i0;
            const float *pc = p.parts + (int64_t)((f.first + i) * 2 + (i == 0 ? 1 : 0)) * kPairPart;
            m[j] = i0 + j < np ? pc[kPairStat + r] : -INFINITY;
            l[j] = pc[kPairStat + 2 * kBM + r];
#pragma unroll
            for (int k = 0; k < 2; ++k) v[j][k] = reinterpret_cast<const float4 *>(pc)[(quad + k) * 2 * kBM + r];
        }
        float mx = ma;
#pragma unroll
        for (int j = 0; j < kFrags; ++j) mx = fmaxf(mx, m[j]);
        const float base_m = mx == -INFINITY ? 0.f : mx;  // nothing seen so far: all weights 0
        const float corr = fast_exp2(ma - base_m);
        ma = mx;
        den *= corr;
#pragma unroll
        for (int k = 0; k < 2; ++k) acc[k] = make_float4(acc[k].x * corr, acc[k].y * corr, acc[k].z * corr, acc[k].w * corr);
#pragma unroll
        for (int j = 0; j < kFrags; ++j) {
            const float w = fast_exp2(m[j] - base_m);
            den += l[j] * w;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                acc[k].x += v[j][k].x * w;
                acc[k].y += v[j][k].y * w;
                acc[k].z += v[j][k].z * w;
                acc[k].w += v[j][k].w * w;
            }
        }
    }
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float *to = &rows_s[lane][warp * 8 + 4 * k];
        to[0] = acc[k].x * inv;
        to[1] = acc[k].y * inv;
        to[2] = acc[k].z * inv;
        to[3] = acc[k].w * inv;
    }
    if (warp == 0 && blockIdx.z == 0 && r < nrows) {
        const int64_t orow = (int64_t)(f.row + r / kGroup) * kNumQHeads + kvh * kGroup + r % kGroup;
        if (p.lse != nullptr) p.lse[orow] = lse_natural(ma, den);
        if (p.lse2 != nullptr) p.lse2[orow] = lse_log2(ma, den);
    }
    __syncthreads();
    // 8 threads a row, 8 dims each
    const int rr = threadIdx.x >> 3, row = blockIdx.y * 32 + rr, d = (threadIdx.x & 7) * 8;
    if (row >= nrows) return;
    const int64_t at = ((int64_t)(f.row + row / kGroup) * kNumQHeads + kvh * kGroup + row % kGroup) * kHeadDim + blockIdx.z * kMergeDims + d;
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = rows_s[rr][d + k];
    if (p.gate != nullptr) {
        const uint4 gq = *reinterpret_cast<const uint4 *>(p.gate + at);
        const uint32_t gw[4] = {gq.x, gq.y, gq.z, gq.w};
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = sigmoid_gate(v[k], (gw[k >> 1] >> ((k & 1) * 16)) & 0xffffu);
    }
    uint4 o;
    o.x = pack_bf16x2(v[0], v[1]);
    o.y = pack_bf16x2(v[2], v[3]);
    o.z = pack_bf16x2(v[4], v[5]);
    o.w = pack_bf16x2(v[6], v[7]);
    *reinterpret_cast<uint4 *>(p.out + at) = o;
}

// One row of a cut unit behind the split kernel, by a block: the fragments (64 and more of a single long
// sequence) are dealt to the warps, four loads of a warp in flight, and the warps' sums joined in
// shared memory. Short straight code: these few blocks run once, so they wait for instructions and
// loads, not for arithmetic.
__device__ __forceinline__ void merge_row(const FinishParams &p, const Fragment &f, int r) {
    __shared__ float2 red_ml[kFinishWarps];
    __shared__ float red[kFinishWarps][kHeadDim + 8];
    constexpr int kBatch = 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int kvh = f.rows_kvh % kNumKvHeads;
    if (r >= f.rows_kvh / kNumKvHeads * kGroup) return;  // uniform
    const float *base = p.parts + (int64_t)f.first * 2 * p.rows * kPartial + (int64_t)r * kPartial;
    const int np = f.last - f.first + 1;
    float ma = -INFINITY, den = 0.f;
    float2 acc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = make_float2(0.f, 0.f);
    for (int i0 = warp; i0 < np; i0 += kFinishWarps * kBatch) {
        float2 ml[kBatch], v[kBatch][4];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            // past the last fragment: the first of this warp again, with weight 0
            const int i = i0 + j * kFinishWarps;
            const float *pc = base + fragment_at(p, i < np ? i : i0);
            ml[j] = *reinterpret_cast<const float2 *>(pc);
            if (i >= np) ml[j].x = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[j][k] = *reinterpret_cast<const float2 *>(pc + 2 + 2 * lane + 64 * k);
        }
        float mx = ma;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) mx = fmaxf(mx, ml[j].x);
        const float base_m = mx == -INFINITY ? 0.f : mx;
        const float corr = fast_exp2(ma - base_m);
        ma = mx;
        den *= corr;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] = __fmul2_rn(acc[k], make_float2(corr, corr));
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const float w = fast_exp2(ml[j].x - base_m);
            den += ml[j].x == -INFINITY ? 0.f : ml[j].y * w;
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] = __ffma2_rn(v[j][k], make_float2(w, w), acc[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<float2 *>(&red[warp][2 * lane + 64 * k]) = acc[k];
    if (lane == 0) red_ml[warp] = make_float2(ma, den);
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= kHeadDim) return;
    const int64_t orow = (int64_t)(f.row + r / kGroup) * kNumQHeads + kvh * kGroup + r % kGroup;
    const float gate = p.gate != nullptr ? sigmoid_gate(1.f, p.gate[orow * kHeadDim + d]) : 1.f;
    // lane w: warp w's statistics
    const float2 mine = lane < kFinishWarps ? red_ml[lane] : make_float2(-INFINITY, 0.f);
    float mx = mine.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float scale = mine.x == -INFINITY ? 0.f : fast_exp2(mine.x - mx);
    den = mine.y * scale;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(0xffffffffu, den, o);
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kFinishWarps; ++w) sum += red[w][d] * __shfl_sync(0xffffffffu, scale, w);
    const float o = den == 0.f ? 0.f : sum / den * gate;
    p.out[orow * kHeadDim + d] = f32_to_bf16_bits(o);
    if (p.lse != nullptr && d == 0) p.lse[orow] = lse_natural(mx, den);
}

// The weights of 2048 tokens of one (sequence, kv head) from the scores that the split kernel left and
// the rows' lse: the split kernel's, or for a cut unit formed from the fragments' (m, l) here, so that
// these blocks need not wait for the merging ones.
__device__ __forceinline__ void add_weights(const FinishParams &p, int blk) {
    __shared__ __align__(16) float lse2[kRows];  // log2 units
    const int chunk = blk % p.add_chunks, unit = blk / p.add_chunks;
    const int kvh = unit % kNumKvHeads, b = unit / kNumKvHeads;
    const Fragment f = read_record(p, unit);  // of a sequence with rows only
    const RaggedSeq sv = ragged_seq(p.rag, b, nullptr);
    const int t0 = chunk * kAddTokens;
    if (b >= *p.live || sv.n == 0 || t0 >= sv.len) return;
    const int64_t slot = ragged_slot(p.w.slots, p.w.num_slots, b, chunk == 0 && kvh == 0 ? &g_chunk_err : nullptr);
    if (slot < 0) return;
    float *w = p.w.weights + (slot * kNumKvHeads + kvh) * p.w.stride;
    const float4 *s = reinterpret_cast<const float4 *>(p.scores) + ((int64_t)sv.row0 * kNumKvHeads + kvh) * p.score_stride;
    constexpr int kEach = kAddTokens / kFinishThreads;
    float sum[kEach];
    float4 x[kEach];
    auto load_scores = [&](int j) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int t = t0 + i * kFinishThreads + threadIdx.x;
            x[i] = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (t <= sv.len - sv.n + j) x[i] = s[(int64_t)j * kNumKvHeads * p.score_stride + t];  // visible to row j
        }
    };
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int t = t0 + i * kFinishThreads + threadIdx.x;
        sum[i] = t < sv.len ? w[t] : 0.f;
    }
    load_scores(0);
    {
        // 16 threads a row (the first half of the block)
        const int r = threadIdx.x >> 4, lane16 = threadIdx.x & 15;
        const bool mine = r < sv.n * kGroup;  // sv.n <= 4
        float m = -INFINITY, l = 0.f;
        if (f.first < f.last) {
            const float *base = p.parts + (int64_t)f.first * 2 * p.rows * kPartial + (int64_t)r * kPartial;
            const int np = mine ? f.last - f.first + 1 : 0;
            for (int i = lane16; i < np; i += 16) {
                const float2 ml = *reinterpret_cast<const float2 *>(base + fragment_at(p, i));
                const float mx = fmaxf(m, ml.x);
                if (mx == -INFINITY) continue;
                l = l * exp2f(m - mx) + ml.y * exp2f(ml.x - mx);
                m = mx;
            }
            float mx = m;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            l = m == -INFINITY ? 0.f : l * exp2f(m - mx);
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
            if (lane16 == 0 && r < kRows) lse2[r] = lse_log2(mx, l);
        } else if (lane16 == 0 && r < kRows) {
            lse2[r] = mine ? p.lse2[(int64_t)(sv.row0 + r / kGroup) * kNumQHeads + kvh * kGroup + r % kGroup] : INFINITY;
        }
    }
    __syncthreads();
    for (int j = 0;;) {
        const float4 l = *reinterpret_cast<const float4 *>(&lse2[j * kGroup]);
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            sum[i] += (fast_exp2(x[i].x - l.x) + fast_exp2(x[i].y - l.y)) + (fast_exp2(x[i].z - l.z) + fast_exp2(x[i].w - l.w));
        if (++j == sv.n) break;
        load_scores(j);
    }
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int t = t0 + i * kFinishThreads + threadIdx.x;
        if (t < sv.len) w[t] = sum[i];
    }
}

// Behind the split kernel: blocks of (record stride, row) merge, the others add weights.
__global__ void __launch_bounds__(kFinishThreads) chunk_finish_kernel(const FinishParams p) {
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x >= p.merge_blocks) {
        add_weights(p, blockIdx.x - p.merge_blocks);
        return;
    }
    const int y = blockIdx.x % p.rows, lanes = p.merge_blocks / p.rows, live = *p.live;
    for (int i = blockIdx.x / p.rows; i < p.records; i += lanes) {
        const Fragment f = read_record(p, i);
        if (i / kNumKvHeads >= live || ragged_seq(p.rag, i / kNumKvHeads, nullptr).n == 0 || f.first >= f.last) continue;  // uniform
        merge_row(p, f, y);
        __syncthreads();  // before the next record's sums
    }
}

// The split form's cluster form: its launch, and the CTAs of a cluster (0: the line form is to be taken). A
// short batch is bound by latency, which the cluster form has less of (one launch); but it takes the
// sequences as they are, so it is for batches whose clusters all run at once, and up to kClusterTokens a
// CTA. Bounds count, not lengths: a call that is to be replayed with up to 65536 tokens takes the line form.
// One row, us: 500 tokens 7.0 against 12.8 of the line form, 4097 10.6 against 15.8, 16000 21.5 against
// 22.5, 32768 36.8 against 33.1; 8 sequences of 1000 9.9 against 15.7, 37 of 300 13.5 against 21.2. Where the
// clusters took two turns: 4 sequences of 300, 8 CTAs each, 11.9 against 12.9, of 2000 16.3 against 16.2.
constexpr int kClusterTokens = 512;
struct ClusterLaunch {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    ClusterLaunch(int clusters, int ctas, cudaStream_t stream) {
        cfg.gridDim = dim3(clusters * ctas);
        cfg.blockDim = dim3(ClusterSmem::kThreads);
        cfg.dynamicSmemBytes = ClusterSmem::kAlloc;
        cfg.stream = stream;
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas;
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
#ifndef PGC_NO_PDL
        cfg.numAttrs = 2;
#else
        cfg.numAttrs = 1;
#endif
    }
};
inline int cluster_of(int dev, int batch, int max_seq_len) {
    static std::atomic<int> held[64][5] = {};  // clusters of 1 << k CTAs that run at once, + 1
    for (int k = 4; k >= 0; --k) {
        int n = dev >= 0 && dev < 64 ? held[dev][k].load() - 1 : -1;
        if (n < 0) {
            ClusterLaunch l(1, 1 << k, nullptr);
            if (cudaOccupancyMaxActiveClusters(&n, chunk_split_kernel<true, true>, &l.cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            if (dev >= 0 && dev < 64) held[dev][k] = n + 1;
        }
        if (batch * kNumKvHeads <= n) return max_seq_len <= kClusterTokens << k ? 1 << k : 0;
    }
    return 0;
}

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace of a call: the shares' records and partials, with weights the rows' lse, and in the split
// form the scores.
struct Layout {
    bool split;
    int shares, rows, records;  // rows: of a partial
    size_t frags = 0, live = 0, parts = 0, lse = 0, scores = 0, total = 0;
    int64_t score_stride = 0;
};
Layout layout(int batch, int total_q, int max_q_len, int max_seq_len, bool weights, int sm_count) {
    Layout l;
    l.split = max_q_len <= PGC_MAX_QUERIES;
    l.shares = l.split ? 2 * sm_count : sm_count / 2;
    l.rows = l.split ? max_q_len * kGroup : 2 * kBM;
    const size_t part = l.split ? (size_t)l.rows * kPartial : kPairPart;
    l.records = l.split ? batch * kNumKvHeads : l.shares;
    l.live = (size_t)l.records * sizeof(Fragment);
    l.parts = align256(l.live + sizeof(int));
    l.lse = align256(l.parts + (size_t)l.shares * 2 * part * sizeof(float));
    l.scores = align256(l.lse + (weights ? (size_t)total_q * kNumQHeads * sizeof(float) : 0));
    l.score_stride = (max_seq_len + kPage - 1) / kPage * kPage;
    l.total = l.scores;
    if (weights && l.split) l.total += (size_t)total_q * kNumKvHeads * l.score_stride * kGroup * sizeof(float);
    return l;
}

}  // namespace

size_t chunk_workspace_bytes(int batch, int total_q, int max_q_len, int max_seq_len, bool weights, int sm_count) {
    return layout(batch, total_q, max_q_len, max_seq_len, weights, sm_count).total;
}

cudaError_t launch_chunk(const uint16_t *q, const CUtensorMap &tk, const CUtensorMap &tv, const uint16_t *v_pages,
                         int64_t num_pages, const int32_t *block_tables, int max_pages_per_seq,
                         const RaggedBatch &rag, float scale, const uint16_t *gate, uint16_t *out, float *lse,
                         const ChunkWeights *weights, void *workspace, int sm_count, cudaStream_t stream) {
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        const auto attr = cudaFuncAttributeMaxDynamicSharedMemorySize;
        cudaError_t e = cudaFuncSetAttribute(chunk_pair_kernel, attr, PairSmem::kBytes);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(chunk_split_kernel<false, false>, attr, LineSmem::kAlloc);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(chunk_split_kernel<true, false>, attr, LineSmem::kAlloc);
        for (auto kern : {chunk_split_kernel<false, true>, chunk_split_kernel<true, true>}) {
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, attr, ClusterSmem::kAlloc);
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        }
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    const Layout lay = layout(rag.batch, rag.total_q, rag.max_q_len, rag.max_seq_len, weights != nullptr, sm_count);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    float *lse2 = weights != nullptr ? reinterpret_cast<float *>(ws + lay.lse) : nullptr;
    FinishParams fp = {};
    fp.frags = reinterpret_cast<const Fragment *>(ws + lay.frags);
    fp.parts = reinterpret_cast<const float *>(ws + lay.parts);
    fp.records = lay.records;
    fp.rows = lay.rows;
    fp.gate = gate;
    fp.out = out;
    fp.lse = lse;
    fp.lse2 = lse2;
    if (lay.split) {
        SplitParams sp = {};
        sp.rag = rag;
        sp.q = q;
        sp.block_tables = block_tables;
        sp.max_pages_per_seq = max_pages_per_seq;
        sp.num_pages = num_pages;
        sp.gate = gate;
        sp.out = out;
        sp.lse = lse;
        sp.lse2 = lse2;
        sp.frags = reinterpret_cast<Fragment *>(ws + lay.frags);
        sp.live = reinterpret_cast<int *>(ws + lay.live);
        sp.parts = reinterpret_cast<float *>(ws + lay.parts);
        sp.scores = weights != nullptr ? reinterpret_cast<float *>(ws + lay.scores) : nullptr;
        sp.score_stride = lay.score_stride;
        sp.scale_log2 = scale * kLog2e;
        sp.cluster = cluster_of(dev, rag.batch, rag.max_seq_len);
        if (sp.cluster != 0) {
            if (weights != nullptr) sp.w = *weights;
            ClusterLaunch l(rag.batch * kNumKvHeads, sp.cluster, stream);
            return cudaLaunchKernelEx(&l.cfg, weights != nullptr ? chunk_split_kernel<true, true> : chunk_split_kernel<false, true>, tk, tv, sp);
        }
        const dim3 grid(lay.shares), block(LineSmem::kThreads);
        cudaError_t e = weights != nullptr ? launch_pdl(chunk_split_kernel<true, false>, grid, block, LineSmem::kAlloc, stream, tk, tv, sp)
                                           : launch_pdl(chunk_split_kernel<false, false>, grid, block, LineSmem::kAlloc, stream, tk, tv, sp);
        if (e != cudaSuccess) return e;
        fp.rag = rag;
        fp.live = sp.live;
        // a few hundred blocks cover the records: most of a large batch's are of units not cut
        fp.merge_blocks = (lay.records < lay.shares ? lay.records : lay.shares) * lay.rows;
        int blocks = fp.merge_blocks;
        if (weights != nullptr) {
            fp.scores = sp.scores;
            fp.score_stride = lay.score_stride;
            fp.w = *weights;
            fp.add_chunks = (rag.max_seq_len + kAddTokens - 1) / kAddTokens;
            blocks += rag.batch * kNumKvHeads * fp.add_chunks;
        }
        return launch_pdl(chunk_finish_kernel, dim3(blocks), dim3(kFinishThreads), 0, stream, fp);
    }
    CUtensorMap tq;
    if (q_tensor_map(q, rag.total_q, &tq) != PGC_OK) return cudaErrorInvalidValue;
    PairParams pp = {};
    pp.rag = rag;
    pp.block_tables = block_tables;
    pp.max_pages_per_seq = max_pages_per_seq;
    pp.num_pages = num_pages;
    pp.v_pages = v_pages;
    pp.gate = gate;
    pp.out = out;
    pp.lse = lse;
    pp.lse2 = lse2;
    pp.frags = reinterpret_cast<Fragment *>(ws + lay.frags);
    pp.parts = reinterpret_cast<float *>(ws + lay.parts);
    pp.scale_log2 = scale * kLog2e;
    cudaError_t e = launch_pdl(chunk_pair_kernel, dim3(2 * lay.shares), dim3(kPairThreads), PairSmem::kBytes, stream, tq, tk, tv, pp);
    if (e == cudaSuccess) e = launch_pdl(chunk_merge_kernel, dim3(lay.shares, lay.rows / 32, kHeadDim / kMergeDims), dim3(kMergeThreads), 0, stream, fp);
    if (e != cudaSuccess || weights == nullptr) return e;
    return launch_chunk_weights(q, tk, num_pages, block_tables, max_pages_per_seq, rag, scale, lse2, *weights, sm_count, stream);
}

cudaError_t chunk_read_error(DevErrorHost *e, bool clear) {
    cudaError_t r = cudaMemcpyFromSymbol(e, g_chunk_err, sizeof(DevError));
    if (r != cudaSuccess || !clear) return r;
    DevErrorHost z = {0, 0, 0};
    return cudaMemcpyToSymbol(g_chunk_err, &z, sizeof(DevError));
}

}  // namespace pgc
