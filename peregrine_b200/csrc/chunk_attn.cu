// chunk_attn.cu — causal GQA attention of a ragged batch of chunks over the paged cache, with the
// log-sum-exp of every row and, on request, each cached token's received attention (sm_100a).
//
// For sequence b with n query rows and L cached tokens (the rows included), row i sits at position
// p = L - n + i and sees tokens [0, p]:
//     s_t = scale q.k_t,  lse = log sum_{t <= p} exp(s_t),  o = sum_t exp(s_t - lse) v_t
// and, with weights, w[kv head][t] += sum over the kv head's 4 query heads and the rows of
// exp(s_t - lse). A row that sees nothing (p < 0) has o = 0 and lse = -inf.
//
// Two forms, chosen by the host bound on the rows of a sequence:
//   * up to PGC_MAX_QUERIES rows: the split decode kernel over the ragged batch (decode_attn.cu),
//     bound by the K/V bytes, then chunk_finish_kernel, which merges the splits and adds the
//     weights from the scores that the split kernel left (one pass over K);
//   * more rows: chunk_pair_kernel on the 5th-gen tensor cores, then chunk_merge_kernel for the
//     rows whose key range was shared out, and chunk_weights.cu for the weights.
#include <cuda.h>

#include "pgc_common.cuh"
#include "pgc_internal.h"
#include "pgc_ragged.cuh"
#include "pgc_tcgen05.cuh"

namespace pgc {

PGC_DEFINE_ERROR_WORD(g_chunk_err);

namespace {

__device__ __forceinline__ float sigmoid_gate(float v, uint32_t gate_bits) {
    return v * (1.0f / (1.0f + expf(-bf16_bits_to_f32(gate_bits))));
}

// =============================================================================================
// Up to 4 rows a sequence: merge of the splits and the weights, one launch. Blocks [0, merge_blocks)
// merge (one per row, head and 32-dim chunk; the 8 warps take every 8th split, as the uniform
// batch's merge does); the rest add the weights of 1024 tokens of one (sequence, kv head) each,
// from the scores in the workspace and the rows' lse, which they form from the splits' (m, l)
// themselves: both halves start as soon as the split kernel has finished.
// =============================================================================================
struct FinishParams {
    RaggedBatch rag;
    const float *parts;  // [total_q * 16][max_splits][258]
    int max_splits;
    int merge_blocks;
    const uint16_t *gate;
    uint16_t *out;
    float *lse;
    // weights
    const float *scores;  // [total_q][4][score_stride][4], scaled by log2(e)
    int64_t score_stride;
    float *weights;
    int64_t weights_stride, num_slots;
    const int32_t *slots;
    int add_chunks;  // blocks per (sequence, kv head)
};

constexpr int kFinishThreads = 256;
constexpr int kAddTokens = 1024;

__device__ __forceinline__ void finish_merge(const FinishParams &p, int blk) {
    __shared__ float red_m[8], red_den[8], red_acc[8][32];
    const int chunk = blk & 7;
    const int head = (blk >> 3) & 15;
    const int j = (blk >> 7) % p.rag.max_q_len;
    const int b = (blk >> 7) / p.rag.max_q_len;
    const RaggedSeq sv = ragged_seq(p.rag, b, nullptr);
    if (j >= sv.n) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)(sv.row0 + j) * kNumQHeads + head;
    const int d = chunk * 32 + lane;
    const float *base = p.parts + row * p.max_splits * kPartial;
    // 10 splits per warp are held in registers (one round of loads); longer rows stream them
    constexpr int kCached = 10;
    float ma = -INFINITY, den = 0.f, acc = 0.f;
    float mc[kCached], lc[kCached], oc[kCached];
#pragma unroll
    for (int i = 0; i < kCached; ++i) {
        const int c = warp + 8 * i;
        mc[i] = -INFINITY;
        lc[i] = oc[i] = 0.f;
        if (c < p.max_splits) {
            const float *pc = base + (int64_t)c * kPartial;
            mc[i] = pc[0];
            lc[i] = pc[1];
            oc[i] = pc[2 + d];  // read even for an empty part: it is not summed
        }
        ma = fmaxf(ma, mc[i]);
    }
    for (int c = warp + 8 * kCached; c < p.max_splits; c += 8) ma = fmaxf(ma, base[(int64_t)c * kPartial]);
    if (lane == 0) red_m[warp] = ma;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) ma = fmaxf(ma, red_m[w]);
#pragma unroll
    for (int i = 0; i < kCached; ++i) {
        if (mc[i] == -INFINITY) continue;
        const float w = exp2f((mc[i] - ma) * kLog2e);
        den += lc[i] * w;
        acc += oc[i] * w;
    }
    for (int c = warp + 8 * kCached; c < p.max_splits; c += 8) {
        const float *pc = base + (int64_t)c * kPartial;
        const float m = pc[0];
        if (m == -INFINITY) continue;
        const float w = exp2f((m - ma) * kLog2e);
        den += pc[1] * w;
        acc += pc[2 + d] * w;
    }
    red_acc[warp][lane] = acc;
    if (lane == 0) red_den[warp] = den;
    __syncthreads();
    if (warp != 0) return;
    acc = den = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
        acc += red_acc[w][lane];
        den += red_den[w];
    }
    float v = (den == 0.f) ? 0.f : acc / den;
    if (p.gate != nullptr) v = sigmoid_gate(v, p.gate[row * kHeadDim + d]);
    p.out[row * kHeadDim + d] = f32_to_bf16_bits(v);
    if (p.lse != nullptr && chunk == 0 && lane == 0) p.lse[row] = (den == 0.f) ? -INFINITY : ma + logf(den);
}

__device__ __forceinline__ void finish_add(const FinishParams &p, int blk) {
    __shared__ float lse2[PGC_MAX_QUERIES * kGroup];
    const int chunk = blk % p.add_chunks;
    const int kvh = (blk / p.add_chunks) % kNumKvHeads;
    const int b = blk / p.add_chunks / kNumKvHeads;
    const RaggedSeq sv = ragged_seq(p.rag, b, nullptr);
    const int t0 = chunk * kAddTokens;
    if (sv.n == 0 || t0 >= sv.len) return;
    const int64_t slot = ragged_slot(p.slots, p.num_slots, b, chunk == 0 && kvh == 0 ? &g_chunk_err : nullptr);
    if (slot < 0) return;
    // 16 threads per row: log2 of the row's sum over all splits; +inf where it is 0, so that a
    // row of -inf scores adds nothing
    {
        const int r = threadIdx.x >> 4, part = threadIdx.x & 15;
        const int np = r < sv.n * kGroup ? p.max_splits : 0;
        const int64_t row = (int64_t)(sv.row0 + r / kGroup) * kNumQHeads + kvh * kGroup + r % kGroup;
        const float *base = p.parts + row * p.max_splits * kPartial;
        float m = -INFINITY, l = 0.f;
        for (int c = part; c < np; c += 16) m = fmaxf(m, base[(int64_t)c * kPartial]);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        for (int c = part; c < np; c += 16) {
            const float mc = base[(int64_t)c * kPartial];
            if (mc != -INFINITY) l += base[(int64_t)c * kPartial + 1] * exp2f((mc - m) * kLog2e);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (part == 0) lse2[r] = l == 0.f ? INFINITY : m * kLog2e + log2f(l);
    }
    __syncthreads();
    float *w = p.weights + (slot * kNumKvHeads + kvh) * p.weights_stride;
    const float4 *s = reinterpret_cast<const float4 *>(p.scores);
#pragma unroll
    for (int i = 0; i < kAddTokens / kFinishThreads; ++i) {
        const int t = t0 + i * kFinishThreads + threadIdx.x;
        if (t >= sv.len) break;
        float add = 0.f;
        for (int j = 0; j < sv.n; ++j) {
            if (t > sv.len - sv.n + j) continue;  // not visible to row j
            const float4 x = s[((int64_t)(sv.row0 + j) * kNumKvHeads + kvh) * p.score_stride + t];
            add += exp2f(x.x - lse2[j * kGroup]);
            add += exp2f(x.y - lse2[j * kGroup + 1]);
            add += exp2f(x.z - lse2[j * kGroup + 2]);
            add += exp2f(x.w - lse2[j * kGroup + 3]);
        }
        w[t] += add;
    }
}

__global__ void __launch_bounds__(kFinishThreads) chunk_finish_kernel(const FinishParams p) {
    pdl_trigger();
    pdl_wait();
    if ((int)blockIdx.x < p.merge_blocks)
        finish_merge(p, blockIdx.x);
    else
        finish_add(p, blockIdx.x - p.merge_blocks);
}

// =============================================================================================
// More rows a sequence: two-SM tcgen05 kernel (cta_group::2). The tile of work and the roles are
// those of the single-sequence prefill kernel: a cluster of two CTAs runs one kv head for 64 query
// tokens (each CTA's 32 tokens x 4 GQA heads stacked into 128 rows, M = 256), each CTA stages its
// own Q, 64 of a 128-key tile's keys and 128 of its value dims, S (two tiles) and O live in TMEM and
// P is written over S. What differs is the schedule. Lengths are on the device, so the launch is a
// fixed grid of one pair per two SMs, and the pairs share out the batch's key tiles: the tiles of
// all (sequence, kv head, 64-token tile) units, in that order, form one line, which is cut into
// equal consecutive shares. A unit cut by a share's border leaves fp32 partials (at most two units a
// pair: its first and its last), which chunk_merge_kernel joins; every other unit is written by its
// pair. The balance is then within one key tile whatever the lengths, and the workspace is fixed.
// Loads, MMAs and softmax run on across units: the next unit's K, V and Q loads and its first S
// products overlap this unit's last products and its epilogue.
// =============================================================================================
constexpr int kBM = 128;  // rows of a CTA: 32 tokens x 4 heads
constexpr int kTokTile = 32;
constexpr int kUnitTok = 2 * kTokTile;
constexpr uint32_t kTmemCols = 512;
constexpr float kLazyRescale = 8.0f;  // log2 units: rescale O only when the max grows by > 2^8
constexpr int kSoftmaxWarps = 16;
constexpr int kProducerWarps = 2;
constexpr int kPairThreads = 32 * (kSoftmaxWarps + 1 + 2 * kProducerWarps);
constexpr int kKeys = 128;                    // keys per tile
constexpr int kQBytes = kBM * kHeadDim * 2;   // [4 dim blocks][128 rows][128 B]
constexpr int kKHalf = 64 * kHeadDim * 2;     // this CTA's 64 keys: [4][64][128 B]
constexpr int kVHalf = kKeys * 128 * 2;       // this CTA's 128 dims: [2][128][128 B]
constexpr int kKSlots = 3;
constexpr int kVSlots = 2;
constexpr uint32_t kTO = 0;    // O: 256 columns
constexpr uint32_t kTS = 256;  // S tiles: 2 x 128 columns; P(j) over the first 64 of S(j)
// A share below this many tiles costs more in its Q load, pipeline fill and partials than it saves.
constexpr int kMinShare = 4;

// A fragment left in the workspace: rows [256][258] fp32 of one unit's tiles [t0, t1) of `tiles`.
struct Fragment {
    int seq;  // -1: none
    int kvh, qt, last;  // last: it holds the unit's last tile
};

struct PairParams {
    RaggedBatch rag;
    const int32_t *block_tables;
    int max_pages_per_seq;
    int64_t num_pages;
    const uint16_t *v_pages;
    const uint16_t *gate;
    uint16_t *out;
    float *lse;
    Fragment *frags;  // [pairs][2]: a share's first unit if cut before its first tile, its last if cut after
    float *parts;     // [pairs][2][256][258]
    float scale_log2;
};

// Key tiles of one unit: the keys that its last row sees, at least one tile (rows that see nothing
// still get their zeros).
__device__ __forceinline__ int unit_tiles(int n, int len, int qt) {
    const int keys = len - n + min((qt + 1) * kUnitTok, n);
    return keys > kKeys ? (keys + kKeys - 1) / kKeys : 1;
}

// A pair's share as a walk over (unit, tile range); every role steps its own copy.
struct Walk {
    int seq, kvh, qt;
    int row0, n, len;  // of the sequence
    int tiles;         // of the unit
    int t0, t1;        // this pair's tiles of it
    int64_t left;      // tiles of the share from t0 on
};

__device__ __forceinline__ void walk_seq(const RaggedBatch &rag, Walk &w) {
    const RaggedSeq s = ragged_seq(rag, w.seq, nullptr);
    w.row0 = s.row0;
    w.n = s.n;
    w.len = s.len;
}
__device__ __forceinline__ void walk_unit(Walk &w, int t0) {
    w.tiles = unit_tiles(w.n, w.len, w.qt);
    w.t0 = t0;
    w.t1 = (int64_t)w.tiles - t0 < w.left ? w.tiles : t0 + (int)w.left;
}
// Next unit; false at the end of the share.
__device__ __forceinline__ bool walk_next(const RaggedBatch &rag, Walk &w) {
    w.left -= w.t1 - w.t0;
    if (w.left <= 0) return false;
    if (++w.qt * kUnitTok >= w.n) {
        w.qt = 0;
        if (++w.kvh == kNumKvHeads) {
            w.kvh = 0;
            do {
                if (++w.seq >= rag.batch) return false;
                walk_seq(rag, w);
            } while (w.n == 0);
        }
    }
    walk_unit(w, 0);
    return true;
}

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
    static constexpr int kTmemSlot = kWalk + 48;
    static constexpr int kAbort = kTmemSlot + 8;
    static constexpr int kBytes = kAbort + 8;
};
static_assert(sizeof(Walk) <= 48 && PairSmem::kWalk % 8 == 0, "walk slot");
static_assert(PairSmem::kBytes <= 232448, "pair shared memory exceeds the sm_100 limit");
static_assert(PGC_CHUNK_MAX_BATCH * 8 <= kKSlots * kKHalf, "the schedule's scratch is the K ring");

// The share of pair `pair` of `pairs`: tiles [total * p / W, total * (p + 1) / W) of the line, over
// W = min(pairs, total / kMinShare) pairs. Run by the whole CTA; `cost` is scratch (one int64 per
// sequence). Returns false when the pair has no share.
__device__ __forceinline__ bool find_share(const RaggedBatch &rag, int64_t *cost, int pair, int pairs, Walk *out,
                                           DevError *err) {
    for (int b = threadIdx.x; b < rag.batch; b += blockDim.x) {
        const RaggedSeq s = ragged_seq(rag, b, err);
        int64_t c = 0;
        for (int qt = 0; qt * kUnitTok < s.n; ++qt) c += unit_tiles(s.n, s.len, qt);
        cost[b] = c * kNumKvHeads;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int64_t total = 0;
        for (int b = lane; b < rag.batch; b += 32) total += cost[b];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        int64_t w = total / kMinShare;
        w = w < 1 ? 1 : w > pairs ? pairs : w;
        const int64_t begin = total * pair / w, end = total * (pair + 1) / w;
        Walk wk = {};
        wk.seq = -1;
        if (pair < w && end > begin) {
            int64_t before = 0;
            for (int b0 = 0; b0 < rag.batch; b0 += 32) {
                const int64_t c = b0 + lane < rag.batch ? cost[b0 + lane] : 0;
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
            const int64_t per = cost[wk.seq] / kNumKvHeads;
            int64_t off = begin - before;
            wk.kvh = (int)(off / per);
            off -= wk.kvh * per;
            for (wk.qt = 0;; ++wk.qt) {
                const int t = unit_tiles(wk.n, wk.len, wk.qt);
                if (off < t) break;
                off -= t;
            }
            wk.left = end - begin;
            walk_unit(wk, (int)off);
        }
        if (lane == 0) *out = wk;
    }
    __syncthreads();
    return out->seq >= 0;
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
    Walk *share = reinterpret_cast<Walk *>(smem + PairSmem::kWalk);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + PairSmem::kAbort);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int pair = blockIdx.x >> 1;

    const bool busy = find_share(p.rag, reinterpret_cast<int64_t *>(smem + PairSmem::kK), pair, gridDim.x >> 1, share,
                                 blockIdx.x == 0 ? &g_chunk_err : nullptr);
    Fragment *frag = p.frags + pair * 2;
    if (leader && threadIdx.x < 2) frag[threadIdx.x].seq = -1;
    if (!busy) return;  // both CTAs of the pair
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
    const uint32_t tmem = *tmem_slot;
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
    Walk w = *share;

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
                if (!walk_next(p.rag, w)) break;
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
            if (!walk_next(p.rag, w)) break;
        }
    } else if (warp == kSoftmaxWarps) {
        // ------------------------------------------------------------ pair MMA issuer (leader)
        if (leader && lane == 0) {
            constexpr uint32_t idesc_s = umma_idesc(2 * kBM, kKeys, false, false);
            constexpr uint32_t idesc_o = umma_idesc(2 * kBM, kHeadDim, false, true);
            const uint32_t q_addr = smem_u32(smem + PairSmem::kQ);
            // `ahead` is the next tile whose S is to be issued: S(g + 2) goes out behind PV(g), but
            // the first S of a unit only behind the last PV of the unit before it, because it waits
            // for that unit's Q to be replaced.
            Walk a = w;
            int at = a.t0, ag = 0, aunit = 0;
            bool more = true, ok = true;
            auto issue_s = [&]() -> bool {
                const int b = ag & 1, sl = ag % kKSlots;
                if (at == a.t0 && !wait(q_full, aunit & 1, 4)) return false;
                if (!wait(&k_full[sl], (ag / kKSlots) & 1, 5)) return false;
                tc_fence_after();
                const uint32_t k_addr = smem_u32(smem + PairSmem::kK + sl * kKHalf);
#pragma unroll
                for (int kk = 0; kk < kHeadDim / 16; ++kk)
                    umma2_ss(tmem + kTS + b * kKeys,
                             umma_desc(q_addr + (kk >> 2) * (kBM * 128) + (kk & 3) * 32, 16, 1024),
                             umma_desc(k_addr + (kk >> 2) * (64 * 128) + (kk & 3) * 32, 16, 1024),
                             idesc_s, kk > 0 ? 1u : 0u);
                umma2_commit_pair(&k_empty[sl]);
                umma2_commit_pair(&s_full[b]);
                ++ag;
                if (++at == a.t1) {
                    umma2_commit_pair(q_empty);
                    more = walk_next(p.rag, a);
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
                    const uint32_t v_addr = smem_u32(smem + PairSmem::kV + sl * kVHalf);
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; ++kk)
                        umma2_ts(tmem + kTO, tmem + kTS + b * kKeys + kk * 8,
                                 umma_desc(v_addr + kk * 2048, kKeys * 128, 1024), idesc_o,
                                 (t > w.t0 || kk > 0) ? 1u : 0u);
                    umma2_commit_pair(&v_empty[sl]);
                    umma2_commit_pair(&pv_done[b]);
                }
                if (!ok || !walk_next(p.rag, w)) break;
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
                    float mq[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
                    for (int i = 4; i < 32; i += 8)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (i + 2 * k + 1 < 32) mq[k] = fmax3(mq[k], sv[i + 2 * k], sv[i + 2 * k + 1]);
                    float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
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
            if (!whole && leader && warp == 0 && lane == 0) {
                frag[slot].kvh = w.kvh;
                frag[slot].qt = w.qt;
                frag[slot].last = w.t1 == w.tiles;
                frag[slot].seq = w.seq;
            }
            if (live) {
                red[cg * kBM + r] = l;
                asm volatile("bar.sync %0, 128;" ::"r"(1 + qd) : "memory");
                const float l_row = (red[r] + red[kBM + r]) + (red[2 * kBM + r] + red[3 * kBM + r]);
                asm volatile("bar.sync %0, 128;" ::"r"(1 + qd) : "memory");  // before the next unit's maxima
                const float inv = l_row == 0.f ? 0.f : 1.f / l_row;
                const int64_t orow = (int64_t)(w.row0 + tok) * kNumQHeads + w.kvh * kGroup + r % kGroup;
                float *part = p.parts + ((int64_t)(pair * 2 + slot) * 2 * kBM + rank * kBM + r) * kPartial;
                if (row_ok && cg == 0) {
                    if (!whole) {
                        part[0] = (m == -INFINITY) ? -INFINITY : m * kLn2;
                        part[1] = l_row;
                    } else if (p.lse != nullptr) {
                        p.lse[orow] = l_row == 0.f ? -INFINITY : m * kLn2 + logf(l_row);
                    }
                }
#pragma unroll 1
                for (int cc = 0; cc < 2; ++cc) {
                    float o[32];
                    const int col = cg * 64 + cc * 32;
                    tmem_ld32(tmem + lane_addr + kTO + col, o);
                    tmem_wait_ld();
                    if (!row_ok) continue;
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            *reinterpret_cast<float2 *>(part + 2 + col + i) = make_float2(o[i], o[i + 1]);
                        continue;
                    }
                    // a row with nothing visible has P = 0 throughout: o = 0 and inv = 0
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] *= inv;
                    if (p.gate != nullptr) {
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
                    uint16_t *dst = p.out + orow * kHeadDim + col;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint4 v;
                        v.x = pack_bf16x2(o[i], o[i + 1]);
                        v.y = pack_bf16x2(o[i + 2], o[i + 3]);
                        v.z = pack_bf16x2(o[i + 4], o[i + 5]);
                        v.w = pack_bf16x2(o[i + 6], o[i + 7]);
                        *reinterpret_cast<uint4 *>(dst + i) = v;
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(obar);
            if (!walk_next(p.rag, w)) break;
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

// Joins the fragments of the units that were cut: block (p, y) takes the unit that pair p left
// unfinished (its last fragment) and the first fragments of the pairs after it, up to the one that
// holds the unit's last tile. A warp per row; lane l owns dims [8 l, 8 l + 8).
constexpr int kMergeY = 16;

__global__ void __launch_bounds__(256) chunk_merge_kernel(const PairParams p) {
    pdl_trigger();
    pdl_wait();
    const int pair = blockIdx.x, pairs = gridDim.x;
    const Fragment f = p.frags[pair * 2 + 1];
    if (f.seq < 0) return;
    int last = pair + 1;  // the pair whose first fragment ends the unit
    while (last < pairs && p.frags[last * 2].seq == f.seq && !p.frags[last * 2].last) ++last;
    if (last >= pairs) return;  // not reached: a cut unit is finished by a later pair
    const RaggedSeq sv = ragged_seq(p.rag, f.seq, nullptr);
    const int lane = threadIdx.x & 31;
    const int64_t slot_floats = (int64_t)2 * kBM * kPartial;
    for (int r = blockIdx.y * 8 + (threadIdx.x >> 5); r < 2 * kBM; r += kMergeY * 8) {
        const int tok = f.qt * kUnitTok + r / kGroup;
        if (tok >= sv.n) break;  // rows are in token order
        const float *first = p.parts + (pair * 2 + 1) * slot_floats + (int64_t)r * kPartial;
        const float *next = p.parts + (int64_t)(pair + 1) * 2 * slot_floats + (int64_t)r * kPartial;
        const int np = last - pair;  // fragments behind the first, one every 2 slots
        float ma = first[0];
        for (int i = 0; i < np; ++i) ma = fmaxf(ma, next[i * 2 * slot_floats]);
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        float den = 0.f;
        for (int i = -1; i < np; ++i) {
            const float *pc = i < 0 ? first : next + i * 2 * slot_floats;
            const float mc = pc[0];
            if (mc == -INFINITY) continue;
            const float w = exp2f((mc - ma) * kLog2e);
            den += pc[1] * w;
            const float2 *o = reinterpret_cast<const float2 *>(pc + 2 + 8 * lane);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 v = o[k];
                acc[2 * k] += v.x * w;
                acc[2 * k + 1] += v.y * w;
            }
        }
        const int64_t orow = (int64_t)(sv.row0 + tok) * kNumQHeads + f.kvh * kGroup + r % kGroup;
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = (den == 0.f) ? 0.f : acc[k] / den;
        if (p.gate != nullptr) {
            const uint4 gq = *reinterpret_cast<const uint4 *>(p.gate + orow * kHeadDim + 8 * lane);
            const uint32_t gw[4] = {gq.x, gq.y, gq.z, gq.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = sigmoid_gate(v[k], (gw[k >> 1] >> ((k & 1) * 16)) & 0xffffu);
        }
        uint4 q;
        q.x = pack_bf16x2(v[0], v[1]);
        q.y = pack_bf16x2(v[2], v[3]);
        q.z = pack_bf16x2(v[4], v[5]);
        q.w = pack_bf16x2(v[6], v[7]);
        *reinterpret_cast<uint4 *>(p.out + orow * kHeadDim + 8 * lane) = q;
        if (p.lse != nullptr && lane == 0) p.lse[orow] = (den == 0.f) ? -INFINITY : ma + logf(den);
    }
}

inline size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }

// Workspace of a call, in order: partials; then, for the split form with weights, the scores; for
// the pair form, the fragment records and, with weights and no caller's lse, the lse.
struct Layout {
    size_t parts = 0, scores = 0, frags = 0, lse = 0, total = 0;
    int64_t score_stride = 0;
};
Layout layout(int batch, int total_q, int max_q_len, int max_seq_len, bool weights, int sm_count) {
    Layout l;
    size_t at = 0;
    if (max_q_len <= PGC_MAX_QUERIES) {
        const DecodePlan plan = decode_plan(batch, max_seq_len, sm_count);
        l.parts = at;
        at = align256(at + (size_t)total_q * kNumQHeads * plan.max_splits * kPartial * sizeof(float));
        if (weights) {
            l.score_stride = (max_seq_len + kPage - 1) / kPage * kPage;
            l.scores = at;
            at = align256(at + (size_t)total_q * kNumKvHeads * l.score_stride * kGroup * sizeof(float));
        }
    } else {
        const size_t pairs = sm_count / 2;
        l.parts = at;
        at = align256(at + pairs * 2 * 2 * kBM * kPartial * sizeof(float));
        l.frags = at;
        at = align256(at + pairs * 2 * sizeof(Fragment));
        if (weights) {
            l.lse = at;
            at = align256(at + (size_t)total_q * kNumQHeads * sizeof(float));
        }
    }
    l.total = at;
    return l;
}

}  // namespace

size_t chunk_workspace_bytes(int batch, int total_q, int max_q_len, int max_seq_len, bool weights, int sm_count) {
    return layout(batch, total_q, max_q_len, max_seq_len, weights, sm_count).total;
}

cudaError_t launch_chunk(const uint16_t *q, const CUtensorMap &tk, const CUtensorMap &tv, const uint16_t *k_pages,
                         const uint16_t *v_pages, int64_t num_pages, const int32_t *block_tables,
                         int max_pages_per_seq, const RaggedBatch &rag, float scale, const uint16_t *gate,
                         uint16_t *out, float *lse, const ChunkWeights *weights, void *workspace, int sm_count,
                         cudaStream_t stream) {
    const Layout lay = layout(rag.batch, rag.total_q, rag.max_q_len, rag.max_seq_len, weights != nullptr, sm_count);
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    float *parts = reinterpret_cast<float *>(ws + lay.parts);
    if (rag.max_q_len <= PGC_MAX_QUERIES) {
        float *scores = weights != nullptr ? reinterpret_cast<float *>(ws + lay.scores) : nullptr;
        cudaError_t e = launch_ragged_split(q, tk, tv, num_pages, block_tables, max_pages_per_seq, rag, scale, parts,
                                            scores, lay.score_stride, k_pages, v_pages, sm_count, stream);
        if (e != cudaSuccess) return e;
        FinishParams fp = {};
        fp.rag = rag;
        fp.parts = parts;
        fp.max_splits = decode_plan(rag.batch, rag.max_seq_len, sm_count).max_splits;
        fp.merge_blocks = rag.batch * rag.max_q_len * kNumQHeads * (kHeadDim / 32);
        fp.gate = gate;
        fp.out = out;
        fp.lse = lse;
        int blocks = fp.merge_blocks;
        if (weights != nullptr) {
            fp.scores = scores;
            fp.score_stride = lay.score_stride;
            fp.weights = weights->weights;
            fp.weights_stride = weights->stride;
            fp.num_slots = weights->num_slots;
            fp.slots = weights->slots;
            fp.add_chunks = (rag.max_seq_len + kAddTokens - 1) / kAddTokens;
            blocks += rag.batch * kNumKvHeads * fp.add_chunks;
        }
        return launch_pdl(chunk_finish_kernel, dim3((unsigned)blocks), dim3(kFinishThreads), 0, stream, fp);
    }
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(chunk_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             PairSmem::kBytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    CUtensorMap tq;
    if (q_tensor_map(q, rag.total_q, &tq) != PGC_OK) return cudaErrorInvalidValue;
    const int pairs = sm_count / 2;
    PairParams pp = {};
    pp.rag = rag;
    pp.block_tables = block_tables;
    pp.max_pages_per_seq = max_pages_per_seq;
    pp.num_pages = num_pages;
    pp.v_pages = v_pages;
    pp.gate = gate;
    pp.out = out;
    pp.lse = lse != nullptr || weights == nullptr ? lse : reinterpret_cast<float *>(ws + lay.lse);
    pp.frags = reinterpret_cast<Fragment *>(ws + lay.frags);
    pp.parts = parts;
    pp.scale_log2 = scale * kLog2e;
    cudaError_t e = launch_pdl(chunk_pair_kernel, dim3(2 * pairs), dim3(kPairThreads), PairSmem::kBytes, stream, tq, tk, tv, pp);
    if (e == cudaSuccess) e = launch_pdl(chunk_merge_kernel, dim3(pairs, kMergeY), dim3(256), 0, stream, pp);
    if (e != cudaSuccess || weights == nullptr) return e;
    return launch_chunk_weights(tq, tk, num_pages, block_tables, max_pages_per_seq, rag, scale, pp.lse, *weights,
                                sm_count, stream);
}

cudaError_t chunk_read_error(DevErrorHost *e, bool clear) {
    cudaError_t r = cudaMemcpyFromSymbol(e, g_chunk_err, sizeof(DevError));
    if (r != cudaSuccess || !clear) return r;
    DevErrorHost z = {0, 0, 0};
    return cudaMemcpyToSymbol(g_chunk_err, &z, sizeof(DevError));
}

}  // namespace pgc
