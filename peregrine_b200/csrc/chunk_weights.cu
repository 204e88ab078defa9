// chunk_weights.cu — the attention that each cached token received from a batch of query rows
// (sm_100a): w[kv head][t] += sum over rows i and the kv head's 4 query heads of exp(s_it - lse_i)
// with the scores recomputed on the 5th-gen tensor cores once the rows' log-sum-exp is known.
//
// The product is taken transposed, S^T = K Q^T: a key is then a TMEM lane, that is one thread, which
// adds its row of exponentials in registers, with no exchange until the key's rows are all done. A
// cluster of two CTAs (cta_group::2) owns 256 keys of one (sequence, kv head) at a time, 128 a CTA,
// resident in shared memory, and streams the query rows past them in tiles of 32 tokens x 4 heads
// (N = 128; each CTA stages half of them, in blocks of 64 dims). One pair adds all of a key's rows
// and is the only writer of its weight, so the sums' order is fixed and no atomics are needed.
// A tile takes 1024 cycles of the tensor pipe and as many of the MUFU pipe (16 exponentials a cycle
// and SM), but three times that from its product to its sums, so TMEM holds four products, each with a
// group of 4 warps of its own. The tensor pipe is 67 % busy on four prompts of 239 to 1600 tokens over
// 4387 to 12000; moving a quarter or more of the exponentials to the FMA pipe (a polynomial) did not
// raise that, two products of 256 columns instead of four of 128 lowered it by 5 %.
// Units (sequence, kv head, 256 keys) are dealt to the pairs in consecutive shares of about equal
// numbers of query tiles.
#include <cuda.h>

#include "pgc_common.cuh"
#include "pgc_internal.h"
#include "pgc_ragged.cuh"
#include "pgc_tcgen05.cuh"

namespace pgc {

PGC_DEFINE_ERROR_WORD(g_cweights_err);

namespace {

constexpr int kUnitKeys = 256;   // keys of a pair's unit, 128 a CTA
constexpr int kTileTok = 32;     // query tokens of a tile (x 4 heads = 128 rows)
constexpr int kCols = kTileTok * kGroup;
constexpr int kBufs = 4;         // products in TMEM, each with a group of 4 warps (a key a thread)
constexpr int kSumWarps = 4 * kBufs;
constexpr int kLoadWarps = 2;    // TMA: one issuing warp delivers about 21 B a cycle to an SM, two 33
constexpr int kThreads = 32 * (kSumWarps + 1 + kLoadWarps);
constexpr int kKBytes = 128 * kHeadDim * 2;  // this CTA's keys: [4 dim blocks][128 rows][128 B]
constexpr int kQBytes = 64 * 128;            // this CTA's 64 query rows x 64 dims
constexpr int kKSlots = 2;
constexpr int kQSlots = 10;
constexpr uint32_t kTmemCols = 512;

struct WeightsParams {
    RaggedBatch rag;
    const int32_t *block_tables;
    int max_pages_per_seq;
    int64_t num_pages;
    const float *lse2;  // of the attention's rows, in log2 units; +inf for a row that sees nothing
    ChunkWeights w;
    float scale_log2;
};

// Walk over the units of a share.
struct Units {
    int seq, kvh, kt;
    int row0, n, len;
    int q0, q1;        // query tiles that see the unit's keys
    int64_t pos, end;  // of this unit's first query tile, of the share
};

// First query tile with a row that sees a key of tile kt: row i sees keys up to len - n + i.
__device__ __forceinline__ int first_tile(int n, int len, int kt) {
    const int i = kt * kUnitKeys - (len - n);
    return i > 0 ? i / kTileTok : 0;
}
// Query tiles of all of a (sequence, kv head)'s units.
__device__ __forceinline__ int64_t head_cost(int n, int len) {
    const int qn = (n + kTileTok - 1) / kTileTok;
    const int kn = (len + kUnitKeys - 1) / kUnitKeys;
    if (n == 0 || kn == 0) return 0;
    // key tiles that every row tile sees, then the diagonal's
    int kt = len >= n ? min(kn, (len - n) / kUnitKeys + 1) : 0;
    int64_t c = (int64_t)kt * qn;
    for (; kt < kn; ++kt) c += qn - first_tile(n, len, kt);
    return c;
}
__device__ __forceinline__ void units_seq(const RaggedBatch &rag, Units &u) {
    const RaggedSeq s = ragged_seq(rag, u.seq, nullptr);
    u.row0 = s.row0;
    u.n = s.n;
    u.len = s.len;
}
__device__ __forceinline__ void units_set(Units &u) {
    u.q0 = first_tile(u.n, u.len, u.kt);
    u.q1 = (u.n + kTileTok - 1) / kTileTok;
}
// Next unit of the share; false behind its last.
__device__ __forceinline__ bool units_next(const RaggedBatch &rag, Units &u) {
    u.pos += u.q1 - u.q0;
    if (u.pos >= u.end) return false;
    if (++u.kt * kUnitKeys >= u.len) {
        u.kt = 0;
        if (++u.kvh == kNumKvHeads) {
            u.kvh = 0;
            do {
                if (++u.seq >= rag.batch) return false;
                units_seq(rag, u);
            } while (u.n == 0 || u.len == 0);
        }
    }
    units_set(u);
    return true;
}

// The units whose first query tile lies in [total * p / pairs, total * (p + 1) / pairs) of the line
// of all units' query tiles. Run by the whole CTA with one int64 of scratch per sequence.
__device__ __forceinline__ bool find_units(const RaggedBatch &rag, int64_t *cost, int pair, int pairs, Units *out) {
    for (int b = threadIdx.x; b < rag.batch; b += blockDim.x) {
        const RaggedSeq s = ragged_seq(rag, b, nullptr);
        cost[b] = s.row0 < 0 ? -1 : head_cost(s.n, s.len) * kNumKvHeads;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int live;
        const int64_t total = ragged_total(cost, rag.batch, live);
        const int64_t begin = total * pair / pairs, end = total * (pair + 1) / pairs;
        Units u = {};
        u.seq = -1;
        if (end > begin) {
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
                    u.seq = b0 + src;
                    before += __shfl_sync(0xffffffffu, incl - c, src);
                    break;
                }
                before += __shfl_sync(0xffffffffu, incl, 31);
            }
            units_seq(rag, u);
            const int64_t per = cost[u.seq] / kNumKvHeads;
            u.kvh = (int)((begin - before) / per);
            int64_t at = before + u.kvh * per;  // the unit's first query tile
            // tiles that all rows see have equal costs; then step
            const int qn = (u.n + kTileTok - 1) / kTileTok;
            const int full = u.len >= u.n ? (u.len - u.n) / kUnitKeys + 1 : 0;
            u.kt = (int)min((int64_t)full, (begin - at) / qn);
            at += (int64_t)u.kt * qn;
            units_set(u);
            while (at + (u.q1 - u.q0) <= begin) {
                at += u.q1 - u.q0;
                ++u.kt;
                units_set(u);
            }
            u.pos = at;
            u.end = end;
            // a unit that began in the share before this one is that share's
            if (at < begin && !units_next(rag, u)) u.seq = -1;
        }
        if (lane == 0) *out = u;
    }
    __syncthreads();
    return out->seq >= 0;
}

struct Smem {
    static constexpr int kK = 0;
    static constexpr int kQ = kK + kKSlots * kKBytes;
    static constexpr int kLse = kQ + kQSlots * kQBytes;  // [groups][2][128] fp32, log2 units
    static constexpr int kSum = kLse + kBufs * 2 * kCols * 4;  // [2][groups][128 keys] fp32
    static constexpr int kBar = kSum + 2 * kBufs * 128 * 4;
    // leader: k_full[2], q_full[10], d_empty[4]; each: k_empty[2], q_empty[10], d_full[4]
    static constexpr int kNumBars = 2 * (kKSlots + kQSlots + kBufs);
    static constexpr int kUnits = kBar + kNumBars * 8;
    static constexpr int kTmemSlot = kUnits + 56;
    static constexpr int kAbort = kTmemSlot + 8;
    static constexpr int kBytes = kAbort + 8;
};
static_assert(sizeof(Units) <= 56 && Smem::kUnits % 8 == 0, "units slot");
static_assert(kBufs * kCols <= (int)kTmemCols, "products");
static_assert(Smem::kBytes <= 232448, "weights kernel shared memory exceeds the sm_100 limit");
static_assert(PGC_CHUNK_MAX_BATCH * 8 <= kKSlots * kKBytes, "the schedule's scratch is the K buffers");

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    chunk_weights_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                         const WeightsParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_trigger();
    pdl_wait();
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    if ((smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) record_error(&g_cweights_err, kErrSmemAlign, 0);
        return;
    }
    uint64_t *k_full = reinterpret_cast<uint64_t *>(smem + Smem::kBar);  // leader: both CTAs' keys
    uint64_t *q_full = k_full + kKSlots;   // leader: both CTAs' query blocks
    uint64_t *d_empty = q_full + kQSlots;  // leader: both CTAs' sum warps have read the product
    uint64_t *k_empty = d_empty + kBufs;
    uint64_t *q_empty = k_empty + kKSlots;
    uint64_t *d_full = q_empty + kQSlots;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + Smem::kTmemSlot);
    Units *share = reinterpret_cast<Units *>(smem + Smem::kUnits);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + Smem::kAbort);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    if (!find_units(p.rag, reinterpret_cast<int64_t *>(smem + Smem::kK), blockIdx.x >> 1, gridDim.x >> 1, share))
        return;  // both CTAs of the pair
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kKSlots; ++s) {
            mbar_init(&k_full[s], 2 * kLoadWarps);
            mbar_init(&k_empty[s], 1);
        }
        for (int s = 0; s < kQSlots; ++s) {
            mbar_init(&q_full[s], 2);
            mbar_init(&q_empty[s], 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&d_full[b], 1);
            mbar_init(&d_empty[b], 8);  // a group of each CTA
        }
        fence_mbar_init();
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    fence_proxy_async_smem();  // the schedule's scratch becomes the K buffers
    tc_fence_before();
    cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    auto leader_addr = [&](uint64_t *bar) { return cluster_map(smem_u32(bar), 0); };
    auto wait = [&](uint64_t *bar, uint32_t parity, int where) {
        return wait_or_abort(bar, parity, abort_flag, &g_cweights_err, where);
    };
    Units u = *share;

    if (warp > kSumWarps) {
        // ------------------------------------------------------------ TMA: keys and query rows
        // Warp lw loads 4 of this CTA's 8 pages of each unit's keys and every second 64-dim block of the
        // query rows. The next unit's keys go out behind the first tiles of this unit: their buffer is
        // free when the unit before this one is done.
        const int lw = warp - kSumWarps - 1;
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_first();
            tma_prefetch_desc(lw == 0 ? &tmk : &tmq);
            auto load_keys = [&](const Units &v, int un) -> bool {
                const int sl = un % kKSlots;
                if (un >= kKSlots && !wait(&k_empty[sl], ((un / kKSlots) - 1) & 1, 1)) return false;
                const int key0 = v.kt * kUnitKeys + (int)rank * 128;
                int npg = 0;
                for (int pp = 4 * lw; pp < 4 * lw + 4; ++pp)
                    if (key0 + pp * kPage < v.len) ++npg;
                const uint32_t kbar = leader_addr(&k_full[sl]);
                mbar_arrive_expect_tx_cluster(kbar, (uint32_t)npg * 4 * 2048);
                uint8_t *dst = smem + Smem::kK + sl * kKBytes;
                for (int pp = 4 * lw; pp < 4 * lw + npg; ++pp) {
                    int page = p.block_tables[(int64_t)v.seq * p.max_pages_per_seq + (key0 >> 4) + pp];
                    if (page < 0 || page >= p.num_pages) {
                        record_error(&g_cweights_err, kErrPageOutOfRange, page);
                        page = 0;
                    }
                    const int row = (page * kNumKvHeads + v.kvh) * kPage;
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        tma_load_2d_pair(dst + c * (128 * 128) + pp * 2048, &tmk, c * 64, row, kbar, pol);
                }
                return true;
            };
            constexpr int kLead = 2;  // tiles of a unit that go out before the next unit's keys
            int g = lw;               // this warp's query blocks: g, g + 2, ...
            bool ok = load_keys(u, 0);
            for (int un = 0; ok; ++un) {
                Units nu = u;
                const bool more = units_next(p.rag, nu);
                for (int qt = u.q0; ok && qt < u.q1; ++qt) {
                    if (qt == u.q0 + kLead && more) ok = load_keys(nu, un + 1);
                    const int tok = u.row0 + qt * kTileTok + (int)rank * (kTileTok / 2);
                    for (int c = lw; ok && c < 4; c += 2, g += 2) {
                        const int sl = g % kQSlots;
                        if (g >= kQSlots && !wait(&q_empty[sl], ((g / kQSlots) - 1) & 1, 2)) {
                            ok = false;
                            break;
                        }
                        const uint32_t qbar = leader_addr(&q_full[sl]);
                        mbar_arrive_expect_tx_cluster(qbar, kQBytes);
                        tma_load_3d_pair(smem + Smem::kQ + sl * kQBytes, &tmq, c * 64, u.kvh * kGroup, tok, qbar);
                    }
                }
                if (!ok || !more) break;
                if (u.q1 - u.q0 <= kLead) ok = load_keys(nu, un + 1);
                u = nu;
            }
        }
    } else if (warp == kSumWarps) {
        // ------------------------------------------------------------ MMA issuer (leader)
        if (leader) {  // the whole warp, of which one lane acts (umma2_ss_elected)
            const uint32_t me = elect_one();
            constexpr uint32_t idesc = umma_idesc(256, kCols, false, false);
            const uint64_t k_desc = umma_desc(smem_u32(smem + Smem::kK), 16, 1024);
            const uint64_t q_desc = umma_desc(smem_u32(smem + Smem::kQ), 16, 1024);
            int g = 0, tile = 0;
            bool ok = true;
            for (int un = 0; ok; ++un) {
                const int ks = un % kKSlots;
                if (!wait(&k_full[ks], (un / kKSlots) & 1, 3)) break;
                const uint64_t kd = k_desc + (uint32_t)(ks * (kKBytes >> 4));
                for (int qt = u.q0; ok && qt < u.q1; ++qt, ++tile) {
                    const int b = tile % kBufs;
                    if (tile >= kBufs && !wait_or_abort_cluster(&d_empty[b], ((tile / kBufs) - 1) & 1, abort_flag,
                                                                &g_cweights_err, 4)) {
                        ok = false;
                        break;
                    }
                    for (int c = 0; c < 4; ++c, ++g) {
                        const int sl = g % kQSlots;
                        if (!wait(&q_full[sl], (g / kQSlots) & 1, 5)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint64_t qd = q_desc + (uint32_t)(sl * (kQBytes >> 4));
#pragma unroll
                        for (int kk = 0; kk < 4; ++kk)
                            umma2_ss_elected(me, tmem + b * kCols, kd + ((c * (128 * 128) + kk * 32) >> 4), qd + ((kk * 32) >> 4),
                                             idesc, (c > 0 || kk > 0) ? 1u : 0u);
                        umma2_commit_pair_elected(me, &q_empty[sl]);
                    }
                    if (ok) umma2_commit_pair_elected(me, &d_full[b]);
                }
                if (!ok) break;
                umma2_commit_pair_elected(me, &k_empty[ks]);
                if (!units_next(p.rag, u)) break;
            }
        }
    } else {
        // ------------------------------------------------------------ exponentials and their sums
        // Group `grp` takes the products of its buffer, every fourth tile; its warp qd the keys
        // 32 qd + lane of this CTA. A wait that gives up does not take a warp out of step with the named
        // barriers (see chunk_attn.cu).
        const int grp = warp >> 2, qd = warp & 3;
        const int gtid = threadIdx.x & 127;
        const uint32_t src = tmem + ((uint32_t)(qd * 32) << 16) + grp * kCols;
        float *lse_s = reinterpret_cast<float *>(smem + Smem::kLse) + grp * 2 * kCols;
        float *sum_s = reinterpret_cast<float *>(smem + Smem::kSum);
        const uint32_t ebar = leader_addr(&d_empty[grp]);
        const float c = p.scale_log2;
        // Column gtid's lse in log2 units; +inf, with which it adds nothing, for the rows that are not the
        // sequence's too.
        auto load_lse = [&](int qt) -> float {
            const int tok = qt * kTileTok + gtid / kGroup;
            if (tok >= u.n) return INFINITY;
            return p.lse2[(int64_t)(u.row0 + tok) * kNumQHeads + u.kvh * kGroup + gtid % kGroup];
        };
        int tile = 0, slot_seq = -1;  // tile: the share's tiles before this unit
        int64_t slot = -1;
        for (int un = 0;; ++un) {
            if (u.seq != slot_seq) {
                slot_seq = u.seq;
                slot = ragged_slot(p.w.slots, p.w.num_slots, u.seq, &g_cweights_err);
            }
            const int key = u.kt * kUnitKeys + (int)rank * 128 + qd * 32 + lane;
            const int P = u.len - u.n;
            float2 sum2 = make_float2(0.f, 0.f);
            const int first = u.q0 + ((grp - tile) & (kBufs - 1));  // this group's first tile of the unit
            int buf = 0;
            if (first < u.q1) {
                lse_s[gtid] = load_lse(first);
                asm volatile("bar.sync %0, 128;" ::"r"(2 + grp) : "memory");
            }
            for (int qt = first; qt < u.q1; qt += kBufs) {
                const int g = tile + qt - u.q0;  // of the share
                // the group's next tile's lse, in flight while this one is summed
                const float next = qt + kBufs < u.q1 ? load_lse(qt + kBufs) : 0.f;
                wait(&d_full[grp], (g / kBufs) & 1, 6);
                tc_fence_after();
                const float *ls = lse_s + buf * kCols;
                const int hi = min(kTileTok, u.n - qt * kTileTok) * kGroup;  // the sequence's columns
                const int lo = (key - P - qt * kTileTok) * kGroup;           // the first that sees this key
                const int lo_warp = (key - lane + 31 - P - qt * kTileTok) * kGroup;
                float sv[2][32];  // the next 32 columns are read while these are summed
                tmem_ld32(src, sv[0]);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < kCols / 32; ++k) {
                    const int col = k * 32;
                    if (col >= hi) break;
                    if (k + 1 < kCols / 32) tmem_ld32(src + col + 32, sv[(k + 1) & 1]);
                    float(&v)[32] = sv[k & 1];
                    if (lo_warp <= col && col + 32 <= hi) {
#pragma unroll
                        for (int i = 0; i < 32; i += 4) {
                            const float4 l4 = *reinterpret_cast<const float4 *>(ls + col + i);
                            const float2 x = __ffma2_rn(make_float2(v[i], v[i + 1]), make_float2(c, c), make_float2(-l4.x, -l4.y));
                            const float2 y = __ffma2_rn(make_float2(v[i + 2], v[i + 3]), make_float2(c, c), make_float2(-l4.z, -l4.w));
                            sum2 = __fadd2_rn(sum2, make_float2(fast_exp2(x.x), fast_exp2(x.y)));
                            sum2 = __fadd2_rn(sum2, make_float2(fast_exp2(y.x), fast_exp2(y.y)));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            const float e = fast_exp2(v[i] * c - ls[col + i]);
                            if (col + i >= lo && col + i < hi) sum2.x += e;
                        }
                    }
                    tmem_wait_ld();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(ebar);
                buf ^= 1;
                if (qt + kBufs < u.q1) {
                    // one barrier a tile: a buffer is written again two tiles on, when all have read it
                    lse_s[buf * kCols + gtid] = next;
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + grp) : "memory");
                }
            }
            // Join: double-buffered by unit, so one barrier also keeps the next writes off these reads
            // and the next unit's lse off this one's.
            float *mine = sum_s + (un & 1) * kBufs * 128;
            mine[grp * 128 + qd * 32 + lane] = sum2.x + sum2.y;
            asm volatile("bar.sync 1, %0;" ::"r"(kSumWarps * 32) : "memory");
            if (warp < 4 && slot >= 0 && key < u.len) {
                const int k = qd * 32 + lane;
                p.w.weights[(slot * kNumKvHeads + u.kvh) * p.w.stride + key] +=
                    (mine[k] + mine[128 + k]) + (mine[256 + k] + mine[384 + k]);
            }
            tile += u.q1 - u.q0;
            if (!units_next(p.rag, u)) break;
        }
    }
    tc_fence_before();
    cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
    }
}

}  // namespace

cudaError_t launch_chunk_weights(const uint16_t *q, const CUtensorMap &tk, int64_t num_pages,
                                 const int32_t *block_tables, int max_pages_per_seq, const RaggedBatch &rag,
                                 float scale, const float *lse2, const ChunkWeights &weights, int sm_count,
                                 cudaStream_t stream) {
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(chunk_weights_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             Smem::kBytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    CUtensorMap tq;
    if (q_tensor_map(q, rag.total_q, &tq, kTileTok / 2) != PGC_OK) return cudaErrorInvalidValue;
    WeightsParams wp = {};
    wp.rag = rag;
    wp.block_tables = block_tables;
    wp.max_pages_per_seq = max_pages_per_seq;
    wp.num_pages = num_pages;
    wp.lse2 = lse2;
    wp.w = weights;
    wp.scale_log2 = scale * kLog2e;
    return launch_pdl(chunk_weights_kernel, dim3(sm_count / 2 * 2), dim3(kThreads), Smem::kBytes, stream, tq, tk, wp);
}

cudaError_t chunk_weights_read_error(DevErrorHost *e, bool clear) {
    cudaError_t r = cudaMemcpyFromSymbol(e, g_cweights_err, sizeof(DevError));
    if (r != cudaSuccess || !clear) return r;
    DevErrorHost z = {0, 0, 0};
    return cudaMemcpyToSymbol(g_cweights_err, &z, sizeof(DevError));
}

}  // namespace pgc
