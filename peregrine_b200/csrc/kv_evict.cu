// kv_evict.cu — eviction from the paged cache by received attention (sm_100a): which tokens of each
// (sequence, kv head) stay, and the gather of their K/V rows into fresh pages.
//
// Selection. A sequence of L tokens with budget B keeps all of them if L <= B; otherwise its first F
// and last R tokens and, of those between, the B - F - R with the greatest weights, equal weights
// going to the lowest index (a NaN weight counts as the smallest). The kept indices are written in
// ascending order and the weights follow them, so that the accumulation goes on over the shorter
// cache. Keys were rotated by their positions when they were appended, so the kept rows need no
// change, and as the pools hold every kv head's rows apart, each kv head keeps tokens of its own.
#include "pgc_common.cuh"
#include "pgc_internal.h"
#include "pgc_ragged.cuh"

namespace pgc {

PGC_DEFINE_ERROR_WORD(g_evict_err);

namespace {

// ---------------------------------------------------------------- selection
// A cluster of 1-8 CTAs per (sequence, kv head); a row that fewer can hold uses fewer. Each warp holds a
// segment of the row in registers, as order-preserving integers, all but the first F and the last R
// tokens, which are kept anyway. The least value kept among the others is searched for in a range that
// shrinks: a histogram over 256 equal parts of it, summed over the cluster through distributed shared
// memory, says which part holds the value. The first range is the non-negative floats (a part is an
// octave). When few values are left in the range, they are listed and ranked against one another; when
// all that are left are kept, the search is over. Then the warps count what they keep, the counts are
// scanned over warps and CTAs, and the tokens are written in order.
// The histogram has a column per lane: lane l adds to hist[part][l], its own bank, so a warp's adds
// never meet however the weights cluster (attention weights share a few exponents; with one shared
// column those adds ran one after the other: 519 us for 64 sequences of up to 65536 tokens).
// Measured: 43 us for those 64 sequences (48 MB, 8 us at the copy rate), 7.0 us for one of 4097, 21.6 us
// for one of 262144. What bounds it are the instructions issued and the ends of the phases: a CTA takes 20
// to 30 thousand cycles, two histograms and the list half of them, a third of that at barriers.
constexpr int kBins = 256;
constexpr int kMaxPer = 32;  // weights a thread
constexpr int kListed = 256;  // values that are ranked against one another
static_assert(8 * 1024 * kMaxPer >= PGC_EVICT_MAX_TOKENS, "the longest row does not fit a cluster");

struct SelectParams {
    const float *weights;
    float *weights_out;  // nullable; may be `weights`
    int64_t stride, num_slots;
    const int32_t *slots;
    const int32_t *seq_lens;
    int max_seq_len;
    int budget, keep_first, keep_last;
    int share;  // weights a CTA takes before another one of its cluster joins in
    int32_t *kept;
    int32_t *new_lens;
};

// A weight as it is held and moved: -0 as +0, every NaN as the one whose order bits are 1.
__device__ __forceinline__ float canonical(float x) { return x == x ? x + 0.f : __uint_as_float(0xfffffffeu); }
// Unsigned integers in the order of the canonical floats, NaN below everything, 0 for none.
__device__ __forceinline__ uint32_t order_bits(float x) {
    const int32_t u = __float_as_int(x);
    return (uint32_t)u ^ ((uint32_t)(u >> 31) | 0x80000000u);
}

__device__ __forceinline__ uint32_t ctas_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cta_in_cluster() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctaid.x;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A word of CTA `cta`'s shared memory at this CTA's address of it.
__device__ __forceinline__ uint32_t load_peer(const void *p, uint32_t cta) {
    uint32_t a, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(cta));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

template <int kSelThreads, int kPer>  // kPer: weights a thread, at most
__global__ void __launch_bounds__(kSelThreads, 1024 / kSelThreads) evict_select_kernel(const SelectParams p) {
    constexpr int kSelWarps = kSelThreads / 32, kPartThreads = kSelThreads / kBins;
    extern __shared__ __align__(16) uint32_t dyn[];
    uint32_t *hist = dyn;                                       // [256][32 lanes]
    float *vals = reinterpret_cast<float *>(dyn + kBins * 32);  // this CTA's share of the weights
    __shared__ uint32_t totals[2][kBins];  // this CTA's histogram, read by the cluster
    __shared__ uint32_t warp_sum[kSelWarps];
    __shared__ uint32_t found[3];  // the part, the values above it and of it
    __shared__ uint32_t cnt[2];    // values above the ties in this CTA, and ties
    __shared__ uint32_t seg_sure[kSelWarps], seg_tie[kSelWarps];
    __shared__ uint32_t listed, list[kListed];  // this CTA's values of the last range, read by the cluster
    __shared__ uint32_t all[kListed];           // the cluster's
    pdl_trigger();
    pdl_wait();
    const uint32_t rank = cta_in_cluster(), cluster = ctas_in_cluster();
    const int h = blockIdx.y, b = blockIdx.z;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const bool reporter = h == 0 && rank == 0;
    int32_t *kept = p.kept + ((int64_t)b * kNumKvHeads + h) * p.budget;

    int L = p.seq_lens[b];
    if (L < 0 || L > p.max_seq_len) {
        if (reporter && tid == 0) record_error(&g_evict_err, kErrLenOutOfRange, b);
        L = 0;
    }
    const int64_t slot = ragged_slot(p.slots, p.num_slots, b, reporter ? &g_evict_err : nullptr);
    if (slot < 0) L = 0;
    const int B = p.budget;
    const int n_new = min(L, B);
    if (reporter && tid == 0 && p.new_lens != nullptr) p.new_lens[b] = n_new;
    for (int i = n_new + (int)rank * kSelThreads + tid; i < B; i += (int)cluster * kSelThreads) kept[i] = -1;
    const int64_t row = (max(slot, (int64_t)0) * kNumKvHeads + h) * p.stride;
    const float *w = p.weights + row;
    float *wo = p.weights_out != nullptr ? p.weights_out + row : nullptr;
    if (L <= B) {  // uniform over the cluster
        for (int i = (int)rank * kSelThreads + tid; i < L; i += (int)cluster * kSelThreads) {
            kept[i] = i;
            if (wo != nullptr && wo != w) wo[i] = w[i];
        }
        return;
    }

    // the CTAs that this row uses; the cluster's barriers do not wait for those that have left
    const uint32_t ctas = (uint32_t)min((int)cluster, (L + p.share - 1) / p.share);
    if (rank >= ctas) return;
    auto sync_all = [&]() {
        if (ctas > 1)
            cluster_sync();
        else
            __syncthreads();
    };

    // warp segments of `per` x 32 consecutive weights; element j of a lane is number j * 32 + lane.
    // `per` is a multiple of 4, so that the loops below test it once per 4 elements.
    const int per = (int)(((int64_t)L + (int64_t)ctas * kSelThreads * 4 - 1) / ((int64_t)ctas * kSelThreads * 4)) * 4;
    const int i0 = warp * per * 32 + lane;        // in the CTA's share
    const int t0 = (int)rank * per * kSelThreads;  // the share's first token
    const int F = p.keep_first, last = L - p.keep_last;
    uint32_t key[kPer];
#define PGC_EACH_KEY \
    _Pragma("unroll") for (int j4 = 0; j4 < kPer; j4 += 4) if (j4 < per) _Pragma("unroll") for (int j = j4; j < j4 + 4; ++j)
    PGC_EACH_KEY {
        const int t = t0 + i0 + j * 32;
        key[j] = t < L ? __float_as_uint(w[t]) : 0;
    }
#pragma unroll
    for (int i = 0; i < kBins * 32 / kSelThreads; ++i) hist[i * kSelThreads + tid] = 0;
    if (tid == 0) listed = 0;
    PGC_EACH_KEY {
        const int t = t0 + i0 + j * 32;
        const float x = canonical(__uint_as_float(key[j]));
        if (wo != nullptr) vals[i0 + j * 32] = x;
        key[j] = (uint32_t)(t - F) < (uint32_t)(last - F) ? order_bits(x) : 0u;
    }
    __syncthreads();

    // The value sought is in [lo, lo + width]: what lies above is kept, and `need` of the `ties` inside,
    // the first in order. With need = 0 the search ends at once, with everything above.
    const uint32_t hist_lane = smem_u32(hist) + lane * 4;
    uint32_t need = (uint32_t)(B - F - p.keep_last), lo = 0x80000000u, width = 0x7fffffffu, ties = ~0u;
    if (need == 0) {
        lo = ~0u;  // no key is as great
        width = 0;
        ties = 0;
    }
#pragma unroll 1
    for (uint32_t buf = 0; ties != need && width != 0; buf ^= 1) {
        if (ties <= (uint32_t)kListed) {
            PGC_EACH_KEY {
                if (key[j] - lo <= width) list[atomicAdd(&listed, 1u)] = key[j] - lo;
            }
            sync_all();
            uint32_t v = 0;
            if (tid < (int)ties) {
                uint32_t q = 0, at = (uint32_t)tid, n = load_peer(&listed, 0);
                while (at >= n) {  // the CTAs' lists have `ties` values between them
                    at -= n;
                    n = load_peer(&listed, ++q);
                }
                v = load_peer(&list[at], q);
                all[tid] = v;
            }
            __syncthreads();
            if (tid < (int)ties) {
                uint32_t above = 0, same = 0;
                for (uint32_t i = 0; i < ties; ++i) {
                    const uint32_t x = all[i];
                    above += x > v;
                    same += x == v;
                }
                if (above < need && above + same >= need) {
                    found[0] = v;
                    found[1] = above;
                    found[2] = same;
                }
            }
            __syncthreads();
            need -= found[1];
            ties = found[2];
            lo += found[0];
            width = 0;
            break;
        }
        const int sh = max(0, 24 - __clz((int)width));
        // predicated adds: a branch around each costs more than the add
        PGC_EACH_KEY {
            asm volatile(
                "{\n\t.reg .pred in;\n\t"
                "setp.le.u32 in, %0, %1;\n\t"
                "@in red.shared.add.u32 [%2], 1;\n\t}"
                ::"r"(key[j] - lo), "r"(width), "r"(hist_lane + ((key[j] - lo) >> sh) * 128)
                : "memory");
        }
        __syncthreads();
        // kPartThreads threads sum a part's columns and clear them for the next round, 16 bytes at a
        // time, each part from another bank group on; the parts go down as the threads go up
        const int part = kBins - 1 - tid / kPartThreads, sub = tid % kPartThreads;
        uint32_t c = 0;
#pragma unroll
        for (int k = 0; k < 8 / kPartThreads; ++k) {
            uint4 *q = reinterpret_cast<uint4 *>(hist + part * 32) + ((sub * (8 / kPartThreads) + k + part) & 7);
            const uint4 x = *q;
            *q = make_uint4(0, 0, 0, 0);
            c += (x.x + x.y) + (x.z + x.w);
        }
        auto part_sum = [](uint32_t x) {
#pragma unroll
            for (int o = 1; o < kPartThreads; o *= 2) x += __shfl_xor_sync(0xffffffffu, x, o);
            return x;
        };
        c = part_sum(c);
        if (ctas > 1) {
            // totals are double-buffered: a peer's reads of a round are over when this CTA writes that
            // buffer again
            if (sub == 0) totals[buf][part] = c;
            cluster_sync();
            c = 0;
#pragma unroll
            for (uint32_t k = 0; k < 8 / kPartThreads; ++k) {
                const uint32_t q = sub + k * kPartThreads;
                if (q < ctas) c += load_peer(&totals[buf][part], q);
            }
            c = part_sum(c);
        }
        // the sum of a part and those above it
        uint32_t incl = sub == 0 ? c : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        incl += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sum[lane] : 0);
        if (sub == 0) {
            if (incl - c < need && incl >= need) {
                found[0] = (uint32_t)part;
                found[1] = incl - c;
                found[2] = c;
            }
            // the first range only: too few there, the value is below it
            if (part == 0 && incl < need) {
                found[1] = incl;
                found[2] = 0;
            }
        }
        __syncthreads();
        need -= found[1];
        if (found[2] == 0) {  // the negative floats and NaN
            lo = 1;
            width = 0x7ffffffeu;
            ties = ~0u;
        } else {
            ties = found[2];
            lo += found[0] << sh;
            width = min(width - (found[0] << sh), (1u << sh) - 1);
        }
    }

    const bool all_ties = ties == need;  // everything from lo on is kept
    uint32_t n_sure = 0, n_tie = 0;
    if (all_ties) {
        PGC_EACH_KEY n_sure += key[j] >= lo;
    } else {
        PGC_EACH_KEY {
            n_tie += key[j] - lo <= width;
            n_sure += key[j] > lo + width;
        }
        n_tie = __reduce_add_sync(0xffffffffu, n_tie);
    }
    n_sure = __reduce_add_sync(0xffffffffu, n_sure);
    if (lane == 0) {
        seg_sure[warp] = n_sure;
        seg_tie[warp] = n_tie;
    }
    __syncthreads();
    const uint32_t ws = lane < kSelWarps ? seg_sure[lane] : 0, wt = lane < kSelWarps ? seg_tie[lane] : 0;
    uint32_t sure_before = __reduce_add_sync(0xffffffffu, lane < warp ? ws : 0);
    uint32_t tie_before = __reduce_add_sync(0xffffffffu, lane < warp ? wt : 0);
    if (warp == 0) {
        const uint32_t s = __reduce_add_sync(0xffffffffu, ws), e = __reduce_add_sync(0xffffffffu, wt);
        if (lane == 0) {
            cnt[0] = s;
            cnt[1] = e;
        }
    }
    // from here on every CTA has read its weights: writing in place is safe
    sync_all();
    {
        const uint32_t s = lane < (int)rank ? load_peer(&cnt[0], lane) : 0;
        const uint32_t e = lane < (int)rank ? load_peer(&cnt[1], lane) : 0;
        sure_before += __reduce_add_sync(0xffffffffu, s);
        tie_before += __reduce_add_sync(0xffffffffu, e);
    }
    const uint32_t lt = (1u << lane) - 1;
    sure_before += (uint32_t)F;
    if (all_ties) {
        uint32_t at = sure_before;
        PGC_EACH_KEY {
            const bool keep = key[j] >= lo;
            const uint32_t m = __ballot_sync(0xffffffffu, keep);
            if (keep) {
                const uint32_t o = at + __popc(m & lt);
                kept[o] = t0 + i0 + j * 32;
                if (wo != nullptr) wo[o] = vals[i0 + j * 32];
            }
            at += __popc(m);
        }
    } else {
        PGC_EACH_KEY {
            const bool sure = key[j] > lo + width, tie = key[j] - lo <= width;
            const uint32_t ms = __ballot_sync(0xffffffffu, sure), mt = __ballot_sync(0xffffffffu, tie);
            const uint32_t rank_t = tie_before + __popc(mt & lt);
            if (sure || (tie && rank_t < need)) {
                const uint32_t o = sure_before + __popc(ms & lt) + min(rank_t, need);
                kept[o] = t0 + i0 + j * 32;
                if (wo != nullptr) wo[o] = vals[i0 + j * 32];
            }
            sure_before += __popc(ms);
            tie_before += __popc(mt);
        }
    }
#undef PGC_EACH_KEY
    // the first and the last tokens of this CTA's share
    const int t1 = min(L, t0 + per * kSelThreads);
    for (int t = t0 + tid; t < min(t1, F); t += kSelThreads) {
        kept[t] = t;
        if (wo != nullptr) wo[t] = vals[t - t0];
    }
    for (int t = max(t0, last) + tid; t < t1; t += kSelThreads) {
        kept[B - L + t] = t;
        if (wo != nullptr) wo[B - L + t] = vals[t - t0];
    }
    if (wo != nullptr)
        for (int i = B + (int)rank * kSelThreads + tid; i < L; i += (int)ctas * kSelThreads) wo[i] = 0.f;
    if (ctas > 1) cluster_sync();  // a peer may still read this CTA's counts
}

// ---------------------------------------------------------------- compaction
// A warp per `rows` consecutive kept tokens of a (sequence, kv head): the lanes look the pages up,
// then each row of K and of V is one 16-byte load and store a lane, 4 rows of both in flight. Bound by the
// bytes, 2 KiB a kept row: 32 sequences cut to 4096 tokens, 1.03 GB, take 161 us (6.4 TB/s, 98 % of a
// plain copy); 1024 rows of one sequence 3.6 us.
struct CompactParams {
    const uint4 *k_src, *v_src;
    uint4 *k_dst, *v_dst;
    int64_t src_pages, dst_pages;
    const int32_t *src_tables, *dst_tables;
    int src_max_pages, dst_max_pages;
    const int32_t *kept;
    int budget, batch;
    int rows;  // <= 32, a multiple of 4
};

__global__ void __launch_bounds__(256) evict_compact_kernel(const CompactParams p) {
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31;
    const int chunks = (p.budget + p.rows - 1) / p.rows;
    const int64_t job = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (job >= (int64_t)p.batch * kNumKvHeads * chunks) return;
    const int i0 = (int)(job % chunks) * p.rows;
    const int h = (int)(job / chunks % kNumKvHeads);
    const int b = (int)(job / chunks / kNumKvHeads);
    // lane i: source and destination rows of kept token i0 + i, in 512-byte rows; -1: none
    int64_t src = -1, dst = -1;
    const int i = i0 + lane;
    if (lane < p.rows && i < p.budget) {
        const int t = p.kept[((int64_t)b * kNumKvHeads + h) * p.budget + i];
        if (t >= 0) {
            const int to = p.dst_tables[(int64_t)b * p.dst_max_pages + i / kPage];
            if (t >= (int64_t)p.src_max_pages * kPage) {
                record_error(&g_evict_err, kErrTableOutOfRange, t);
            } else {
                const int from = p.src_tables[(int64_t)b * p.src_max_pages + t / kPage];
                if (from < 0 || from >= p.src_pages)
                    record_error(&g_evict_err, kErrPageOutOfRange, from);
                else if (to < 0 || to >= p.dst_pages)
                    record_error(&g_evict_err, kErrPageOutOfRange, to);
                else {
                    src = ((int64_t)from * kNumKvHeads + h) * kPage + t % kPage;
                    dst = ((int64_t)to * kNumKvHeads + h) * kPage + i % kPage;
                }
            }
        }
    }
    constexpr int kUnits = kHeadDim * 2 / 16;  // 16-byte units of a row: one a lane
    static_assert(kUnits == 32, "a row is one 16-byte unit a lane");
    for (int r = 0; r < p.rows; r += 4) {
        uint4 k[4], v[4];
        int64_t d[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t s = __shfl_sync(0xffffffffu, src, r + j);
            d[j] = __shfl_sync(0xffffffffu, dst, r + j);
            if (s >= 0) {
                k[j] = p.k_src[s * kUnits + lane];
                v[j] = p.v_src[s * kUnits + lane];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (d[j] >= 0) {
                p.k_dst[d[j] * kUnits + lane] = k[j];
                p.v_dst[d[j] * kUnits + lane] = v[j];
            }
        }
    }
}

}  // namespace

cudaError_t launch_evict_select(const float *weights, float *weights_out, int64_t stride, int64_t num_slots,
                                const int32_t *slots, const int32_t *seq_lens, int batch, int max_seq_len,
                                int budget, int keep_first, int keep_last, int32_t *kept, int32_t *new_lens,
                                cudaStream_t stream) {
    SelectParams p = {};
    p.weights = weights;
    p.weights_out = weights_out;
    p.stride = stride;
    p.num_slots = num_slots;
    p.slots = slots;
    p.seq_lens = seq_lens;
    p.max_seq_len = max_seq_len;
    p.budget = budget;
    p.keep_first = keep_first;
    p.keep_last = keep_last;
    p.kept = kept;
    p.new_lens = new_lens;
    // Threads and CTAs per row: at least what keeps a thread within kMaxPer weights, 512 threads a CTA (two
    // CTAs an SM: 43.0 us against 45.4 with 1024 for 64 rows of up to 65536, 28 against 50 for 800 rows of
    // up to 8192) except above kLongRow tokens, which only 1024 hold; a batch that leaves SMs free takes
    // more CTAs, up to 8, down to kSplitPer weights a thread, below which the cluster's barriers cost more
    // than they save (8, 12, 16 a thread, us: one sequence of 4097 8.1, 7.0, 7.0, of 16000 8.9, 8.8, 10.2, of
    // 32000 10.0, 10.0, 10.9; 16 of 6000 10.1, 8.0, 8.2). Clusters of 16 CTAs took 20 us instead of 21.6 for one sequence of 262144, but 62.7
    // instead of 60.5 for eight and 12.9 instead of 11.3 for one of 65536. A CTA a row that reads it from
    // L2 in every round took 51 us for one sequence of 262144 and 146 us for the 64 rows.
    constexpr int kSplitPer = 12, kLongRow = 8 * 512 * kMaxPer;
    int sms = 148, dev = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const int threads = max_seq_len > kLongRow ? 1024 : 512;
    auto weights_per_thread = [&](int c) { return (int)(((int64_t)max_seq_len + (int64_t)c * threads - 1) / ((int64_t)c * threads)); };
    int ctas = 1;
    while (ctas < 8 && (weights_per_thread(ctas) > kMaxPer ||
                        ((int64_t)batch * kNumKvHeads * ctas * 2 <= sms && weights_per_thread(ctas) > kSplitPer)))
        ctas *= 2;
    const int per = weights_per_thread(ctas);
    struct Variant {
        void (*kern)(const SelectParams);
        int threads, per;
    };
    const Variant variants[] = {{evict_select_kernel<512, 8>, 512, 8}, {evict_select_kernel<512, 16>, 512, 16},
                                {evict_select_kernel<512, 32>, 512, 32}, {evict_select_kernel<1024, 32>, 1024, 32}};
    const size_t hist_bytes = kBins * 32 * sizeof(uint32_t);
    static std::atomic<bool> attr_set[64] = {};
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        for (const Variant &v : variants) {
            cudaError_t e = cudaFuncSetAttribute(v.kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)(hist_bytes + v.threads * v.per * sizeof(float)));
            if (e != cudaSuccess) return e;
        }
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    const Variant &v = variants[threads == 1024 ? 3 : per <= 8 ? 0 : per <= 16 ? 1 : 2];
    // A row takes the fewest CTAs that hold it where the grid fills the device, so that the others leave
    // at once and make room; else as many as have kSplitPer weights a thread.
    const bool fills = (int64_t)batch * kNumKvHeads * ctas * threads > (int64_t)sms * 1024;
    p.share = threads * (fills ? v.per : std::min(v.per, kSplitPer));
    const int held = std::max((per + 3) / 4 * 4, p.share / threads);  // weights a thread, at most
    const size_t smem = hist_bytes + (weights_out != nullptr ? (size_t)held * threads * sizeof(float) : 0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, kNumKvHeads, batch);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[3];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[2].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[2].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    // the default policy left a third of the SMs idle where CTAs leave early: 51.4 us instead of 43.0 for 64
    // rows of up to 65536
    attr[1].id = cudaLaunchAttributeClusterSchedulingPolicyPreference;
    attr[1].val.clusterSchedulingPolicyPreference =
        fills ? cudaClusterSchedulingPolicyLoadBalancing : cudaClusterSchedulingPolicyDefault;
#ifndef PGC_NO_PDL
    cfg.numAttrs = 3;
#else
    cfg.numAttrs = 2;
#endif
    return cudaLaunchKernelEx(&cfg, v.kern, p);
}

cudaError_t launch_evict_compact(const uint16_t *k_src, const uint16_t *v_src, int64_t src_pages,
                                 const int32_t *src_tables, int src_max_pages, const int32_t *kept, int batch,
                                 int budget, uint16_t *k_dst, uint16_t *v_dst, int64_t dst_pages,
                                 const int32_t *dst_tables, int dst_max_pages, cudaStream_t stream) {
    CompactParams p = {};
    p.k_src = reinterpret_cast<const uint4 *>(k_src);
    p.v_src = reinterpret_cast<const uint4 *>(v_src);
    p.k_dst = reinterpret_cast<uint4 *>(k_dst);
    p.v_dst = reinterpret_cast<uint4 *>(v_dst);
    p.src_pages = src_pages;
    p.dst_pages = dst_pages;
    p.src_tables = src_tables;
    p.dst_tables = dst_tables;
    p.src_max_pages = src_max_pages;
    p.dst_max_pages = dst_max_pages;
    p.kept = kept;
    p.budget = budget;
    p.batch = batch;
    p.rows = 8;
    const int64_t jobs = (int64_t)batch * kNumKvHeads * ((budget + p.rows - 1) / p.rows);
    return launch_pdl(evict_compact_kernel, dim3((unsigned)((jobs + 7) / 8)), dim3(256), 0, stream, p);
}

cudaError_t evict_read_error(DevErrorHost *e, bool clear) {
    cudaError_t r = cudaMemcpyFromSymbol(e, g_evict_err, sizeof(DevError));
    if (r != cudaSuccess || !clear) return r;
    DevErrorHost z = {0, 0, 0};
    return cudaMemcpyToSymbol(g_evict_err, &z, sizeof(DevError));
}

}  // namespace pgc
