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
// A cluster of 1-8 CTAs per (sequence, kv head); each CTA keeps its consecutive share of the weights
// in shared memory, so they are read from HBM once. The weight of rank B - F - R is found from the
// top bits down: three histograms (11, 11 and 10 bits of the weight's bits in an order-preserving
// form) of the candidates that share the bits found so far, summed over the cluster through
// distributed shared memory. Then each warp counts its segment's kept tokens with ballots, the
// counts are scanned over warps and CTAs, and the tokens are written in order.
constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kBins = 2048;

struct SelectParams {
    const float *weights;
    float *weights_out;  // nullable; may be `weights`
    int64_t stride, num_slots;
    const int32_t *slots;
    const int32_t *seq_lens;
    int max_seq_len;
    int budget, keep_first, keep_last;
    int32_t *kept;
    int32_t *new_lens;
};

// Unsigned integers in the order of the floats, -0 and +0 alike, NaN below everything.
__device__ __forceinline__ uint32_t order_bits(float x) {
    if (x != x) return 0;
    const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
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

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const SelectParams p) {
    extern __shared__ float vals[];  // this CTA's share of the weights
    __shared__ uint32_t hist[2][kBins];
    __shared__ uint32_t warp_sum[kSelWarps];
    __shared__ uint32_t found[2];                // the bin and the candidates above it
    __shared__ uint32_t cnt[2];                  // this CTA's kept tokens apart from ties, and its ties
    __shared__ uint32_t seg_sure[kSelWarps], seg_tie[kSelWarps];
    pdl_trigger();
    pdl_wait();
    const uint32_t rank = cta_in_cluster(), ctas = ctas_in_cluster();
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
    for (int i = n_new + (int)rank * kSelThreads + tid; i < B; i += (int)ctas * kSelThreads) kept[i] = -1;
    const float *w = p.weights + (slot * kNumKvHeads + h) * p.stride;
    float *wo = p.weights_out + (slot * kNumKvHeads + h) * p.stride;
    if (L <= B) {  // uniform over the cluster
        for (int i = (int)rank * kSelThreads + tid; i < L; i += (int)ctas * kSelThreads) {
            kept[i] = i;
            if (p.weights_out != nullptr && p.weights_out != p.weights) wo[i] = w[i];
        }
        return;
    }

    // shares of whole warp segments
    const int seg = (int)(((int64_t)L + (int64_t)ctas * kSelThreads - 1) / ((int64_t)ctas * kSelThreads)) * 32;
    const int share = seg * kSelWarps;
    const int t0 = min(L, (int)rank * share), n = min(L, t0 + share) - t0;
#pragma unroll 4
    for (int i = tid; i < n; i += kSelThreads) vals[i] = w[t0 + i];
    for (int i = tid; i < 2 * kBins; i += kSelThreads) (&hist[0][0])[i] = 0;
    __syncthreads();

    const int lo = p.keep_first, hi = L - p.keep_last;  // candidates
    uint32_t need = (uint32_t)(B - p.keep_first - p.keep_last);
    uint32_t prefix = 0;  // bits found so far
    if (need > 0) {
        int known = 0;  // how many
#pragma unroll 1
        for (int pass = 0; pass < 3; ++pass) {
            const int bits = pass < 2 ? 11 : 10, shift = 32 - known - bits;
            uint32_t *hh = hist[pass & 1];
            for (int i = tid; i < n; i += kSelThreads) {
                const int t = t0 + i;
                const uint32_t k = order_bits(vals[i]);
                if (t >= lo && t < hi && (pass == 0 || (k >> (32 - known)) == prefix))
                    atomicAdd(&hh[(k >> shift) & ((1u << bits) - 1)], 1u);
            }
            cluster_sync();
            // Sum over the cluster, bins from the top: thread i holds bins top - 4 i .. - 3.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int bin = kBins - 1 - (tid * 4 + k);
                c[k] = 0;
                for (uint32_t q = 0; q < ctas; ++q) c[k] += q == rank ? hh[bin] : load_peer(&hh[bin], q);
                sum += c[k];
            }
            uint32_t incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            if (lane == 31) warp_sum[warp] = incl;
            // the other buffer is cleared for the next pass: its last readers were the pass before
            // this one's cluster barrier
            for (int i = tid; i < kBins; i += kSelThreads) hist[(pass & 1) ^ 1][i] = 0;
            __syncthreads();
            uint32_t above = incl - sum;
            for (int q = 0; q < warp; ++q) above += warp_sum[q];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (above < need && above + c[k] >= need) {
                    found[0] = (uint32_t)(kBins - 1 - (tid * 4 + k));
                    found[1] = above;
                }
                above += c[k];
            }
            __syncthreads();
            prefix = (prefix << bits) | found[0];
            need -= found[1];
            known += bits;
        }
    }
    // Kept: the first and last, candidates above `prefix`, and the first `need` equal to it.
    const bool middle = B > p.keep_first + p.keep_last;
    auto classify = [&](int i, bool &sure, bool &tie) {
        const int t = t0 + i;
        const bool in = i < n;
        const uint32_t k = in ? order_bits(vals[i]) : 0;
        const bool cand = in && t >= lo && t < hi;
        sure = in && (t < lo || t >= hi || (middle && k > prefix));
        tie = cand && middle && k == prefix;
    };
    uint32_t n_sure = 0, n_tie = 0;
    for (int s = 0; s < seg; s += 32) {
        bool sure, tie;
        classify(warp * seg + s + lane, sure, tie);
        n_sure += __popc(__ballot_sync(0xffffffffu, sure));
        n_tie += __popc(__ballot_sync(0xffffffffu, tie));
    }
    if (lane == 0) {
        seg_sure[warp] = n_sure;
        seg_tie[warp] = n_tie;
    }
    __syncthreads();
    if (tid == 0) {
        uint32_t s = 0, e = 0;
        for (int q = 0; q < kSelWarps; ++q) {
            s += seg_sure[q];
            e += seg_tie[q];
        }
        cnt[0] = s;
        cnt[1] = e;
    }
    cluster_sync();
    uint32_t sure_before = 0, tie_before = 0;
    for (uint32_t q = 0; q < rank; ++q) {
        sure_before += load_peer(&cnt[0], q);
        tie_before += load_peer(&cnt[1], q);
    }
    for (int q = 0; q < warp; ++q) {
        sure_before += seg_sure[q];
        tie_before += seg_tie[q];
    }
    const uint32_t lt = (1u << lane) - 1;
    for (int s = 0; s < seg; s += 32) {
        const int i = warp * seg + s + lane;
        bool sure, tie;
        classify(i, sure, tie);
        const uint32_t ms = __ballot_sync(0xffffffffu, sure), mt = __ballot_sync(0xffffffffu, tie);
        const uint32_t rank_t = tie_before + __popc(mt & lt);
        if (sure || (tie && rank_t < need)) {
            const uint32_t at = sure_before + __popc(ms & lt) + min(rank_t, need);
            kept[at] = t0 + i;
            if (p.weights_out != nullptr) wo[at] = vals[i];
        }
        sure_before += __popc(ms);
        tie_before += __popc(mt);
    }
    // every CTA has read its share (the cluster barriers above), so in place is safe
    if (p.weights_out != nullptr)
        for (int i = B + (int)rank * kSelThreads + tid; i < L; i += (int)ctas * kSelThreads) wo[i] = 0.f;
    cluster_sync();  // a peer may still read this CTA's counts
}

// ---------------------------------------------------------------- compaction
// A warp per `rows` consecutive kept tokens of a (sequence, kv head): the lanes look the pages up,
// then each row of K and of V is one 16-byte load and store a lane, 4 rows of both in flight.
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
    // CTAs per row: enough that a CTA's share is at most 8192 weights
    int ctas = 1;
    while (ctas < 8 && max_seq_len > ctas * 8192) ctas *= 2;
    // the largest share: whole warp segments of ceil(L / (ctas * threads)) x 32
    const int64_t per = ((int64_t)max_seq_len + (int64_t)ctas * kSelThreads - 1) / ((int64_t)ctas * kSelThreads);
    const size_t smem = (size_t)per * kSelThreads * sizeof(float);
    static std::atomic<bool> attr_set[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_set[dev]) {
        cudaError_t e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             PGC_EVICT_MAX_TOKENS / 8 * (int)sizeof(float));
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas, kNumKvHeads, batch);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
#ifndef PGC_NO_PDL
    cfg.numAttrs = 2;
#else
    cfg.numAttrs = 1;
#endif
    return cudaLaunchKernelEx(&cfg, evict_select_kernel, p);
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
