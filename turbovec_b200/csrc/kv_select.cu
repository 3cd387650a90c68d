// Which pages of its sequence a token attends to: the first ones, the most recent ones, and the best of the others by a score: what a key at
// the page's bounds would give the query, rounded to int8.  (Not quite a bound of what its keys give: the query's rounding may go either way.)
//
// The score of a page for a key head is the largest, over the query heads that share it, of sum_d max(q_d lo_d, q_d hi_d) with q in
// int8 (multiples of a power of two per head, nearest, ties to even) and the page's int8 bounds: a contraction of (min(q, 0), max(q, 0))
// with (lo, hi), exact in whole numbers below 2^22, times powers of two (2^-24 to 2^40 each): nothing is rounded after the query, so the choice does
// not depend on the order of any sum, and equal scores go to the lower page.
//
// The kernel is a chain of dependent steps (sequence, quantised queries, scores, histogram, list), each a latency of its own; the bounds alone
// (2 D bytes a page and head) would be a fraction of its time.  selected_48x65536, 830 pages to each of 192 (token, head) pairs, 41 MB of
// bounds: 21.8 us, 1.9 TB/s; selected_16_ragged, 23 MB: 22.4 us; selected_1x32000, 1 MB: 7.7 us.
//
// A cluster of blocks takes one token and key head: all of them score pages, into the shared memory of the first, which chooses.
// Scores: int8 MMAs, query heads on the M side, 8 pages on the N side; a lane's 16-byte
// pieces of a page's bounds feed four register operands, with the queries' channels permuted to match.  Choice: the k-th largest
// score by a histogram of its leading digit and a comparison of those that share it, then one pass that keeps the pages' order.
#include <cfloat>

#include "kv_cache.cuh"
#include "scan_tc_common.cuh"

namespace tv {
namespace {

constexpr int kSelectThreads = 256;
constexpr int kSelectWarps = kSelectThreads / 32;

__device__ __forceinline__ uint32_t ascending(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void store_cluster(uint32_t addr, uint32_t x) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(x) : "memory"); }
__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(addr) : "memory");
    return x;
}

__device__ __forceinline__ void copy16(uint32_t to, const void *from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }

constexpr int kBinBits = 11, kBins = 1 << kBinBits;
// Runs of 8 pages that a warp has under way.  1, 2, 3, 4: selected_1x32000 18.3, 18.5, 18.9, 19.2 us a call, selected_16_ragged 51.8, 49.3, 49.8, 50.4,
// selected_48x65536 93.3, 90.7, 91.5, 91.6: 16 warps on a multiprocessor hide the latency with two, and more is more to begin.
constexpr int kDepth = 2;
template <int D>
constexpr int kRingBytes = kSelectWarps * kDepth * 8 * 2 * D;   // bounds on their way: [warp][run][8 pages][2 D]
struct SelectShared {
    union {
        uint32_t counts[kBins];
        uint32_t few[kSelectThreads];                     // the keys of one bin
    };
    uint32_t found[3];
    uint32_t sums[2][kSelectWarps], least[kSelectWarps], most[kSelectWarps];
    int seq[4];                                           // sequence of the token, its first row and count, its length
    float q_scale[kKvRows];
};

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 2) kv_select_kernel(const KvSelectParams p, int blocks) {
    extern __shared__ __align__(16) uint8_t dynamic[];
    uint32_t *keys = reinterpret_cast<uint32_t *>(dynamic + kRingBytes<D>);     // scores in ascending order of their bits; 0: no such page in the pool
    __shared__ __align__(16) int8_t q8[kKvRows][2 * D];
    __shared__ SelectShared sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, item = blockIdx.x / blocks, token = item / p.kv_heads, h = item % p.kv_heads;
    const int rank = blocks > 1 ? int(cluster_ctarank()) : 0;              // clusters lie along x

    if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this block has begun: others may write into it
    auto others_begun = [&] { if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); };
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    // a warp's first row of queries comes while the sequence is being looked for
    auto query = [&](int r, uint32_t (&x)[D / 64]) {
        const T *src = static_cast<const T *>(p.q.data) + int64_t(token) * p.q.token_stride + int64_t(h * p.group + r) * p.q.head_stride;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) x[i] = *reinterpret_cast<const uint32_t *>(src + 64 * i + 2 * lane);
    };
    uint32_t q_first[D / 64] = {};
    if (warp < p.group) query(warp, q_first);
    if (tid == 0) { sh.seq[0] = INT_MAX; sh.seq[2] = 0; }
    __syncthreads();
    // Offsets that decrease give sequences that overlap: the lowest of them, for the blocks of a cluster must all take the same one (a block
    // that had nothing to score would have left when the others write into its memory).
    int mine = INT_MAX, len_of_mine = 0;
    KvSpan span_of_mine{0, 0};
    for (int i = tid; i < p.batch.sequences && mine == INT_MAX; i += kSelectThreads) {
        const int from = p.batch.offsets[i], to = p.batch.offsets[i + 1];
        len_of_mine = p.batch.lens[i];
        span_of_mine = kv_span(from, to, p.tokens);
        if (token >= span_of_mine.first && token < span_of_mine.first + span_of_mine.count) mine = i;
    }
    if (mine != INT_MAX) atomicMin(&sh.seq[0], mine);
    __syncthreads();
    if (mine != INT_MAX && mine == sh.seq[0]) { sh.seq[1] = span_of_mine.first; sh.seq[2] = span_of_mine.count; sh.seq[3] = len_of_mine; }
    __syncthreads();
    const int b = sh.seq[0], first_row = sh.seq[1], count = sh.seq[2], len = sh.seq[3];
    if (count == 0) {                                                      // behind the last sequence
        others_begun();
        return;
    }
    const int64_t pos = int64_t(len) - count + (token - first_row);
    const int seen = kv_visible(pos, kv_capacity(p.batch.table_width, p.page_shift));
    const int n = int((int64_t(seen) + (1 << p.page_shift) - 1) >> p.page_shift);
    if (h == 0 && rank == 0 && tid == 0) p.token_pos[token] = seen - 1;
    const int32_t *table = p.batch.table + int64_t(b) * p.batch.table_stride;
    int32_t *list = p.chosen + (int64_t(token) * p.kv_heads + h) * p.budget, *pool = p.chosen_pool + (int64_t(token) * p.kv_heads + h) * p.budget;
    auto put = [&](int at, int page) {
        list[at] = page;
        pool[at] = page >= 0 ? __ldg(table + page) : -1;
    };
    if (n <= p.budget) {
        if (rank == 0)
            for (int i = tid; i < p.budget; i += kSelectThreads) put(i, i < n ? i : -1);
        others_begun();
        return;
    }
    const int begin = p.first, end = n - p.recent, want = p.budget - p.first - p.recent;
    auto put_taken = [&] {
        for (int i = tid; i < p.first; i += kSelectThreads) put(i, i);
        for (int i = tid; i < p.recent; i += kSelectThreads) put(p.budget - p.recent + i, end + i);
    };
    if (want == 0) {
        if (rank == 0) put_taken();
        others_begun();
        return;
    }
    const uint32_t keys_at = blocks > 1 ? map_to_cta(smem_u32(keys), 0) : smem_u32(keys);
    const int r0 = lane >> 2, c = lane & 3;
    const uint8_t *ring = dynamic + warp * (kRingBytes<D> / kSelectWarps);
    const uint32_t ring_at = smem_u32(ring);

    for (int g0 = 0; g0 < p.group; g0 += kKvRows) {
        if (g0 > 0) __syncthreads();
        for (int r = warp; r < kKvRows; r += kSelectWarps) {
            const bool have = g0 + r < p.group;
            uint32_t raw[D / 64] = {};
            if (g0 == 0 && r == warp) {
#pragma unroll
                for (int i = 0; i < D / 64; ++i) raw[i] = q_first[i];
            } else if (have) {
                query(g0 + r, raw);
            }
            float x[D / 32], top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const float2 y = KvType<T>::unpack(raw[i]);
                x[2 * i] = y.x; x[2 * i + 1] = y.y;
                top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));           // NaN left out
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
            const int e = kv_exponent(top);
            const float inverse = kv_pow2(-e);                             // exact, and so is the product
            if (lane == 0) sh.q_scale[r] = kv_pow2(e);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const float y = rintf(x[i] * inverse);
                const int v = y == y ? int(fminf(fmaxf(y, -127.0f), 127.0f)) : 0;
                const int ch = 64 * (i >> 1) + 2 * lane + (i & 1);
                q8[r][ch] = int8_t(min(v, 0));
                q8[r][D + ch] = int8_t(max(v, 0));
            }
        }
        __syncthreads();
        const bool have0 = g0 + r0 < p.group, have1 = g0 + r0 + 8 < p.group;
        const float f0 = sh.q_scale[r0], f1 = sh.q_scale[r0 + 8];
        uint4 a0[D / 32], a1[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            a0[i] = *reinterpret_cast<const uint4 *>(&q8[r0][64 * i + 16 * c]);
            a1[i] = *reinterpret_cast<const uint4 *>(&q8[r0 + 8][64 * i + 16 * c]);
        }
        if (g0 == 0) others_begun();
        // Runs of 8 pages, kDepth of them under way: page numbers, then bounds (into shared memory) and scales, then products.  A row of
        // bounds keeps its 16-byte pieces in order, odd rows with neighbouring fours swapped: eight lanes read two rows at once.
        const int step = kSelectWarps * 8 * blocks, p0 = begin + (rank * kSelectWarps + warp) * 8;
        auto page_of = [&](int run) {
            const int mine = p0 + run * step + r0;
            return mine < end ? __ldg(table + mine) : -1;
        };
        const int swap = (r0 & 1) << 2;
        float scale[kDepth] = {};
        bool good[kDepth];
        auto fetch = [&](int k, int page) {
            good[k] = page >= 0 && page < p.pages;
            if (good[k]) {                                 // (no load in the place of a page that is not there: they would all meet in one line)
                const int64_t at = int64_t(page) * p.kv_heads + h;
                const uint8_t *row = reinterpret_cast<const uint8_t *>(p.bounds + at * 2 * D);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) copy16(ring_at + (k * 8 + r0) * 2 * D + (((4 * i + c) ^ swap) << 4), row + ((4 * i + c) << 4));
                scale[k] = __ldcg(p.scales + at);          // (not by the read-only path: an append may still run when this kernel begins)
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        int ahead[kDepth];
#pragma unroll
        for (int k = 0; k < kDepth; ++k) ahead[k] = page_of(k);
#pragma unroll
        for (int k = 0; k < kDepth; ++k) fetch(k, ahead[k]);
#pragma unroll
        for (int k = 0; k < kDepth; ++k) ahead[k] = page_of(kDepth + k);
        for (int run0 = 0; p0 + run0 * step < end; run0 += kDepth) {
#pragma unroll
            for (int k = 0; k < kDepth; ++k) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
                __syncwarp();
                int d[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    const uint4 w = *reinterpret_cast<const uint4 *>(ring + (k * 8 + r0) * 2 * D + (((4 * i + c) ^ swap) << 4));
                    mma_s8(d, a0[i].x, a1[i].x, a0[i].y, a1[i].y, w.x, w.y);
                    mma_s8(d, a0[i].z, a1[i].z, a0[i].w, a1[i].w, w.z, w.w);
                }
                const bool is_good = good[k];
                const float page_scale = scale[k];
                __syncwarp();
                fetch(k, ahead[k]);
                ahead[k] = page_of(run0 + 2 * kDepth + k);
                float s0 = -FLT_MAX, s1 = -FLT_MAX;
                if (have0) { s0 = float(d[0]) * f0; s1 = float(d[1]) * f0; }
                if (have1) { s0 = fmaxf(s0, float(d[2]) * f1); s1 = fmaxf(s1, float(d[3]) * f1); }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    s0 = fmaxf(s0, __shfl_xor_sync(kFullMask, s0, o));
                    s1 = fmaxf(s1, __shfl_xor_sync(kFullMask, s1, o));
                }
                // lanes 0 .. 3 hold pages 2 lane and 2 lane + 1; hand page r0 to lane 4 r0
                const float from0 = __shfl_sync(kFullMask, s0, r0 >> 1), from1 = __shfl_sync(kFullMask, s1, r0 >> 1);
                const int mine = p0 + (run0 + k) * step + r0;
                if (c == 0 && mine < end) {
                    const uint32_t to = keys_at + 4 * (mine - begin);
                    uint32_t key = is_good ? max(ascending(((r0 & 1) ? from1 : from0) * page_scale), 1u) : 0u;
                    if (g0 > 0) key = max(key, load_cluster(to));          // this lane wrote it for the heads before
                    store_cluster(to, key);
                }
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (blocks > 1) {
        cluster_sync_all();
        if (rank > 0) return;
    } else {
        __syncthreads();
    }

    put_taken();
    // The want-th largest key.  Between the smallest and the largest key the leading digit of kBinBits bits mostly leaves a handful of candidates,
    // which are ranked by comparing them all; where it leaves more, the next digit of the bin that holds the key is looked at.
    const int m = end - begin;
    uint32_t lo = ~0u, hi = 0u;
    for (int i = tid; i < m; i += kSelectThreads) { lo = min(lo, keys[i]); hi = max(hi, keys[i]); }
    lo = __reduce_min_sync(kFullMask, lo);
    hi = __reduce_max_sync(kFullMask, hi);
    if (lane == 0) { sh.least[warp] = lo; sh.most[warp] = hi; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWarps; ++w) { lo = min(lo, sh.least[w]); hi = max(hi, sh.most[w]); }
    int bits = 32 - __clz(int(hi - lo));                   // keys lo .. lo + 2^bits - 1 are looked at
    uint32_t limit = lo;
    int left = want;                                       // places left for keys from `limit` on, below those taken already
#pragma unroll 1
    while (true) {
        const int shift = max(0, bits - kBinBits);
#pragma unroll
        for (int j = 0; j < kBins / kSelectThreads; ++j) sh.counts[tid + j * kSelectThreads] = 0;
        __syncthreads();
        const uint32_t inside = bits >= 32 ? ~0u : (1u << bits) - 1u;
        for (int i = tid; i < m; i += kSelectThreads) {
            const uint32_t x = keys[i] - limit;
            if (keys[i] >= limit && x <= inside) atomicAdd(&sh.counts[x >> shift], 1u);
        }
        __syncthreads();
        constexpr int kOwn = kBins / kSelectThreads;       // bins of a thread, the highest to thread 0
        uint32_t own[kOwn], mine = 0;
#pragma unroll
        for (int j = 0; j < kOwn; ++j) { own[j] = sh.counts[kBins - 1 - tid * kOwn - j]; mine += own[j]; }
        uint32_t upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t up = __shfl_up_sync(kFullMask, upto, o);
            if (lane >= o) upto += up;
        }
        if (lane == 31) sh.sums[0][warp] = upto;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) if (w < warp) upto += sh.sums[0][w];
        uint32_t above = upto - mine;
        if (above < uint32_t(left) && upto >= uint32_t(left)) {
#pragma unroll
            for (int j = 0; j < kOwn; ++j) {
                if (above < uint32_t(left) && above + own[j] >= uint32_t(left)) { sh.found[0] = uint32_t(kBins - 1 - tid * kOwn - j); sh.found[1] = above; sh.found[2] = own[j]; }
                above += own[j];
            }
        }
        __syncthreads();
        const uint32_t bin = sh.found[0], size = sh.found[2];
        left -= int(sh.found[1]);
        limit += bin << shift;
        bits = shift;
        if (shift == 0) break;                             // all of the bin are the same key
        if (size > uint32_t(kSelectThreads)) continue;
        __syncthreads();                                   // the counts have been read: their place is used for the candidates
        if (tid == 0) sh.found[0] = 0;
        __syncthreads();
        for (int i = tid; i < m; i += kSelectThreads)
            if (keys[i] >= limit && keys[i] - limit < (1u << shift)) sh.few[atomicAdd(&sh.found[0], 1u)] = keys[i];
        __syncthreads();
        if (tid < int(size)) {
            const uint32_t key = sh.few[tid];
            int over = 0, same = 0;
            for (uint32_t i = 0; i < size; ++i) { over += sh.few[i] > key; same += sh.few[i] == key; }
            if (over < left && over + same >= left) { sh.found[1] = key; sh.found[2] = uint32_t(over); }      // (the same for all equal keys)
        }
        __syncthreads();
        limit = sh.found[1];
        left -= int(sh.found[2]);
        break;
    }
    // keys above that, and the first `left` of those equal to it, in the pages' order
    uint32_t taken = 0, equal = 0;
    for (int i0 = 0, turn = 0; i0 < m; i0 += kSelectThreads, turn ^= 1) {
        const int i = i0 + tid;
        const uint32_t key = i < m ? keys[i] : 0u;
        const bool over = i < m && key > limit, same = i < m && key == limit;
        const uint32_t bo = __ballot_sync(kFullMask, over), bs = __ballot_sync(kFullMask, same), under = (1u << lane) - 1u;
        if (lane == 0) sh.sums[turn][warp] = uint32_t(__popc(bo)) | uint32_t(__popc(bs)) << 16;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) {
            const uint32_t x = sh.sums[turn][w];
            if (w < warp) before += x;
            all += x;
        }
        const uint32_t o = taken + (before & 0xffffu) + __popc(bo & under), e = equal + (before >> 16) + __popc(bs & under);
        if (over || (same && e < uint32_t(left))) put(p.first + int(o + min(e, uint32_t(left))), begin + i);
        taken += all & 0xffffu;
        equal += all >> 16;
    }
}

template <typename T, int D>
cudaError_t launch(const KvSelectParams &p, int device, int sm_count, cudaStream_t s) {
    constexpr int kStatic = kKvRows * 2 * D + sizeof(SelectShared) + 256;
    static_assert(kRingBytes<D> + 4 * kKvMaxScored + kStatic <= kBlockSharedBytes, "more shared memory than a block can have");
    auto *kern = kv_select_kernel<T, D>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = kv_allow_shared(kern, allowed, device, kStatic);
    if (e != cudaSuccess) return e;
    // as many blocks to a token and key head as the device holds at once (two to a multiprocessor), none with less than a round of pages
    const int64_t items = int64_t(p.tokens) * p.kv_heads;
    int blocks = 1;
    while (blocks < 8 && items * blocks * 2 <= 2 * sm_count && blocks * kSelectWarps * 8 < p.batch.table_width) blocks *= 2;
    cudaLaunchAttribute attrs[2];
    attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[0].val.programmaticStreamSerializationAllowed = 1;
    attrs[1].id = cudaLaunchAttributeClusterDimension;
    attrs[1].val.clusterDim.x = unsigned(blocks); attrs[1].val.clusterDim.y = 1; attrs[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(items * blocks));       // the heads of a token side by side: their bounds lie side by side in every page
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = kRingBytes<D> + size_t(p.batch.table_width) * 4;
    cfg.stream = s;
    cfg.attrs = attrs;
    cfg.numAttrs = blocks > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, p, blocks);
}

}  // namespace

cudaError_t launch_kv_select(const KvSelectParams &p, int dtype, int head_dim, int device, int sm_count, cudaStream_t s) {
    if (p.tokens == 0 || p.batch.sequences == 0) return cudaSuccess;
    if (dtype == TV_KV_BF16) return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, device, sm_count, s) : launch<__nv_bfloat16, 64>(p, device, sm_count, s);
    return head_dim == 128 ? launch<__half, 128>(p, device, sm_count, s) : launch<__half, 64>(p, device, sm_count, s);
}

}  // namespace tv
