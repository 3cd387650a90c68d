// Which pages of its sequence a token attends to: the first ones, the most recent ones, and the best of the others by a score that
// bounds what any key of a page can give.
//
// The score of a page for a key head is the largest, over the query heads that share it, of sum_d max(q_d lo_d, q_d hi_d) with q in
// int8 (multiples of a power of two per head, nearest, ties to even) and the page's int8 bounds: a contraction of (min(q, 0), max(q, 0))
// with (lo, hi), exact in whole numbers below 2^22, times powers of two (2^-24 to 2^40 each): no rounding anywhere, so the choice does not depend on the
// order of any sum, and equal scores go to the lower page.
//
// A cluster of blocks takes one token and key head: all of them score pages, into the shared memory of the first, which chooses.
// Scores: int8 MMAs, query heads on the M side, 8 pages on the N side; a lane's 16-byte
// loads of a page's bounds feed four register operands, with the queries' channels permuted to match.  Choice: the k-th largest
// score digit by digit (four counts of 8 bits), then one pass that keeps the pages' order.
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

template <typename T, int D>
__global__ void __launch_bounds__(kSelectThreads, 2) kv_select_kernel(const KvSelectParams p, int blocks) {
    extern __shared__ uint32_t keys[];                    // scores in ascending order of their bits; 0: no such page in the pool
    __shared__ __align__(16) int8_t q8[kKvRows][2 * D];
    __shared__ float q_scale[kKvRows];
    __shared__ uint32_t counts[256];
    __shared__ uint32_t found[2];
    __shared__ uint32_t sums[kSelectWarps];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, token = blockIdx.x / blocks, h = blockIdx.y;
    const int rank = blocks > 1 ? int(cluster_ctarank()) : 0;              // clusters lie along x

    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // this block has begun: others may write into it
    auto others_begun = [&] { if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory"); };
    int b = 0;
    {
        int hi = p.batch.sequences;
        while (hi - b > 1) {
            const int mid = (b + hi) >> 1;
            if (p.batch.offsets[mid] <= token) b = mid; else hi = mid;
        }
    }
    const KvSpan sp = kv_span(p.batch.offsets[b], p.batch.offsets[b + 1], p.tokens);
    if (token < sp.first || token >= sp.first + sp.count) {                // behind the last sequence
        others_begun();
        return;
    }
    const int64_t pos = int64_t(p.batch.lens[b]) - sp.count + (token - sp.first);
    const int seen = kv_visible(pos, kv_capacity(p.batch.table_width, p.page_shift));
    const int n = int((int64_t(seen) + (1 << p.page_shift) - 1) >> p.page_shift);
    if (h == 0 && rank == 0 && tid == 0) p.token_pos[token] = seen - 1;
    const int32_t *table = p.batch.table + int64_t(b) * p.batch.table_stride;
    int32_t *list = p.chosen + (int64_t(token) * p.kv_heads + h) * p.budget, *pool = p.chosen_pool + (int64_t(token) * p.kv_heads + h) * p.budget;
    auto put = [&](int at, int page) {
        list[at] = page;
        pool[at] = page >= 0 ? table[page] : -1;
    };
    if (n <= p.budget) {
        if (rank == 0)
            for (int i = tid; i < p.budget; i += kSelectThreads) put(i, i < n ? i : -1);
        others_begun();
        return;
    }
    const int begin = p.first, end = n - p.recent, want = p.budget - p.first - p.recent;
    if (rank == 0) {
        for (int i = tid; i < p.first; i += kSelectThreads) put(i, i);
        for (int i = tid; i < p.recent; i += kSelectThreads) put(p.budget - p.recent + i, end + i);
    }
    if (want == 0) {
        others_begun();
        return;
    }
    const uint32_t keys_at = blocks > 1 ? map_to_cta(smem_u32(keys), 0) : smem_u32(keys);

    for (int g0 = 0; g0 < p.group; g0 += kKvRows) {
        __syncthreads();
        for (int r = warp; r < kKvRows; r += kSelectWarps) {
            const bool have = g0 + r < p.group;
            const T *src = static_cast<const T *>(p.q.data) + int64_t(token) * p.q.token_stride + int64_t(h * p.group + g0 + (have ? r : 0)) * p.q.head_stride;
            float x[D / 32], top = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 64; ++i) {
                const float2 y = KvType<T>::unpack(*reinterpret_cast<const uint32_t *>(src + 64 * i + 2 * lane));
                x[2 * i] = y.x; x[2 * i + 1] = y.y;
                top = fmaxf(top, fmaxf(fabsf(y.x), fabsf(y.y)));           // NaN left out
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
            const float scale = kv_pow2(kv_exponent(top));
            if (lane == 0) q_scale[r] = scale;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                const float y = rintf(x[i] / scale);
                const int v = have && y == y ? int(fminf(fmaxf(y, -127.0f), 127.0f)) : 0;
                const int ch = 64 * (i >> 1) + 2 * lane + (i & 1);
                q8[r][ch] = int8_t(min(v, 0));
                q8[r][D + ch] = int8_t(max(v, 0));
            }
        }
        __syncthreads();
        const int r0 = lane >> 2, c = lane & 3;
        const bool have0 = g0 + r0 < p.group, have1 = g0 + r0 + 8 < p.group;
        const float f0 = q_scale[r0], f1 = q_scale[r0 + 8];
        uint4 a0[D / 32], a1[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            a0[i] = *reinterpret_cast<const uint4 *>(&q8[r0][64 * i + 16 * c]);
            a1[i] = *reinterpret_cast<const uint4 *>(&q8[r0 + 8][64 * i + 16 * c]);
        }
        if (g0 == 0) others_begun();
        // two runs of 8 pages at a time: their loads overlap
        constexpr int kRuns = 2;
        const int step = kSelectWarps * 8 * blocks;
        for (int p0 = begin + (rank * kSelectWarps + warp) * 8; p0 < end; p0 += kRuns * step) {
            bool good[kRuns];
            int64_t at[kRuns];
            uint4 w[kRuns][D / 32];
#pragma unroll
            for (int k = 0; k < kRuns; ++k) {
                const int mine = p0 + k * step + r0;
                const int page = mine < end ? __ldg(table + mine) : -1;
                good[k] = page >= 0 && page < p.pages;
                at[k] = (good[k] ? int64_t(page) : 0) * p.kv_heads + h;
            }
            float scale[kRuns];
#pragma unroll
            for (int k = 0; k < kRuns; ++k) {
                const uint4 *row = reinterpret_cast<const uint4 *>(p.bounds + at[k] * 2 * D) + c;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) w[k][i] = __ldg(row + 4 * i);
                scale[k] = __ldg(p.scales + at[k]);
            }
#pragma unroll
            for (int k = 0; k < kRuns; ++k) {
                int d[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    mma_s8(d, a0[i].x, a1[i].x, a0[i].y, a1[i].y, w[k][i].x, w[k][i].y);
                    mma_s8(d, a0[i].z, a1[i].z, a0[i].w, a1[i].w, w[k][i].z, w[k][i].w);
                }
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
                const int mine = p0 + k * step + r0;
                if (c == 0 && mine < end) {
                    const uint32_t to = keys_at + 4 * (mine - begin);
                    uint32_t key = good[k] ? max(ascending(((r0 & 1) ? from1 : from0) * scale[k]), 1u) : 0u;
                    if (g0 > 0) key = max(key, load_cluster(to));          // this lane wrote it for the heads before
                    store_cluster(to, key);
                }
            }
        }
    }
    if (blocks > 1) {
        cluster_sync_all();
        if (rank > 0) return;
    }
    __syncthreads();

    // the want-th largest key, digit by digit
    const int m = end - begin;
    uint32_t prefix = 0;
    int left = want;                                       // places left for keys that agree with `prefix` so far
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
        counts[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : ~0u << (shift + 8);
        for (int i0 = 0; i0 < m; i0 += kSelectThreads) {
            const int i = i0 + tid;
            const uint32_t key = i < m ? keys[i] : 0u;
            const bool on = i < m && (key & mask) == prefix;
            const uint32_t digit = on ? (key >> shift) & 255u : 256u;
            const uint32_t same = __match_any_sync(kFullMask, digit);
            if (on && lane == __ffs(int(same)) - 1) atomicAdd(&counts[digit], uint32_t(__popc(same)));
        }
        __syncthreads();
        if (warp == 0) {                                   // lane l looks after the digits 255 - 8 l .. 248 - 8 l
            uint32_t mine = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) mine += counts[255 - 8 * lane - j];
            uint32_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t up = __shfl_up_sync(kFullMask, upto, o);
                if (lane >= o) upto += up;
            }
            uint32_t above = upto - mine;
            if (above < uint32_t(left) && upto >= uint32_t(left)) {
                for (int j = 0; j < 8; ++j) {
                    const uint32_t cnt = counts[255 - 8 * lane - j];
                    if (above + cnt >= uint32_t(left)) { found[0] = uint32_t(255 - 8 * lane - j); found[1] = above; break; }
                    above += cnt;
                }
            }
        }
        __syncthreads();
        prefix |= found[0] << shift;
        left -= int(found[1]);
        __syncthreads();
    }
    // keys above the want-th, and the first `left` of those equal to it, in the pages' order
    uint32_t taken = 0, equal = 0;
    for (int i0 = 0; i0 < m; i0 += kSelectThreads) {
        const int i = i0 + tid;
        const uint32_t key = i < m ? keys[i] : 0u;
        const bool over = i < m && key > prefix, same = i < m && key == prefix;
        const uint32_t bo = __ballot_sync(kFullMask, over), bs = __ballot_sync(kFullMask, same), under = (1u << lane) - 1u;
        if (lane == 0) sums[warp] = uint32_t(__popc(bo)) | uint32_t(__popc(bs)) << 16;
        __syncthreads();
        uint32_t before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < kSelectWarps; ++w) {
            if (w < warp) before += sums[w];
            all += sums[w];
        }
        const uint32_t o = taken + (before & 0xffffu) + __popc(bo & under), e = equal + (before >> 16) + __popc(bs & under);
        if (over || (same && e < uint32_t(left))) put(p.first + int(o + min(e, uint32_t(left))), begin + i);
        taken += all & 0xffffu;
        equal += all >> 16;
        __syncthreads();
    }
}

template <typename T, int D>
cudaError_t launch(const KvSelectParams &p, int device, int sm_count, cudaStream_t s) {
    constexpr int kStatic = 8 * 1024;
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
    cfg.gridDim = dim3(unsigned(p.tokens) * unsigned(blocks), unsigned(p.kv_heads));
    cfg.blockDim = dim3(kSelectThreads);
    cfg.dynamicSmemBytes = size_t(p.batch.table_width) * 4;
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
