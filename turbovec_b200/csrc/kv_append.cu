// Appending keys and values to the pages of a cache, with the position rotation and the pages' bounds.
//
// A block takes one page that a sequence's new tokens touch, and one key head: it rotates the page's new keys and the queries of
// that head's group, copies the values, and brings the page's bounds up to date.  A page belongs to one block, so bounds need no
// atomics and no order matters.
//
// Rotation: (y1, y2) = (x1 cos - x2 sin, x2 cos + x1 sin) in 32 bits, each product and sum rounded by itself, then to the type.
// Bounds: for every channel the lowest and highest key of the page, as int8 multiples of one power of two 2^e per page and key head,
// rounded outwards: hi = ceil(max / 2^e), lo = floor(min / 2^e), e the smallest with max |key| <= 127 * 2^e.  Because
// ceil(ceil(x / 2^a) / 2^b) = ceil(x / 2^(a+b)) and rounding is monotone, widening the 8-bit bounds by new keys gives what the
// bounds of all keys together would be: tokens may come in any pieces, and the page is not read again.
#include "kv_cache.cuh"

namespace tv {
namespace {

constexpr int kAppendThreads = 256;

template <typename T>
__device__ __forceinline__ void rotate8(const uint4 &a, const uint4 &b, const float (&c)[8], const float (&s)[8], uint4 &ya, uint4 &yb) {
    const uint32_t *pa = reinterpret_cast<const uint32_t *>(&a), *pb = reinterpret_cast<const uint32_t *>(&b);
    uint32_t *qa = reinterpret_cast<uint32_t *>(&ya), *qb = reinterpret_cast<uint32_t *>(&yb);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x1 = KvType<T>::unpack(pa[i]), x2 = KvType<T>::unpack(pb[i]);
        qa[i] = KvType<T>::pack(__fsub_rn(__fmul_rn(x1.x, c[2 * i]), __fmul_rn(x2.x, s[2 * i])),
                                __fsub_rn(__fmul_rn(x1.y, c[2 * i + 1]), __fmul_rn(x2.y, s[2 * i + 1])));
        qb[i] = KvType<T>::pack(__fadd_rn(__fmul_rn(x2.x, c[2 * i]), __fmul_rn(x1.x, s[2 * i])),
                                __fadd_rn(__fmul_rn(x2.y, c[2 * i + 1]), __fmul_rn(x1.y, s[2 * i + 1])));
    }
}
// pairs of neighbours: the 16 channels of (a, b) are the pairs of angles 0 .. 7
template <typename T>
__device__ __forceinline__ void rotate_pairs(const uint4 &a, const uint4 &b, const float (&c)[8], const float (&s)[8], uint4 &ya, uint4 &yb) {
    const uint32_t *pa = reinterpret_cast<const uint32_t *>(&a), *pb = reinterpret_cast<const uint32_t *>(&b);
    uint32_t *qa = reinterpret_cast<uint32_t *>(&ya), *qb = reinterpret_cast<uint32_t *>(&yb);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 x = KvType<T>::unpack(i < 4 ? pa[i] : pb[i - 4]);
        const uint32_t y = KvType<T>::pack(__fsub_rn(__fmul_rn(x.x, c[i]), __fmul_rn(x.y, s[i])), __fadd_rn(__fmul_rn(x.y, c[i]), __fmul_rn(x.x, s[i])));
        if (i < 4) qa[i] = y; else qb[i - 4] = y;
    }
}

// Channels of unit u of a row: two runs of 8, which the rotation mixes (half-split: i and i + rotary / 2) or which are neighbours.
struct Unit {
    int a, b;
    bool turned;
};
__device__ __forceinline__ Unit unit_of(int u, int rotary, int interleaved) {
    const int turned = rotary >> 4;
    if (u < turned && !interleaved) return {8 * u, (rotary >> 1) + 8 * u, true};
    return {16 * u, 16 * u + 8, u < turned};
}

template <typename T>
__device__ __forceinline__ void unit_through(const T *src, T *dst, const Unit &un, int u, bool turn, int interleaved, const float *cos_row,
                                             const float *sin_row, uint4 &ya, uint4 &yb) {
    const uint4 a = *reinterpret_cast<const uint4 *>(src + un.a), b = *reinterpret_cast<const uint4 *>(src + un.b);
    ya = a; yb = b;
    if (turn && un.turned) {
        float c[8], s[8];
        const float4 *pc = reinterpret_cast<const float4 *>(cos_row + 8 * u), *ps = reinterpret_cast<const float4 *>(sin_row + 8 * u);
        *reinterpret_cast<float4 *>(c) = pc[0]; *reinterpret_cast<float4 *>(c + 4) = pc[1];
        *reinterpret_cast<float4 *>(s) = ps[0]; *reinterpret_cast<float4 *>(s + 4) = ps[1];
        if (interleaved) rotate_pairs<T>(a, b, c, s, ya, yb);
        else rotate8<T>(a, b, c, s, ya, yb);
    }
    *reinterpret_cast<uint4 *>(dst + un.a) = ya;
    *reinterpret_cast<uint4 *>(dst + un.b) = yb;
}

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const KvAppendParams p) {
    constexpr int kUnits = D / 16;                          // threads of one row, 16 channels each
    constexpr int kLanes = kAppendThreads / kUnits;         // rows at a time
    constexpr int kWarps = kAppendThreads / 32;
    __shared__ int64_t scratch[kWarps + 2];
    __shared__ float lows[kWarps][D], highs[kWarps][D];
    __shared__ float tops[D / 32];
    const int tid = threadIdx.x, h = blockIdx.y, page_size = 1 << p.page_shift;

    int b;
    int64_t place;
    auto first_position = [&](int i, const KvSpan &sp) { return int64_t(p.batch.lens[i]) - sp.count; };
    // pages that sequence i's tokens touch; positions before 0 belong to no page
    auto touched = [&](int i) -> int64_t {
        const KvSpan sp = kv_span(p.batch.offsets[i], p.batch.offsets[i + 1], p.tokens);
        const int64_t from = first_position(i, sp), to = from + sp.count;
        if (sp.count == 0 || to <= 0) return 0;
        return ((to - 1) >> p.page_shift) - ((from < 0 ? 0 : from) >> p.page_shift) + 1;
    };
    kv_locate<kAppendThreads>(int64_t(blockIdx.x), p.batch.sequences, touched, scratch, b, place);
    if (b >= p.batch.sequences) return;
    const KvSpan sp = kv_span(p.batch.offsets[b], p.batch.offsets[b + 1], p.tokens);
    const int64_t from = first_position(b, sp), to = from + sp.count;
    const int64_t page_index = ((from < 0 ? 0 : from) >> p.page_shift) + place, page_from = page_index << p.page_shift;
    const int64_t begin = from > page_from ? from : page_from;                                  // positions of this block
    const int64_t end = to < page_from + page_size ? to : page_from + page_size;
    const int64_t page = page_index < p.batch.table_width ? int64_t(p.batch.table[int64_t(b) * p.batch.table_stride + page_index]) : -1;
    const bool stored = page >= 0 && page < p.pages;
    const int count = int(end - begin), row0 = sp.first + int(begin - from), at0 = int(begin - page_from);
    const int half = p.rotary >> 1;
    // a position outside the tables has no angle: its token is neither stored nor rotated
    auto angled = [&](int i) {
        const int64_t a = begin + i + p.position_offset;
        return p.rotary == 0 || (a >= 0 && a < p.positions);
    };

    const int u = tid % kUnits, lane_row = tid / kUnits;
    const Unit un = unit_of(u, p.rotary, p.interleaved);
    float lo[16], hi[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) { lo[i] = INFINITY; hi[i] = -INFINITY; }
    if (stored) {
        T *dst = reinterpret_cast<T *>(p.k) + page * p.k_page + int64_t(h) * p.k_head;
        const T *src = static_cast<const T *>(p.k_new.data) + int64_t(h) * p.k_new.head_stride;
        for (int i = lane_row; i < count; i += kLanes) {
            if (!angled(i)) continue;
            const int64_t a = (begin + i + p.position_offset) * half;
            uint4 ya, yb;
            unit_through<T>(src + int64_t(row0 + i) * p.k_new.token_stride, dst + int64_t(at0 + i) * p.k_token, un, u, true, p.interleaved, p.cos + a, p.sin + a, ya, yb);
            const uint32_t *wa = reinterpret_cast<const uint32_t *>(&ya), *wb = reinterpret_cast<const uint32_t *>(&yb);
#pragma unroll
            for (int j = 0; j < 4; ++j) {                    // fminf and fmaxf leave NaN out
                const float2 x = KvType<T>::unpack(wa[j]), y = KvType<T>::unpack(wb[j]);
                lo[2 * j] = fminf(lo[2 * j], x.x); hi[2 * j] = fmaxf(hi[2 * j], x.x);
                lo[2 * j + 1] = fminf(lo[2 * j + 1], x.y); hi[2 * j + 1] = fmaxf(hi[2 * j + 1], x.y);
                lo[8 + 2 * j] = fminf(lo[8 + 2 * j], y.x); hi[8 + 2 * j] = fmaxf(hi[8 + 2 * j], y.x);
                lo[9 + 2 * j] = fminf(lo[9 + 2 * j], y.y); hi[9 + 2 * j] = fmaxf(hi[9 + 2 * j], y.y);
            }
        }
    }
    // values and queries: rows of the same shape, G + 1 to a token
    const int per_token = (p.q.data ? p.group : 0) + 1;
    for (int i = lane_row; i < count * per_token; i += kLanes) {
        const int t = i / per_token, r = i - t * per_token;
        if (!angled(t)) continue;
        const int64_t row = row0 + t;
        uint4 ya, yb;
        if (r == 0) {
            if (stored)
                unit_through<T>(static_cast<const T *>(p.v_new.data) + row * p.v_new.token_stride + int64_t(h) * p.v_new.head_stride,
                                reinterpret_cast<T *>(p.v) + page * p.v_page + int64_t(h) * p.v_head + int64_t(at0 + t) * p.v_token, un, u, false, 0, nullptr, nullptr, ya, yb);
        } else {
            const int64_t head = int64_t(h) * p.group + r - 1, a = (begin + t + p.position_offset) * half;
            unit_through<T>(static_cast<const T *>(p.q.data) + row * p.q.token_stride + head * p.q.head_stride,
                            static_cast<T *>(p.q_out.data) + row * p.q_out.token_stride + head * p.q_out.head_stride, un, u, true, p.interleaved, p.cos + a, p.sin + a, ya, yb);
        }
    }
    if (p.bounds == nullptr || !stored) return;
    const int64_t at = page * p.kv_heads + h;
    const bool widen = at0 > 0;                             // the page holds earlier keys
    const float old_scale = widen ? p.scales[at] : 0.0f;    // before a barrier that comes before its new value

    // lowest and highest new key of every channel: over the rows of a warp, then over the warps
#pragma unroll
    for (int o = kUnits; o < 32; o <<= 1)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            lo[i] = fminf(lo[i], __shfl_xor_sync(kFullMask, lo[i], o));
            hi[i] = fmaxf(hi[i], __shfl_xor_sync(kFullMask, hi[i], o));
        }
    const int warp = tid >> 5, lane = tid & 31;
    if (lane < kUnits)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int ch = i < 8 ? un.a + i : un.b + i - 8;
            lows[warp][ch] = lo[i];
            highs[warp][ch] = hi[i];
        }
    __syncthreads();
    float low = INFINITY, high = -INFINITY;
    if (tid < D) {
#pragma unroll
        for (int w = 0; w < kWarps; ++w) { low = fminf(low, lows[w][tid]); high = fmaxf(high, highs[w][tid]); }
        float top = low > high ? 0.0f : fmaxf(fabsf(low), fabsf(high));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, o));
        if (lane == 0) tops[warp] = top;
    }
    __syncthreads();
    if (tid >= D) return;
    float top = tops[0];
#pragma unroll
    for (int w = 1; w < D / 32; ++w) top = fmaxf(top, tops[w]);
    int8_t *row = p.bounds + at * 2 * D;
    const float scale = fmaxf(kv_pow2(kv_exponent(top)), old_scale);
    const bool none = low > high;                           // no new key with a value in this channel
    float qlo = none ? 127.0f : fminf(fmaxf(floorf(low / scale), -127.0f), 127.0f);
    float qhi = none ? -127.0f : fminf(fmaxf(ceilf(high / scale), -127.0f), 127.0f);
    if (widen) {
        const float ratio = old_scale / scale;
        qlo = fminf(qlo, floorf(float(row[tid]) * ratio));
        qhi = fmaxf(qhi, ceilf(float(row[D + tid]) * ratio));
    } else if (none) {
        qlo = qhi = 0.0f;
    }
    row[tid] = int8_t(int(qlo));
    row[D + tid] = int8_t(int(qhi));
    if (tid == 0) p.scales[at] = scale;
}

template <typename T, int D>
cudaError_t launch(const KvAppendParams &p, cudaStream_t s) {
    // pages touched: at most one per token, and at most two partial ones beside the full ones of a sequence
    const int64_t most = (int64_t(p.tokens) >> p.page_shift) + 2 * int64_t(p.batch.sequences);
    const int64_t blocks = most < p.tokens ? most : p.tokens;
    kv_append_kernel<T, D><<<dim3(unsigned(blocks), unsigned(p.kv_heads)), kAppendThreads, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams &p, int dtype, int head_dim, cudaStream_t s) {
    if (p.tokens == 0 || p.batch.sequences == 0) return cudaSuccess;
    if (dtype == TV_KV_BF16) return head_dim == 128 ? launch<__nv_bfloat16, 128>(p, s) : launch<__nv_bfloat16, 64>(p, s);
    return head_dim == 128 ? launch<__half, 128>(p, s) : launch<__half, 64>(p, s);
}

}  // namespace tv
