/*
 * kv_cache.hip - Writing rows of keys and values into the paged cache, quantised on the way, and
 * reading them back; the checks of a cache and a batch.
 */
#include "kv.h"

using namespace w4a16;

namespace {

constexpr float kSmallest = 0x1p-117f; /* 448 / kSmallest is still finite in FP32 */

/* The sequence of a row and its place in the cache: found by a whole wave, the same on all lanes.
 * The sequences whose rows end at or before `row` are counted 64 at a time. */
struct Place {
    int seq, page, inside; /* seq < 0: no sequence's row; page < 0: a row without a place */
};

__device__ __forceinline__ Place find_place(const KvView &kv, int row) {
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int base = 0; base < kv.seqs; base += 64) {
        const int s = base + lane;
        const bool ends = s < kv.seqs && kv.starts[s + 1] <= row;
        const int n = __popcll(__ballot(ends));
        before += n;
        if (n < 64) break;
    }
    if (before >= kv.seqs) return {-1, -1, 0};
    const int first = kv.starts[before], last = kv.starts[before + 1];
    if (row < first || row >= last) return {-1, -1, 0};
    /* kv_lens and the number of rows may be anything up to 2^31: the difference in 64 bits */
    const long long at = (long long)kv.kv_lens[before] - last + row;
    if (at < 0 || (at >> kv.shift) >= kv.table_pages) return {before, -1, 0};
    const int page = kv.table[(long long)before * kv.table_stride + (at >> kv.shift)];
    if ((unsigned)page >= (unsigned)kv.pages) return {before, -1, 0};
    return {before, page, (int)(at & ((1 << kv.shift) - 1))};
}

/* The largest of v over groups of N lanes (8, 16 or 32). */
template <int N>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int m = 1; m < N; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

/* One wave a row of K (blockIdx.y = 0) or V (1): D / 8 lanes a head, eight values a lane. Bound by
 * memory: a row is read once with 16 bytes a lane and its codes are written once. The row's
 * largest value is found over the head's lanes by shuffles; the scale and its inverse are each
 * one division a row, and a value costs a product and a conversion. 8198 rows of 8 heads of 128 to FP8:
 * 12.6 us, 51 MB at 4.0 TB/s (a large copy: 4.9); four rows: 3.4, a launch and three round trips. */
template <int D, int FMT>
__global__ __launch_bounds__(256) void kv_write_kernel(KvView kv, const uint16_t *k, long long k_row,
                                                       long long k_head, const uint16_t *v,
                                                       long long v_row, long long v_head) {
    constexpr int kLanes = D / 8, kHeads = 64 / kLanes;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= kv.rows) return;
    const Place at = find_place(kv, row);
    if (at.page < 0) return;
    const bool is_v = blockIdx.y != 0;
    const uint16_t *src = is_v ? v + row * v_row : k + row * k_row;
    const long long head_stride = is_v ? v_head : k_head;
    void *codes = is_v ? kv.v : kv.k;
    float *scales = is_v ? kv.v_scale : kv.k_scale;
    const int part = (lane % kLanes) * 8;
    for (int h = lane / kLanes; h < kv.heads; h += kHeads) {
        const uint4 x = *reinterpret_cast<const uint4 *>(src + h * head_stride + part);
        const long long slot = (((long long)at.page * kv.heads + h) << kv.shift) + at.inside;
        if constexpr (FMT == W4A16_KV_BF16) {
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(codes) + slot * D + part) = x;
        } else {
            constexpr float kTop = FMT == W4A16_KV_INT8 ? 127.0f : 448.0f;
            const uint32_t w[4] = {x.x, x.y, x.z, x.w};
            float f[8], most = 0.0f;
            bool finite = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[2 * i] = __builtin_bit_cast(float, w[i] << 16);
                f[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xFFFF0000u);
                finite = finite && (w[i] & 0x7F800000u) != 0x7F800000u && (w[i] & 0x7F80u) != 0x7F80u;
                most = fmaxf(most, fmaxf(fabsf(f[2 * i]), fabsf(f[2 * i + 1])));
            }
            most = group_max<kLanes>(finite ? most : __builtin_inff());
            const bool held = most >= kSmallest && most < __builtin_inff();
            const float inverse = held ? kTop / most : 0.0f;
            uint32_t out[2] = {0u, 0u};
            if (held) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = __builtin_amdgcn_fmed3f(f[i] * inverse, -kTop, kTop);
                if constexpr (FMT == W4A16_KV_FP8) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        int word = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
                        out[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], word, true);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        out[i / 4] |= ((uint32_t)(int)__builtin_rintf(f[i]) & 0xFFu) << (8 * (i % 4));
                }
            }
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(codes) + slot * D + part) =
                make_uint2(out[0], out[1]);
            if (lane % kLanes == 0)
                scales[slot] = held ? most / kTop : most < kSmallest ? 0.0f : __builtin_nanf("");
        }
    }
}

/* The reverse, with the same split: codes read once, BF16 rows written once. 82258 rows of 8 heads of 128
 * from FP8: 111 us, 511 MB at 4.6 TB/s. */
template <int D, int FMT>
__global__ __launch_bounds__(256) void kv_read_kernel(KvView kv, uint16_t *k, uint16_t *v) {
    constexpr int kLanes = D / 8, kHeads = 64 / kLanes;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (row >= kv.rows) return;
    const Place at = find_place(kv, row);
    if (at.seq < 0) return;
    const bool is_v = blockIdx.y != 0;
    const void *codes = is_v ? kv.v : kv.k;
    const float *scales = is_v ? kv.v_scale : kv.k_scale;
    uint16_t *dst = (is_v ? v : k) + (long long)row * kv.heads * D;
    const int part = (lane % kLanes) * 8;
    for (int h = lane / kLanes; h < kv.heads; h += kHeads) {
        uint4 x = make_uint4(0u, 0u, 0u, 0u);
        if (at.page >= 0) {
            const long long slot = (((long long)at.page * kv.heads + h) << kv.shift) + at.inside;
            if constexpr (FMT == W4A16_KV_BF16) {
                x = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(codes) + slot * D + part);
            } else {
                const uint2 c = *reinterpret_cast<const uint2 *>(static_cast<const uint8_t *>(codes) + slot * D + part);
                const float s = scales[slot];
                const uint32_t w[4] = {kv_widen<FMT, 0>(c.x), kv_widen<FMT, 1>(c.x), kv_widen<FMT, 0>(c.y),
                                       kv_widen<FMT, 1>(c.y)};
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = kv_pack_bf16(__builtin_bit_cast(float, w[i] << 16) * s,
                                        __builtin_bit_cast(float, w[i] & 0xFFFF0000u) * s);
                x = make_uint4(o[0], o[1], o[2], o[3]);
            }
        }
        *reinterpret_cast<uint4 *>(dst + (long long)h * D + part) = x;
    }
}

template <int D>
void launch_write(int format, const KvView &kv, const uint16_t *k, long long k_row, long long k_head,
                  const uint16_t *v, long long v_row, long long v_head, hipStream_t s) {
    const dim3 grid((kv.rows + 3) / 4, 2), block(256);
    auto kernel = format == W4A16_KV_BF16   ? kv_write_kernel<D, W4A16_KV_BF16>
                  : format == W4A16_KV_INT8 ? kv_write_kernel<D, W4A16_KV_INT8>
                                            : kv_write_kernel<D, W4A16_KV_FP8>;
    launch_k(kernel, grid, block, 0, s, kv, k, k_row, k_head, v, v_row, v_head);
}

template <int D>
void launch_read(int format, const KvView &kv, uint16_t *k, uint16_t *v, hipStream_t s) {
    const dim3 grid((kv.rows + 3) / 4, 2), block(256);
    auto kernel = format == W4A16_KV_BF16   ? kv_read_kernel<D, W4A16_KV_BF16>
                  : format == W4A16_KV_INT8 ? kv_read_kernel<D, W4A16_KV_INT8>
                                            : kv_read_kernel<D, W4A16_KV_FP8>;
    launch_k(kernel, grid, block, 0, s, kv, k, v);
}

} // namespace

namespace w4a16 {

size_t kv_bytes(const W4A16KvCache *c) {
    return (size_t)c->num_pages * c->kv_heads * c->page_size * c->head_dim * (c->format == W4A16_KV_BF16 ? 2 : 1);
}

size_t kv_scale_bytes(const W4A16KvCache *c) {
    return c->format == W4A16_KV_BF16 ? 0 : (size_t)c->num_pages * c->kv_heads * c->page_size * 4;
}

size_t strided_bytes(long long rows, long long row_stride, long long heads, long long head_stride, int dim) {
    constexpr long long kMost = 1LL << 60;
    if (row_stride < 0 || head_stride < 0 || row_stride % 8 || head_stride % 8) return 0;
    if (rows > 1 && row_stride > kMost / (rows - 1)) return 0;
    if (heads > 1 && head_stride > kMost / (heads - 1)) return 0;
    return ((size_t)(rows - 1) * row_stride + (size_t)(heads - 1) * head_stride + dim) * 2;
}

int kv_check(const W4A16KvCache *c, const W4A16KvBatch *b, const char *what, KvView *view) {
    if (!c || !b) return set_error(W4A16_ERR_CONFIG, "%s: null cache or batch", what);
    if (c->format != W4A16_KV_BF16 && c->format != W4A16_KV_INT8 && c->format != W4A16_KV_FP8)
        return set_error(W4A16_ERR_CONFIG, "%s: cache format %d is none of W4A16_KV_*", what, c->format);
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return set_error(W4A16_ERR_CONFIG, "%s: head_dim=%d is not 64, 128 or 256", what, c->head_dim);
    if (c->page_size < 8 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
        return set_error(W4A16_ERR_CONFIG, "%s: page_size=%d is not a power of two from 8 to 65536", what,
                         c->page_size);
    if (c->kv_heads < 1 || c->kv_heads > 65535 || c->num_pages < 1 ||
        (long long)c->num_pages * c->page_size > INT32_MAX)
        return set_error(W4A16_ERR_CONFIG, "%s: bad extents num_pages=%d page_size=%d kv_heads=%d", what,
                         c->num_pages, c->page_size, c->kv_heads);
    if ((long long)c->kv_heads * c->page_size * c->head_dim * 2 > INT32_MAX)
        return set_error(W4A16_ERR_CONFIG, "%s: a page of kv_heads=%d page_size=%d passes 2 GiB", what, c->kv_heads,
                         c->page_size);
    if (!c->k || !c->v) return set_error(W4A16_ERR_CONFIG, "%s: null cache buffer", what);
    const bool coded = c->format != W4A16_KV_BF16;
    if (coded && (!c->k_scale || !c->v_scale))
        return set_error(W4A16_ERR_CONFIG, "%s: an 8-bit cache without scales", what);
    if (misaligned(c->k) || misaligned(c->v) || (coded && (misaligned(c->k_scale) || misaligned(c->v_scale))))
        return set_error(W4A16_ERR_CONFIG, "%s: cache buffers must be 16-byte aligned", what);
    if (b->seqs < 0 || b->rows < 0 || b->rows > 1 << 25 || b->table_pages < 0 || b->table_stride < b->table_pages || b->max_new < 0 ||
        b->max_kv < 0)
        return set_error(W4A16_ERR_CONFIG, "%s: bad extents seqs=%d rows=%d table_pages=%d table_stride=%d max_new=%d "
                         "max_kv=%d", what, b->seqs, b->rows, b->table_pages, b->table_stride, b->max_new, b->max_kv);
    if (b->seqs > 0 && b->rows > 0) {
        if (!b->kv_lens || !b->starts || (b->table_pages > 0 && !b->page_table))
            return set_error(W4A16_ERR_CONFIG, "%s: null batch array", what);
        if (((uintptr_t)b->kv_lens | (uintptr_t)b->starts | (uintptr_t)b->page_table) & 3)
            return set_error(W4A16_ERR_CONFIG, "%s: batch arrays must be 4-byte aligned", what);
    }
    const int32_t *table = b->page_table;
    int shift = 0;
    while ((1 << shift) < c->page_size) ++shift;
    *view = {c->k, c->v, coded ? c->k_scale : nullptr, coded ? c->v_scale : nullptr, table, b->kv_lens, b->starts,
             c->kv_heads, c->num_pages, shift, (uint32_t)(c->kv_heads * c->page_size), b->seqs, b->rows, b->table_pages, b->table_stride};
    /* positions are 32-bit in the kernels, and so are the tiles' ends behind them */
    if (view->table_pages > (1 << 30) >> shift) view->table_pages = (1 << 30) >> shift;
    return W4A16_OK;
}

} // namespace w4a16

extern "C" int w4a16_kv_write_bf16(const W4A16KvCache *cache, const W4A16KvBatch *batch, const uint16_t *k,
                                   long long k_row_stride, long long k_head_stride, const uint16_t *v,
                                   long long v_row_stride, long long v_head_stride, void *stream) {
    const char *what = "w4a16_kv_write_bf16";
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (st) return st;
    if (kv.rows == 0 || kv.seqs == 0) return W4A16_OK;
    if (!k || !v) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (misaligned(k) || misaligned(v))
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 16-byte aligned", what);
    drop_strides_of_one(kv.rows, &k_row_stride, kv.heads, &k_head_stride);
    drop_strides_of_one(kv.rows, &v_row_stride, kv.heads, &v_head_stride);
    const size_t kb = strided_bytes(kv.rows, k_row_stride, kv.heads, k_head_stride, cache->head_dim);
    const size_t vb = strided_bytes(kv.rows, v_row_stride, kv.heads, v_head_stride, cache->head_dim);
    if (!kb || !vb)
        return set_error(W4A16_ERR_CONFIG, "%s: strides must be multiples of 8 elements from 0", what);
    const size_t cb = kv_bytes(cache), sb = kv_scale_bytes(cache);
    for (const void *dst : {(const void *)cache->k, (const void *)cache->v})
        if (overlap(dst, cb, k, kb) || overlap(dst, cb, v, vb))
            return set_error(W4A16_ERR_CONFIG, "%s: the rows overlap the cache", what);
    for (const void *dst : {(const void *)kv.k_scale, (const void *)kv.v_scale})
        if (overlap(dst, sb, k, kb) || overlap(dst, sb, v, vb))
            return set_error(W4A16_ERR_CONFIG, "%s: the rows overlap the cache's scales", what);
    const struct { const void *p; size_t n; } parts[] = {{cache->k, cb}, {cache->v, cb}, {kv.k_scale, sb}, {kv.v_scale, sb}};
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < i; ++j)
            if (overlap(parts[i].p, parts[i].n, parts[j].p, parts[j].n))
                return set_error(W4A16_ERR_CONFIG, "%s: the cache's keys, values and scales overlap", what);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = cache->head_dim == 64 ? launch_write<64> : cache->head_dim == 128 ? launch_write<128> : launch_write<256>;
    launch(cache->format, kv, k, k_row_stride, k_head_stride, v, v_row_stride, v_head_stride, s);
    return hip_status(hipGetLastError(), "kv write launch");
}

extern "C" int w4a16_kv_read_bf16(const W4A16KvCache *cache, const W4A16KvBatch *batch, uint16_t *k, uint16_t *v,
                                  void *stream) {
    const char *what = "w4a16_kv_read_bf16";
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (st) return st;
    if (kv.rows == 0 || kv.seqs == 0) return W4A16_OK;
    if (!k || !v) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (misaligned(k) || misaligned(v))
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 16-byte aligned", what);
    const size_t n = (size_t)kv.rows * kv.heads * cache->head_dim * 2;
    const size_t cb = kv_bytes(cache), sb = kv_scale_bytes(cache);
    if (overlap(k, n, v, n)) return set_error(W4A16_ERR_CONFIG, "%s: the outputs overlap", what);
    for (const void *dst : {(const void *)k, (const void *)v})
        if (overlap(dst, n, cache->k, cb) || overlap(dst, n, cache->v, cb) || overlap(dst, n, kv.k_scale, sb) ||
            overlap(dst, n, kv.v_scale, sb))
            return set_error(W4A16_ERR_CONFIG, "%s: an output overlaps the cache", what);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = cache->head_dim == 64 ? launch_read<64> : cache->head_dim == 128 ? launch_read<128> : launch_read<256>;
    launch(cache->format, kv, k, v, s);
    return hip_status(hipGetLastError(), "kv read launch");
}
