/*
 * kv_move.hip - Tokens that move inside the paged cache: a tree's path to the front of its tokens, and beams that go on from their
 * parents: their tables, and the last pages that they cannot share. Bytes are moved as they are, codes with their scales.
 */
#include "kv.h"

using namespace w4a16;

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

/* The page of a token, or -1 where there is none. */
__device__ __forceinline__ int page_of(const KvView &kv, int seq, int at) {
    if (at < 0 || (at >> kv.shift) >= kv.table_pages) return -1;
    const int page = kv.table[(long long)seq * kv.table_stride + (at >> kv.shift)];
    return (unsigned)page < (unsigned)kv.pages ? page : -1;
}

/*
 * One wave a sequence, head and matrix: K or V. Token j of the sequence's new ones takes what token from[j] >= j holds. A wave
 * goes through them in their order, kAhead loads and then as many stores: what a later one takes stands behind everything that was
 * stored so far, so nothing is overwritten before it is taken. A few tokens a sequence: four dependent loads (starts, the path,
 * the pages, the rows) are what it takes: one path of 26 nodes of which four are kept and three move, BF16, 3.7 us (2.8 where none moves); 24 of
 * 40 of which two move each, FP8, 4.3 (3.7).
 */
template <int BYTES> /* of a token's row of one head */
__global__ __launch_bounds__(256) void keep_path_kernel(KvView kv, const int32_t *path, int width) {
    constexpr int kLanes = BYTES / 16, kTokens = 64 / kLanes, kAhead = 4;
    const int seq = blockIdx.x, lane = threadIdx.x & 63, pair = blockIdx.y * 4 + (threadIdx.x >> 6), head = pair >> 1;
    if (head >= kv.heads) return;
    const int first = kv.starts[seq], last = kv.starts[seq + 1];
    if (first < 0 || last > kv.rows || last <= first) return;
    const int news = last - first, old = kv_length(kv, seq) - news, sub = lane % kLanes, most = width < news ? width : news;
    uint8_t *codes = static_cast<uint8_t *>(pair & 1 ? kv.v : kv.k);
    float *scales = pair & 1 ? kv.v_scale : kv.k_scale;
    auto slot = [&](int page, int at) { return (((long long)page * kv.heads + head) << kv.shift) + (at & ((1 << kv.shift) - 1)); };
    for (int j0 = 0; j0 < most; j0 += kAhead * kTokens) {
        u4 row[kAhead];
        float scale[kAhead];
        long long to[kAhead];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int j = j0 + n * kTokens + lane / kLanes;
            const int from = j < most ? path[(long long)seq * width + j] : -1;
            to[n] = -1;
            if (from > j && from < news) {
                const int here = page_of(kv, seq, old + j), there = page_of(kv, seq, old + from);
                if (here >= 0 && there >= 0) {
                    to[n] = slot(here, old + j);
                    const long long of = slot(there, old + from);
                    row[n] = *reinterpret_cast<const u4 *>(codes + of * BYTES + sub * 16);
                    if (scales && sub == 0) scale[n] = scales[of];
                }
            }
        }
#pragma unroll
        for (int n = 0; n < kAhead; ++n)
            if (to[n] >= 0) {
                *reinterpret_cast<u4 *>(codes + to[n] * BYTES + sub * 16) = row[n];
                if (scales && sub == 0) scales[to[n]] = scale[n];
            }
    }
}

/* The tokens of a sequence's last page, as far as it is filled, from another sequence's, whose length is the same: a head's
 * are one run of memory. A block a sequence, head and matrix, bound by its dependent loads: 16 groups of 8 beams, 8 heads of 128, BF16, pages of
 * 64, 6.1 us (up to 17 MB move, 3.4 us of memory's time). */
template <int BYTES>
__global__ __launch_bounds__(256) void copy_tails_kernel(KvView kv, const int32_t *source) {
    const int seq = blockIdx.x, head = blockIdx.y >> 1, from = source[seq];
    if ((unsigned)from >= (unsigned)kv.seqs || from == seq) return;
    const int length = kv_length(kv, seq), tail = length & ((1 << kv.shift) - 1);
    const int to_page = page_of(kv, seq, length), page = page_of(kv, from, length);
    if (to_page < 0 || page < 0 || to_page == page) return;
    const long long to = ((long long)to_page * kv.heads + head) << kv.shift, of = ((long long)page * kv.heads + head) << kv.shift;
    uint8_t *codes = static_cast<uint8_t *>(blockIdx.y & 1 ? kv.v : kv.k);
    float *scales = blockIdx.y & 1 ? kv.v_scale : kv.k_scale;
    const u4 *src = reinterpret_cast<const u4 *>(codes + of * BYTES);
    u4 *dst = reinterpret_cast<u4 *>(codes + to * BYTES);
    const int n = tail * (BYTES / 16);
    for (int i0 = threadIdx.x; i0 < n; i0 += 4 * 256) {
        u4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * 256 < n) x[j] = src[i0 + j * 256];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (i0 + j * 256 < n) dst[i0 + j * 256] = x[j];
    }
    if (scales)
        for (int i = threadIdx.x; i < tail; i += 256) scales[to + i] = scales[of + i];
}

constexpr int kMostBeams = 1024;

/*
 * A group of beams goes on from its parents. Full pages are shared: their entries are the parent's. The pages from the first that is not
 * full on are a beam's own: the first child of a parent goes on with the parent's, and the other children take those of the
 * beams that no one goes on from, the nth the nth's; there are as many of the one as of the other. So only the latter have
 * anything to copy, and out of pages that no one writes to. A block's dependent steps: 16 groups of 8 beams and 47 pages 3.8 us.
 */
__global__ __launch_bounds__(256) void beam_tables_kernel(const int32_t *table, int stride, int pages, const int32_t *kv_lens,
                                                          const int32_t *parents, int beams, int shift, int32_t *to, int to_stride,
                                                          int32_t *source) {
    __shared__ int parent[kMostBeams], keeper[kMostBeams], own[kMostBeams], gone[kMostBeams];
    const int group = blockIdx.x, tid = threadIdx.x;
    const long long first = (long long)group * beams;
    for (int b = tid; b < beams; b += 256) {
        const int p = parents[first + b];
        parent[b] = (unsigned)p < (unsigned)beams ? p : b;
        keeper[b] = beams;
    }
    __syncthreads();
    for (int b = tid; b < beams; b += 256) atomicMin(&keeper[parent[b]], b);
    __syncthreads();
    if (tid < 64) {
        int n = 0;
        for (int b0 = 0; b0 < beams; b0 += 64) {
            const bool is = b0 + tid < beams && keeper[b0 + tid] == beams;
            const unsigned long long all = __ballot(is);
            if (is) gone[n + __popcll(all & ((1ULL << tid) - 1))] = b0 + tid;
            n += __popcll(all);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        n = 0;
        for (int b0 = 0; b0 < beams; b0 += 64) {
            const int b = b0 + tid;
            const bool real = b < beams, is = real && keeper[parent[b]] != b;
            const unsigned long long all = __ballot(is);
            if (real) own[b] = is ? gone[n + __popcll(all & ((1ULL << tid) - 1))] : parent[b];
            n += __popcll(all);
        }
    }
    __syncthreads();
    if (blockIdx.y == 0)
        for (int b = tid; b < beams; b += 256) source[first + b] = keeper[parent[b]] == b ? -1 : (int)first + keeper[parent[b]];
    const int length = kv_lens[first], full = length < 0 ? 0 : length >> shift;
    for (long long i = blockIdx.y * 256 + tid; i < (long long)beams * pages; i += 256 * gridDim.y) {
        const int b = (int)(i / pages), page = (int)(i - (long long)b * pages);
        to[(first + b) * to_stride + page] = table[(first + (page < full ? parent[b] : own[b])) * stride + page];
    }
}

int cache_parts_apart(const W4A16KvCache *cache, const KvView &kv, const void *p, size_t n, const char *name, const char *what) {
    const size_t cb = kv_bytes(cache), sb = kv_scale_bytes(cache);
    const struct { const void *p; size_t n; } parts[] = {{cache->k, cb}, {cache->v, cb}, {kv.k_scale, sb}, {kv.v_scale, sb}};
    for (int i = 0; i < 4; ++i) {
        if (overlap(parts[i].p, parts[i].n, p, n)) return set_error(W4A16_ERR_CONFIG, "%s: %s overlaps the cache", what, name);
        for (int j = 0; j < i; ++j)
            if (overlap(parts[i].p, parts[i].n, parts[j].p, parts[j].n))
                return set_error(W4A16_ERR_CONFIG, "%s: the cache's keys, values and scales overlap", what);
    }
    return W4A16_OK;
}

/* A head's row of the cache in bytes: 64 to 512. */
int row_bytes(const W4A16KvCache *cache) { return cache->head_dim * (cache->format == W4A16_KV_BF16 ? 2 : 1); }

} // namespace

extern "C" int w4a16_kv_keep_path(const W4A16KvCache *cache, const W4A16KvBatch *batch, const int32_t *path, int width, void *stream) {
    const char *what = "w4a16_kv_keep_path";
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (st) return st;
    if (width < 0) return set_error(W4A16_ERR_CONFIG, "%s: width=%d is negative", what, width);
    if (kv.rows == 0 || kv.seqs == 0 || width == 0) return W4A16_OK;
    if (!path) return set_error(W4A16_ERR_CONFIG, "%s: null path", what);
    if ((uintptr_t)path & 3) return set_error(W4A16_ERR_CONFIG, "%s: the path must be 4-byte aligned", what);
    st = cache_parts_apart(cache, kv, path, (size_t)kv.seqs * width * 4, "the path", what);
    if (st) return st;
    const dim3 grid(kv.seqs, (2 * kv.heads + 3) / 4), block(256);
    const int bytes = row_bytes(cache);
    const auto kernel = bytes == 64    ? keep_path_kernel<64>
                        : bytes == 128 ? keep_path_kernel<128>
                        : bytes == 256 ? keep_path_kernel<256>
                                       : keep_path_kernel<512>;
    launch_k(kernel, grid, block, 0, static_cast<hipStream_t>(stream), kv, path, width);
    return hip_status(hipGetLastError(), "keep path launch");
}

extern "C" int w4a16_kv_copy_tails(const W4A16KvCache *cache, const int32_t *page_table, int table_stride, int table_pages,
                                   const int32_t *kv_lens, const int32_t *source, int seqs, void *stream) {
    const char *what = "w4a16_kv_copy_tails";
    W4A16KvBatch batch = {page_table, kv_lens, nullptr, seqs, 0, table_pages, table_stride, 0, 0};
    KvView kv;
    int st = kv_check(cache, &batch, what, &kv);
    if (st) return st;
    if (kv.heads > 32767) return set_error(W4A16_ERR_CONFIG, "%s: kv_heads=%d: at most 32767", what, kv.heads);
    if (seqs == 0 || table_pages == 0) return W4A16_OK;
    if (!page_table || !kv_lens || !source) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (((uintptr_t)page_table | (uintptr_t)kv_lens | (uintptr_t)source) & 3)
        return set_error(W4A16_ERR_CONFIG, "%s: arrays must be 4-byte aligned", what);
    const size_t n = (size_t)seqs * 4;
    st = cache_parts_apart(cache, kv, source, n, "the source", what);
    if (!st) st = cache_parts_apart(cache, kv, kv_lens, n, "kv_lens", what);
    if (!st) st = cache_parts_apart(cache, kv, page_table, ((size_t)(seqs - 1) * table_stride + table_pages) * 4, "the table", what);
    if (st) return st;
    const dim3 grid(seqs, 2 * kv.heads), block(256);
    const int bytes = row_bytes(cache);
    const auto kernel = bytes == 64    ? copy_tails_kernel<64>
                        : bytes == 128 ? copy_tails_kernel<128>
                        : bytes == 256 ? copy_tails_kernel<256>
                                       : copy_tails_kernel<512>;
    launch_k(kernel, grid, block, 0, static_cast<hipStream_t>(stream), kv, source);
    return hip_status(hipGetLastError(), "copy tails launch");
}

extern "C" int w4a16_beam_tables(const int32_t *page_table, int table_stride, int table_pages, const int32_t *kv_lens,
                                 const int32_t *parents, int groups, int beams, int page_size, int32_t *new_table, int new_stride,
                                 int32_t *source, void *stream) {
    const char *what = "w4a16_beam_tables";
    if (groups < 0 || groups > 65535 || beams < 1 || beams > kMostBeams || (long long)groups * beams > INT32_MAX / 2 || table_pages < 0 ||
        table_stride < table_pages || new_stride < table_pages)
        return set_error(W4A16_ERR_CONFIG, "%s: bad extents groups=%d beams=%d (1 to %d) table_pages=%d table_stride=%d new_stride=%d", what,
                         groups, beams, kMostBeams, table_pages, table_stride, new_stride);
    if (page_size < 8 || page_size > 65536 || (page_size & (page_size - 1)))
        return set_error(W4A16_ERR_CONFIG, "%s: page_size=%d is not a power of two from 8 to 65536", what, page_size);
    if (groups == 0) return W4A16_OK;
    if (!kv_lens || !parents || !source || (table_pages && (!page_table || !new_table)))
        return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (((uintptr_t)page_table | (uintptr_t)kv_lens | (uintptr_t)parents | (uintptr_t)new_table | (uintptr_t)source) & 3)
        return set_error(W4A16_ERR_CONFIG, "%s: arrays must be 4-byte aligned", what);
    const size_t seqs = (size_t)groups * beams;
    auto extent = [&](long long stride) { return table_pages ? ((seqs - 1) * (size_t)stride + table_pages) * 4 : 0; };
    const struct { const void *p; size_t n; } writes[] = {{new_table, extent(new_stride)}, {source, seqs * 4}},
        reads[] = {{page_table, extent(table_stride)}, {kv_lens, seqs * 4}, {parents, seqs * 4}};
    bool clash = overlap(writes[0].p, writes[0].n, writes[1].p, writes[1].n);
    for (const auto &w : writes)
        for (const auto &r : reads) clash = clash || overlap(w.p, w.n, r.p, r.n);
    if (clash) return set_error(W4A16_ERR_CONFIG, "%s: an output overlaps another buffer", what);
    int shift = 0;
    while ((1 << shift) < page_size) ++shift;
    /* a block for every 1024 entries, at most 64 of them a group */
    const long long parts = ((long long)beams * table_pages + 1023) / 1024;
    launch_k(beam_tables_kernel, dim3(groups, parts < 1 ? 1 : parts > 64 ? 64 : (unsigned)parts), dim3(256), 0,
             static_cast<hipStream_t>(stream), page_table, table_stride, table_pages, kv_lens, parents, beams, shift, new_table, new_stride,
             source);
    return hip_status(hipGetLastError(), "beam tables launch");
}
