/*
 * kv_cache.hip - Writing rows of keys and values into the paged cache, turned by their positions and
 * quantised on the way, and reading them back; the checks of a cache and a batch.
 */
#include "kv.h"

using namespace w4a16;

namespace {

constexpr float kSmallest = 0x1p-117f; /* 448 / kSmallest is still finite in FP32 */

/* The sequence of a row and its place in the cache: found by a whole wave, the same on all lanes.
 * The sequences whose rows end at or before `row` are counted 64 at a time. */
struct Place {
    int seq, page, inside; /* seq < 0: no sequence's row; page < 0: a row without a place */
    int at;                /* the row's token in its sequence */
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
    if (before >= kv.seqs) return {-1, -1, 0, 0};
    const int first = kv.starts[before], last = kv.starts[before + 1];
    if (row < first || row >= last) return {-1, -1, 0, 0};
    /* kv_lens and the number of rows may be anything up to 2^31: the difference in 64 bits */
    const long long at = (long long)kv.kv_lens[before] - last + row;
    if (at < 0 || (at >> kv.shift) >= kv.table_pages) return {before, -1, 0, (int)at};
    const int page = kv.table[(long long)before * kv.table_stride + (at >> kv.shift)];
    if ((unsigned)page >= (unsigned)kv.pages) return {before, -1, 0, (int)at};
    return {before, page, (int)(at & ((1 << kv.shift) - 1)), (int)at};
}

/* The largest of v over groups of N lanes (8, 16 or 32). */
template <int N>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
    for (int m = 1; m < N; m *= 2) v = fmaxf(v, __shfl_xor(v, m));
    return v;
}

/* A lane's eight of a row's values as codes, and the row's scale. `most`: the largest of them in size, infinity if one is
 * none that is finite. The scale and its inverse are each one division a row, and a value costs a product
 * and a conversion. */
template <int FMT, int LANES>
__device__ __forceinline__ float encode(float (&f)[8], float most, uint32_t (&out)[2]) {
    constexpr float kTop = FMT == W4A16_KV_INT8 ? 127.0f : 448.0f;
    most = group_max<LANES>(most);
    const bool held = most >= kSmallest && most < __builtin_inff();
    const float inverse = held ? kTop / most : 0.0f;
    out[0] = out[1] = 0u;
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
    return held ? most / kTop : most < kSmallest ? 0.0f : __builtin_nanf("");
}

/* One wave a row of K (blockIdx.y = 0) or V (1): D / 8 lanes a head, eight values a lane. Bound by
 * memory: a row is read once with 16 bytes a lane and its codes are written once. The row's
 * largest value is found over the head's lanes by shuffles. 8198 rows of 8 heads of 128 to FP8:
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
            uint32_t out[2];
            const float scale = encode<FMT, kLanes>(f, finite ? most : __builtin_inff(), out);
            *reinterpret_cast<uint2 *>(static_cast<uint8_t *>(codes) + slot * D + part) =
                make_uint2(out[0], out[1]);
            if (lane % kLanes == 0) scales[slot] = scale;
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

/*
 * Keys turned by their positions and quantised, values quantised, queries turned: y = R(position * inv_freq) x.
 *
 * One wave a row and part of its heads. The row's angles are worked out first, one or two pairs a lane, into
 * a table of the wave's own in LDS, from which a lane takes the four pairs that it turns in
 * every head: the sines of a row cost 1 / heads of what they would beside each value. An angle is
 * reduced in FP64 to a part of a turn (position * inv_freq is exact to 2^-53, so at 2^30 to 2^-23), and
 * from there FP32 is enough. A head has D / 8 lanes of eight values; in halves a lane has four values of the one and
 * their partners of the other, so that a turn stays in its registers and q_out may be q.
 *
 * Work beyond the row's place comes in steps of 64 lanes (1 KiB): heads of K, of V, of q, in this order, kAhead of them on
 * their way at a time.
 *
 * Bound by memory: 8198 rows of 32 queries and 8 keys of 128, BF16, 40 us, 203 MB at 5.0 TB/s (a large copy's rate). 592 rows
 * of 24 + 4 heads of 256, INT8, 6.2 us; four rows 3.8, a launch and four dependent round trips.
 */
struct AppendArgs {
    const uint16_t *k, *v, *q;
    uint16_t *q_out;
    long long k_row, k_head, v_row, v_head, q_row, q_head, o_row, o_head;
    const float *inv_freq;
    const int32_t *positions;
    int q_heads, pairs, interleaved;
};

constexpr double kTurns = 0.15915494309189535; /* 1 / (2 pi) */

template <int D, int FMT>
__global__ __launch_bounds__(256) void kv_append_kernel(KvView kv, AppendArgs a) {
    constexpr int kLanes = D / 8, kHeads = 64 / kLanes, kAhead = 4;
    __shared__ float2 turns[4][D / 2];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, row = blockIdx.x * 4 + wave, sub = lane % kLanes;
    if (row >= kv.rows) return;
    const Place at = find_place(kv, row);
    if (at.seq < 0) return;
    const double position = a.positions ? a.positions[row] : at.at;
    for (int i = lane; i < a.pairs; i += 64) {
        const double turn = position * (double)a.inv_freq[i] * kTurns;
        float s, c;
        sincospif(2.0f * (float)(turn - __builtin_rint(turn)), &s, &c);
        turns[wave][i] = make_float2(c, s);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* the wave's own table: no other reads it */
    const bool turned = 4 * sub < a.pairs;
    float c[4], s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = turns[wave][turned ? 4 * sub + i : 0];
        c[i] = t.x;
        s[i] = t.y;
    }
    /* this lane's values of a head: four from `first` and four from `second` */
    const int first = a.interleaved ? 8 * sub : turned ? 4 * sub : 2 * a.pairs + 8 * (sub - a.pairs / 4);
    const int second = a.interleaved || !turned ? first + 4 : first + a.pairs;
    const int of_kv = (kv.heads + kHeads - 1) / kHeads, of_q = (a.q_heads + kHeads - 1) / kHeads, steps = 2 * of_kv + of_q;
    for (int step0 = blockIdx.y; step0 < steps; step0 += kAhead * gridDim.y) {
        uint2 x[kAhead][2];
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int step = step0 + n * gridDim.y;
            const int which = step < of_kv ? 0 : step < 2 * of_kv ? 1 : 2;
            const int h = (step - which * of_kv) * kHeads + lane / kLanes;
            x[n][0] = x[n][1] = make_uint2(0u, 0u);
            if (step < steps && h < (which == 2 ? a.q_heads : kv.heads)) {
                const uint16_t *from = which == 0   ? a.k + row * a.k_row + h * a.k_head
                                       : which == 1 ? a.v + row * a.v_row + h * a.v_head
                                                    : a.q + row * a.q_row + h * a.q_head;
                x[n][0] = *reinterpret_cast<const uint2 *>(from + first);
                x[n][1] = *reinterpret_cast<const uint2 *>(from + second);
            }
        }
#pragma unroll
        for (int n = 0; n < kAhead; ++n) {
            const int step = step0 + n * gridDim.y;
            if (step >= steps) break;
            const int which = step < of_kv ? 0 : step < 2 * of_kv ? 1 : 2;
            const int h = (step - which * of_kv) * kHeads + lane / kLanes;
            const bool is_v = which == 1;
            if (which < 2 && at.page < 0) continue;
            const uint32_t w[4] = {x[n][0].x, x[n][0].y, x[n][1].x, x[n][1].y};
            float f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                f[2 * i] = __builtin_bit_cast(float, w[i] << 16);
                f[2 * i + 1] = __builtin_bit_cast(float, w[i] & 0xFFFF0000u);
            }
            float y[8];
            auto turn = [&] {
                if (a.interleaved) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[2 * i] = f[2 * i] * c[i] - f[2 * i + 1] * s[i];
                        y[2 * i + 1] = f[2 * i + 1] * c[i] + f[2 * i] * s[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        y[i] = f[i] * c[i] - f[4 + i] * s[i];
                        y[4 + i] = f[4 + i] * c[i] + f[i] * s[i];
                    }
                }
            };
            if (FMT != W4A16_KV_BF16 && !is_v) {
                turn();
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = turned ? y[i] : f[i];
            }
            if (which == 2 || FMT == W4A16_KV_BF16) {
                if (h >= (which == 2 ? a.q_heads : kv.heads)) continue;
                const long long slot = (((long long)at.page * kv.heads + h) << kv.shift) + at.inside;
                uint16_t *to = which == 2 ? a.q_out + row * a.o_row + h * a.o_head
                                          : static_cast<uint16_t *>(is_v ? kv.v : kv.k) + slot * D;
                uint32_t o[4] = {w[0], w[1], w[2], w[3]}; /* what is not turned goes as it came: a conversion would quiet a NaN */
                if (!is_v) {
                    if constexpr (FMT == W4A16_KV_BF16) turn();
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] = turned ? kv_pack_bf16(y[2 * i], y[2 * i + 1]) : w[i];
                }
                *reinterpret_cast<uint2 *>(to + first) = make_uint2(o[0], o[1]);
                *reinterpret_cast<uint2 *>(to + second) = make_uint2(o[2], o[3]);
            } else {
                float most = 0.0f;
                bool finite = true;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    finite = finite && fabsf(f[i]) < __builtin_inff();
                    most = fmaxf(most, fabsf(f[i]));
                }
                uint32_t out[2];
                const float scale = encode<FMT, kLanes>(f, finite ? most : __builtin_inff(), out);
                if (h >= kv.heads) continue;
                const long long slot = (((long long)at.page * kv.heads + h) << kv.shift) + at.inside;
                uint8_t *to = static_cast<uint8_t *>(is_v ? kv.v : kv.k) + slot * D;
                *reinterpret_cast<uint32_t *>(to + first) = out[0];
                *reinterpret_cast<uint32_t *>(to + second) = out[1];
                if (sub == 0) (is_v ? kv.v_scale : kv.k_scale)[slot] = scale;
            }
        }
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
void launch_append(int format, const KvView &kv, const AppendArgs &a, hipStream_t s) {
    constexpr int kHeads = 512 / D;
    const int steps = 2 * ((kv.heads + kHeads - 1) / kHeads) + (a.q_heads + kHeads - 1) / kHeads;
    /* Every step a wave of its own where there are few rows; where there are many, a wave's angles serve all of its steps. 32 + 8 + 8 heads of
     * 128, BF16, one wave a row, four, a step each (12): 4 rows 7.5, 3.8, 3.1 us; 2048 rows 12.0, 10.0, 13.9; 8192 rows 33.4, 33.2, 43.5. */
    const int blocks = (kv.rows + 3) / 4, most = (8 * device_cus() + blocks - 1) / blocks;
    const dim3 grid(blocks, steps < most ? steps : most), block(256);
    auto kernel = format == W4A16_KV_BF16   ? kv_append_kernel<D, W4A16_KV_BF16>
                  : format == W4A16_KV_INT8 ? kv_append_kernel<D, W4A16_KV_INT8>
                                            : kv_append_kernel<D, W4A16_KV_FP8>;
    launch_k(kernel, grid, block, 0, s, kv, a);
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

bool rows_apart(int rows, const RowsView &x, int dim) {
    const long long by_row = (long long)(x.heads - 1) * x.head + dim, by_head = (long long)(rows - 1) * x.row + dim;
    return ((x.heads == 1 || x.head >= dim) && (rows == 1 || x.row >= by_row)) ||
           ((rows == 1 || x.row >= dim) && (x.heads == 1 || x.head >= by_head));
}

bool rows_beside(int rows, const RowsView &x, const RowsView &y, int dim) {
    if (!overlap(x.p, x.bytes, y.p, y.bytes)) return true;
    if (x.row != y.row || rows == 1) return false;
    const long long off = ((const uint8_t *)x.p - (const uint8_t *)y.p) / 2;
    const long long x_wide = (long long)(x.heads - 1) * x.head + dim, y_wide = (long long)(y.heads - 1) * y.head + dim;
    return off > 0 ? off >= y_wide && off + x_wide <= x.row : off < 0 && -off >= x_wide && -off + y_wide <= x.row;
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

namespace {

/* Rows that are read share no memory with the cache, nor its parts with each other. */
int check_apart(const W4A16KvCache *cache, const KvView &kv, const void *k, size_t kb, const void *v, size_t vb, const char *what) {
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
    return W4A16_OK;
}

} // namespace

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
    st = check_apart(cache, kv, k, kb, v, vb, what);
    if (st) return st;
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

extern "C" int w4a16_kv_append_rope_bf16(const W4A16KvCache *cache, const W4A16KvBatch *batch, const uint16_t *k,
                                         long long k_row_stride, long long k_head_stride, const uint16_t *v,
                                         long long v_row_stride, long long v_head_stride, const uint16_t *q,
                                         long long q_row_stride, long long q_head_stride, int q_heads, uint16_t *q_out,
                                         long long q_out_row_stride, long long q_out_head_stride,
                                         const float *inv_freq, int rotary_dim, int interleaved,
                                         const int32_t *positions, void *stream) {
    const char *what = "w4a16_kv_append_rope_bf16";
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (st) return st;
    const int dim = cache->head_dim;
    if (rotary_dim < 8 || rotary_dim > dim || rotary_dim % 8)
        return set_error(W4A16_ERR_CONFIG, "%s: rotary_dim=%d is no multiple of 8 from 8 to head_dim=%d", what, rotary_dim, dim);
    if (q_heads < 0 || q_heads > 65535 || (q == nullptr) != (q_heads == 0) || (q == nullptr) != (q_out == nullptr))
        return set_error(W4A16_ERR_CONFIG, "%s: q_heads=%d (0 to 65535) for queries that are %s and %s", what, q_heads,
                         q ? "given" : "null", q_out ? "wanted" : "not");
    if (kv.rows == 0 || kv.seqs == 0) return W4A16_OK;
    if (!k || !v || !inv_freq) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (misaligned(k) || misaligned(v) || misaligned(q) || misaligned(q_out))
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 16-byte aligned", what);
    if (((uintptr_t)inv_freq | (uintptr_t)positions) & 3)
        return set_error(W4A16_ERR_CONFIG, "%s: inv_freq and positions must be 4-byte aligned", what);
    drop_strides_of_one(kv.rows, &k_row_stride, kv.heads, &k_head_stride);
    drop_strides_of_one(kv.rows, &v_row_stride, kv.heads, &v_head_stride);
    const size_t kb = strided_bytes(kv.rows, k_row_stride, kv.heads, k_head_stride, dim);
    const size_t vb = strided_bytes(kv.rows, v_row_stride, kv.heads, v_head_stride, dim);
    size_t qb = 0, ob = 0;
    if (q) {
        drop_strides_of_one(kv.rows, &q_row_stride, q_heads, &q_head_stride);
        drop_strides_of_one(kv.rows, &q_out_row_stride, q_heads, &q_out_head_stride);
        qb = strided_bytes(kv.rows, q_row_stride, q_heads, q_head_stride, dim);
        ob = strided_bytes(kv.rows, q_out_row_stride, q_heads, q_out_head_stride, dim);
    }
    if (!kb || !vb || (q && (!qb || !ob)))
        return set_error(W4A16_ERR_CONFIG, "%s: strides must be multiples of 8 elements from 0", what);
    st = check_apart(cache, kv, k, kb, v, vb, what);
    if (st) return st;
    const size_t cb = kv_bytes(cache), sb = kv_scale_bytes(cache), fb = (size_t)rotary_dim * 2,
                 pb = positions ? (size_t)kv.rows * 4 : 0;
    const struct { const void *p; size_t n; } held[] = {{cache->k, cb}, {cache->v, cb}, {kv.k_scale, sb}, {kv.v_scale, sb}},
        others[] = {{q, qb}, {inv_freq, fb}, {positions, pb}, {q_out, ob}};
    for (const auto &h : held)
        for (const auto &o : others)
            if (overlap(h.p, h.n, o.p, o.n))
                return set_error(W4A16_ERR_CONFIG, "%s: queries, frequencies or positions overlap the cache", what);
    if (q) {
        const RowsView kr = {k, kb, k_row_stride, k_head_stride, kv.heads}, vr = {v, vb, v_row_stride, v_head_stride, kv.heads},
                       qr = {q, qb, q_row_stride, q_head_stride, q_heads},
                       out = {q_out, ob, q_out_row_stride, q_out_head_stride, q_heads};
        if (!rows_apart(kv.rows, out, dim)) return set_error(W4A16_ERR_CONFIG, "%s: output rows overlap each other", what);
        if ((!rows_same(out, qr) && !rows_beside(kv.rows, out, qr, dim)) || !rows_beside(kv.rows, out, kr, dim) ||
            !rows_beside(kv.rows, out, vr, dim) || overlap(q_out, ob, inv_freq, fb) || overlap(q_out, ob, positions, pb))
            return set_error(W4A16_ERR_CONFIG, "%s: q_out overlaps another tensor of the call", what);
    }
    const AppendArgs a = {k, v, q, q_out, k_row_stride, k_head_stride, v_row_stride, v_head_stride, q_row_stride, q_head_stride,
                          q_out_row_stride, q_out_head_stride, inv_freq, positions, q_heads, rotary_dim / 2, interleaved != 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = dim == 64 ? launch_append<64> : dim == 128 ? launch_append<128> : launch_append<256>;
    launch(cache->format, kv, a, s);
    return hip_status(hipGetLastError(), "kv append launch");
}
