/*
 * kv.h - The paged cache and the batch as kernels see them, and the checks of both (kv_cache.hip).
 */
#ifndef W4A16_KV_H
#define W4A16_KV_H

#include "common.h"
#include "launch.h"

namespace w4a16 {

struct KvView {
    void *k, *v;
    float *k_scale, *v_scale;
    const int32_t *table, *kv_lens, *starts;
    int heads, pages, shift; /* page_size = 1 << shift */
    uint32_t page_tokens;    /* heads << shift: rows of a page, under 2^31 bytes of them */
    int seqs, rows, table_pages, table_stride;
};

/* Refuses what the kernels do not take; *view is filled otherwise. */
int kv_check(const W4A16KvCache *cache, const W4A16KvBatch *batch, const char *what, KvView *view);

/* Bytes from the first to the last element of a [rows][heads][dim] tensor of 2-byte elements; 0 if
 * its strides are not the multiples of 8 from 0 that the kernels' 16-byte moves need, or if their
 * sums pass 62 bits. */
size_t strided_bytes(long long rows, long long row_stride, long long heads, long long head_stride,
                     int dim);

/* An axis of one has no stride: whatever its caller's says is 0 from here on. */
inline void drop_strides_of_one(int rows, long long *row_stride, int heads, long long *head_stride) {
    if (rows == 1) *row_stride = 0;
    if (heads == 1) *head_stride = 0;
}

/* Bytes of one of the cache's code and scale buffers. */
size_t kv_bytes(const W4A16KvCache *cache);
size_t kv_scale_bytes(const W4A16KvCache *cache);

} // namespace w4a16

#ifdef __HIPCC__

namespace w4a16 {

typedef __bf16 kv_bf2 __attribute__((ext_vector_type(2)));
typedef float kv_f2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t kv_pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(kv_f2{a, b}, kv_bf2));
}

/* Codes 2 * HALF and 2 * HALF + 1 of a dword as BF16 pairs: both formats' codes are BF16 values. */
template <int FMT, int HALF>
__device__ __forceinline__ uint32_t kv_widen(uint32_t codes) {
    if constexpr (FMT == W4A16_KV_FP8) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, HALF));
    } else {
        return kv_pack_bf16((float)(int8_t)(codes >> (16 * HALF)), (float)(int8_t)(codes >> (16 * HALF + 8)));
    }
}

/* Tokens of sequence s: its rows are the last of them, whether the cache has room for them or not. */
__device__ __forceinline__ int kv_length(const KvView &kv, int s) {
    const int n = kv.kv_lens[s];
    return n < 0 ? 0 : n;
}

/* Of `length` tokens those that the table has room for: the keys that may be there. */
__device__ __forceinline__ int kv_held(const KvView &kv, int length) {
    const int room = kv.table_pages << kv.shift; /* up to 2^30 */
    return length > room ? room : length;
}

} // namespace w4a16

#endif

#endif /* W4A16_KV_H */
