/*
 * tree.hip - Trees of drafted tokens in the paged cache: what each node sees and where it stands, from the trees' links.
 */
#include "kv.h"

using namespace w4a16;

namespace {

constexpr int kMostNodes = 256, kMostWords = kMostNodes / 64;

/*
 * One block a sequence, a thread a node. A node's bits are its own and its parent's, which begin as each node's own: with
 * jump_j the node that many links above, seen_j |= seen_jump_j and jump_j = jump_jump_j doubles the links
 * that are covered, so that 8 rounds cover 256 nodes in a chain. The nodes above are as many as the depth: positions are counts of bits.
 * A launch, three dependent loads and the rounds in LDS: a tree of 26 takes 2.2 us, 16 of 37 3.2, 8 of 251 3.8.
 */
__global__ __launch_bounds__(kMostNodes) void tree_plan_kernel(const int32_t *kv_lens, const int32_t *starts, int rows, const int32_t *parents,
                                                               int parents_stride, const int32_t *sizes, int nodes,
                                                               unsigned long long *seen, int32_t *positions) {
    __shared__ unsigned long long bits[kMostWords][kMostNodes];
    __shared__ int jumps[kMostNodes];
    const int seq = blockIdx.x, tid = threadIdx.x, words = (nodes + 63) >> 6;
    const int first = starts[seq], last = starts[seq + 1];
    int size = sizes ? sizes[seq] : nodes, length = kv_lens[seq];
    int parent = tid < nodes ? parents[(long long)seq * parents_stride + tid] : -1;
    size = size < 0 ? 0 : size > nodes ? nodes : size;
    length = length < 0 ? 0 : length;
    if (first < 0 || last > rows || last <= first) return; /* the same in every thread */
    int jump = parent >= 0 && parent < tid && tid < size ? parent : -1;
    unsigned long long mine[kMostWords];
#pragma unroll
    for (int w = 0; w < kMostWords; ++w) bits[w][tid] = mine[w] = tid >> 6 == w ? 1ULL << (tid & 63) : 0ULL;
    jumps[tid] = jump;
    __syncthreads();
    for (int reach = 1; reach < size; reach *= 2) {
        int next = -1;
        if (jump >= 0) {
#pragma unroll
            for (int w = 0; w < kMostWords; ++w) mine[w] |= bits[w][jump];
            next = jumps[jump];
        }
        __syncthreads();
        if (jump >= 0) {
#pragma unroll
            for (int w = 0; w < kMostWords; ++w) bits[w][tid] = mine[w];
            jumps[tid] = next;
        }
        jump = next;
        __syncthreads();
    }
    const int news = last - first, base = length - size;
    for (int i = tid; i < news; i += kMostNodes) {
        const int node = size - news + i;
        int above = 0;
        for (int w = 0; w < words; ++w) {
            const unsigned long long x = node >= 0 ? bits[w][node] : 0ULL;
            above += __popcll(x);
            seen[(long long)(first + i) * words + w] = x;
        }
        positions[first + i] = node >= 0 ? base + above - 1 : base + node;
    }
}

} // namespace

extern "C" int w4a16_kv_tree_plan(const W4A16KvBatch *b, const int32_t *parents, int parents_stride, const int32_t *sizes,
                                  int nodes, uint64_t *seen, int32_t *positions, void *stream) {
    const char *what = "w4a16_kv_tree_plan";
    if (!b) return set_error(W4A16_ERR_CONFIG, "%s: null batch", what);
    if (b->seqs < 0 || b->rows < 0 || b->rows > 1 << 25)
        return set_error(W4A16_ERR_CONFIG, "%s: bad extents seqs=%d rows=%d", what, b->seqs, b->rows);
    if (nodes < 1 || nodes > kMostNodes) return set_error(W4A16_ERR_CONFIG, "%s: trees of nodes=%d are not of 1 to %d", what, nodes, kMostNodes);
    if (parents_stride < 0) return set_error(W4A16_ERR_CONFIG, "%s: parents_stride=%d is negative", what, parents_stride);
    if (b->seqs == 0 || b->rows == 0) return W4A16_OK;
    if (!b->kv_lens || !b->starts || !parents || !seen || !positions) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if ((((uintptr_t)b->kv_lens | (uintptr_t)b->starts | (uintptr_t)parents | (uintptr_t)sizes | (uintptr_t)positions) & 3) ||
        ((uintptr_t)seen & 7))
        return set_error(W4A16_ERR_CONFIG, "%s: arrays must be 4-byte aligned, the bits 8-byte", what);
    const size_t words = (nodes + 63) / 64, n = (size_t)b->seqs * 4;
    const struct { const void *p; size_t n; } writes[] = {{seen, (size_t)b->rows * words * 8}, {positions, (size_t)b->rows * 4}},
        reads[] = {{b->kv_lens, n}, {b->starts, n + 4}, {sizes, sizes ? n : 0},
                   {parents, ((size_t)(b->seqs - 1) * parents_stride + nodes) * 4}};
    bool clash = overlap(writes[0].p, writes[0].n, writes[1].p, writes[1].n);
    for (const auto &w : writes)
        for (const auto &r : reads) clash = clash || overlap(w.p, w.n, r.p, r.n);
    if (clash) return set_error(W4A16_ERR_CONFIG, "%s: an output overlaps another buffer", what);
    launch_k(tree_plan_kernel, dim3(b->seqs), dim3(kMostNodes), 0, static_cast<hipStream_t>(stream), b->kv_lens, b->starts, b->rows,
             parents, parents_stride, sizes, nodes, (unsigned long long *)seen, positions);
    return hip_status(hipGetLastError(), "tree plan launch");
}
