/*
 * drafts.hip - Verification of drafted tokens against the target's probabilities.
 *
 * A token x drafted from q is taken with probability min(1, p(x) / q(x)); the first that is not is
 * replaced by a draw from max(p - q, 0), after which the sequence's tokens are distributed as if
 * drawn from p. The random numbers are given, so the whole call is a function of its arguments.
 *
 * TREE: the drafted tokens are the nodes of a tree, chosen and not drawn. A node's children are asked in their order; each is taken with
 * the probability that it has among what its refused siblings leave, p(x) / (1 - sum of theirs), and behind the last taken
 * node one token is drawn from its row without its children. Every wave goes through the tree by itself: a
 * lane has a node (four with more than 64) and its probability, all gathered at once, and a step down is ballots and lane reads. A tree of
 * 26 over 151936 words, four of them taken: 5.5 + 3.8 us (none: 5.0 + 4.2); 24 of 40 over 100003, three taken: 9.4 + 4.2 (none: 8.5 + 4.4, and 7.0
 * where the targets stand in a cache); bound as below.
 *
 * Up to kSmall words: one launch of one block a sequence that holds the row's weights in registers.
 * More: two launches. drafts_sum_kernel: every block finds its sequence's first refused token (a few
 * gathers, the same in all of them) and sums one piece of that one row's weights in FP64.
 * drafts_draw_kernel: one block a sequence runs over the pieces' sums to the one in which the
 * running sum passes the drawn threshold, and through that piece alone. Bound by memory for many
 * sequences (two rows of the vocabulary each), by the two launches and their few dependent round
 * trips for few: 64 sequences of 128257 words 17.2 us (66 MB, 3.8 TB/s), one of 151936 7.6 in a
 * graph.
 *
 * The sums are FP64. A weight goes through fewer than 40 additions to the total (16 in its thread, 6 in a
 * wave's scan, up to 16 over the waves, 6 over the pieces) and fewer than 60 to a running sum (up to its piece's
 * start 33, and the piece's scan behind it), one more of each every 2^18 words. Each is off by at most 2^-53 of its own
 * result, which is no more than the total. So the order of the additions decides the drawn index only
 * where a running sum lies within 2^-46 of the total from the threshold.
 */
#include "launch.h"
#include "wave.h"

using namespace w4a16;

namespace {

constexpr int kThreads = 256;
constexpr int kQuads = 4;                     /* of neighbouring weights, a thread's: quad j of thread t is at 4 (256 j + t) */
constexpr int kPiece = kThreads * kQuads * 4; /* weights a block sums */

constexpr int kSmallThreads = 1024, kSmallQuads = 4;
constexpr int kSmall = kSmallThreads * kSmallQuads * 4;

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f4_loose __attribute__((ext_vector_type(4), aligned(4))); /* rows start anywhere */

struct DraftArgs {
    const float *target, *draft;
    long long target_seq, target_row, draft_seq, draft_row;
    const int32_t *draft_tokens, *lens;
    const float *uniforms;
    int32_t *accepted, *tokens;
    double *sums; /* [seqs][pieces][2]: of the weights, of the target's row */
    int2 *found;  /* [seqs]: tokens taken; where one was refused, it (INT32_MIN: none) */
    int steps, vocab, pieces;
    const int32_t *parents; /* TREE: [seqs][steps + 1], as draft_tokens; node 0 is the root. lens: of nodes */
    int32_t *path;
};

constexpr int kNone = INT32_MIN;
constexpr int kMostNodes = 256, kNodeWords = kMostNodes / 64;

/* How many of the sequence's tokens are taken, and the one refused behind them (kNone: all taken):
 * by one wave, 64 tokens at a time. */
__device__ __forceinline__ int taken_of(const DraftArgs &a, int seq, int *refused) {
    const int lane = threadIdx.x & 63;
    /* the first 64 tokens are fetched beside their number, not after it */
    const int asked = a.lens ? a.lens[seq] : a.steps;
    int n = a.steps;
    for (int base = 0; base < n; base += 64) {
        const int i = base + lane;
        bool take = true;
        int x = 0;
        if (i < n) {
            x = a.draft_tokens[(long long)seq * a.steps + i];
            const float u = a.uniforms[(long long)seq * (a.steps + 1) + i];
            const bool inside = (unsigned)x < (unsigned)a.vocab;
            const int at = inside ? x : 0;
            const double p = a.target[seq * a.target_seq + i * a.target_row + at];
            const double q = a.draft ? a.draft[seq * a.draft_seq + i * a.draft_row + at] : 1.0f;
            take = inside && (double)u * q < p;
            x = x == kNone ? -1 : x; /* outside the vocabulary either way */
        }
        if (base == 0) n = asked < 0 ? 0 : asked > a.steps ? a.steps : asked;
        take = take || i >= n;
        const unsigned long long no = __ballot(!take);
        if (no) {
            const int l = __ffsll((long long)no) - 1;
            *refused = __builtin_amdgcn_readlane(x, l);
            return base + l;
        }
    }
    *refused = kNone;
    return n;
}

__device__ __forceinline__ float weight(float w) { return w > 0.0f && w < __builtin_inff() ? w : 0.0f; }

/* The weight of token i in the row that is drawn from, and the target's own. */
__device__ __forceinline__ float rest_of(float p, float q, bool has_q, int i, int chosen) {
    return has_q ? weight(p - q) : i == chosen ? 0.0f : weight(p);
}

/* A tree's nodes, 64 w + lane on a lane. */
struct Nodes {
    int parent[kNodeWords], token[kNodeWords]; /* parent: -1 where there is no node, or none that is reached */
    float p[kNodeWords], u[kNodeWords];        /* p: of the node's token in its parent's row */
};

/* The links and tokens, which are enough to find a node's children. */
__device__ __forceinline__ void load_links(const DraftArgs &a, int seq, Nodes *n) {
    const int lane = threadIdx.x & 63, nodes = a.steps + 1;
    int size = a.lens ? a.lens[seq] : nodes;
    size = size > nodes ? nodes : size;
#pragma unroll
    for (int w = 0; w < kNodeWords; ++w) {
        const int i = 64 * w + lane;
        n->parent[w] = -1;
        n->token[w] = -1;
        if (64 * w < nodes && i < nodes) {
            const long long at = (long long)seq * nodes + i;
            const int parent = a.parents[at];
            n->token[w] = a.draft_tokens[at];
            if (i < size && (unsigned)parent < (unsigned)i) n->parent[w] = parent;
        }
    }
}

/* How many nodes behind the root are taken, and the last of them. RECORD: the path and its tokens are written. */
template <bool RECORD>
__device__ __forceinline__ int walk_tree(const DraftArgs &a, int seq, Nodes *n, int *last) {
    const int lane = threadIdx.x & 63, nodes = a.steps + 1;
    const long long first = (long long)seq * nodes;
    load_links(a, seq, n);
#pragma unroll
    for (int w = 0; w < kNodeWords; ++w) {
        n->p[w] = n->u[w] = 0.0f;
        if (n->parent[w] >= 0) {
            n->u[w] = a.uniforms[first + 64 * w + lane];
            if ((unsigned)n->token[w] < (unsigned)a.vocab)
                n->p[w] = weight(a.target[seq * a.target_seq + n->parent[w] * a.target_row + n->token[w]]);
        }
    }
    int node = 0, taken = 0;
    if (RECORD && threadIdx.x == 0) a.path[first] = 0;
    for (;;) {
        double left = 1.0;
        int next = -1, chosen = 0;
#pragma unroll
        for (int w = 0; w < kNodeWords; ++w) {
            unsigned long long children = __ballot(n->parent[w] == node);
            while (children && next < 0) {
                const int l = __ffsll((long long)children) - 1;
                children &= children - 1;
                const int token = __builtin_amdgcn_readlane(n->token[w], l);
                const float p = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, n->p[w]), l));
                const float u = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, n->u[w]), l));
                /* a token that a sibling before it had is refused with it */
                unsigned long long again = __ballot(n->parent[w] == node && n->token[w] == token) & ((1ULL << l) - 1);
#pragma unroll
                for (int x = 0; x < w; ++x) again |= __ballot(n->parent[x] == node && n->token[x] == token);
                if (again) continue;
                if ((double)u * left < (double)p) {
                    next = 64 * w + l;
                    chosen = token;
                } else {
                    left -= (double)p;
                    left = left > 0.0 ? left : 0.0;
                }
            }
        }
        if (next < 0) break;
        node = next; /* behind its parent: the walk ends */
        ++taken;
        if (RECORD && threadIdx.x == 0) {
            a.path[first + taken] = node;
            a.tokens[first + taken - 1] = chosen;
        }
    }
    *last = node;
    return taken;
}

/* The tokens of a node's children, by the block's first wave; count of them. */
__device__ __forceinline__ void list_children(const Nodes &n, int node, int *list, int *count) {
    const int lane = threadIdx.x & 63;
    if (threadIdx.x >= 64) return;
    int total = 0;
#pragma unroll
    for (int w = 0; w < kNodeWords; ++w) {
        const bool is = n.parent[w] == node;
        const unsigned long long all = __ballot(is);
        if (is) list[total + __popcll(all & ((1ULL << lane) - 1))] = n.token[w];
        total += __popcll(all);
    }
    if (lane == 0) *count = total;
}

/* Weights i .. i + 3 of a row of n; zeros behind it. */
__device__ __forceinline__ f4 load_quad(const float *row, int i, int n) {
    if (i + 4 <= n) return *reinterpret_cast<const f4_loose *>(row + i);
    f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < 3; ++c)
        if (i + c < n) v[c] = row[i + c];
    return v;
}

/* The row drawn from: the target's, what is taken off it, and the one token that is where the
 * drafted one was chosen. */
struct Row {
    const float *p, *q;
    int chosen;
};

__device__ __forceinline__ Row row_of(const DraftArgs &a, int seq, int taken, int refused) {
    Row r = {a.target + seq * a.target_seq + taken * a.target_row, nullptr, -1};
    if (refused != kNone) {
        if (a.draft)
            r.q = a.draft + seq * a.draft_seq + taken * a.draft_row;
        else
            r.chosen = refused;
    }
    return r;
}

/* Takes a list of tokens out of quads of weights, quad j from weight first + j * step on: those of the block's weights from `begin` to
 * `end` are looked at. */
template <int QUADS>
__device__ __forceinline__ void take_out(f4 (&own)[QUADS], int first, int step, int begin, int end, const int *list, int count) {
    for (int i = 0; i < count; ++i) {
        const int token = __builtin_amdgcn_readfirstlane(list[i]);
        if (token < begin || token >= end) continue;
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) own[j][c] = token == first + j * step + c ? 0.0f : own[j][c];
    }
}

/* The block's smallest `mine` and largest `behind`, a wave's first: 64 lanes at one LDS word take turns. */
__device__ __forceinline__ void join_found(int mine, int behind, int *found, int *last) {
    const int first = INT32_MAX - wave_most(INT32_MAX - mine), end = wave_most(behind + 1) - 1;
    if ((threadIdx.x & 63) == 0) {
        if (first != INT32_MAX) atomicMin(found, first);
        if (end >= 0) atomicMax(last, end);
    }
}

/* The block's walk through a sequence's tree: the nodes taken and the last one's row; its children in the list. `writes`: this block
 * writes what is known then. */
__device__ __forceinline__ int walk_by_block(const DraftArgs &a, int seq, bool writes, int *node, int *list, int *count) {
    Nodes n;
    const int taken = writes ? walk_tree<true>(a, seq, &n, node) : walk_tree<false>(a, seq, &n, node);
    list_children(n, *node, list, count);
    if (writes) {
        if (threadIdx.x == 0) a.accepted[seq] = taken;
        for (int i = threadIdx.x; i <= a.steps; i += blockDim.x)
            if (i > taken) a.tokens[(long long)seq * (a.steps + 1) + i] = a.path[(long long)seq * (a.steps + 1) + i] = -1;
    }
    __syncthreads();
    return taken;
}

template <bool TREE>
__global__ __launch_bounds__(kThreads) void drafts_sum_kernel(DraftArgs a) {
    const int seq = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x;
    __shared__ int list[TREE ? kMostNodes : 1], count;
    int refused, taken;
    Row r;
    if constexpr (TREE) {
        taken = walk_by_block(a, seq, piece == 0, &refused, list, &count);
        if (piece == 0 && tid == 0) a.found[seq] = make_int2(taken, refused); /* the last node */
        r = {a.target + seq * a.target_seq + refused * a.target_row, nullptr, -1};
    } else {
        taken = taken_of(a, seq, &refused);
        if (piece == 0) {
            if (tid == 0) {
                a.accepted[seq] = taken;
                a.found[seq] = make_int2(taken, refused);
            }
            for (int i = tid; i <= a.steps; i += kThreads)
                if (i != taken)
                    a.tokens[(long long)seq * (a.steps + 1) + i] =
                        i < taken ? a.draft_tokens[(long long)seq * a.steps + i] : -1;
        }
        r = row_of(a, seq, taken, refused);
    }
    f4 p[kQuads], q[kQuads];
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
        const int i = piece * kPiece + (j * kThreads + tid) * 4;
        p[j] = load_quad(r.p, i, a.vocab);
        q[j] = r.q ? load_quad(r.q, i, a.vocab) : f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    double rest = 0.0, all = 0.0;
    if constexpr (TREE) {
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) all += (double)weight(p[j][c]);
        take_out(p, piece * kPiece + tid * 4, kThreads * 4, piece * kPiece, (piece + 1) * kPiece, list, count);
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) rest += (double)weight(p[j][c]);
    } else {
#pragma unroll
        for (int j = 0; j < kQuads; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = piece * kPiece + (j * kThreads + tid) * 4 + c;
                rest += (double)rest_of(p[j][c], q[j][c], r.q != nullptr, i, r.chosen);
                all += (double)weight(p[j][c]);
            }
    }
    __shared__ double part[2][kThreads / 64];
    rest = wave_sum(rest);
    all = wave_sum(all);
    if ((tid & 63) == 0) {
        part[0][tid >> 6] = rest;
        part[1][tid >> 6] = all;
    }
    __syncthreads();
    if (tid < 2) {
        double s = 0.0;
        for (int w = 0; w < kThreads / 64; ++w) s += part[tid][w];
        a.sums[((long long)seq * a.pieces + piece) * 2 + tid] = s;
    }
}

template <bool TREE>
__global__ __launch_bounds__(kThreads) void drafts_draw_kernel(DraftArgs a) {
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    __shared__ int list[TREE ? kMostNodes : 1], count;
    Nodes n;
    if constexpr (TREE) load_links(a, seq, &n); /* on their way beside what was found */
    const double2 *sums = reinterpret_cast<const double2 *>(a.sums) + (long long)seq * a.pieces;
    const int2 got = a.found[seq];
    const float uniform = a.uniforms[(long long)seq * (a.steps + 1) + (TREE ? 0 : a.steps)];
    /* every wave does the same over the pieces' sums */
    double2 first_sums = lane < a.pieces ? sums[lane] : double2{0.0, 0.0};
    double rest = first_sums.x, all = first_sums.y;
    for (int i = lane + 64; i < a.pieces; i += 64) {
        const double2 s = sums[i];
        rest += s.x;
        all += s.y;
    }
    rest = wave_sum(rest);
    all = wave_sum(all);
    const Row r = TREE ? Row{a.target + seq * a.target_seq + got.y * a.target_row, nullptr, -1} : row_of(a, seq, got.x, got.y);
    const bool which = !(rest > 0.0); /* from the target's own weights */
    const double total = which ? all : rest;
    const double pass = (double)uniform * total;
    int32_t *out = a.tokens + (long long)seq * (a.steps + 1) + got.x;
    if (!(total > 0.0)) {
        if (tid == 0) *out = -1;
        return;
    }
    /* the first piece whose running sum passes, or the last that holds anything */
    double before = 0.0, start = 0.0;
    int piece = -1;
    for (int base = 0; base < a.pieces; base += 64) {
        if (base) first_sums = base + lane < a.pieces ? sums[base + lane] : double2{0.0, 0.0};
        const double v = which ? first_sums.y : first_sums.x;
        const double upto = before + wave_scan(v);
        const unsigned long long here = __ballot(v > 0.0), passing = __ballot(v > 0.0 && upto > pass);
        const unsigned long long pick = passing ? passing & -passing : here ? 1ULL << (63 - __clzll((long long)here)) : 0ULL;
        if (pick) {
            const int l = __ffsll((long long)pick) - 1;
            piece = base + l;
            start = l ? lane_f64(upto, l - 1) : before;
        }
        before = lane_f64(upto, 63);
        if (passing) break;
    }
    /* Through that piece in order: 1024 weights a round j, of them 256 a wave, of them 4 a lane. A
     * quad's running sum is what stands before the piece, the (round, wave) pairs before its own,
     * the lanes before it. */
    f4 own[kQuads], q[kQuads];
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
        const int i = piece * kPiece + (j * kThreads + tid) * 4;
        own[j] = load_quad(r.p, i, a.vocab);
        q[j] = r.q && !which ? load_quad(r.q, i, a.vocab) : f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if constexpr (TREE) {
        list_children(n, got.y, list, &count);
        __syncthreads();
        if (!which) take_out(own, piece * kPiece + tid * 4, kThreads * 4, piece * kPiece, (piece + 1) * kPiece, list, count);
    }
    constexpr int kWaves = kThreads / 64;
    __shared__ double before_of[kQuads * kWaves];
    __shared__ int found, last;
    double upto[kQuads];
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = piece * kPiece + (j * kThreads + tid) * 4 + c;
            own[j][c] = which ? weight(own[j][c]) : rest_of(own[j][c], q[j][c], r.q != nullptr, i, r.chosen);
            sum += (double)own[j][c];
        }
        upto[j] = wave_scan(sum);
        if (lane == 63) before_of[j * kWaves + (tid >> 6)] = upto[j];
        upto[j] -= sum; /* before this quad */
    }
    if (tid == 0) {
        found = INT32_MAX;
        last = -1;
    }
    __syncthreads();
    int mine = INT32_MAX, behind = -1;
    double run_before = start;
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
        double run = run_before + upto[j];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const double of = before_of[j * kWaves + w];
            if (w < (tid >> 6)) run += of;
            run_before += of;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = piece * kPiece + (j * kThreads + tid) * 4 + c;
            run += (double)own[j][c];
            if (own[j][c] > 0.0f) {
                behind = i;
                if (run > pass && mine == INT32_MAX) mine = i;
            }
        }
    }
    join_found(mine, behind, &found, &last);
    __syncthreads();
    if (tid == 0) *out = found != INT32_MAX ? found : last;
}

/* Everything in one block. A quad's place in the order is (round, wave, lane), as above; one wave sums
 * the (round, wave) pairs. */
template <int QUADS, bool TREE>
__global__ __launch_bounds__(kSmallThreads) void drafts_small_kernel(DraftArgs a) {
    constexpr int kWaves = kSmallThreads / 64, kPairs = QUADS * kWaves;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ double sums[2][kWaves], before_of[kPairs];
    __shared__ int found, last, list[TREE ? kMostNodes : 1], count;
    int refused, taken;
    if constexpr (TREE) taken = walk_by_block(a, seq, true, &refused, list, &count);
    else taken = taken_of(a, seq, &refused);
    const float uniform = a.uniforms[(long long)seq * (a.steps + 1) + (TREE ? 0 : a.steps)];
    int32_t *out = a.tokens + (long long)seq * (a.steps + 1);
    if constexpr (!TREE)
        for (int i = tid; i <= a.steps; i += kSmallThreads)
            if (i != taken) out[i] = i < taken ? a.draft_tokens[(long long)seq * a.steps + i] : -1;
    if (tid == 0) {
        if constexpr (!TREE) a.accepted[seq] = taken;
        found = INT32_MAX;
        last = -1;
    }
    Row r;
    if constexpr (TREE) r = {a.target + seq * a.target_seq + refused * a.target_row, nullptr, -1};
    else r = row_of(a, seq, taken, refused);
    f4 own[QUADS];
    double rest = 0.0, all = 0.0;
#pragma unroll
    for (int half = 0; half < QUADS; half += 2) { /* as many rows' loads at a time as there are registers for */
        f4 p[2], q[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = ((half + j) * kSmallThreads + tid) * 4;
            p[j] = load_quad(r.p, i, a.vocab);
            q[j] = r.q ? load_quad(r.q, i, a.vocab) : f4{0.0f, 0.0f, 0.0f, 0.0f};
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int i = ((half + j) * kSmallThreads + tid) * 4 + c;
                own[half + j][c] = rest_of(p[j][c], q[j][c], r.q != nullptr, i, r.chosen);
                if constexpr (!TREE) rest += (double)own[half + j][c];
                all += (double)weight(p[j][c]);
            }
    }
    if constexpr (TREE) {
        take_out(own, tid * 4, kSmallThreads * 4, 0, a.vocab, list, count);
#pragma unroll
        for (int j = 0; j < QUADS; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) rest += (double)own[j][c];
    }
    rest = wave_sum(rest);
    all = wave_sum(all);
    if (lane == 0) {
        sums[0][wave] = rest;
        sums[1][wave] = all;
    }
    __syncthreads();
    rest = all = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        rest += sums[0][w];
        all += sums[1][w];
    }
    const bool which = !(rest > 0.0); /* from the target's own weights */
    const double total = which ? all : rest, pass = (double)uniform * total;
    if (!(total > 0.0)) {
        if (tid == 0) out[taken] = -1;
        return;
    }
    if (which) {
#pragma unroll
        for (int j = 0; j < QUADS; ++j) {
            const f4 p = load_quad(r.p, (j * kSmallThreads + tid) * 4, a.vocab);
#pragma unroll
            for (int c = 0; c < 4; ++c) own[j][c] = weight(p[c]);
        }
    }
    double upto[QUADS];
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        double sum = 0.0;
#pragma unroll
        for (int c = 0; c < 4; ++c) sum += (double)own[j][c];
        upto[j] = wave_scan(sum);
        if (lane == 63) before_of[j * kWaves + wave] = upto[j];
        upto[j] -= sum; /* before this quad */
    }
    __syncthreads();
    if (wave == 0) {
        double before = 0.0;
        for (int base = 0; base < kPairs; base += 64) {
            const double v = base + lane < kPairs ? before_of[base + lane] : 0.0;
            const double to = before + wave_scan(v);
            before = lane_f64(to, 63);
            if (base + lane < kPairs) before_of[base + lane] = to - v;
        }
    }
    __syncthreads();
    int mine = INT32_MAX, behind = -1;
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
        double run = before_of[j * kWaves + wave] + upto[j];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = (j * kSmallThreads + tid) * 4 + c;
            run += (double)own[j][c];
            if (own[j][c] > 0.0f) {
                behind = i;
                if (run > pass && mine == INT32_MAX) mine = i;
            }
        }
    }
    join_found(mine, behind, &found, &last);
    __syncthreads();
    if (tid == 0) out[taken] = found != INT32_MAX ? found : last;
}

template <bool TREE>
void launch_all(const DraftArgs &a, int seqs, hipStream_t s) {
    /* 8000 words: 5.2 us in one launch, as many as a 1000; 16000: 7.0, and 7.6 for two (32000: 7.7),
     * whose second call costs the host 2 more. */
    if (a.vocab <= kSmall) {
        const auto kernel = a.vocab <= kSmall / 2 ? drafts_small_kernel<kSmallQuads / 2, TREE> : drafts_small_kernel<kSmallQuads, TREE>;
        launch_k(kernel, dim3(seqs), dim3(kSmallThreads), 0, s, a);
        return;
    }
    launch_k(drafts_sum_kernel<TREE>, dim3(a.pieces, seqs), dim3(kThreads), 0, s, a);
    launch_k(drafts_draw_kernel<TREE>, dim3(seqs), dim3(kThreads), 0, s, a);
}

} // namespace

extern "C" int w4a16_verify_drafts_workspace(int seqs, int steps, int vocab, size_t *bytes) {
    if (!bytes) return set_error(W4A16_ERR_CONFIG, "w4a16_verify_drafts_workspace: null result");
    if (seqs < 0 || seqs > 65535 || steps < 0 || steps > 65535 || vocab < 1 || vocab > (1 << 28))
        return set_error(W4A16_ERR_CONFIG, "w4a16_verify_drafts: bad extents seqs=%d steps=%d vocab=%d (seqs and steps "
                         "up to 65535, vocab 1 to 2^28)", seqs, steps, vocab);
    *bytes = vocab <= kSmall ? 0 : (size_t)seqs * ((size_t)((vocab + kPiece - 1) / kPiece) * 16 + 16);
    return W4A16_OK;
}

extern "C" int w4a16_verify_drafts_f32(const float *target, long long target_seq_stride, long long target_row_stride,
                                       const float *draft, long long draft_seq_stride, long long draft_row_stride,
                                       const int32_t *draft_tokens, const int32_t *lens, const float *uniforms,
                                       int32_t *accepted, int32_t *tokens, int seqs, int steps, int vocab, void *ws,
                                       size_t ws_bytes, void *stream) {
    const char *what = "w4a16_verify_drafts_f32";
    size_t need = 0;
    int st = w4a16_verify_drafts_workspace(seqs, steps, vocab, &need);
    if (st) return st;
    if (seqs == 0) return W4A16_OK;
    if (!target || !uniforms || !accepted || !tokens || (need && !ws) || (steps > 0 && !draft_tokens))
        return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (((uintptr_t)target | (uintptr_t)draft | (uintptr_t)draft_tokens | (uintptr_t)lens | (uintptr_t)uniforms |
         (uintptr_t)accepted | (uintptr_t)tokens) & 3)
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 4-byte aligned", what);
    if (misaligned(ws)) return set_error(W4A16_ERR_CONFIG, "%s: the workspace must be 16-byte aligned", what);
    if (ws_bytes < need)
        return set_error(W4A16_ERR_CONFIG, "%s: a workspace of %zu bytes, the call needs %zu", what, ws_bytes, need);
    constexpr long long kMost = 1LL << 43;
    for (long long s : {target_seq_stride, target_row_stride, draft_seq_stride, draft_row_stride})
        if (s < 0 || s > kMost) return set_error(W4A16_ERR_CONFIG, "%s: stride %lld outside 0 to 2^43", what, s);
    const size_t one = (size_t)vocab * 4;
    const size_t tb = ((size_t)(seqs - 1) * target_seq_stride + (size_t)steps * target_row_stride) * 4 + one;
    const size_t db = draft && steps > 0
                          ? ((size_t)(seqs - 1) * draft_seq_stride + (size_t)(steps - 1) * draft_row_stride) * 4 + one
                          : 0;
    const size_t out = (size_t)seqs * (steps + 1) * 4, in = (size_t)seqs * steps * 4;
    const struct { const void *p; size_t n; } reads[] = {{target, tb}, {draft, db}, {draft_tokens, in},
                                                         {lens, lens ? (size_t)seqs * 4 : 0}, {uniforms, out}},
        writes[] = {{accepted, (size_t)seqs * 4}, {tokens, out}, {ws, need}};
    for (int i = 0; i < 3; ++i) {
        for (const auto &r : reads)
            if (overlap(writes[i].p, writes[i].n, r.p, r.n))
                return set_error(W4A16_ERR_CONFIG, "%s: an output or the workspace overlaps an input", what);
        for (int j = 0; j < i; ++j)
            if (overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n))
                return set_error(W4A16_ERR_CONFIG, "%s: the outputs and the workspace overlap", what);
    }
    const int pieces = (vocab + kPiece - 1) / kPiece;
    double *const sums = static_cast<double *>(ws);
    const DraftArgs a = {target, steps > 0 ? draft : nullptr, target_seq_stride, target_row_stride, draft_seq_stride,
                         draft_row_stride, draft_tokens, lens, uniforms, accepted, tokens, sums,
                         need ? reinterpret_cast<int2 *>(sums + (size_t)seqs * pieces * 2) : nullptr, steps, vocab, pieces, nullptr, nullptr};
    launch_all<false>(a, seqs, static_cast<hipStream_t>(stream));
    return hip_status(hipGetLastError(), "verify drafts launch");
}

extern "C" int w4a16_verify_tree_workspace(int seqs, int nodes, int vocab, size_t *bytes) {
    if (!bytes) return set_error(W4A16_ERR_CONFIG, "w4a16_verify_tree_workspace: null result");
    if (seqs < 0 || seqs > 65535 || nodes < 1 || nodes > kMostNodes || vocab < 1 || vocab > (1 << 28))
        return set_error(W4A16_ERR_CONFIG, "w4a16_verify_tree: bad extents seqs=%d nodes=%d vocab=%d (seqs up to 65535, nodes 1 to %d, "
                         "vocab 1 to 2^28)", seqs, nodes, vocab, kMostNodes);
    return w4a16_verify_drafts_workspace(seqs, nodes - 1, vocab, bytes);
}

extern "C" int w4a16_verify_tree_f32(const float *target, long long target_seq_stride, long long target_row_stride,
                                     const int32_t *node_tokens, const int32_t *parents, const int32_t *sizes, const float *uniforms,
                                     int32_t *accepted, int32_t *path, int32_t *tokens, int seqs, int nodes, int vocab,
                                     void *ws, size_t ws_bytes, void *stream) {
    const char *what = "w4a16_verify_tree_f32";
    size_t need = 0;
    int st = w4a16_verify_tree_workspace(seqs, nodes, vocab, &need);
    if (st) return st;
    if (seqs == 0) return W4A16_OK;
    if (!target || !node_tokens || !parents || !uniforms || !accepted || !path || !tokens || (need && !ws))
        return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (((uintptr_t)target | (uintptr_t)node_tokens | (uintptr_t)parents | (uintptr_t)sizes | (uintptr_t)uniforms | (uintptr_t)accepted |
         (uintptr_t)path | (uintptr_t)tokens) & 3)
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 4-byte aligned", what);
    if (misaligned(ws)) return set_error(W4A16_ERR_CONFIG, "%s: the workspace must be 16-byte aligned", what);
    if (ws_bytes < need)
        return set_error(W4A16_ERR_CONFIG, "%s: a workspace of %zu bytes, the call needs %zu", what, ws_bytes, need);
    constexpr long long kMost = 1LL << 43;
    for (long long s : {target_seq_stride, target_row_stride})
        if (s < 0 || s > kMost) return set_error(W4A16_ERR_CONFIG, "%s: stride %lld outside 0 to 2^43", what, s);
    const size_t n = (size_t)seqs * 4, each = n * nodes;
    const struct { const void *p; size_t n; } reads[] = {
        {target, ((size_t)(seqs - 1) * target_seq_stride + (size_t)(nodes - 1) * target_row_stride + vocab) * 4},
        {node_tokens, each}, {parents, each}, {sizes, sizes ? n : 0}, {uniforms, each}},
        writes[] = {{accepted, n}, {path, each}, {tokens, each}, {ws, need}};
    for (int i = 0; i < 4; ++i) {
        for (const auto &r : reads)
            if (overlap(writes[i].p, writes[i].n, r.p, r.n))
                return set_error(W4A16_ERR_CONFIG, "%s: an output or the workspace overlaps an input", what);
        for (int j = 0; j < i; ++j)
            if (overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n))
                return set_error(W4A16_ERR_CONFIG, "%s: the outputs and the workspace overlap", what);
    }
    const int pieces = (vocab + kPiece - 1) / kPiece;
    double *const sums = static_cast<double *>(ws);
    const DraftArgs a = {target, nullptr, target_seq_stride, target_row_stride, 0, 0, node_tokens, sizes, uniforms, accepted, tokens, sums,
                         need ? reinterpret_cast<int2 *>(sums + (size_t)seqs * pieces * 2) : nullptr, nodes - 1, vocab, pieces, parents,
                         path};
    launch_all<true>(a, seqs, static_cast<hipStream_t>(stream));
    return hip_status(hipGetLastError(), "verify tree launch");
}
