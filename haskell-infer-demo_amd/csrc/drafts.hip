/*
 * drafts.hip - Verification of drafted tokens against the target's probabilities.
 *
 * A token x drafted from q is taken with probability min(1, p(x) / q(x)); the first that is not is
 * replaced by a draw from max(p - q, 0), after which the sequence's tokens are distributed as if
 * drawn from p. The random numbers are given, so the whole call is a function of its arguments.
 *
 * Two launches. drafts_sum_kernel: every block finds its sequence's first refused token (a few
 * gathers, the same in all of them) and sums one piece of that one row's weights in FP64.
 * drafts_draw_kernel: one block a sequence runs over the pieces' sums to the one in which the
 * running sum passes the drawn threshold, and through that piece alone. Bound by memory for many
 * sequences (two rows of the vocabulary each), by the two launches and their few dependent round
 * trips for few. FP64 sums put the threshold within 2^-52 of its exact place, so that the drawn
 * index does not hang on the order in which a vocabulary's many small weights are added.
 */
#include "launch.h"

using namespace w4a16;

namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 16;
constexpr int kPiece = kThreads * kPerThread; /* weights a block sums */

struct DraftArgs {
    const float *target, *draft;
    long long target_seq, target_row, draft_seq, draft_row;
    const int32_t *draft_tokens, *lens;
    const float *uniforms;
    int32_t *accepted, *tokens;
    double *sums; /* [seqs][pieces][2]: of the weights, of the target's row */
    int steps, vocab, pieces;
};

/* How many of the sequence's tokens are taken, and whether one was refused behind them: by one
 * wave, 64 tokens at a time. */
__device__ __forceinline__ int taken_of(const DraftArgs &a, int seq, int *refused) {
    const int lane = threadIdx.x & 63;
    int n = a.lens ? a.lens[seq] : a.steps;
    n = n < 0 ? 0 : n > a.steps ? a.steps : n;
    for (int base = 0; base < n; base += 64) {
        const int i = base + lane;
        bool take = true;
        if (i < n) {
            const int x = a.draft_tokens[(long long)seq * a.steps + i];
            take = false;
            if ((unsigned)x < (unsigned)a.vocab) {
                const double p = a.target[seq * a.target_seq + i * a.target_row + x];
                const double q = a.draft ? a.draft[seq * a.draft_seq + i * a.draft_row + x] : 1.0f;
                take = (double)a.uniforms[(long long)seq * (a.steps + 1) + i] * q < p;
            }
        }
        const unsigned long long no = __ballot(!take);
        if (no) {
            *refused = 1;
            return base + __ffsll(no) - 1;
        }
    }
    *refused = 0;
    return n;
}

__device__ __forceinline__ float weight(float w) { return w > 0.0f && w < __builtin_inff() ? w : 0.0f; }

/* The weight of token i in the row that is drawn from, and the target's own. */
__device__ __forceinline__ float rest_of(float p, float q, bool has_q, int i, int chosen) {
    return has_q ? weight(p - q) : i == chosen ? 0.0f : weight(p);
}

/* The row drawn from: the target's, what is taken off it, and the one token that is where the
 * drafted one was chosen. */
struct Row {
    const float *p, *q;
    int chosen;
};

__device__ __forceinline__ Row row_of(const DraftArgs &a, int seq, int taken, int refused) {
    Row r = {a.target + seq * a.target_seq + taken * a.target_row, nullptr, -1};
    if (refused) {
        const int x = a.draft_tokens[(long long)seq * a.steps + taken];
        if (a.draft)
            r.q = a.draft + seq * a.draft_seq + taken * a.draft_row;
        else
            r.chosen = x;
    }
    return r;
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 32; m; m /= 2) v += __shfl_xor(v, m);
    return v;
}

/* Sum of v over the lanes up to and with this one. */
__device__ __forceinline__ double wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int m = 1; m < 64; m *= 2) {
        const double o = __shfl_up(v, m);
        if (lane >= m) v += o;
    }
    return v;
}

__global__ __launch_bounds__(kThreads) void drafts_sum_kernel(DraftArgs a) {
    const int seq = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x;
    int refused;
    const int taken = taken_of(a, seq, &refused);
    if (piece == 0) {
        if (tid == 0) a.accepted[seq] = taken;
        for (int i = tid; i <= a.steps; i += kThreads)
            if (i != taken)
                a.tokens[(long long)seq * (a.steps + 1) + i] =
                    i < taken ? a.draft_tokens[(long long)seq * a.steps + i] : -1;
    }
    const Row r = row_of(a, seq, taken, refused);
    float p[kPerThread], q[kPerThread];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = piece * kPiece + j * kThreads + tid;
        p[j] = i < a.vocab ? r.p[i] : 0.0f;
        q[j] = r.q && i < a.vocab ? r.q[i] : 0.0f;
    }
    double rest = 0.0, all = 0.0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = piece * kPiece + j * kThreads + tid;
        rest += (double)rest_of(p[j], q[j], r.q != nullptr, i, r.chosen);
        all += (double)weight(p[j]);
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

__global__ __launch_bounds__(kThreads) void drafts_draw_kernel(DraftArgs a) {
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const double *sums = a.sums + (long long)seq * a.pieces * 2;
    int refused;
    const int taken = taken_of(a, seq, &refused);
    const Row r = row_of(a, seq, taken, refused);
    /* every wave does the same over the pieces' sums */
    double rest = 0.0, all = 0.0;
    for (int i = lane; i < a.pieces; i += 64) {
        rest += sums[2 * i];
        all += sums[2 * i + 1];
    }
    rest = wave_sum(rest);
    all = wave_sum(all);
    const int which = rest > 0.0 ? 0 : 1;
    const double total = which ? all : rest;
    const double pass = (double)a.uniforms[(long long)seq * (a.steps + 1) + a.steps] * total;
    int32_t *out = a.tokens + (long long)seq * (a.steps + 1) + taken;
    if (!(total > 0.0)) {
        if (tid == 0) *out = -1;
        return;
    }
    /* the first piece whose running sum passes, or the last that holds anything */
    double before = 0.0, start = 0.0;
    int piece = -1;
    for (int base = 0; base < a.pieces; base += 64) {
        const double v = base + lane < a.pieces ? sums[2 * (base + lane) + which] : 0.0;
        const double upto = before + wave_scan(v);
        const unsigned long long here = __ballot(v > 0.0), passing = __ballot(v > 0.0 && upto > pass);
        const unsigned long long pick = passing ? passing & -passing : here ? 1ULL << (63 - __clzll(here)) : 0ULL;
        if (pick) {
            const int l = __ffsll(pick) - 1;
            piece = base + l;
            const double previous = l ? __shfl(upto, l - 1) : before;
            start = previous;
        }
        before = __shfl(upto, 63);
        if (passing) break;
    }
    /* through that piece: a thread's own neighbours in order, then the waves, then the block */
    const int first = piece * kPiece + tid * kPerThread;
    double own[kPerThread], sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = first + j;
        float w = 0.0f;
        if (i < a.vocab) w = which ? weight(r.p[i]) : rest_of(r.p[i], r.q ? r.q[i] : 0.0f, r.q != nullptr, i, r.chosen);
        own[j] = w;
        sum += own[j];
    }
    __shared__ double waves[kThreads / 64];
    __shared__ int found, last;
    const double upto = wave_scan(sum);
    if (lane == 63) waves[tid >> 6] = upto;
    if (tid == 0) {
        found = INT32_MAX;
        last = -1;
    }
    __syncthreads();
    double run = start + upto - sum;
    for (int w = 0; w < (tid >> 6); ++w) run += waves[w];
    int mine = INT32_MAX, behind = -1;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        run += own[j];
        if (own[j] > 0.0) {
            behind = first + j;
            if (run > pass && mine == INT32_MAX) mine = first + j;
        }
    }
    if (mine != INT32_MAX) atomicMin(&found, mine);
    if (behind >= 0) atomicMax(&last, behind);
    __syncthreads();
    if (tid == 0) *out = found != INT32_MAX ? found : last;
}

} // namespace

extern "C" int w4a16_verify_drafts_workspace(int seqs, int steps, int vocab, size_t *bytes) {
    if (!bytes) return set_error(W4A16_ERR_CONFIG, "w4a16_verify_drafts_workspace: null result");
    if (seqs < 0 || seqs > 65535 || steps < 0 || steps > 65535 || vocab < 1 || vocab > (1 << 28))
        return set_error(W4A16_ERR_CONFIG, "w4a16_verify_drafts: bad extents seqs=%d steps=%d vocab=%d (seqs and steps "
                         "up to 65535, vocab 1 to 2^28)", seqs, steps, vocab);
    *bytes = (size_t)seqs * ((vocab + kPiece - 1) / kPiece) * 16;
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
    if (!target || !uniforms || !accepted || !tokens || !ws || (steps > 0 && !draft_tokens))
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
    const DraftArgs a = {target, steps > 0 ? draft : nullptr, target_seq_stride, target_row_stride, draft_seq_stride,
                         draft_row_stride, draft_tokens, lens, uniforms, accepted, tokens, static_cast<double *>(ws),
                         steps, vocab, pieces};
    hipStream_t s = static_cast<hipStream_t>(stream);
    launch_k(drafts_sum_kernel, dim3(pieces, seqs), dim3(kThreads), 0, s, a);
    launch_k(drafts_draw_kernel, dim3(seqs), dim3(kThreads), 0, s, a);
    return hip_status(hipGetLastError(), "verify drafts launch");
}
