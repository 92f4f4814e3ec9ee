/*
 * drafts.hip - Verification of drafted tokens against the target's probabilities.
 *
 * A token x drafted from q is taken with probability min(1, p(x) / q(x)); the first that is not is
 * replaced by a draw from max(p - q, 0), after which the sequence's tokens are distributed as if
 * drawn from p. The random numbers are given, so the whole call is a function of its arguments.
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
};

constexpr int kNone = INT32_MIN;

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

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
    const uint2 b = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_update_dpp(0, (int)b.x, CTRL, ROWS, 0xF, false),
                                                 (uint32_t)__builtin_amdgcn_update_dpp(0, (int)b.y, CTRL, ROWS, 0xF, false)));
}

/* Sum of v over the lanes up to and with this one, by VALU moves: row shifts within 16 lanes, then the
 * rows' last lanes carried to the rows behind. */
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_or_zero<0x111, 0xF>(v);
    v += dpp_or_zero<0x112, 0xF>(v);
    v += dpp_or_zero<0x114, 0xF>(v);
    v += dpp_or_zero<0x118, 0xF>(v);
    v += dpp_or_zero<0x142, 0xA>(v); /* row_bcast:15 into rows 1 and 3 */
    v += dpp_or_zero<0x143, 0xC>(v); /* row_bcast:31 into rows 2 and 3 */
    return v;
}

__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint2 b = __builtin_bit_cast(uint2, v);
    return __builtin_bit_cast(double, make_uint2((uint32_t)__builtin_amdgcn_readlane((int)b.x, lane),
                                                 (uint32_t)__builtin_amdgcn_readlane((int)b.y, lane)));
}

/* The block's smallest `mine` and largest `behind`, a wave's first: 64 lanes at one LDS word take turns. */
__device__ __forceinline__ void join_found(int mine, int behind, int *found, int *last) {
    const int first = INT32_MAX - wave_most(INT32_MAX - mine), end = wave_most(behind + 1) - 1;
    if ((threadIdx.x & 63) == 0) {
        if (first != INT32_MAX) atomicMin(found, first);
        if (end >= 0) atomicMax(last, end);
    }
}

__device__ __forceinline__ double wave_sum(double v) { return lane_f64(wave_scan(v), 63); }

__global__ __launch_bounds__(kThreads) void drafts_sum_kernel(DraftArgs a) {
    const int seq = blockIdx.y, piece = blockIdx.x, tid = threadIdx.x;
    int refused;
    const int taken = taken_of(a, seq, &refused);
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
    const Row r = row_of(a, seq, taken, refused);
    f4 p[kQuads], q[kQuads];
#pragma unroll
    for (int j = 0; j < kQuads; ++j) {
        const int i = piece * kPiece + (j * kThreads + tid) * 4;
        p[j] = load_quad(r.p, i, a.vocab);
        q[j] = r.q ? load_quad(r.q, i, a.vocab) : f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    double rest = 0.0, all = 0.0;
#pragma unroll
    for (int j = 0; j < kQuads; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int i = piece * kPiece + (j * kThreads + tid) * 4 + c;
            rest += (double)rest_of(p[j][c], q[j][c], r.q != nullptr, i, r.chosen);
            all += (double)weight(p[j][c]);
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
    const double2 *sums = reinterpret_cast<const double2 *>(a.sums) + (long long)seq * a.pieces;
    const int2 got = a.found[seq];
    const float uniform = a.uniforms[(long long)seq * (a.steps + 1) + a.steps];
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
    const Row r = row_of(a, seq, got.x, got.y);
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
template <int QUADS>
__global__ __launch_bounds__(kSmallThreads) void drafts_small_kernel(DraftArgs a) {
    constexpr int kWaves = kSmallThreads / 64, kPairs = QUADS * kWaves;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ double sums[2][kWaves], before_of[kPairs];
    __shared__ int found, last;
    int refused;
    const int taken = taken_of(a, seq, &refused);
    const float uniform = a.uniforms[(long long)seq * (a.steps + 1) + a.steps];
    int32_t *out = a.tokens + (long long)seq * (a.steps + 1);
    for (int i = tid; i <= a.steps; i += kSmallThreads)
        if (i != taken) out[i] = i < taken ? a.draft_tokens[(long long)seq * a.steps + i] : -1;
    if (tid == 0) {
        a.accepted[seq] = taken;
        found = INT32_MAX;
        last = -1;
    }
    const Row r = row_of(a, seq, taken, refused);
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
                rest += (double)own[half + j][c];
                all += (double)weight(p[j][c]);
            }
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
                         need ? reinterpret_cast<int2 *>(sums + (size_t)seqs * pieces * 2) : nullptr, steps, vocab, pieces};
    hipStream_t s = static_cast<hipStream_t>(stream);
    /* 8000 words: 5.2 us in one launch, as many as a 1000; 16000: 7.0, and 7.6 for two (32000: 7.7),
     * whose second call costs the host 2 more. */
    if (vocab <= kSmall) {
        const auto kernel = vocab <= kSmall / 2 ? drafts_small_kernel<kSmallQuads / 2> : drafts_small_kernel<kSmallQuads>;
        launch_k(kernel, dim3(seqs), dim3(kSmallThreads), 0, s, a);
        return hip_status(hipGetLastError(), "verify drafts launch");
    }
    launch_k(drafts_sum_kernel, dim3(pieces, seqs), dim3(kThreads), 0, s, a);
    launch_k(drafts_draw_kernel, dim3(seqs), dim3(kThreads), 0, s, a);
    return hip_status(hipGetLastError(), "verify drafts launch");
}
