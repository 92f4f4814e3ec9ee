/*
 * beams.hip - Beam search's step: the best continuations over a group's beams and the vocabulary, and where the beams' caches go on.
 *
 *   candidate (b, v) scores  score_b + x_bv - log sum_w exp(x_bw)
 *
 * beams_scan_kernel reads the logits once: it leaves the sum of each wave's piece of a row and the largest value of every
 * chunk (what a wave loads at once: 256 FP32 values or 512 BF16 ones). beams_pick_kernel, one block a group, has then little to read: the `take`
 * best candidates lie in the `take` best chunks, by their largest values and, where those are equal, their numbers: a
 * candidate outside of them stands behind the largest of each, all of which are better or equal with a lower number. So it
 * picks chunks by their largest values, and candidates out of those.
 *
 * Either pick is of a few out of many: each wave gives a lower bound of the last one that is picked (with 16 waves, the least of their
 * ceil(take / 16)th largest: there are `take` values at or above it), what reaches the bound is collected (not many more than
 * are picked, if the values are not alike), and each of these counts those before it, which is its place. Scores are FP64
 * and numbers unique, so the order is too. Where more are collected than there is room for, which takes rows of equal values, the
 * picks are made one after another instead.
 *
 * The scan is bound by memory: 16 groups of 10 beams, 128257 words in FP32, 16.2 us (82 MB at 5.1 TB/s, a large copy's rate), 94 % of the VALU's
 * cycles beside it. The pick is one block's chain of dependent steps: 8 of 4 beams' words 9.2 us, 40 of 10 beams' 16.4; four BF16 rows of 151936
 * words are scanned in 4.3.
 *
 * Exponentials are FP32 (1.5 * 2^-23 with their product's rounding made good; of FP32 logits' difference from their piece's largest another 2^-22
 * at most, over those of a piece that count), the sums of a load's four or eight too (2^-24 for each of two or three additions), the sums of
 * those FP64: 2^-20 in all.
 */
#include "launch.h"
#include "wave.h"

using namespace w4a16;

namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4_loose __attribute__((ext_vector_type(4), aligned(2))); /* rows start anywhere */

constexpr int kMostTake = 128, kMostBeams = 1024;
constexpr int kScanThreads = 256, kLoads = 4;   /* 16-byte loads of a scanning wave's piece: chunks of it */
constexpr int kPickThreads = 1024, kPickWaves = kPickThreads / 64, kRoom = 512;

constexpr int values_a_load(bool bf16) { return bf16 ? 8 : 4; }
constexpr int chunk_values(bool bf16) { return 64 * values_a_load(bf16); }

struct SelectArgs {
    const void *logits;
    long long group_stride, beam_stride;
    const float *scores;
    int beams, vocab, take, chunks, pieces; /* of a row */
    float *tops;                            /* [groups][beams][chunks] */
    double *sums;                           /* [groups][beams][pieces]: of exp(x - the piece's largest) */
    float *mosts;                           /* [groups][beams][pieces]: the piece's largest, -infinity where it is nothing else */
    float *out_scores;
    int32_t *out_parents, *out_tokens;
};

/* 16 bytes of a row of n values from value i on; -infinity behind it. */
template <bool BF16>
__device__ __forceinline__ u4 load_raw(const void *row, int i, int n) {
    constexpr int kValues = values_a_load(BF16);
    if (i <= n - kValues) return *reinterpret_cast<const u4_loose *>(static_cast<const uint8_t *>(row) + (long long)i * (BF16 ? 2 : 4));
    constexpr uint32_t kLeast = BF16 ? 0xFF80FF80u : 0xFF800000u;
    u4 v = {kLeast, kLeast, kLeast, kLeast};
#pragma unroll
    for (int j = 0; j < kValues; ++j)
        if (i + j < n) {
            if constexpr (BF16) {
                const uint32_t x = static_cast<const uint16_t *>(row)[i + j];
                v[j / 2] = j % 2 ? (v[j / 2] & 0xFFFFu) | x << 16 : (v[j / 2] & 0xFFFF0000u) | x;
            } else {
                v[j] = static_cast<const uint32_t *>(row)[i + j];
            }
        }
    return v;
}

template <bool BF16>
__device__ __forceinline__ float value_of(u4 raw, int j) {
    const uint32_t word = raw[BF16 ? j / 2 : j]; /* an element itself is no operand of a bit cast: it gives the first one */
    return __builtin_bit_cast(float, !BF16 ? word : j % 2 ? word & 0xFFFF0000u : word << 16);
}

template <bool BF16>
__device__ __forceinline__ const void *row_of(const SelectArgs &a, int group, int beam) {
    return static_cast<const uint8_t *>(a.logits) + (group * a.group_stride + beam * a.beam_stride) * (BF16 ? 2 : 4);
}

/* exp(x - most) for x <= most: the product with log2(e) in two parts, the second for what the first rounds off. */
__device__ __forceinline__ float exp_below(float x, float most) {
    constexpr float kHigh = 1.44269502162933349609375f, kLow = 1.92596299112661746887e-8f;
    const float d = fmaxf(x - most, -128.0f); /* its exponential is nothing beside 1 */
    const float high = d * kHigh, low = fmaf(d, kHigh, -high) + d * kLow;
    const float e = __builtin_amdgcn_exp2f(high);
    return fmaf(e, low * 0.693147182464599609375f, e);
}

/* One wave a piece of kLoads chunks. */
template <bool BF16>
__global__ __launch_bounds__(kScanThreads) void beams_scan_kernel(SelectArgs a) {
    constexpr int kValues = values_a_load(BF16), kChunk = chunk_values(BF16);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, beam = blockIdx.y, group = blockIdx.z;
    const int piece = blockIdx.x * (kScanThreads / 64) + wave;
    if (piece >= a.pieces) return;
    const void *row = row_of<BF16>(a, group, beam);
    const long long which = (long long)group * a.beams + beam;
    u4 raw[kLoads];
    float top[kLoads], most = -__builtin_inff();
#pragma unroll
    for (int j = 0; j < kLoads; ++j) raw[j] = load_raw<BF16>(row, (piece * kLoads + j) * kChunk + lane * kValues, a.vocab);
    bool odd = false; /* a NaN, which no maximum sees */
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        top[j] = value_of<BF16>(raw[j], 0);
#pragma unroll
        for (int i = 0; i < kValues; ++i) {
            const float x = value_of<BF16>(raw[j], i);
            top[j] = fmaxf(top[j], x);
            odd = odd | (x != x);
        }
        top[j] = wave_most(top[j]);
        most = fmaxf(most, top[j]);
    }
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        float part[kValues];
#pragma unroll
        for (int i = 0; i < kValues; ++i) part[i] = exp_below(value_of<BF16>(raw[j], i), most);
#pragma unroll
        for (int n = kValues / 2; n > 0; n /= 2)
#pragma unroll
            for (int i = 0; i < n; ++i) part[i] += part[i + n];
        sum += (double)part[0];
    }
    sum = most == -__builtin_inff() ? 0.0 : wave_sum(sum);
    if (__any(odd) || most == __builtin_inff()) sum = __builtin_nan("");
    if (lane == 0) {
        a.sums[which * a.pieces + piece] = sum;
        a.mosts[which * a.pieces + piece] = most;
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
        if (lane == j && piece * kLoads + j < a.chunks) a.tops[which * a.chunks + piece * kLoads + j] = top[j];
}

/* What is picked from: a score and its number, among all of a group. The one is before the other if it scores more, or the
 * same with a lower number. Scores of -infinity and NaN are none. */
struct Entry {
    double score;
    int index;
};

__device__ __forceinline__ bool before(double score, int index, const Entry &than) {
    return score > than.score || (score == than.score && index < than.index);
}

struct PickShared {
    Entry list[kRoom], picked[kMostTake], wave_best[kPickWaves];
    double offsets[kMostBeams];
    float bounds[kPickWaves];
    int count;
};

/* An FP32 number that is not above v: a bound may be less than it need be. */
__device__ __forceinline__ float not_above(double v) {
    const float f = (float)v;
    return f - fabsf(f) * 0x1p-22f - 0x1p-140f;
}

/* The `rank`th largest of the lanes' values, -infinity where there are fewer. */
__device__ __forceinline__ float wave_bound(float mine, int rank) {
    float bound = -__builtin_inff();
    for (int r = 0; r < rank; ++r) {
        bound = wave_most(mine);
        if (!(bound > -__builtin_inff())) break;
        /* one lane of those that have it */
        const unsigned long long have = __ballot(mine == bound);
        if ((int)(threadIdx.x & 63) == __ffsll((long long)have) - 1) mine = -__builtin_inff();
    }
    return bound;
}

/*
 * Picks the `take` first of the entries that each(from, f) gives to f(score, index): all whose score is at least `from`, and others if it
 * likes, in whatever order and on whatever thread, the same ones each time. They come into s.picked in their order; returns how many
 * there are. most(): the largest score of a thread's. The first `waves` waves have all of them, evenly, and `least` is a bound
 * that is known. Called by the whole block; s.picked is its own until the next call.
 */
template <typename MOST, typename EACH>
__device__ __forceinline__ int pick(PickShared &s, int take, int waves, double least, MOST most, EACH each) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, rank = (take + waves - 1) / waves;
    float bound = __builtin_inff();
    if (wave < waves) bound = rank <= 64 ? wave_bound(not_above(most()), rank) : -__builtin_inff();
    if (lane == 0) s.bounds[wave] = bound;
    if (tid == 0) s.count = 0;
    __syncthreads();
    bound = s.bounds[lane % kPickWaves];
    bound = -wave_most(-bound);
    const double from = bound > least ? (double)bound : least;
    if (wave < waves)
        each(from, [&](double score, int index) {
            if (score >= from && score > -__builtin_inf()) {
                const int at = atomicAdd(&s.count, 1);
                if (at < kRoom) s.list[at] = {score, index};
            }
        });
    __syncthreads();
    const int count = s.count;
    if (count <= kRoom) {
        /* eight threads an entry, each with an eighth of the others */
        const int part = tid & 7;
        for (int i0 = 0; i0 < count; i0 += kPickThreads / 8) {
            const int i = i0 + (tid >> 3);
            const Entry own = s.list[i < count ? i : 0];
            int place = 0;
#pragma unroll 4
            for (int j = part; j < count; j += 8) {
                const Entry other = s.list[j];
                place += before(other.score, other.index, own);
            }
            place += __shfl_xor(place, 1);
            place += __shfl_xor(place, 2);
            place += __shfl_xor(place, 4);
            if (part == 0 && i < count && place < take) s.picked[place] = own;
        }
        __syncthreads();
        return count < take ? count : take;
    }
    /* more than there is room for: one after another */
    Entry last = {__builtin_inf(), -1};
    for (int n = 0; n < take; ++n) {
        Entry best = {-__builtin_inf(), INT32_MAX};
        if (wave < waves)
            each(-__builtin_inf(), [&](double score, int index) {
                if (before(last.score, last.index, Entry{score, index}) && before(score, index, best)) best = {score, index};
            });
        for (int m = 1; m < 64; m *= 2) {
            const Entry o = {__shfl_xor(best.score, m), __shfl_xor(best.index, m)};
            if (before(o.score, o.index, best)) best = o;
        }
        if (lane == 0) s.wave_best[wave] = best;
        __syncthreads();
        best = s.wave_best[0];
        for (int w = 1; w < kPickWaves; ++w)
            if (before(s.wave_best[w].score, s.wave_best[w].index, best)) best = s.wave_best[w];
        if (tid == 0) s.picked[n] = best;
        last = best;
        __syncthreads();
        if (!(best.score > -__builtin_inf())) return n;
    }
    return take;
}

template <bool BF16>
__global__ __launch_bounds__(kPickThreads) void beams_pick_kernel(SelectArgs a) {
    constexpr int kValues = values_a_load(BF16), kChunk = chunk_values(BF16), kHeld = 8;
    __shared__ PickShared s;
    const int group = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    /* Chunks, by their numbers in the group: neighbours, which are of one beam, go to different waves. A thread's first ones are on
     * their way from the start. More of them than that are looked at by pieces first, in the same way. */
    const float *tops = a.tops + (long long)group * a.beams * a.chunks, *mosts = a.mosts + (long long)group * a.beams * a.pieces;
    const bool by_pieces = a.beams * a.chunks > kHeld * kPickThreads;
    const float *const of = by_pieces ? mosts : tops;
    const int each_beam = by_pieces ? a.pieces : a.chunks, all = a.beams * each_beam, first = wave + kPickWaves * lane;
    float top[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) top[i] = first + i * kPickThreads < all ? of[first + i * kPickThreads] : -__builtin_inff();
    /* what a beam's logits are moved by: its score less the logarithm of its sum; NaN, which no comparison passes, where it has none */
    for (int b = wave; b < a.beams; b += kPickWaves) {
        const long long which = (long long)group * a.beams + b;
        float most = -__builtin_inff();
        double sum = 0.0; /* of exp(x - most) */
        const double score = a.scores[which];
        for (int p0 = 0; p0 < a.pieces; p0 += 4 * 64) {
            double part[4];
            float of[4], next = most;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int p = p0 + 64 * j + lane;
                part[j] = p < a.pieces ? a.sums[which * a.pieces + p] : 0.0;
                of[j] = p < a.pieces ? a.mosts[which * a.pieces + p] : 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) next = part[j] == 0.0 ? next : fmaxf(next, of[j]);
            next = wave_most(next);
            sum = most == next ? sum : sum * exp((double)most - (double)next);
            most = next;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum += part[j] == 0.0 ? 0.0 : part[j] * exp((double)of[j] - (double)most); /* 0: nothing but -infinity */
        }
        sum = wave_sum(sum);
        const double offset = score - ((double)most + log(sum));
        if (lane == 0) s.offsets[b] = fabs(offset) < __builtin_inf() ? offset : __builtin_nan("");
    }
    __syncthreads();
    double held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int e = first + i * kPickThreads;
        held[i] = e < all ? s.offsets[e / each_beam] + (double)top[i] : -__builtin_inf();
    }
    auto each = [&](double, auto &&f) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) f(held[i], first + i * kPickThreads);
        for (int e = first + kHeld * kPickThreads; e < all; e += kPickThreads) f(s.offsets[e / each_beam] + (double)of[e], e);
    };
    auto largest = [&] {
        double most = -__builtin_inf();
        each(0.0, [&](double score, int) { most = score > most ? score : most; });
        return most;
    };
    int chunks = pick(s, a.take, kPickWaves, -__builtin_inf(), largest, each);
    if (by_pieces) {
        /* the chunks of `chunks` pieces, a thread each */
        static_assert(kMostTake * kLoads <= kPickThreads, "one chunk a thread");
        const double least = chunks == a.take ? s.picked[chunks - 1].score : -__builtin_inf();
        double score = -__builtin_inf();
        int number = 0;
        if (first < chunks * kLoads) {
            const int e = s.picked[first / kLoads].index, beam = e / a.pieces, chunk = (e - beam * a.pieces) * kLoads + first % kLoads;
            number = beam * a.chunks + chunk;
            if (chunk < a.chunks) score = s.offsets[beam] + (double)tops[number];
        }
        __syncthreads();
        chunks = pick(s, a.take, kPickWaves, least, [&] { return score; }, [&](double, auto &&f) { f(score, number); });
    }
    /* Their values: a wave's load is a chunk, all of a wave's on their way at once. The last of `take` chunks' largest value is a bound. */
    const double least = chunks == a.take ? s.picked[chunks - 1].score : -__builtin_inf();
    constexpr int kMost = kMostTake / kPickWaves;
    u4 raw[kMost];
    int base[kMost]; /* number of the lane's first value; -1: none */
    double offset[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int c = wave + i * kPickWaves;
        base[i] = -1;
        if (c < chunks) {
            const int e = s.picked[c].index, beam = e / a.chunks, at = (e - beam * a.chunks) * kChunk + lane * kValues;
            offset[i] = s.offsets[beam];
            base[i] = beam * a.vocab + at;
            raw[i] = load_raw<BF16>(row_of<BF16>(a, group, beam), at, a.vocab);
        }
    }
    float most[kMost]; /* of the lane's values of a chunk; values behind a row's end are -infinity, and never picked */
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        most[i] = -__builtin_inff();
        if (base[i] >= 0)
#pragma unroll
            for (int j = 0; j < kValues; ++j) most[i] = fmaxf(most[i], value_of<BF16>(raw[i], j));
    }
    __syncthreads();
    const int found = pick(
        s, a.take, chunks < kPickWaves ? (chunks ? chunks : 1) : kPickWaves, least,
        [&] {
            double largest = -__builtin_inf();
#pragma unroll
            for (int i = 0; i < kMost; ++i)
                if (base[i] >= 0) {
                    const double score = offset[i] + (double)most[i];
                    largest = score > largest ? score : largest;
                }
            return largest;
        },
        [&](double from, auto &&f) {
#pragma unroll
            for (int i = 0; i < kMost; ++i)
                if (base[i] >= 0 && offset[i] + (double)most[i] >= from)
#pragma unroll
                    for (int j = 0; j < kValues; ++j) {
                        u4 own = raw[i];
                        asm volatile("" : "+v"(own)); /* or scores are kept for where they are needed again, in more registers than there are */
                        const double score = offset[i] + (double)value_of<BF16>(own, j);
                        if (score >= from) f(score, base[i] + j);
                    }
        });
    for (int i = tid; i < a.take; i += kPickThreads) {
        const bool real = i < found;
        const Entry own = s.picked[real ? i : 0];
        const int parent = own.index / a.vocab;
        const long long to = (long long)group * a.take + i;
        a.out_scores[to] = real ? (float)own.score : -__builtin_inff();
        a.out_parents[to] = real ? parent : -1;
        a.out_tokens[to] = real ? own.index - parent * a.vocab : -1;
    }
}

template <bool BF16>
void launch_select(const SelectArgs &a, int groups, hipStream_t s) {
    constexpr int kWaves = kScanThreads / 64;
    launch_k(beams_scan_kernel<BF16>, dim3((a.pieces + kWaves - 1) / kWaves, a.beams, groups), dim3(kScanThreads), 0, s, a);
    launch_k(beams_pick_kernel<BF16>, dim3(groups), dim3(kPickThreads), 0, s, a);
}

} // namespace

namespace {

int select(const char *what, bool bf16, const void *logits, long long group_stride, long long beam_stride, const float *scores, int groups,
           int beams, int vocab, int take, float *out_scores, int32_t *parents, int32_t *tokens, void *ws, size_t ws_bytes, void *stream) {
    size_t need = 0;
    int st = w4a16_beam_select_workspace(groups, beams, vocab, &need);
    if (st) return st;
    if (take < 1 || take > kMostTake) return set_error(W4A16_ERR_CONFIG, "%s: take=%d is not 1 to %d", what, take, kMostTake);
    if (groups == 0) return W4A16_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens || !ws) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (((uintptr_t)logits & (bf16 ? 1 : 3)) ||
        (((uintptr_t)scores | (uintptr_t)out_scores | (uintptr_t)parents | (uintptr_t)tokens) & 3))
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 4-byte aligned (BF16 logits: 2)", what);
    if (misaligned(ws)) return set_error(W4A16_ERR_CONFIG, "%s: the workspace must be 16-byte aligned", what);
    if (ws_bytes < need)
        return set_error(W4A16_ERR_CONFIG, "%s: a workspace of %zu bytes, the call needs %zu", what, ws_bytes, need);
    constexpr long long kMost = 1LL << 43;
    for (long long x : {group_stride, beam_stride})
        if (x < 0 || x > kMost) return set_error(W4A16_ERR_CONFIG, "%s: stride %lld outside 0 to 2^43", what, x);
    const size_t size = bf16 ? 2 : 4, out = (size_t)groups * take * 4;
    const struct { const void *p; size_t n; } reads[] = {
        {logits, ((size_t)(groups - 1) * group_stride + (size_t)(beams - 1) * beam_stride + vocab) * size},
        {scores, (size_t)groups * beams * 4}}, writes[] = {{out_scores, out}, {parents, out}, {tokens, out}, {ws, need}};
    bool clash = false;
    for (int i = 0; i < 4; ++i) {
        for (const auto &r : reads) clash = clash || overlap(writes[i].p, writes[i].n, r.p, r.n);
        for (int j = 0; j < i; ++j) clash = clash || overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n);
    }
    if (clash) return set_error(W4A16_ERR_CONFIG, "%s: an output or the workspace overlaps another buffer", what);
    SelectArgs a;
    a.logits = logits;
    a.group_stride = group_stride;
    a.beam_stride = beam_stride;
    a.scores = scores;
    a.beams = beams;
    a.vocab = vocab;
    a.take = take;
    a.chunks = (vocab - 1) / chunk_values(bf16) + 1;
    a.pieces = (a.chunks + kLoads - 1) / kLoads;
    const size_t rows = (size_t)groups * beams;
    a.sums = static_cast<double *>(ws);
    a.mosts = reinterpret_cast<float *>(a.sums + rows * a.pieces);
    a.tops = a.mosts + rows * a.pieces;
    a.out_scores = out_scores;
    a.out_parents = parents;
    a.out_tokens = tokens;
    (bf16 ? launch_select<true> : launch_select<false>)(a, groups, static_cast<hipStream_t>(stream));
    return hip_status(hipGetLastError(), "beam select launch");
}

} // namespace

extern "C" int w4a16_beam_select_workspace(int groups, int beams, int vocab, size_t *bytes) {
    if (!bytes) return set_error(W4A16_ERR_CONFIG, "w4a16_beam_select_workspace: null result");
    if (groups < 0 || groups > 65535 || beams < 1 || beams > kMostBeams || vocab < 1 || (long long)beams * vocab > INT32_MAX)
        return set_error(W4A16_ERR_CONFIG, "w4a16_beam_select: bad extents groups=%d beams=%d vocab=%d (groups up to 65535, beams 1 to "
                         "%d, beams * vocab up to 2^31 - 1)", groups, beams, vocab, kMostBeams);
    /* of FP32 logits, whose chunks are the smaller */
    const size_t chunks = ((size_t)vocab + chunk_values(false) - 1) / chunk_values(false), pieces = (chunks + kLoads - 1) / kLoads;
    *bytes = (size_t)groups * beams * (pieces * 12 + chunks * 4);
    return W4A16_OK;
}

extern "C" int w4a16_beam_select_f32(const float *logits, long long group_stride, long long beam_stride, const float *scores, int groups,
                                     int beams, int vocab, int take, float *out_scores, int32_t *parents, int32_t *tokens,
                                     void *ws, size_t ws_bytes, void *stream) {
    return select("w4a16_beam_select_f32", false, logits, group_stride, beam_stride, scores, groups, beams, vocab, take, out_scores, parents,
                  tokens, ws, ws_bytes, stream);
}

extern "C" int w4a16_beam_select_bf16(const uint16_t *logits, long long group_stride, long long beam_stride, const float *scores,
                                      int groups, int beams, int vocab, int take, float *out_scores, int32_t *parents,
                                      int32_t *tokens, void *ws, size_t ws_bytes, void *stream) {
    return select("w4a16_beam_select_bf16", true, logits, group_stride, beam_stride, scores, groups, beams, vocab, take, out_scores, parents,
                  tokens, ws, ws_bytes, stream);
}
