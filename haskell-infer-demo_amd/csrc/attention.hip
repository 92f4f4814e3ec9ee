/*
 * attention.hip - Attention of a batch's new tokens over the paged cache.
 *
 *   out_i = sum_j p_ij v_j / l_i,  p_ij = exp(s_ij - m_i),  l_i = sum_j p_ij,  s_ij = scale <q_i, k_j>
 *
 * in one pass over the keys with a running maximum m and sum l (FP32, in units of log 2). The
 * query heads that share a key head are rows of one tile, (token, head) in order, so a key is
 * read once for all of them.
 *
 * Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, so that a lane's column is
 * a row of the tile in both: the weights leave the first product in the registers that the
 * second takes them from, and the statistics of a row are a lane's own but for the exchange
 * between the lane groups that hold its other tokens. The order of the tokens inside a product is
 * free as long as both operands keep it, which is what makes the two layouts meet.
 *
 * An 8-bit cache's codes are BF16 values; their scales multiply the scores (K) and the weights (V)
 * in FP32.
 */
#include "kv.h"

using namespace w4a16;

namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
    KvView kv;
    const uint16_t *q;
    uint16_t *out;
    float *lse, *ws;
    long long q_row, q_head, out_row, out_head;
    int group, q_heads, causal, window;
    int splits, items;
    float scale; /* times log2(e) */
};

constexpr int kFewestTokens = 256; /* of a split */
constexpr float kLn2 = 0.69314718055994531f;

/* What a tile's block works on: a sequence, its rows in the tile, the keys that any of them
 * sees and its own split of those. The same on every lane. */
struct Tile {
    int first_row;          /* the sequence's first row in q */
    int rows, news;         /* (token, head) rows of the tile from `start`; the sequence's new tokens */
    int start;              /* first (token, head) row of the tile in the sequence */
    int length;             /* the sequence's cached tokens */
    int lo, hi;             /* keys that some row sees: [lo, hi) */
    int all_lo, all_hi;     /* keys that every row sees */
    int begin, end, active; /* this split's keys; how many splits have any */
    int window;             /* 0 where it cuts nothing */
    int seq;
};

/* Finds the `item`th tile of RM rows: the sequences' tiles are counted 64 sequences at a time.
 * Sequences whose rows do not lie in the call's tensors have none. */
template <int RM>
__device__ __forceinline__ bool find_tile(const AttnArgs &a, int item, int split, Tile *t) {
    const int lane = threadIdx.x & 63;
    int left = item;
    for (int base = 0; base < a.kv.seqs; base += 64) {
        const int s = base + lane;
        int first = 0, news = 0;
        if (s < a.kv.seqs) {
            first = a.kv.starts[s];
            const int last = a.kv.starts[s + 1];
            if (first >= 0 && last <= a.kv.rows && last > first) news = last - first;
        }
        const int tiles = (news * a.group + RM - 1) / RM;
        int upto = tiles;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            const int o = __shfl_up(upto, m);
            if (lane >= m) upto += o;
        }
        const unsigned long long here = __ballot(upto > left);
        if (here) {
            const int l = __ffsll(here) - 1;
            t->seq = base + l;
            t->first_row = __builtin_amdgcn_readlane(first, l);
            t->news = __builtin_amdgcn_readlane(news, l);
            t->start = (left - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l))) * RM;
            break;
        }
        left -= __builtin_amdgcn_readlane(upto, 63);
        if (base + 64 >= a.kv.seqs) return false;
    }
    t->seq = __builtin_amdgcn_readfirstlane(t->seq);
    const int all = t->news * a.group;
    t->rows = all - t->start < RM ? all - t->start : RM;
    t->length = __builtin_amdgcn_readfirstlane(kv_length(a.kv, t->seq));
    const int t0 = t->start / a.group, t1 = (t->start + t->rows - 1) / a.group, old = t->length - t->news;
    t->window = a.window <= t->length ? a.window : 0;
    t->hi = a.causal ? old + t1 + 1 : t->length;
    t->all_hi = a.causal ? old + t0 + 1 : t->length;
    t->lo = t->window ? old + t0 - t->window + 1 : 0;
    t->all_lo = t->window ? old + t1 - t->window + 1 : 0;
    if (t->lo < 0) t->lo = 0;
    if (t->hi < t->lo) t->hi = t->lo;
    /* splits begin at multiples of 32 tokens and have at least kFewestTokens */
    const int from = t->lo & ~31, span = t->hi - from;
    int per = (span + a.splits - 1) / a.splits;
    per = (per + 127) & ~127;
    if (per < kFewestTokens) per = kFewestTokens;
    t->active = (span + per - 1) / per;
    if (t->active < 1) t->active = 1;
    t->begin = from + split * per;
    t->end = t->begin + per < t->hi ? t->begin + per : t->hi;
    return true;
}

/* max of v and its value in lanes l ^ 16, l ^ 32 (as the sums of kernels.hip by lane swaps). */
__device__ __forceinline__ float lane_max16(float v) {
    float x = v, y = v;
    asm volatile("s_nop 1\n v_permlane16_swap_b32 %0, %1\n s_nop 1" : "+v"(x), "+v"(y));
    return fmaxf(x, y);
}
__device__ __forceinline__ float lane_max32(float v) {
    float x = v, y = v;
    asm volatile("s_nop 1\n v_permlane32_swap_b32 %0, %1\n s_nop 1" : "+v"(x), "+v"(y));
    return fmaxf(x, y);
}
__device__ __forceinline__ float lane_sum16(float v) {
    float x = v, y = v;
    asm volatile("s_nop 1\n v_permlane16_swap_b32 %0, %1\n s_nop 1" : "+v"(x), "+v"(y));
    return x + y;
}
__device__ __forceinline__ float lane_sum32(float v) {
    float x = v, y = v;
    asm volatile("s_nop 1\n v_permlane32_swap_b32 %0, %1\n s_nop 1" : "+v"(x), "+v"(y));
    return x + y;
}

__device__ __forceinline__ bf8 as_bf8(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(bf8, make_uint4(a, b, c, d));
}

__device__ __forceinline__ bool nonfinite2(uint32_t pair) {
    return (pair & 0x7F80u) == 0x7F80u || (pair & 0x7F800000u) == 0x7F800000u;
}

/* Where a partial result of (tile item, key head, split) stands in the workspace: RM rows of D
 * values, then RM pairs (m, l). */
template <int D, int RM>
__device__ __forceinline__ float *partial_of(const AttnArgs &a, int item, int head, int split) {
    return a.ws + (((long long)item * a.kv.heads + head) * a.splits + split) * (RM * (D + 2));
}

/*
 * Few rows: a block of four waves has RT tiles of 16 rows and one split of the keys; its waves
 * take 32 tokens at a time in turn, each with statistics of its own, and are joined in LDS at the
 * end. K and V go from memory into the registers that the products take them from; no LDS in the
 * loop.
 *
 * v_mfma_f32_16x16x32_bf16. K: a lane's row is token l % 16 of two groups of 16, its values the
 * 8 or 16 that lane group g = l / 16 has of each step. S^T gives a lane tokens 16 a + 4 g + i of row
 * l % 16, and those are the eight that it holds of P^T (a, i from 0 to 1, 3) and has to load of V^T: 16
 * lanes load a token's whole row, E = D / 16 values each, which stand at E neighbouring
 * columns; a transposition of 8 tokens x 2 values at a time by byte permutations makes them the
 * operand of value e's product.
 */
template <int D, int FMT, int RT>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
    constexpr int RM = 16 * RT, E = D / 16, KS = D / 32; /* values of V a lane has; steps of the K product */
    constexpr bool kCoded = FMT != W4A16_KV_BF16;
    constexpr int kVWords = kCoded ? E / 4 : E / 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.kv.heads, item = blockIdx.x / a.kv.heads, split = blockIdx.y;
    Tile t;
    if (!find_tile<RM>(a, item, split, &t)) return;
    if (split >= t.active) return;

    /* this lane's rows: their queries as the products' operand, and the keys they see */
    bf8 q[RT][KS];
    int lo[RT], hi[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int i = r * 16 + n, token = (t.start + i) / a.group, h = head * a.group + (t.start + i) % a.group;
        const bool real = i < t.rows;
        const int place = t.length - t.news + token;
        hi[r] = !real ? 0 : a.causal ? place + 1 : t.length;
        lo[r] = t.window ? place - t.window + 1 : 0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = kCoded ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
            uint4 x = make_uint4(0u, 0u, 0u, 0u);
            if (real) x = *reinterpret_cast<const uint4 *>(a.q + (t.first_row + token) * a.q_row + h * a.q_head + d);
            q[r][s] = __builtin_bit_cast(bf8, x);
        }
    }

    f4 acc[RT][E];
    float m[RT], l[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        m[r] = -__builtin_inff();
        l[r] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const int32_t *table = a.kv.table + (long long)t.seq * a.kv.table_stride;
    const int mask = (1 << a.kv.shift) - 1;
    for (int t0 = t.begin + 32 * wave; t0 < t.end; t0 += 128) {
        /* pages of this lane's K tokens and V tokens (page sizes are multiples of 8, so four
         * neighbours from a multiple of 4 share one); tokens out of range read token 0 of page 0
         * and are masked below */
        long long kslot[2], vslot[2];
        bool there[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int kt = t0 + 16 * c + n, vt = t0 + 16 * c + 4 * g;
            const int kp = kt < t.length ? table[kt >> a.kv.shift] : -1;
            const int vp = vt < t.length ? table[vt >> a.kv.shift] : -1;
            const bool kin = (unsigned)kp < (unsigned)a.kv.pages;
            there[c] = (unsigned)vp < (unsigned)a.kv.pages;
            kslot[c] = kin ? (((long long)kp * a.kv.heads + head) << a.kv.shift) + (kt & mask) : 0;
            vslot[c] = there[c] ? (((long long)vp * a.kv.heads + head) << a.kv.shift) + (vt & mask) : 0;
        }
        /* K */
        bf8 k[2][KS];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if constexpr (kCoded) {
                const uint8_t *p = static_cast<const uint8_t *>(a.kv.k) + kslot[c] * D + 16 * g;
#pragma unroll
                for (int s = 0; s < KS / 2; ++s) {
                    const uint4 x = *reinterpret_cast<const uint4 *>(p + 64 * s);
                    k[c][2 * s] = as_bf8(kv_widen<FMT, 0>(x.x), kv_widen<FMT, 1>(x.x), kv_widen<FMT, 0>(x.y), kv_widen<FMT, 1>(x.y));
                    k[c][2 * s + 1] = as_bf8(kv_widen<FMT, 0>(x.z), kv_widen<FMT, 1>(x.z), kv_widen<FMT, 0>(x.w), kv_widen<FMT, 1>(x.w));
                }
            } else {
                const uint16_t *p = static_cast<const uint16_t *>(a.kv.k) + kslot[c] * D + 8 * g;
#pragma unroll
                for (int s = 0; s < KS; ++s) k[c][s] = *reinterpret_cast<const bf8 *>(p + 32 * s);
            }
        }
        /* V: tokens vt, vt + 1, .. of both groups, E values of each */
        uint32_t v[8][kVWords];
        f4 ks[2], vs[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t *p = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(a.kv.v) +
                                        (vslot[c] + i) * (kCoded ? D : 2 * D)) + n * kVWords;
#pragma unroll
                for (int w = 0; w < kVWords; ++w) v[4 * c + i][w] = p[w];
            }
            if constexpr (kCoded) {
                ks[c] = *reinterpret_cast<const f4 *>(a.kv.k_scale + vslot[c]) * a.scale;
                vs[c] = *reinterpret_cast<const f4 *>(a.kv.v_scale + vslot[c]);
            }
        }
        /* tokens that some row does not see, or that are not there: their V is not multiplied */
        const bool cut = t0 < t.all_lo || t0 + 32 > t.all_hi || __any(!there[0] || !there[1]);
        bool odd = false;
        if (cut) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = t0 + 16 * c + 4 * g + i;
                    if (!there[c] || at < t.lo || at >= t.hi)
#pragma unroll
                        for (int w = 0; w < kVWords; ++w) v[4 * c + i][w] = 0u;
                    if constexpr (!kCoded)
#pragma unroll
                        for (int w = 0; w < kVWords; ++w) odd = odd || nonfinite2(v[4 * c + i][w]);
                }
            odd = __any(odd);
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            f4 s[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                s[c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KS; ++j) s[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[c][j], q[r][j], s[c], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[c][i] *= kCoded ? ks[c][i] : a.scale;
                    if (cut) {
                        const int at = t0 + 16 * c + 4 * g + i;
                        if (!there[c] || at < lo[r] || at >= hi[r]) s[c][i] = -__builtin_inff();
                    }
                }
            }
            float most = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                               fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
            most = lane_max32(lane_max16(most));
            const float next = fmaxf(m[r], most);
            const float base = next == -__builtin_inff() ? 0.0f : next;
            const float grow = __builtin_amdgcn_exp2f(m[r] - base);
            m[r] = next;
            uint32_t p[4];
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = __builtin_amdgcn_exp2f(s[c][i] - base);
                    sum += w[i];
                    if constexpr (kCoded) {
                        w[i] *= vs[c][i];
                        if (cut && s[c][i] == -__builtin_inff()) w[i] = 0.0f;
                    }
                }
                p[2 * c] = kv_pack_bf16(w[0], w[1]);
                p[2 * c + 1] = kv_pack_bf16(w[2], w[3]);
            }
            l[r] = l[r] * grow + sum;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] *= grow;
            const bf8 weights = as_bf8(p[0], p[1], p[2], p[3]);
            if (!odd) {
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    uint32_t even[4], odds[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t x, y; /* values e, e + 1 of tokens 2 j and 2 j + 1 */
                        if constexpr (kCoded) {
                            x = e % 4 ? kv_widen<FMT, 1>(v[2 * j][e / 4]) : kv_widen<FMT, 0>(v[2 * j][e / 4]);
                            y = e % 4 ? kv_widen<FMT, 1>(v[2 * j + 1][e / 4]) : kv_widen<FMT, 0>(v[2 * j + 1][e / 4]);
                        } else {
                            x = v[2 * j][e / 2];
                            y = v[2 * j + 1][e / 2];
                        }
                        even[j] = __builtin_amdgcn_perm(y, x, 0x05040100u);
                        odds[j] = __builtin_amdgcn_perm(y, x, 0x07060302u);
                    }
                    acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(even[0], even[1], even[2], even[3]), weights, acc[r][e], 0, 0, 0);
                    acc[r][e + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(odds[0], odds[1], odds[2], odds[3]), weights, acc[r][e + 1], 0, 0, 0);
                }
            } else if constexpr (!kCoded) {
                /* an infinity or a NaN among values that not every row sees: 0 times it would
                 * reach the rows that do not, so each row's product is formed apart, without
                 * the tokens that it does not see */
                for (int one = 0; one < 16; ++one) {
                    const int o_lo = __shfl(lo[r], one), o_hi = __shfl(hi[r], one);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        uint32_t pair[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int at = t0 + 16 * (j / 2) + 4 * g + 2 * (j % 2);
                            const uint32_t x = at >= o_lo && at < o_hi ? v[2 * j][e / 2] : 0u;
                            const uint32_t y = at + 1 >= o_lo && at + 1 < o_hi ? v[2 * j + 1][e / 2] : 0u;
                            pair[j] = e % 2 ? __builtin_amdgcn_perm(y, x, 0x07060302u) : __builtin_amdgcn_perm(y, x, 0x05040100u);
                        }
                        const f4 got = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(pair[0], pair[1], pair[2], pair[3]), weights, acc[r][e], 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[r][e][i] = n == one ? got[i] : acc[r][e][i];
                    }
                }
            }
        }
    }

    /* the four waves together: 128 values of 16 rows at a time */
    constexpr int kPart = D < 128 ? D : 128, kPad = kPart + 4, kPer = kPart / 16;
    __shared__ float o_all[4][16][kPad];
    __shared__ float m_all[4][16], l_all[4][16];
    float *partial = t.active > 1 ? partial_of<D, RM>(a, item, head, split) : nullptr;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const float sum = lane_sum32(lane_sum16(l[r]));
#pragma unroll
        for (int half = 0; half < D / kPart; ++half) {
            __syncthreads();
            if (g == 0) {
                m_all[wave][n] = m[r];
                l_all[wave][n] = sum;
            }
            /* a lane has values 4 E g .. of its row: E e-neighbours for each i */
            const int d0 = 4 * E * g - half * kPart;
            if (d0 >= 0 && d0 < kPart) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *reinterpret_cast<f4 *>(&o_all[wave][n][d0 + E * i + e]) =
                            f4{acc[r][e][i], acc[r][e + 1][i], acc[r][e + 2][i], acc[r][e + 3][i]};
            }
            __syncthreads();
            const int row = tid >> 4, part = (tid & 15) * kPer, i = r * 16 + row;
            if (i < t.rows) {
                float top = -__builtin_inff();
#pragma unroll
                for (int w = 0; w < 4; ++w) top = fmaxf(top, m_all[w][row]);
                const float base = top == -__builtin_inff() ? 0.0f : top;
                float total = 0.0f, o[kPer];
#pragma unroll
                for (int j = 0; j < kPer; ++j) o[j] = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = __builtin_amdgcn_exp2f(m_all[w][row] - base);
                    total += f * l_all[w][row];
#pragma unroll
                    for (int j = 0; j < kPer; ++j) o[j] += f * o_all[w][row][part + j];
                }
                if (partial) {
                    float *to = partial + (long long)i * D + half * kPart + part;
#pragma unroll
                    for (int j = 0; j < kPer; j += 4) *reinterpret_cast<f4 *>(to + j) = f4{o[j], o[j + 1], o[j + 2], o[j + 3]};
                    if (part == 0 && half == 0) {
                        partial[RM * D + 2 * i] = top;
                        partial[RM * D + 2 * i + 1] = total;
                    }
                } else {
                    const int token = (t.start + i) / a.group, h = head * a.group + (t.start + i) % a.group;
                    const float by = total == 0.0f ? 0.0f : 1.0f / total;
                    uint32_t *to = reinterpret_cast<uint32_t *>(a.out + (t.first_row + token) * a.out_row + h * a.out_head +
                                                                half * kPart + part);
#pragma unroll
                    for (int j = 0; j < kPer; j += 2) to[j / 2] = kv_pack_bf16(o[j] * by, o[j + 1] * by);
                    if (a.lse && part == 0 && half == 0)
                        a.lse[(long long)(t.first_row + token) * a.q_heads + h] =
                            total == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * kLn2;
                }
            }
        }
    }
}

/* Joins the splits of a tile that has more than one: 16 lanes a row. */
template <int D, int RM>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    constexpr int kPer = D / 16;
    const int head = blockIdx.x % a.kv.heads, item = blockIdx.x / a.kv.heads;
    Tile t;
    if (!find_tile<RM>(a, item, 0, &t) || t.active < 2) return;
    for (int i = threadIdx.x >> 4; i < t.rows; i += 16) {
        const float *from = partial_of<D, RM>(a, item, head, 0);
        float top = -__builtin_inff();
        for (int s = 0; s < t.active; ++s) top = fmaxf(top, from[s * (RM * (D + 2)) + RM * D + 2 * i]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float total = 0.0f, o[kPer];
#pragma unroll
        for (int j = 0; j < kPer; ++j) o[j] = 0.0f;
        const int part = (threadIdx.x & 15) * kPer;
        for (int s = 0; s < t.active; ++s) {
            const float *p = from + (long long)s * (RM * (D + 2));
            const float f = __builtin_amdgcn_exp2f(p[RM * D + 2 * i] - base);
            total += f * p[RM * D + 2 * i + 1];
#pragma unroll
            for (int j = 0; j < kPer; j += 4) {
                const f4 x = *reinterpret_cast<const f4 *>(p + (long long)i * D + part + j);
#pragma unroll
                for (int c = 0; c < 4; ++c) o[j + c] += f * x[c];
            }
        }
        const int token = (t.start + i) / a.group, h = head * a.group + (t.start + i) % a.group;
        const float by = total == 0.0f ? 0.0f : 1.0f / total;
        uint32_t *to = reinterpret_cast<uint32_t *>(a.out + (t.first_row + token) * a.out_row + h * a.out_head + part);
#pragma unroll
        for (int j = 0; j < kPer; j += 2) to[j / 2] = kv_pack_bf16(o[j] * by, o[j + 1] * by);
        if (a.lse && part == 0)
            a.lse[(long long)(t.first_row + token) * a.q_heads + h] =
                total == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * kLn2;
    }
}

/* How a call is cut: tiles of 16 rt rows, at most `items` of them a key head, `splits` a tile. */
struct Plan {
    int rt, items, splits;
    size_t ws_bytes;
};

Plan plan_of(const W4A16KvCache *c, const W4A16KvBatch *b, int q_heads) {
    Plan p;
    const int group = q_heads / c->kv_heads;
    const long long most = (long long)(b->max_new ? b->max_new : b->rows) * group;
    p.rt = most <= 16 ? 1 : most <= 32 ? 2 : 4;
    const int rm = 16 * p.rt;
    p.items = (int)((long long)b->rows * group / rm + (b->seqs < b->rows ? b->seqs : b->rows));
    /* four blocks a CU */
    const long long blocks = (long long)p.items * c->kv_heads, wanted = 4LL * device_cus();
    const long long tokens = b->max_kv ? b->max_kv : (long long)b->table_pages * c->page_size;
    const long long longest = (tokens + kFewestTokens - 1) / kFewestTokens;
    long long splits = blocks > 0 ? (wanted + blocks - 1) / blocks : 1;
    if (splits > longest) splits = longest;
    if (splits > 256) splits = 256;
    p.splits = splits < 1 ? 1 : (int)splits;
    p.ws_bytes = p.splits > 1 ? (size_t)blocks * p.splits * rm * (c->head_dim + 2) * 4 : 0;
    return p;
}

template <int D, int RT>
void launch_rows(int format, const Plan &p, const AttnArgs &a, hipStream_t s) {
    auto kernel = format == W4A16_KV_BF16   ? attn_rows_kernel<D, W4A16_KV_BF16, RT>
                  : format == W4A16_KV_INT8 ? attn_rows_kernel<D, W4A16_KV_INT8, RT>
                                            : attn_rows_kernel<D, W4A16_KV_FP8, RT>;
    launch_k(kernel, dim3(a.kv.heads * p.items, p.splits), dim3(256), 0, s, a);
    if (p.splits > 1) launch_k(attn_join_kernel<D, 16 * RT>, dim3(a.kv.heads * p.items), dim3(256), 0, s, a);
}

template <int D>
void launch_dim(int format, const Plan &p, const AttnArgs &a, hipStream_t s) {
    if (p.rt == 1) launch_rows<D, 1>(format, p, a, s);
    else if (p.rt == 2) launch_rows<D, 2>(format, p, a, s);
    else launch_rows<D, 4>(format, p, a, s);
}

int check_heads(const KvView &kv, int q_heads, const char *what) {
    if (q_heads < 1 || q_heads % kv.heads || (long long)q_heads * kv.rows > INT32_MAX / 2)
        return set_error(W4A16_ERR_CONFIG, "%s: q_heads=%d is no multiple of the cache's %d heads, or %d rows of them "
                         "are too many", what, q_heads, kv.heads, kv.rows);
    return W4A16_OK;
}

} // namespace

extern "C" int w4a16_paged_attention_workspace(const W4A16KvCache *cache, const W4A16KvBatch *batch, int q_heads,
                                               size_t *bytes) {
    const char *what = "w4a16_paged_attention_workspace";
    if (!bytes) return set_error(W4A16_ERR_CONFIG, "%s: null result", what);
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (!st) st = check_heads(kv, q_heads, what);
    if (st) return st;
    *bytes = kv.rows && kv.seqs ? plan_of(cache, batch, q_heads).ws_bytes : 0;
    return W4A16_OK;
}

extern "C" int w4a16_paged_attention_bf16(const W4A16KvCache *cache, const W4A16KvBatch *batch, const uint16_t *q,
                                          long long q_row_stride, long long q_head_stride, int q_heads, float scale,
                                          int causal, int window, uint16_t *out, long long out_row_stride,
                                          long long out_head_stride, float *lse, void *ws, size_t ws_bytes,
                                          void *stream) {
    const char *what = "w4a16_paged_attention_bf16";
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (!st) st = check_heads(kv, q_heads, what);
    if (st) return st;
    if (!(scale - scale == 0.0f)) return set_error(W4A16_ERR_CONFIG, "%s: the scale is not finite", what);
    if (window < 0) return set_error(W4A16_ERR_CONFIG, "%s: window=%d is negative", what, window);
    if (kv.rows == 0 || kv.seqs == 0) return W4A16_OK;
    if (!q || !out) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (misaligned(q) || misaligned(out) || misaligned(ws) || ((uintptr_t)lse & 3))
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 16-byte aligned (lse: 4)", what);
    const int dim = cache->head_dim;
    const size_t qb = strided_bytes(kv.rows, q_row_stride, q_heads, q_head_stride, dim);
    const size_t ob = strided_bytes(kv.rows, out_row_stride, q_heads, out_head_stride, dim);
    if (!qb || !ob) return set_error(W4A16_ERR_CONFIG, "%s: strides must be multiples of 8 elements from 0", what);
    const long long by_row = (long long)(q_heads - 1) * out_head_stride + dim;
    const long long by_head = (long long)(kv.rows - 1) * out_row_stride + dim;
    const bool apart = ((q_heads == 1 || out_head_stride >= dim) && (kv.rows == 1 || out_row_stride >= by_row)) ||
                       ((kv.rows == 1 || out_row_stride >= dim) && (q_heads == 1 || out_head_stride >= by_head));
    if (!apart) return set_error(W4A16_ERR_CONFIG, "%s: output rows overlap each other", what);
    const Plan p = plan_of(cache, batch, q_heads);
    if (p.ws_bytes > 0 && (!ws || ws_bytes < p.ws_bytes))
        return set_error(W4A16_ERR_CONFIG, "%s: a workspace of %zu bytes, the call needs %zu", what, ws ? ws_bytes : 0,
                         p.ws_bytes);
    /* q and out may be the same tensor, or heads of the same rows side by side */
    bool clash = overlap(q, qb, out, ob);
    if (clash && q_row_stride == out_row_stride && kv.rows > 0) {
        const long long q_wide = (long long)(q_heads - 1) * q_head_stride + dim, o_wide = by_row;
        const long long off = ((const uint8_t *)out - (const uint8_t *)q) / 2;
        if (off == 0 && q_head_stride == out_head_stride) clash = false;
        else if (off > 0) clash = !(off >= q_wide && off + o_wide <= q_row_stride);
        else clash = !(-off >= o_wide && -off + q_wide <= q_row_stride);
    }
    const size_t lb = lse ? (size_t)kv.rows * q_heads * 4 : 0, cb = kv_bytes(cache), sb = kv_scale_bytes(cache);
    const struct { const void *p; size_t n; } writes[] = {{out, ob}, {lse, lb}, {ws, p.ws_bytes}};
    const struct { const void *p; size_t n; } reads[] = {{cache->k, cb}, {cache->v, cb}, {kv.k_scale, sb}, {kv.v_scale, sb}};
    for (int i = 0; i < 3; ++i) {
        for (const auto &r : reads) clash = clash || overlap(writes[i].p, writes[i].n, r.p, r.n);
        if (i) clash = clash || overlap(writes[i].p, writes[i].n, q, qb);
        for (int j = 0; j < i; ++j) clash = clash || overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n);
    }
    if (clash) return set_error(W4A16_ERR_CONFIG, "%s: an output or the workspace overlaps another buffer", what);
    if ((long long)p.items * kv.heads > 1 << 23)
        return set_error(W4A16_ERR_CONFIG, "%s: %lld tiles of rows: at most 2^23 a call", what,
                         (long long)p.items * kv.heads);
    AttnArgs a;
    a.kv = kv;
    a.q = q;
    a.out = out;
    a.lse = lse;
    a.ws = static_cast<float *>(ws);
    a.q_row = q_row_stride;
    a.q_head = q_head_stride;
    a.out_row = out_row_stride;
    a.out_head = out_head_stride;
    a.group = q_heads / kv.heads;
    a.q_heads = q_heads;
    a.causal = causal != 0;
    a.window = window;
    a.splits = p.splits;
    a.items = p.items;
    a.scale = scale * 1.4426950408889634f;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dim == 64) launch_dim<64>(cache->format, p, a, s);
    else if (dim == 128) launch_dim<128>(cache->format, p, a, s);
    else launch_dim<256>(cache->format, p, a, s);
    return hip_status(hipGetLastError(), "paged attention launch");
}
