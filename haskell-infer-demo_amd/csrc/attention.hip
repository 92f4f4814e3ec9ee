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
 * An 8-bit cache's codes are BF16 and FP16 values; their scales multiply the scores (K) and the weights
 * (V) in FP32.
 *
 * TREE: a sequence's last tokens are the nodes of a tree, and a row sees of them those that its bits name. The tokens before
 * them and those that no row of a tile may see are found as without; a step that holds nodes is one that is
 * cut, in which a lane has the bits of its row's next tokens in one word.
 */
#include <cmath>

#include "kv.h"
#include "wave.h"

using namespace w4a16;

namespace {

typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct AttnArgs {
    KvView kv;
    const uint16_t *q;
    uint16_t *out;
    float *lse, *ws;
    long long q_row, q_head, out_row, out_head;
    int group, q_heads, causal, window;
    int splits, items;
    int blocks;       /* few rows: as many parts have a place in the workspace */
    int over, upto;   /* only sequences of over < rows <= upto (token, head) rows */
    float scale;      /* |scale| log2(e) */
    uint32_t flip;    /* sign bits of a BF16 pair of q: a negative scale turns its sign over */
    W4A16KvTree tree; /* of the kernels with TREE */
    int least;        /* units of a part at least, where pairs are cut */
};

constexpr int kFewestTokens = 256; /* of a split of the chunk kernel */
constexpr int kUnit = 128;         /* tokens that a block of the few-row kernel takes at a time */
constexpr float kLn2 = 0.69314718055994531f;

/* What a tile's block works on: a sequence, its rows in the tile, the keys that any of them
 * sees and its own split of those. The same on every lane. */
struct Tile {
    int first_row;          /* the sequence's first row in q */
    int rows, news;         /* (token, head) rows of the tile from `start`; the sequence's new tokens */
    int start;              /* first (token, head) row of the tile in the sequence */
    int old;                /* position of the sequence's first row: its tokens less the new ones */
    int length;             /* the sequence's keys: its tokens that the table has room for */
    int lo, hi;             /* keys that some row sees: [lo, hi) */
    int all_lo, all_hi;     /* keys that every row sees */
    int begin, end, active; /* this split's keys; how many splits have any */
    int window;             /* 0 where it cuts nothing */
    int seq;
    int base, nodes;        /* TREE: the tree's first token, and how many it has */
};

/* The end of the keys that a row at `place` sees; with trees, none behind its own place. */
template <bool TREE>
__device__ __forceinline__ int row_end(const AttnArgs &a, const Tile &t, int place) {
    const int end = TREE || a.causal ? place + 1 : t.length;
    return end < t.length ? end : t.length;
}

/* Nodes that a sequence's tree has. */
__device__ __forceinline__ int tree_nodes(const AttnArgs &a, int seq) {
    const int n = a.tree.sizes ? a.tree.sizes[seq] : a.tree.nodes;
    return n < 0 ? 0 : n > a.tree.nodes ? a.tree.nodes : n;
}

/* The rest of a tile from its sequence's tokens (old + news) and rows, and its start. */
template <int RM, bool TREE>
__device__ __forceinline__ void fill_tile(const AttnArgs &a, Tile *t) {
    const int all = t->news * a.group;
    t->rows = all - t->start < RM ? all - t->start : RM;
    const int t0 = t->start / a.group, t1 = (t->start + t->rows - 1) / a.group;
    /* the same on every lane, and kept as such: in lanes it costs the few-row kernels registers that they do not have */
    t->length = __builtin_amdgcn_readfirstlane(kv_held(a.kv, t->old + t->news));
    t->window = a.window <= t->old + t->news ? a.window : 0;
    t->hi = row_end<TREE>(a, *t, t->old + t1);
    t->all_hi = row_end<TREE>(a, *t, t->old + t0);
    int least = t->old + t0; /* position of any of the tile's rows */
    if constexpr (TREE) {
        t->base = t->old + t->news - t->nodes;
        if (t->base < t->all_hi) t->all_hi = t->base;
        if (t->base < least) least = t->base;
    }
    t->lo = t->window ? least - t->window + 1 : 0;
    t->all_lo = t->window ? t->old + t1 - t->window + 1 : 0;
    if (t->lo < 0) t->lo = 0;
    if (t->hi <= t->lo) t->hi = t->lo = 0; /* the window may begin behind the last key */
}

/* TREE: what a tile's rows see of their tree, in LDS: a row's words of bits, its position and its token in the sequence (-1: no row). Steps
 * that hold nodes come last, when nothing is left to hide a load behind. */
constexpr int kTreeWords = 8, kTreePosition = kTreeWords, kTreeToken = kTreeWords + 1, kTreeRow = kTreeWords + 2;

/* Fills the ROWS rows from row `first` of a tile on, by the wave that reads them: GROUPS lanes a row. In two parts, for the loads to be
 * on their way meanwhile. */
template <int ROWS>
struct TreeLoad {
    static constexpr int kGroups = 64 / ROWS, kWords = kTreeWords / kGroups;
    uint32_t words[kWords];
    int position, token;

    __device__ __forceinline__ void load(const AttnArgs &a, const Tile &t, int first) {
        const int lane = threadIdx.x & 63, i = first + lane % ROWS, group = lane / ROWS;
        token = i < t.rows ? (t.start + i) / a.group : -1;
        const long long row = t.first_row + (token < 0 ? 0 : token);
        const int held = (a.tree.nodes + 63) >> 6 << 1;
        const uint32_t *bits = reinterpret_cast<const uint32_t *>(a.tree.seen) + row * held;
#pragma unroll
        for (int w = 0; w < kWords; ++w) words[w] = group + w * kGroups < held ? bits[group + w * kGroups] : 0u;
        position = t.window ? a.tree.positions[row] : 0;
    }
    __device__ __forceinline__ void store(uint32_t *rows, int first) const {
        const int lane = threadIdx.x & 63, group = lane / ROWS;
        uint32_t *to = rows + (first + lane % ROWS) * kTreeRow;
#pragma unroll
        for (int w = 0; w < kWords; ++w) to[group + w * kGroups] = words[w];
        if (group == 0) {
            to[kTreePosition] = position;
            to[kTreeToken] = token;
        }
    }
};

/* Which of the 32 tokens from `at` on a row sees, bit k for token at + k. What it follows from is found anew at each step that needs it: kept
 * over a loop it would cost registers that there are not. */
__device__ __forceinline__ uint32_t tree_sees(const AttnArgs &a, const Tile &t, const uint32_t *row, int at) {
    const int token = (int)row[kTreeToken], place = t.old + token;
    /* [from, to) of the 32 */
    const int to = token < 0 ? 0 : row_end<true>(a, t, place) - at;
    int from = 0;
    if (t.window) {
        /* a node's position lies between its tree's first token and its place */
        const int p = (int)row[kTreePosition];
        from = (place < t.base || p > place ? place : p < t.base ? t.base : p) - t.window + 1 - at;
    }
    uint32_t sees = (to >= 32 ? 0xFFFFFFFFu : to > 0 ? (1u << to) - 1u : 0u) & (from <= 0 ? 0xFFFFFFFFu : from < 32 ? 0xFFFFFFFFu << from : 0u);
    const int node = at - t.base; /* of the first of them; the tokens before node 0 are no nodes */
    if (node > -32) {
        const int w = node >> 5;
        const uint32_t low = w < 0 ? 0xFFFFFFFFu : w < kTreeWords ? row[w] : 0u, high = w + 1 < kTreeWords ? row[w + 1] : 0u;
        sees &= __builtin_amdgcn_alignbit(high, low, node & 31);
    }
    return sees;
}

constexpr int kMostUnits = 1 << 23; /* of 2^30 tokens */

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
            if (news * a.group <= a.over || news * a.group > a.upto) news = 0;
        }
        const int tiles = (news * a.group + RM - 1) / RM, upto = wave_upto(tiles);
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
    t->old = __builtin_amdgcn_readfirstlane(kv_length(a.kv, t->seq)) - t->news;
    fill_tile<RM, false>(a, t);
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

/*
 * The few-row kernel's work, and with trees the chunk kernel's too, is cut by the lengths that it finds: with N units of kUnit tokens over
 * all (tile, head) pairs and a.splits blocks wanted, every pair is cut into parts of
 * ceil(N / a.splits) units, so that long sequences have many parts and none is much longer
 * than another. The parts are counted through the sequences; a part is a block's, and its place in
 * the workspace. With trees only the parts of pairs that are cut have places: ceil(u / each) of a pair of u > each units are fewer than
 * 2 u / each, so all of them fewer than 2 N / each <= 2 a.splits, however many pairs there are, and such pairs fewer than a.splits.
 */
struct Seqs { /* 64 sequences, one a lane */
    int first, news, old, from; /* old: position of its first row; from: where the first key that any of its rows sees is cut */
    int pairs, units;              /* its (tile, head) pairs, units of each */
    int nodes;                     /* TREE */
};

template <int RM, bool TREE>
__device__ __forceinline__ Seqs load_seqs(const AttnArgs &a, int base) {
    const int s = base + (threadIdx.x & 63);
    Seqs q = {0, 0, 0, 0, 0, 1, 0};
    if (s < a.kv.seqs) {
        q.first = a.kv.starts[s];
        const int last = a.kv.starts[s + 1];
        const int length = kv_length(a.kv, s), held = kv_held(a.kv, length);
        if (q.first >= 0 && last <= a.kv.rows && last > q.first) q.news = last - q.first;
        if (q.news * a.group <= a.over || q.news * a.group > a.upto) q.news = 0;
        q.old = length - q.news;
        int least = q.old;
        if constexpr (TREE) {
            q.nodes = tree_nodes(a, s);
            if (length - q.nodes < least) least = length - q.nodes;
        }
        if (a.window && a.window <= length && least - a.window + 1 > 0) q.from = (least - a.window + 1) & ~31;
        if (held > q.from) q.units = (held - q.from + kUnit - 1) / kUnit;
        else q.from = 0; /* no row sees any */
        q.pairs = (q.news * a.group + RM - 1) / RM * a.kv.heads;
    }
    return q;
}

/* Units of a part; *q is left with the first 64 sequences. N / (blocks wanted) where that makes no
 * more parts than blocks; each pair's last part is on average half as long. */
template <int RM, bool TREE>
__device__ __forceinline__ int part_units(const AttnArgs &a, Seqs *q, bool *equal) {
    *q = load_seqs<RM, TREE>(a, 0);
    *equal = false;
    if (a.splits == 0) return kMostUnits; /* pairs are whole */
    /* n < 2^47 in two pieces, whose sums over 64 lanes fit 32 bits */
    unsigned long long total = 0;
    long long pairs = 0;
    Seqs s = *q;
    for (int base = 0;;) {
        const unsigned long long n = (unsigned long long)s.pairs * s.units;
        total += (uint32_t)__builtin_amdgcn_readlane(wave_upto((int)(n & 0xFFFFFF)), 63);
        total += (unsigned long long)(uint32_t)__builtin_amdgcn_readlane(wave_upto((int)(n >> 24)), 63) << 24;
        pairs += __builtin_amdgcn_readlane(wave_upto(s.pairs), 63);
        base += 64;
        if (base >= a.kv.seqs) break;
        s = load_seqs<RM, TREE>(a, base);
    }
    const unsigned long long wanted = pairs < a.splits ? a.splits - pairs / 2 : a.splits;
    const unsigned long long each = (total + wanted - 1) / wanted;
    if constexpr (TREE) {
        if (RM == 128 && a.kv.seqs <= 64 && pairs > 0 && pairs < a.splits) {
            /* Sequences that are about as long as each other: as many equal parts of each pair as are one round of blocks. 250 nodes over
             * 16384 tokens: four of 32 units, not three of 37 and one of 17, 189 and 215 us. Of ragged ones the short rests fill the gaps. */
            const long long most = wave_most(q->pairs ? q->units : 0);
            if (8 * most * pairs <= 9 * (long long)total) {
                *equal = true;
                const int parts = a.splits / (int)pairs, size = ((int)most + parts - 1) / parts;
                return size < a.least ? a.least : size;
            }
        }
        return each < a.least ? a.least : each > kMostUnits ? kMostUnits : (int)each;
    }
    return each < 1 ? 1 : each > kMostUnits ? kMostUnits : (int)each;
}

/* The part of this block (PAIR false) or the (tile, head) pair of number `index` (true; with trees, among those that are cut): the
 * tile, its head, its number of parts, and the number of its first one. TREE: *place is the part's (PAIR: its first part's) in the workspace, -1
 * where it has none. */
template <int RM, bool PAIR, bool TREE>
__device__ __forceinline__ bool find_part(const AttnArgs &a, int index, Tile *t, int *head, int *first_part, int *place) {
    Seqs q;
    bool equal; /* TREE: a pair's parts are alike */
    const int each = part_units<RM, TREE>(a, &q, &equal);
    int left = index, before = 0, places = 0; /* parts of the sequences before, and those that have places */
    for (int base = 0;;) {
        const int per = (q.units + each - 1) / each, parts = q.pairs * per;
        const int pairs = TREE && per < 2 ? 0 : q.pairs, stored = pairs * per; /* TREE: that are cut */
        const int upto_parts = wave_upto(parts), upto = PAIR ? wave_upto(pairs) : upto_parts, upto_stored = TREE ? wave_upto(stored) : 0;
        const unsigned long long here = __ballot(upto > left);
        if (here) {
            const int l = __ffsll((long long)here) - 1;
            t->seq = base + l;
            t->first_row = __builtin_amdgcn_readlane(q.first, l);
            t->news = __builtin_amdgcn_readlane(q.news, l);
            t->old = __builtin_amdgcn_readlane(q.old, l);
            if constexpr (TREE) t->nodes = __builtin_amdgcn_readlane(q.nodes, l);
            const int from = __builtin_amdgcn_readlane(q.from, l);
            t->active = __builtin_amdgcn_readlane(per, l);
            const int in_seq = left - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(PAIR ? pairs : parts, l));
            const int pair = PAIR ? in_seq : in_seq / t->active, part = PAIR ? 0 : in_seq - pair * t->active;
            *first_part = before + __builtin_amdgcn_readlane(upto_parts, l) - __builtin_amdgcn_readlane(parts, l) + pair * t->active;
            if constexpr (TREE)
                *place = t->active < 2 ? -1 : places + __builtin_amdgcn_readlane(upto_stored, l) - __builtin_amdgcn_readlane(stored, l) + pair * t->active + part;
            *head = pair % a.kv.heads;
            t->start = pair / a.kv.heads * RM;
            fill_tile<RM, TREE>(a, t);
            int size = each;
            if constexpr (TREE)
                if (equal) size = (__builtin_amdgcn_readlane(q.units, l) + t->active - 1) / t->active;
            t->begin = from + part * size * kUnit;
            t->end = part + 1 < t->active && t->begin + size * kUnit < t->hi ? t->begin + size * kUnit : t->hi;
            if constexpr (TREE) {
                /* Rows before the tree: a tile's window may begin far behind its sequence's. By whole steps (of 64 tokens at most), which end with
                 * the part, and what is left of it may be nothing. 4096 rows over 8192 tokens, window 256, 32 heads over 8 of 128, BF16:
                 * 60 us, and 491 from the part's own begin. */
                if (t->begin < t->lo) t->begin += (t->lo - t->begin) & ~63;
            }
            return true;
        }
        left -= __builtin_amdgcn_readlane(upto, 63);
        before += __builtin_amdgcn_readlane(upto_parts, 63);
        if constexpr (TREE) places += __builtin_amdgcn_readlane(upto_stored, 63);
        base += 64;
        if (base >= a.kv.seqs) return false;
        q = load_seqs<RM, TREE>(a, base);
    }
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
    return ((pair & 0x7F80u) == 0x7F80u) | ((pair & 0x7F800000u) == 0x7F800000u);
}

/* A partial result in the workspace: RM rows of D values, then RM pairs (m, l). */
template <int D, int RM>
__device__ __forceinline__ float *partial_at(const AttnArgs &a, long long index) {
    return a.ws + index * (RM * (D + 2));
}

/* Codes 2 * HALF and 2 * HALF + 1 of one token's dword x and its neighbour's y, as pairs of one value of
 * both tokens: FP16, in which the codes of both formats are exact. An INT8 code's bits with the sign
 * flipped, 0 to 255, are the low bits of 1024 + 128 + code. */
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <int FMT, int HALF>
__device__ __forceinline__ void code_pairs(uint32_t x, uint32_t y, uint32_t *even, uint32_t *odd) {
    if constexpr (FMT == W4A16_KV_FP8) {
        const uint32_t a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, HALF));
        const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.0f, HALF));
        *even = __builtin_amdgcn_perm(b, a, 0x05040100u);
        *odd = __builtin_amdgcn_perm(b, a, 0x07060302u);
    } else {
        const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const uint32_t a = __builtin_amdgcn_perm(y, x, HALF ? 0x0C060C02u : 0x0C040C00u) ^ 0x64806480u;
        const uint32_t b = __builtin_amdgcn_perm(y, x, HALF ? 0x0C070C03u : 0x0C050C01u) ^ 0x64806480u;
        *even = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, a) + off);
        *odd = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, b) + off);
    }
}

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(kv_f2{a, b}, h2));
}

/* The V product: BF16 values with BF16 weights, or codes with FP16 weights. */
template <bool CODED>
__device__ __forceinline__ f4 mfma_v(const uint32_t *v, const uint32_t *w, f4 acc) {
    if constexpr (CODED)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, make_uint4(v[0], v[1], v[2], v[3])),
                                                      __builtin_bit_cast(h8, make_uint4(w[0], w[1], w[2], w[3])), acc, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf8(v[0], v[1], v[2], v[3]), as_bf8(w[0], w[1], w[2], w[3]), acc, 0, 0, 0);
}

/* A pair of BF16 weights and a pair of what they leave of a and b: a weight is then off by 2^-15 of itself
 * (cut to 8 bits, and the rest rounded to 8), not 2^-8. The rest is positive, as the weight is, and not
 * zero: an infinity among V's values stays one, it meets no product of the other sign or of zero. A last bit
 * set beforehand (2^-23) sees to that, for weights from 2^-100 of the largest. */
__device__ __forceinline__ void split_weights(float a, float b, uint32_t *first, uint32_t *rest) {
    const uint32_t x = __builtin_bit_cast(uint32_t, a), y = __builtin_bit_cast(uint32_t, b);
    *first = __builtin_amdgcn_perm(y, x, 0x07060302u);
    *rest = kv_pack_bf16(__builtin_bit_cast(float, x | 1u) - __builtin_bit_cast(float, x & 0xFFFF0000u),
                         __builtin_bit_cast(float, y | 1u) - __builtin_bit_cast(float, y & 0xFFFF0000u));
}

__device__ __forceinline__ float power_of_two(int biased) { return __builtin_bit_cast(float, (uint32_t)biased << 23); }

/* The weights of an 8-bit cache carry V's scale, so they are FP16 (in which codes are exact), over a
 * power of two that holds the largest scale so far in [1, 2), and times 2^kLift: at most 2^8 (a weight
 * over the last maximum) * 2 * 2^kLift, half of what FP16 holds. A weight's rounding is 2^-11 of
 * itself, or 2^-31 of the largest weight times the largest scale where that is more; BF16 would be 2^-8.
 * Biased exponents below kLift + 1 are raised to it, for the factor to be a number. */
constexpr int kLift = 6;
__device__ __forceinline__ float over_power(int biased) { return power_of_two(254 + kLift - biased); }
__device__ __forceinline__ float times_power(int biased) { return power_of_two(biased - kLift); }

/* Blocks of attn_rows_kernel that a CU is to hold: as many as its registers allow without spilling.
 * More waves are what hides the latency of its loads. At one block and at these (the join included): 48
 * ragged sequences of up to 8192 tokens, D = 128, INT8, 129 and 93.5 us; 16 of 4096 with five rows each, FP8,
 * RT = 2, 31.0 and 25.4; 64 of 8192, D = 256, FP8, 152 and 109, though 2 of 100003 take 91 and 94. */
constexpr int rows_blocks(int dim, int format, int rt) {
    return dim == 256 && rt == 2 ? 1 : dim == 256 ? (format == W4A16_KV_BF16 ? 1 : 2) : dim == 128 ? (rt == 1 ? 3 : 2) : rt == 1 ? 4 : 3;
}

/*
 * Few rows: a block of four waves has RT tiles of 16 rows and one split of the keys; its waves
 * take 32 tokens at a time in turn, each with statistics of its own, and are joined in LDS at the
 * end. K and V go from memory into the registers that the products take them from; no LDS in the
 * loop. The next tokens' K is loaded into its registers as soon as the score product has read
 * them, V behind the second product, and the page entries two steps ahead, so that a load has most
 * of a step to arrive and none waits for one behind it (loads arrive in order).
 *
 * v_mfma_f32_16x16x32. K: a lane's row is token l % 16 of two groups of 16, its values the
 * 8 or 16 that lane group g = l / 16 has of each step. S^T gives a lane tokens 16 c + 4 g + i of row
 * l % 16, and those are the eight that it holds of P^T (c, i from 0 to 1, 3) and has to load of V^T: 16
 * lanes load a token's whole row, E = D / 16 values each, which stand at E neighbouring
 * columns; a transposition of 8 tokens x 2 values at a time by byte permutations makes them the
 * operand of value e's product.
 *
 * A BF16 cache's weights are two BF16 numbers each (split_weights), 2^-15: the second product takes 0 to 0.3 % (16
 * sequences of 4096 with five rows each, D = 128 39.5 and 39.9 us, D = 64 24.4 and 25.3), and one user's output of 1337 tokens is off
 * by 1.7e-3, its own rounding, where it was by 1.8e-3 to 2.2e-3. Those of an 8-bit cache are rounded to FP16
 * (kLift), which also takes fewer instructions to widen INT8.
 *
 * Bound by memory: 32 sequences of 8192 tokens, one row of 32 heads each (16 of 256 values), the join included:
 * BF16 D = 64 102 us (5.2 TB/s), D = 128 192 (5.6), D = 256 200 (5.4); FP8 66 (4.4), 108 (5.1), 107 (5.1); INT8
 * 70, 110, 109. Trees: two of which 5 rows grow over 100003 tokens, 24 heads over 4 of 256, INT8, 100 us (4.2 TB/s; VALU 52 %, one
 * block a CU) and 7.2 for the join; one of 26 over 1500 tokens, 32 over 8 heads of 128, BF16, 12.9 and 4.0.
 */
template <int D, int FMT, int RT, bool TREE>
__global__ __launch_bounds__(256, rows_blocks(D, FMT, RT)) void attn_rows_kernel(AttnArgs a) {
    constexpr int RM = 16 * RT, E = D / 16, KS = D / 32; /* values of V a lane has; steps of the K product */
    constexpr bool kCoded = FMT != W4A16_KV_BF16;
    constexpr int kVWords = kCoded ? E / 4 : E / 2, kKLoads = kCoded ? KS / 2 : KS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int mask = (1 << a.kv.shift) - 1;
    Tile t;
    int head, first_part, place_of_part;
    if (!find_part<RM, false, TREE>(a, blockIdx.x, &t, &head, &first_part, &place_of_part)) return;

    const int32_t *table = a.kv.table + (long long)t.seq * a.kv.table_stride;
    /* Pages of this lane's K tokens and V tokens (page sizes are multiples of 8, so four
     * neighbours from a multiple of 4 share one). Tokens that are not there read page 0 and are
     * masked. */
    /* Table entries; vnext those of the tokens whose V is next. The entries are loaded two steps ahead
     * (INT8 and FP8, BF16 of 256 values: 2 to 5 % less time), or one, where the two registers more
     * would spill. */
    constexpr bool kAhead = kCoded || D != 128;
    int kpage[2], vpage[2], ahead[2];
    int(&vnext)[2] = kAhead ? ahead : vpage;
    auto load_pages = [&](int t0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int kt = t0 + 16 * c + n, vt = t0 + 16 * c + 4 * g;
            kpage[c] = table[(kt < t.length ? kt : 0) >> a.kv.shift];
            vpage[c] = table[(vt < t.length ? vt : 0) >> a.kv.shift];
        }
    };
    auto is_there = [&](int page, int token) { return (token < t.length) & ((unsigned)page < (unsigned)a.kv.pages); };
    auto offset_of = [&](int page, int token, uint32_t row) -> unsigned long long { /* rows of that many bytes */
        const uint32_t safe = is_there(page, token) ? page : 0;
        return (unsigned long long)safe * (a.kv.page_tokens * row) + (uint32_t)((head << a.kv.shift) + (token & mask)) * row;
    };
    constexpr uint32_t kRow = D * (kCoded ? 1 : 2);
    u4 kraw[2][kKLoads];
    uint32_t v[8][kVWords];
    f4 ks[2], vs[2];
    auto load_k = [&](int t0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint8_t *p = static_cast<const uint8_t *>(a.kv.k) + offset_of(kpage[c], t0 + 16 * c + n, kRow) + 16 * g;
#pragma unroll
            for (int s = 0; s < kKLoads; ++s) kraw[c][s] = *reinterpret_cast<const u4 *>(p + 64 * s);
        }
    };
    auto load_v = [&](int t0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint8_t *first = static_cast<const uint8_t *>(a.kv.v) + offset_of(vnext[c], t0 + 16 * c + 4 * g, kRow) + n * (4 * kVWords);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint8_t *p = first + i * kRow;
                if constexpr (kVWords == 1) {
                    v[4 * c + i][0] = *reinterpret_cast<const uint32_t *>(p);
                } else if constexpr (kVWords == 2) {
                    const uint2 x = *reinterpret_cast<const uint2 *>(p);
                    v[4 * c + i][0] = x.x;
                    v[4 * c + i][1] = x.y;
                } else {
#pragma unroll
                    for (int w = 0; w < kVWords; w += 4) {
                        const u4 x = *reinterpret_cast<const u4 *>(p + 4 * w);
                        v[4 * c + i][w] = x.x;
                        v[4 * c + i][w + 1] = x.y;
                        v[4 * c + i][w + 2] = x.z;
                        v[4 * c + i][w + 3] = x.w;
                    }
                }
            }
        }
    };
    auto load_scales = [&](int t0, f4 *k_of, f4 *v_of) {
        if constexpr (kCoded) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const unsigned long long from = offset_of(vpage[c], t0 + 16 * c + 4 * g, 1);
                k_of[c] = *reinterpret_cast<const f4 *>(a.kv.k_scale + from);
                v_of[c] = *reinterpret_cast<const f4 *>(a.kv.v_scale + from);
            }
        }
    };
    /* TREE: the rows of the tile that this wave's steps are cut for, if they are; a copy for each wave. They set out ahead of keys and values. */
    __shared__ uint32_t tree_rows[TREE ? 4 * RM * kTreeRow : 1];
    uint32_t *const own_rows = tree_rows + (TREE ? wave * RM * kTreeRow : 0);
    TreeLoad<RM> of_tree;
    if constexpr (TREE) of_tree.load(a, t, 0);
    int t0 = t.begin + 32 * wave;
    if (t0 < t.end) {
        load_pages(t0);
        load_k(t0);
        load_scales(t0, ks, vs);
        if constexpr (kAhead) {
            vnext[0] = vpage[0];
            vnext[1] = vpage[1];
            load_pages(t0 + 128);
        }
        load_v(t0);
    }

    /* this lane's rows: their queries as the products' operand, and the keys they see */
    /* 32 rows of 256 values: in LDS, beside sums that take half of the registers */
    constexpr bool kStored = D == 256 && RT == 2;
    __shared__ bf8 q_stored[kStored ? RT * KS * 64 : 1];
    bf8 q[RT][kStored ? 1 : KS];
    int lo[RT], hi[RT]; /* TREE: unused, tree_sees instead */
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        const int i = r * 16 + n, token = (t.start + i) / a.group, h = head * a.group + (t.start + i) % a.group;
        const bool real = i < t.rows;
        const int place = t.old + token;
        const uint16_t *row = a.q + (t.first_row + (real ? token : 0)) * a.q_row + h * a.q_head;
        hi[r] = !real ? 0 : row_end<TREE>(a, t, place);
        lo[r] = t.window ? place - t.window + 1 : 0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            const int d = kCoded ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
            if (kStored && s % 4 != wave) continue;
            const u4 x = *reinterpret_cast<const u4 *>(row + d);
            const bf8 y = as_bf8(real ? x.x ^ a.flip : 0u, real ? x.y ^ a.flip : 0u, real ? x.z ^ a.flip : 0u, real ? x.w ^ a.flip : 0u);
            if constexpr (kStored) q_stored[(r * KS + s) * 64 + lane] = y;
            else q[r][s] = y;
        }
    }
    if constexpr (kStored) __syncthreads();

    f4 acc[RT][E];
    float m[RT], l[RT];
    if constexpr (TREE) {
        of_tree.store(own_rows, 0);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); /* the wave's own: no other reads it */
    }
    auto tree_row = [&](int r) { /* TREE: of this lane's row */
        int i = r * 16 + n;
        asm volatile("" : "+v"(i)); /* or it is kept */
        return own_rows + i * kTreeRow;
    };
    float spoiled[RT] = {}; /* 1: this lane's row has seen a scale that is no number */
    int v_exp = kLift + 1; /* biased exponent of the power of two that the weights are over (8-bit caches) */
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        m[r] = -__builtin_inff();
        l[r] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (; t0 < t.end; t0 += 128) {
        bool there[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) there[c] = is_there(vnext[c], t0 + 16 * c + 4 * g);
        /* Loads are waited for by their number: with trees the next step's set out in any case (behind the last, as that one's again), or
         * V's would be waited for as if K's behind them had not been asked for. 30 rows over 100003 tokens, D = 256, INT8: 132 and
         * 101 us. 16 rows of 256 values have no registers for it. */
        constexpr bool kAlways = TREE && !(D == 256 && RT == 1);
        const bool more = kAlways || t0 + 128 < t.end;
        const int next = kAlways && t0 + 128 >= t.end ? t0 : t0 + 128;
        const bool cut = (t0 < t.all_lo) | (t0 + 32 > t.all_hi) | (__any(!there[0] | !there[1]) != 0);
        if constexpr (kCoded)
            if (cut) {
                bool odd_scale = false;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = t0 + 16 * c + 4 * g + i;
                        const bool none = !there[c] | (at < t.lo) | (at >= t.hi);
                        vs[c][i] = none ? 0.0f : vs[c][i];
                        odd_scale = odd_scale | !(fabsf(vs[c][i]) < __builtin_inff());
                    }
                if (__any(odd_scale)) {
                    /* a scale that is no number, at a token that not every row sees: 0 times it would
                     * reach the rows that do not. Those that do are noted, and the product goes
                     * without it. */
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        uint32_t row_sees = 0;
                        if constexpr (TREE) row_sees = tree_sees(a, t, tree_row(r), t0) >> (4 * g);
#pragma unroll
                        for (int c = 0; c < 2; ++c)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const int at = t0 + 16 * c + 4 * g + i;
                                const bool shown = TREE ? row_sees >> (16 * c + i) & 1u : (at >= lo[r]) & (at < hi[r]);
                                const bool sees = shown & !(fabsf(vs[c][i]) < __builtin_inff());
                                spoiled[r] = sees ? 1.0f : spoiled[r];
                            }
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c)
#pragma unroll
                        for (int i = 0; i < 4; ++i) vs[c][i] = fabsf(vs[c][i]) < __builtin_inff() ? vs[c][i] : 0.0f;
                }
            }
        if constexpr (!kAhead)
            if (more) load_pages(next);
        f4 s[RT][2];
        int q_lane = lane;
        if constexpr (kStored) asm volatile("" : "+v"(q_lane)); /* or what is read is kept */
        auto query = [&](int r, int step) {
            if constexpr (kStored) return q_stored[(r * KS + step) * 64 + q_lane];
            else return q[r][step];
        };
#pragma unroll
        for (int c = 0; c < 2; ++c) {
#pragma unroll
            for (int r = 0; r < RT; ++r) s[r][c] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 0; j < kKLoads; ++j) {
                u4 x = kraw[c][j];
                if constexpr (kCoded) {
                    asm volatile("" : "+v"(x)); /* or the bytes are carried apart, each in a register */
                    const bf8 k0 = as_bf8(kv_widen<FMT, 0>(x.x), kv_widen<FMT, 1>(x.x), kv_widen<FMT, 0>(x.y), kv_widen<FMT, 1>(x.y));
                    const bf8 k1 = as_bf8(kv_widen<FMT, 0>(x.z), kv_widen<FMT, 1>(x.z), kv_widen<FMT, 0>(x.w), kv_widen<FMT, 1>(x.w));
#pragma unroll
                    for (int r = 0; r < RT; ++r) {
                        s[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k0, query(r, 2 * j), s[r][c], 0, 0, 0);
                        s[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k1, query(r, 2 * j + 1), s[r][c], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < RT; ++r) s[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf8, x), query(r, j), s[r][c], 0, 0, 0);
                }
            }
        }
        f4 ks_next[2], vs_next[2];
        if (more) {
            load_k(next);
            load_scales(next, ks_next, vs_next);
            if constexpr (kAhead) {
                vnext[0] = vpage[0];
                vnext[1] = vpage[1];
                load_pages(next + 128);
            }
        }
        if constexpr (kCoded)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int w = 0; w < kVWords; ++w) asm volatile("" : "+v"(v[i][w]));
        /* tokens that some row does not see, or that are not there: their V is not multiplied */
        bool odd = false;
        if (cut) {
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = t0 + 16 * c + 4 * g + i;
                    const bool none = !there[c] | (at < t.lo) | (at >= t.hi);
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) v[4 * c + i][w] = none ? 0u : v[4 * c + i][w];
                    if constexpr (!kCoded)
#pragma unroll
                        for (int w = 0; w < kVWords; ++w) odd = odd | nonfinite2(v[4 * c + i][w]);
                }
            odd = __any(odd);
        }
        if constexpr (kCoded) {
            /* the largest scale's size; infinities and NaN are no measure of the others */
            float most = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) most = fmaxf(most, fabsf(vs[c][i]) < __builtin_inff() ? fabsf(vs[c][i]) : 0.0f);
            most = lane_max32(lane_max16(most));
            int exp = (int)(__builtin_bit_cast(uint32_t, most) >> 23);
            exp = __builtin_amdgcn_readfirstlane(exp > 253 ? 1 : exp);
            if (exp > v_exp) {
                const int fall = exp - v_exp > 126 ? 126 : exp - v_exp;
                const float by = power_of_two(127 - fall);
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[r][e] *= by;
                v_exp = exp;
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                vs[c] *= over_power(v_exp);
                ks[c] *= a.scale;
            }
        }
        uint32_t p[RT][4], p_rest[kCoded ? 1 : RT][4];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            uint32_t row_sees = 0;
            if constexpr (TREE)
                if (cut) row_sees = tree_sees(a, t, tree_row(r), t0) >> (4 * g);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                if constexpr (kCoded) s[r][c] *= ks[c];
                else s[r][c] *= a.scale;
                if (cut)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = t0 + 16 * c + 4 * g + i;
                        const bool hidden = TREE ? !there[c] | !(row_sees >> (16 * c + i) & 1u) : !there[c] | (at < lo[r]) | (at >= hi[r]);
                        s[r][c][i] = hidden ? -__builtin_inff() : s[r][c][i];
                    }
            }
            float most = fmaxf(fmaxf(fmaxf(s[r][0][0], s[r][0][1]), fmaxf(s[r][0][2], s[r][0][3])),
                               fmaxf(fmaxf(s[r][1][0], s[r][1][1]), fmaxf(s[r][1][2], s[r][1][3])));
            most = lane_max32(lane_max16(most));
            if (__any(most > m[r] + 8.0f)) {
                const float upto = fmaxf(m[r], most);
                const float grow = __builtin_amdgcn_exp2f(m[r] - (upto == -__builtin_inff() ? 0.0f : upto));
                m[r] = upto;
                l[r] *= grow;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[r][e] *= grow;
            }
            const float base = m[r] == -__builtin_inff() ? 0.0f : m[r];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = __builtin_amdgcn_exp2f(s[r][c][i] - base);
                    l[r] += w[i];
                    if constexpr (kCoded) w[i] *= vs[c][i];
                }
                if constexpr (kCoded) {
                    p[r][2 * c] = pack_f16(w[0], w[1]);
                    p[r][2 * c + 1] = pack_f16(w[2], w[3]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; i += 2) split_weights(w[i], w[i + 1], &p[r][2 * c + i / 2], &p_rest[r][2 * c + i / 2]);
                }
            }
        }
        if constexpr (!kCoded)
            if (odd) {
                /* An infinity or a NaN among values that not every row sees: 0 times it would reach the
                 * rows that do not. Those that do have it added as it is, and the products go without it.
                 * Value E (4 g + i) + e of a token, which is acc[][e][i], is lane 4 g + i's of its 16. */
                uint32_t row_sees[RT];
                if constexpr (TREE)
#pragma unroll
                    for (int r = 0; r < RT; ++r) row_sees[r] = tree_sees(a, t, tree_row(r), t0);
#pragma unroll
                for (int x = 0; x < 8; ++x) {
                    bool some = false;
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) some = some | nonfinite2(v[x][w]);
                    const unsigned long long where = __ballot(some);
                    if (where == 0) continue;
#pragma unroll 1
                    for (int of = 0; of < 4; ++of) {
                        if ((where >> (16 * of) & 0xFFFF) == 0) continue;
                        const int at = t0 + 16 * (x / 4) + 4 * of + x % 4;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int w = 0; w < kVWords; ++w) {
                                const uint32_t pair = __shfl(v[x][w], 16 * of + 4 * g + i);
                                const uint32_t f[2] = {pair << 16, pair & 0xFFFF0000u};
#pragma unroll
                                for (int r = 0; r < RT; ++r)
#pragma unroll
                                    for (int half = 0; half < 2; ++half) {
                                        const bool shown = TREE ? row_sees[r] >> (at - t0) & 1u : (at >= lo[r]) & (at < hi[r]);
                                        const bool adds = shown & ((f[half] & 0x7F800000u) == 0x7F800000u);
                                        acc[r][2 * w + half][i] += adds ? __builtin_bit_cast(float, f[half]) : 0.0f;
                                    }
                            }
                    }
#pragma unroll
                    for (int w = 0; w < kVWords; ++w) {
                        const uint32_t pair = v[x][w];
                        v[x][w] = ((pair & 0x7F80u) == 0x7F80u ? 0u : pair & 0xFFFFu) | ((pair & 0x7F800000u) == 0x7F800000u ? 0u : pair & 0xFFFF0000u);
                    }
                }
            }
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            uint32_t even[4], odds[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) { /* values e, e + 1 of tokens 2 j and 2 j + 1 */
                if constexpr (kCoded) {
                    if (e % 4) code_pairs<FMT, 1>(v[2 * j][e / 4], v[2 * j + 1][e / 4], &even[j], &odds[j]);
                    else code_pairs<FMT, 0>(v[2 * j][e / 4], v[2 * j + 1][e / 4], &even[j], &odds[j]);
                } else {
                    even[j] = __builtin_amdgcn_perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], 0x05040100u);
                    odds[j] = __builtin_amdgcn_perm(v[2 * j + 1][e / 2], v[2 * j][e / 2], 0x07060302u);
                }
            }
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                acc[r][e] = mfma_v<kCoded>(even, p[r], acc[r][e]);
                acc[r][e + 1] = mfma_v<kCoded>(odds, p[r], acc[r][e + 1]);
                if constexpr (!kCoded) {
                    acc[r][e] = mfma_v<kCoded>(even, p_rest[r], acc[r][e]);
                    acc[r][e + 1] = mfma_v<kCoded>(odds, p_rest[r], acc[r][e + 1]);
                }
            }
        }
        if (more) load_v(next);
        if constexpr (kCoded) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                ks[c] = ks_next[c];
                vs[c] = vs_next[c];
            }
        }
    }
    if constexpr (kCoded) {
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const float by = lane_max32(lane_max16(spoiled[r])) > 0.0f ? __builtin_nanf("") : times_power(v_exp);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[r][e] *= by;
        }
    }

    /* the four waves together: 128 values of 16 rows at a time */
    constexpr int kPart = D < 128 ? D : 128, kPad = kPart + 4, kPer = kPart / 16;
    __shared__ float o_all[4][16][kPad];
    __shared__ float m_all[4][16], l_all[4][16];
    float *partial = (TREE ? place_of_part >= 0 : t.active > 1) ? partial_at<D, RM>(a, TREE ? place_of_part : blockIdx.x) : nullptr;
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

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

/* Codes 2 * HALF and 2 * HALF + 1 of a dword as an FP16 pair. */
template <int FMT, int HALF>
__device__ __forceinline__ uint32_t widen_f16(uint32_t codes) {
    if constexpr (FMT == W4A16_KV_FP8) {
        return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, HALF));
    } else {
        const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
        const uint32_t x = __builtin_amdgcn_perm(codes, codes, HALF ? 0x0C030C02u : 0x0C010C00u) ^ 0x64806480u;
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, x) + off);
    }
}

/*
 * Many rows: a block of four waves has 128 (token, head) rows, 32 a wave, and goes through its
 * keys BN at a time. The tile's K and V stand in LDS, BF16 (V of an 8-bit cache FP16), twice:
 * while one is multiplied the next is on its way from memory into registers, widened there once
 * for all four waves and written behind the products; one barrier a step.
 *
 * v_mfma_f32_32x32x16. S^T = K Q^T: a lane's column is row l % 32, its 16 values tokens
 * 8 (i / 4) + 4 (l / 32) + i % 4 of 32, so that the first eight of them are what the lane holds of
 * P^T in a product over 16 tokens, and the next eight in the following one; V^T comes out
 * of LDS with the transposing read (four tokens of a column to each lane). A row's maximum is over
 * a lane's own values and those of lane l ^ 32. The sums are rescaled only when a maximum has
 * grown by more than 2^8 since the last time, which rounds nothing more: weights up to 2^8
 * are as exact in BF16, FP16 and FP32 as those up to 1.
 *
 * 16-byte pieces of a token's K are exchanged by its number (XOR), pairs of pieces of its V by
 * the same, so that the eight lanes of a step of a read fall on different banks.
 *
 * Every wave reads the whole tile, so the LDS reads of 32 rows take as long as their products; above
 * that it is bound by the weights' VALU work (five instructions each, and for 8-bit caches the widening
 * of a tile over 128 rows). 4096 rows over 16384 tokens, 32 heads (16 of 256 values): BF16 D = 64 671 us, 717
 * TFLOP/s; D = 128 979, 983; D = 256 1017, 946; INT8 859, 1193, 1308; FP8 748, 1134, 1269. Trees: 16 of up to 60 over up to
 * 8192 tokens, 32 heads over 8 of 128, FP8, 86.9 us, VALU 39 % and MFMA 22 % busy, 1.7 waves a SIMD: a tile's way through the registers to
 * LDS is waited for; 8 of up to 251 over up to 16384, window 4096, 32 over 4 of 64, BF16, 88.2, VALU 58 %.
 */
template <int D, int FMT, bool TIGHT, bool TREE>
struct Chunk {
    static constexpr bool kCoded = FMT != W4A16_KV_BF16;
    static constexpr int kRows = 128, BN = D == 256 ? 32 : 64;
    static constexpr int kPieces = D / 8;                              /* of 8 values a token */
    static constexpr int kLoads = BN * D * (kCoded ? 1 : 2) / (256 * 16); /* 16-byte loads a thread and matrix */
    static constexpr int kSwizzle = kPieces < 16 ? kPieces - 1 : 15;
    /* LDS: [2]{K, V}, then scales [2][2][BN], pages [3][BN], flags, queries, rows of the tree (TREE) */
    static constexpr int kTile = BN * D * 2;
    static constexpr int kScales = 4 * kTile, kPages = kScales + (kCoded ? 4 * BN * 4 : 0);
    static constexpr int kFlags = kPages + 3 * BN * 4, kQueries = kFlags + 32; /* bad[3], exponents[2] */
    /* the last steps' queries of a K product that stand in LDS, [step][half][row]: the registers of 8-bit
     * codes on their way leave no room for all of 256 values, or of 64 where four blocks are to fit */
    static constexpr int kStored = !kCoded || (!TIGHT && !TREE) ? 0 : D == 256 ? TREE ? 2 : 3 : D == 64 ? TREE ? 2 : 1 : 0;
    static constexpr int kTree = kQueries + kStored * 2 * kRows * 16, kBytes = kTree + (TREE ? kRows * kTreeRow * 4 : 0);
};

/* 16 bytes a lane from memory to LDS, lane after lane from `to` (the same on every lane). */
__device__ __forceinline__ void load_to_lds(const uint8_t *from, uint8_t *to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)from,
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

/* Before the barrier behind which other waves read what load_to_lds wrote. */
__device__ __forceinline__ void wait_for_lds_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

/* Asks the scheduler for the LDS reads (READS for each of COUNT products) FAR products before their
 * use. 4096 rows over 16384 tokens, without and with FAR = 2: BF16 D = 128 1024 and 997 us, D = 64 720 and 697,
 * FP8 D = 128 1241 and 1221; at D = 256, where the registers are for FAR = 1: BF16 1099 and 1086, FP8 1296 and
 * 1259. */
template <int COUNT, int READS, int FAR>
__device__ __forceinline__ void interleave() {
    if constexpr (FAR > 0) {
        __builtin_amdgcn_sched_group_barrier(0x100, READS * FAR, 0);
#pragma unroll
        for (int i = 0; i < COUNT - FAR; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, FAR, 0);
    }
}

/* Blocks of attn_chunk_kernel that a CU is to hold, without spilling: the waves of one multiply while those
 * of another find their weights. TIGHT: addresses are worked out at every step, for one block more. At D =
 * 256 that is two instead of one, and 4096 rows over 16384 tokens take BF16 1022 us instead of 1610, FP8
 * 1260 instead of 2074. 64 values of 8 bits: four instead of three, INT8 856 instead of 917 us, but 624 tiles
 * of ragged sequences, for which three have room, 85 instead of 78, so those go without (BF16 needs the
 * registers, and gains nothing: 680 and 685). */
constexpr int chunk_blocks(int dim, bool tight) { return dim > 64 ? 2 : tight ? 4 : 3; }

template <int D, int FMT, bool TIGHT, bool TREE>
__global__ __launch_bounds__(256, chunk_blocks(D, TIGHT)) void attn_chunk_kernel(AttnArgs a) {
    using C = Chunk<D, FMT, TIGHT, TREE>;
    constexpr bool kCoded = C::kCoded;
    constexpr int BN = C::BN, RM = C::kRows, kHalves = BN / 32, KS = D / 16, DB = D / 32;
    constexpr int kFar = D == 256 ? 1 : 2;
    extern __shared__ uint4 smem4[];
    uint8_t *smem = reinterpret_cast<uint8_t *>(smem4);
    float *scales = reinterpret_cast<float *>(smem + C::kScales); /* [buffer][k, v][BN] */
    int *pages = reinterpret_cast<int *>(smem + C::kPages);       /* [step % 3][BN] */
    int *bad = reinterpret_cast<int *>(smem + C::kFlags);         /* [step % 3]: a token without a page */
    int *exponents = bad + 3;                                      /* [step % 2]: V's scales are over 2 to this, biased; + 256: one is not finite */
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, half = lane >> 5;
    /* the last tiles of a sequence see the most keys: those first */
    int head = blockIdx.x % a.kv.heads, split = blockIdx.y, item = a.items - 1 - (int)(blockIdx.x / a.kv.heads);
    int first_part, place_of_part;
    Tile t;
    if constexpr (TREE) {
        if (!find_part<RM, false, TREE>(a, blockIdx.x, &t, &head, &first_part, &place_of_part)) return;
    } else {
        if (!find_tile<RM>(a, item, split, &t)) return;
        if (split >= t.active) return;
    }

    const int32_t *table = a.kv.table + (long long)t.seq * a.kv.table_stride;
    const int mask = (1 << a.kv.shift) - 1;
    const int steps = t.end > t.begin ? (t.end - t.begin + BN - 1) / BN : 0;

    /* Token tid % BN of a step: its entry of the page table, unread until put_page, so that nothing waits
     * for it (and, loads arriving in order, for the tile's before it) at the start of a step. */
    auto entry_of = [&](int step) {
        const int at = t.begin + step * BN + tid % BN;
        return table[(at >= t.lo && at < t.hi ? at : t.lo) >> a.kv.shift];
    };
    auto put_page = [&](int step, int entry) { /* by the first wave: -1 where there is no token */
        const int at = t.begin + step * BN + tid % BN;
        const bool ok = (at >= t.lo) & (at < t.hi) & ((unsigned)entry < (unsigned)a.kv.pages);
        if (tid < BN) pages[(step % 3) * BN + tid] = ok ? entry : -1;
        const bool none = __any(!ok);
        if (lane == 0) bad[step % 3] = none;
    };
    /* 8-bit: through registers, widened on the way into LDS. BF16: straight into LDS, a wave's 1 KiB at
     * a time; a lane fetches the piece that belongs where it writes. */
    u4 kr[C::kLoads], vr[C::kLoads];
    float scale_r = 0.0f;
    bool scale_there = false;
    int v_run = kLift + 1;
    bool there_r[C::kLoads];
    constexpr int kLanes = D * (kCoded ? 1 : 2) / 16; /* a token's 16-byte loads */
    /* the place in its page and head of token `at` of a step; rows of it that many bytes apart */
    auto inside = [&](int step, int at) { return (uint32_t)((head << a.kv.shift) + ((t.begin + step * BN + at) & mask)); };
    constexpr uint32_t kRow = D * (kCoded ? 1 : 2);
    auto offset_of = [&](int step, int at, int page, uint32_t row) -> unsigned long long {
        return (unsigned long long)(uint32_t)(page >= 0 ? page : 0) * (a.kv.page_tokens * row) + inside(step, at) * row;
    };
    auto load_tile = [&](int step) {
        int tid = threadIdx.x;
        if constexpr (TIGHT) asm volatile("" : "+v"(tid)); /* or what follows from it is kept over the loop */
        const uint8_t *k = static_cast<const uint8_t *>(a.kv.k), *v = static_cast<const uint8_t *>(a.kv.v);
        if constexpr (kCoded) {
#pragma unroll
            for (int x = 0; x < C::kLoads; ++x) {
                const int at = (x * 256 + tid) / kLanes, part = (x * 256 + tid) % kLanes;
                const int page = pages[(step % 3) * BN + at];
                there_r[x] = page >= 0;
                const unsigned long long from = offset_of(step, at, page, kRow) + part * 16;
                kr[x] = *reinterpret_cast<const u4 *>(k + from);
                vr[x] = *reinterpret_cast<const u4 *>(v + from);
            }
            /* K's scales by threads 0 .. BN - 1 of each 2 BN, V's by the others; unread here, as entries are */
            const int at = tid % BN, page = pages[(step % 3) * BN + at];
            scale_there = page >= 0;
            scale_r = (tid % (2 * BN) < BN ? a.kv.k_scale : a.kv.v_scale)[offset_of(step, at, page, 1)];
        } else {
            const int wave_u = __builtin_amdgcn_readfirstlane(wave);
            uint8_t *to = smem + (step & 1) * 2 * C::kTile + wave_u * 1024;
#pragma unroll
            for (int x = 0; x < C::kLoads; ++x) {
                const int at = (x * 256 + tid) / kLanes, part = (x * 256 + tid) % kLanes;
                const unsigned long long from = offset_of(step, at, pages[(step % 3) * BN + at], kRow);
                load_to_lds(k + from + (part ^ (at & C::kSwizzle)) * 16, to + x * 4096);
                load_to_lds(v + from + (part ^ ((2 * at) & C::kSwizzle)) * 16, to + C::kTile + x * 4096);
            }
        }
    };
    auto store_tile = [&](int step) {
        if constexpr (kCoded) {
            int tid = threadIdx.x;
            if constexpr (TIGHT) asm volatile("" : "+v"(tid));
            uint8_t *k = smem + (step & 1) * 2 * C::kTile, *v = k + C::kTile;
#pragma unroll
            for (int x = 0; x < C::kLoads; ++x) {
                const int at = (x * 256 + tid) / kLanes, part = (x * 256 + tid) % kLanes;
                asm volatile("" : "+v"(kr[x]), "+v"(vr[x])); /* or the bytes are carried apart from the load on */
                const u4 vx = there_r[x] ? vr[x] : u4{0u, 0u, 0u, 0u};
                const int ks = at & C::kSwizzle, vs = (2 * at) & C::kSwizzle;
                const u4 k0 = {kv_widen<FMT, 0>(kr[x].x), kv_widen<FMT, 1>(kr[x].x), kv_widen<FMT, 0>(kr[x].y), kv_widen<FMT, 1>(kr[x].y)};
                const u4 k1 = {kv_widen<FMT, 0>(kr[x].z), kv_widen<FMT, 1>(kr[x].z), kv_widen<FMT, 0>(kr[x].w), kv_widen<FMT, 1>(kr[x].w)};
                *reinterpret_cast<u4 *>(k + at * 2 * D + ((2 * part) ^ ks) * 16) = k0;
                *reinterpret_cast<u4 *>(k + at * 2 * D + ((2 * part + 1) ^ ks) * 16) = k1;
                const u4 v0 = {widen_f16<FMT, 0>(vx.x), widen_f16<FMT, 1>(vx.x), widen_f16<FMT, 0>(vx.y), widen_f16<FMT, 1>(vx.y)};
                const u4 v1 = {widen_f16<FMT, 0>(vx.z), widen_f16<FMT, 1>(vx.z), widen_f16<FMT, 0>(vx.w), widen_f16<FMT, 1>(vx.w)};
                *reinterpret_cast<u4 *>(v + at * 2 * D + ((2 * part) ^ vs) * 16) = v0;
                *reinterpret_cast<u4 *>(v + at * 2 * D + ((2 * part + 1) ^ vs) * 16) = v1;
            }
            /* V's scales over a power of two that holds the largest so far in [1, 2), as in
             * attn_rows_kernel; the wave that has them keeps it for the block. Infinities and NaN are
             * no measure of the others. */
            scale_r = !scale_there ? 0.0f : tid % (2 * BN) < BN ? scale_r * a.scale : scale_r;
            if (wave == BN / 64) {
                const int e = (int)(__builtin_bit_cast(uint32_t, scale_r) >> 23) & 255;
                const int most = wave_most(tid >= BN && e <= 253 ? e : 0);
                v_run = most > v_run ? most : v_run;
                if (tid >= BN) scale_r *= over_power(v_run);
                const bool odd = __any((tid >= BN) & (e == 255));
                if (lane == 0) exponents[step & 1] = v_run + (odd ? 256 : 0);
            }
            if (tid < 2 * BN) scales[(step & 1) * 2 * BN + tid] = scale_r;
        } else {
            wait_for_lds_loads();
        }
    };

    /* TREE: a wave without any rows only helps with the tiles. Which waves have the rows goes round with the blocks, so that those of the
     * blocks that share a CU are on different SIMDs. */
    const int turn = TREE ? (blockIdx.x + 2 * (blockIdx.x >> 8)) & 3 : 0;
    TreeLoad<32> of_tree;
    if constexpr (TREE) of_tree.load(a, t, ((wave + turn) & 3) * 32);
    if (steps > 0) {
        if (tid < 64) {
            const int first = entry_of(0), second = entry_of(steps > 1 ? 1 : 0);
            put_page(0, first);
            if (steps > 1) put_page(1, second);
        }
        __syncthreads();
        load_tile(0);
    }

    /* this lane's row: its queries and the keys it sees */
    int i_row = ((wave + turn) & 3) * 32 + n, token = (t.start + i_row) / a.group, h = head * a.group + (t.start + i_row) % a.group;
    bool real = i_row < t.rows;
    const int place = t.old + token;
    /* TREE: unused, tree_sees instead */
    const int hi = !real ? 0 : row_end<TREE>(a, t, place), lo = t.window ? place - t.window + 1 : 0;
    const uint32_t seen = hi > lo ? hi - lo : 0; /* this row sees a key where its place less lo, unsigned, is below this */
    uint32_t *const tree_rows = reinterpret_cast<uint32_t *>(smem + C::kTree); /* TREE; read by the waves that wrote them */
    auto row_of = [&] {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid)); /* or it is kept over the loop, and what follows from it */
        return (((tid >> 6) + turn) & 3) * 32 + (tid & 31);
    };
    const bool idle = TREE && __builtin_amdgcn_readfirstlane(i_row) >= t.rows;
    auto tree_row = [&] { return tree_rows + row_of() * kTreeRow; };
    if constexpr (TREE) {
        of_tree.store(tree_rows, __builtin_amdgcn_readfirstlane(i_row) & ~31);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    constexpr int kHeld = KS - C::kStored;
    bf8 q[kHeld], *const q_stored = reinterpret_cast<bf8 *>(smem + C::kQueries) + half * RM + i_row;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
        const u4 x = *reinterpret_cast<const u4 *>(a.q + (t.first_row + (real ? token : 0)) * a.q_row + h * a.q_head + 16 * s + 8 * half);
        const bf8 y = as_bf8(real ? x.x ^ a.flip : 0u, real ? x.y ^ a.flip : 0u, real ? x.z ^ a.flip : 0u, real ? x.w ^ a.flip : 0u);
        if (s < kHeld) q[s < kHeld ? s : 0] = y;
        else q_stored[(s - kHeld) * 2 * RM] = y;
    }
    f16v acc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[d][i] = 0.0f;
    float m = real ? -__builtin_inff() : 0.0f, l = 0.0f;
    int v_exp = kLift + 1;
    bool spoiled = false; /* this lane's row has seen a scale that is no number */
    if (steps > 0) {
        store_tile(0);
        __syncthreads();
    }

    /* This lane's places in a tile of K: piece `half` of token n (that of step j, 2 j + half, is an XOR
     * away); and in one of V, for the transposing read: row (lane % 16) / 4 of four tokens, four of
     * 16 columns. */
    int k_at = n * 2 * D + ((half ^ (n & C::kSwizzle)) * 16);
    const int v_row = 4 * half + ((lane >> 2) & 3), v_piece = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    int v_at = v_row * 2 * D + ((v_piece ^ ((2 * v_row) & C::kSwizzle)) * 16) + 8 * (lane & 1);
    for (int step = 0; step < steps; ++step) {
        const bool more = step + 1 < steps;
        const bool look = step + 2 < steps;
        const int t0 = t.begin + step * BN;
        const bool cut = (t0 < t.all_lo) | (t0 + BN > t.all_hi) | (__builtin_amdgcn_readfirstlane(bad[step % 3]) != 0);
        if constexpr (kCoded) {
            if (cut & (__builtin_amdgcn_readfirstlane(exponents[step & 1]) > 255)) {
                /* a scale that is no number, at a token that not every row sees: as in attn_rows_kernel */
                float *of = scales + (step & 1) * 2 * BN + BN;
#pragma unroll 1
                for (int in = 0; in < BN; ++in) {
                    const bool shown = TREE ? tree_sees(a, t, tree_row(), t0 + in) & 1u : (uint32_t)(t0 + in - lo) < seen;
                    spoiled |= shown & !(fabsf(of[in]) < __builtin_inff());
                }
                __syncthreads();
                if (tid < BN) of[tid] = fabsf(of[tid]) < __builtin_inff() ? of[tid] : 0.0f;
                __syncthreads();
            }
        }
        if (more) load_tile(step + 1);
        const int entry = entry_of(look ? step + 2 : step);
        if constexpr (TIGHT) asm volatile("" : "+v"(k_at), "+v"(v_at));
        const uint8_t *kt = smem + (step & 1) * 2 * C::kTile, *vt = kt + C::kTile;
        const float *sc = scales + (step & 1) * 2 * BN;
        uint32_t p[kHalves][8];
        if (!idle) {
            f16v s[kHalves];
#pragma unroll
            for (int c = 0; c < kHalves; ++c) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[c][i] = 0.0f;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const bf8 k = *reinterpret_cast<const bf8 *>(kt + (k_at ^ (32 * j)) + 32 * c * 2 * D);
                    const bf8 y = j < kHeld ? q[j < kHeld ? j : 0] : q_stored[(j - kHeld) * 2 * RM];
                    s[c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, y, s[c], 0, 0, 0);
                }
            }
            interleave<kHalves * KS, 1, kFar>();
            /* scores over the maximum that the sums stand at: the exponents of the weights */
            float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    f4 x = {a.scale, a.scale, a.scale, a.scale};
                    if constexpr (kCoded) x = *reinterpret_cast<const f4 *>(sc + 32 * c + 8 * b + 4 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[c][4 * b + i] = fmaf(s[c][4 * b + i], x[i], -base);
                }
            if (cut) {
                const uint32_t at = t0 - lo;
#pragma unroll
                for (int c = 0; c < kHalves; ++c) {
                    uint32_t row_sees = 0;
                    if constexpr (TREE) row_sees = tree_sees(a, t, tree_row(), t0 + 32 * c) >> (4 * half);
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int in = 32 * c + 8 * b + 4 * half;
                        const int4 page = *reinterpret_cast<const int4 *>(pages + (step % 3) * BN + in);
                        const int each[4] = {page.x, page.y, page.z, page.w};
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const bool hidden = TREE ? (each[i] < 0) | !(row_sees >> (8 * b + i) & 1u)
                                                     : ((at + in + i) | (each[i] & 0x80000000u)) >= seen; /* a page of -1 as well */
                            s[c][4 * b + i] = hidden ? -__builtin_inff() : s[c][4 * b + i];
                        }
                    }
                }
            }
            float most = s[0][0];
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) most = fmaxf(most, s[c][i]);
            if (__any((most > 8.0f) | (m == -__builtin_inff()))) {
                /* a new maximum: for rows that have none yet, or whose weights would pass 2^8 */
                most = lane_max32(most);
                const bool none = m == -__builtin_inff();
                const float rise = most > (none ? -__builtin_inff() : 8.0f) ? most : 0.0f;
                const float grow = none ? 0.0f : __builtin_amdgcn_exp2f(-rise);
                m = none && rise == 0.0f && most != 0.0f ? m : base + rise;
                l *= grow;
#pragma unroll
                for (int d = 0; d < DB; ++d) acc[d] *= grow;
#pragma unroll
                for (int c = 0; c < kHalves; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[c][i] -= rise;
            }
            if constexpr (kCoded) {
                const int now = __builtin_amdgcn_readfirstlane(exponents[step & 1]) & 255;
                if (now != v_exp) {
                    const float by = power_of_two(now - v_exp > 126 ? 1 : 127 - (now - v_exp));
#pragma unroll
                    for (int d = 0; d < DB; ++d) acc[d] *= by;
                    v_exp = now;
                }
            }
#pragma unroll
            for (int c = 0; c < kHalves; ++c)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    float w[4];
                    f4 x = {1.0f, 1.0f, 1.0f, 1.0f};
                    if constexpr (kCoded) x = *reinterpret_cast<const f4 *>(sc + BN + 32 * c + 8 * b + 4 * half);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w[i] = __builtin_amdgcn_exp2f(s[c][4 * b + i]);
                        l += w[i];
                        if constexpr (kCoded) w[i] *= x[i];
                    }
                    p[c][2 * b] = kCoded ? pack_f16(w[0], w[1]) : kv_pack_bf16(w[0], w[1]);
                    p[c][2 * b + 1] = kCoded ? pack_f16(w[2], w[3]) : kv_pack_bf16(w[2], w[3]);
                }
        }
        if constexpr (!kCoded) {
            /* Tokens that are not there weigh nothing, and what memory holds for them is taken
             * out. An infinity or a NaN among values that not every row sees: 0 times it would
             * reach the rows that do not. Those that do have it added as it is, and the product
             * goes without it. */
            if (cut) {
                uint32_t *tile = reinterpret_cast<uint32_t *>(smem + (step & 1) * 2 * C::kTile + C::kTile);
                bool odd = false;
                for (int x = tid; x < C::kTile / 4; x += 256) {
                    if (pages[(step % 3) * BN + x / (D / 2)] < 0) tile[x] = 0u;
                    else odd = odd | nonfinite2(tile[x]);
                }
                if (__syncthreads_or(odd)) {
                    for (int in = 0; in < BN; ++in) {
                        const bool sees = TREE ? tree_sees(a, t, tree_row(), t0 + in) & 1u : (uint32_t)(t0 + in - lo) < seen;
#pragma unroll
                        for (int d = 0; d < DB; ++d)
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                __builtin_amdgcn_sched_barrier(0); /* one piece at a time: registers */
                                const uint2 x = *reinterpret_cast<const uint2 *>(vt + in * 2 * D + ((4 * d + b) ^ ((2 * in) & C::kSwizzle)) * 16 + 8 * half);
                                if (!__any((int)nonfinite2(x.x) | (int)nonfinite2(x.y))) continue;
                                const uint32_t f[4] = {x.x << 16, x.x & 0xFFFF0000u, x.y << 16, x.y & 0xFFFF0000u};
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    const bool adds = sees & ((f[i] & 0x7F800000u) == 0x7F800000u);
                                    acc[d][4 * b + i] += adds ? __builtin_bit_cast(float, f[i]) : 0.0f;
                                }
                            }
                    }
                    __syncthreads();
                    for (int x = tid; x < C::kTile / 4; x += 256) {
                        const uint32_t pair = tile[x];
                        tile[x] = ((pair & 0x7F80u) == 0x7F80u ? 0u : pair & 0xFFFFu) | ((pair & 0x7F800000u) == 0x7F800000u ? 0u : pair & 0xFFFF0000u);
                    }
                    __syncthreads();
                }
            }
        }
        /* O^T: 16 tokens and 32 values a product */
        if (!idle) {
#pragma unroll
            for (int u = 0; u < BN / 16; ++u) {
                const uint32_t *w = &p[u / 2][4 * (u % 2)];
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    uint32_t v[4];
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const uint2 got = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) s4 *)(vt + (v_at ^ (64 * d)) + (16 * u + 8 * y) * 2 * D)));
                        v[2 * y] = got.x;
                        v[2 * y + 1] = got.y;
                    }
                    if constexpr (kCoded) {
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, make_uint4(v[0], v[1], v[2], v[3])),
                                                                        __builtin_bit_cast(h8, make_uint4(w[0], w[1], w[2], w[3])), acc[d], 0, 0, 0);
                    } else {
                        acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(v[0], v[1], v[2], v[3]), as_bf8(w[0], w[1], w[2], w[3]), acc[d], 0, 0, 0);
                    }
                }
            }
            interleave<BN / 16 * DB, 2, kFar>();
        }
        if (more) store_tile(step + 1);
        if (look && tid < 64) put_page(step + 2, entry);
        __syncthreads();
    }

    /* a lane has values 32 d + 8 b + 4 half .. + 3 of its row; so does lane ^ 32 the four between */
    const float total = lane_sum32(l);
    if constexpr (TREE) {
        i_row = row_of();
        token = (t.start + i_row) / a.group;
        h = head * a.group + (t.start + i_row) % a.group;
        real = i_row < t.rows;
    }
    if (!real) return;
    float by = !kCoded ? 1.0f : spoiled ? __builtin_nanf("") : times_power(v_exp);
    float *partial = (TREE ? place_of_part >= 0 : t.active > 1)
                         ? partial_at<D, RM>(a, TREE ? place_of_part : ((long long)item * a.kv.heads + head) * a.splits + split) : nullptr;
    if (partial) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int b = 0; b < 4; ++b)
                *reinterpret_cast<f4 *>(partial + (long long)i_row * D + 32 * d + 8 * b + 4 * half) =
                    f4{acc[d][4 * b], acc[d][4 * b + 1], acc[d][4 * b + 2], acc[d][4 * b + 3]} * by;
        if (half == 0) {
            partial[RM * D + 2 * i_row] = m;
            partial[RM * D + 2 * i_row + 1] = total;
        }
        return;
    }
    by = total == 0.0f ? 0.0f : by / total;
    uint16_t *to = a.out + (t.first_row + token) * a.out_row + h * a.out_head + 4 * half;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int b = 0; b < 4; ++b)
            *reinterpret_cast<uint2 *>(to + 32 * d + 8 * b) = make_uint2(kv_pack_bf16(acc[d][4 * b] * by, acc[d][4 * b + 1] * by),
                                                                        kv_pack_bf16(acc[d][4 * b + 2] * by, acc[d][4 * b + 3] * by));
    if (a.lse && half == 0)
        a.lse[(long long)(t.first_row + token) * a.q_heads + h] =
            total == 0.0f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(total)) * kLn2;
}

/* Joins the parts of a (tile, head) that has more than one: the splits of the chunk kernel, or the
 * parts of the few-row kernel (EVEN). A block has 16 / SUB rows (blockIdx.y of
 * them), 16 lanes a row and part of its splits: with many splits the sum over them is what takes
 * time, so SUB parts of it run side by side and meet in LDS. */
template <int D, int RM, int SUB, bool EVEN, bool TREE>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    constexpr int kPer = D / 16, kRows = 16 / SUB;
    Tile t;
    int head, first_part = 0, first_place = 0;
    if constexpr (EVEN) {
        if (!find_part<RM, true, TREE>(a, blockIdx.x, &t, &head, &first_part, &first_place)) return;
        if (first_part + t.active > a.blocks) return; /* sequences that overlap: not all parts were worked on */
        if constexpr (!TREE) first_place = first_part;
    } else {
        head = blockIdx.x % a.kv.heads;
        if (!find_tile<RM>(a, blockIdx.x / a.kv.heads, 0, &t)) return;
    }
    if (t.active < 2 || (int)blockIdx.y * kRows >= t.rows) return;
    const int lane = threadIdx.x & 15, unit = threadIdx.x >> 4, sub = unit / kRows, i = blockIdx.y * kRows + unit % kRows;
    const int row = i < t.rows ? i : t.rows - 1;
    auto part_of = [&](int s) { return partial_at<D, RM>(a, (EVEN ? first_place : (long long)blockIdx.x * a.splits) + s); };
    /* Of many parts the first ones' values are on their way beside the maxima: 64 parts of 256 values 8.6
     * and 7.4 us; of few that costs more than it gives. */
    constexpr int kFirst = SUB == 16 ? 2 : 0;
    f4 x[kFirst + 1][kPer / 4];
    float m[kFirst + 1], l[kFirst + 1];
#pragma unroll
    for (int k = 0; k < kFirst; ++k) {
        const int s = sub + k * SUB;
        const float *from = part_of(s < t.active ? s : 0), *ml = from + RM * D + 2 * row, *values = from + row * D + lane * kPer;
        m[k] = ml[0];
        l[k] = ml[1];
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) x[k][j] = *reinterpret_cast<const f4 *>(values + 4 * j);
    }
    float top = -__builtin_inff();
    for (int s = lane; s < t.active; s += 16) top = fmaxf(top, part_of(s)[RM * D + 2 * row]);
#pragma unroll
    for (int x = 1; x < 16; x *= 2) top = fmaxf(top, __shfl_xor(top, x));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float total = 0.0f, o[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) o[j] = 0.0f;
#pragma unroll
    for (int k = 0; k < kFirst; ++k)
        if (sub + k * SUB < t.active) {
            const float f = __builtin_amdgcn_exp2f(m[k] - base);
            total += f * l[k];
#pragma unroll
            for (int j = 0; j < kPer; ++j) o[j] += f * x[k][j / 4][j % 4];
        }
#pragma unroll 4
    for (int s = sub + kFirst * SUB; s < t.active; s += SUB) {
        const float *from = part_of(s), *ml = from + RM * D + 2 * row, *values = from + row * D + lane * kPer;
        const float f = __builtin_amdgcn_exp2f(ml[0] - base);
        total += f * ml[1];
#pragma unroll
        for (int j = 0; j < kPer; j += 4) {
            const f4 x = *reinterpret_cast<const f4 *>(values + j);
#pragma unroll
            for (int c = 0; c < 4; ++c) o[j + c] += f * x[c];
        }
    }
    if constexpr (SUB > 1) {
        __shared__ float parts[16][D + 4], totals[16];
#pragma unroll
        for (int j = 0; j < kPer; ++j) parts[unit][lane * kPer + j] = o[j];
        if (lane == 0) totals[unit] = total;
        __syncthreads();
        if (sub) return;
#pragma unroll
        for (int s = 1; s < SUB; ++s) {
            total += totals[unit + s * kRows];
#pragma unroll
            for (int j = 0; j < kPer; ++j) o[j] += parts[unit + s * kRows][lane * kPer + j];
        }
    }
    if (i >= t.rows) return;
    const int token = (t.start + i) / a.group, h = head * a.group + (t.start + i) % a.group;
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    uint32_t *to = reinterpret_cast<uint32_t *>(a.out + (t.first_row + token) * a.out_row + h * a.out_head + lane * kPer);
#pragma unroll
    for (int j = 0; j < kPer; j += 2) to[j / 2] = kv_pack_bf16(o[j] * by, o[j + 1] * by);
    if (a.lse && lane == 0)
        a.lse[(long long)(t.first_row + token) * a.q_heads + h] =
            total == 0.0f ? -__builtin_inff() : (top + __builtin_amdgcn_logf(total)) * kLn2;
}

/* How a call is cut: sequences of few (token, head) rows into tiles of 16 rt rows, the others into
 * tiles of 128; at most `items` tiles a key head, `splits` of each (for few rows, of all), and
 * where their partial results begin in the workspace. */
struct Part {
    int items, splits, over, upto;
    size_t ws_at;
    long long blocks; /* few rows, and with trees */
    int least;
};
struct Plan {
    int rt;
    Part few, many; /* items 0: not launched */
    size_t ws_bytes;
};

constexpr int kChunkRows = 128;

/* Places that parts of a call with trees may need: of those that are cut (find_part), and no more than there are blocks. */
long long tree_places(const Part &p) { return 2LL * p.splits < p.blocks ? 2LL * p.splits : p.blocks; }

Plan plan_of(const W4A16KvCache *c, const W4A16KvBatch *b, int q_heads, bool tree) {
    Plan p = {};
    const int group = q_heads / c->kv_heads, dim = c->head_dim;
    const int max_new = b->max_new ? b->max_new : b->rows;
    const long long rows = (long long)b->rows * group, longest = (long long)max_new * group;
    const long long seqs = b->seqs < b->rows ? b->seqs : b->rows;
    /* attn_rows_kernel has registers for 32 rows, or 16 of 256 values at two blocks a CU; trees have more than 16 more often
     * than not, and one block is better than the chunk kernel there */
    const int limit = dim == 256 && !tree ? 16 : 32;
    p.rt = longest <= 16 || limit == 16 ? 1 : 2;
    const int rm = 16 * p.rt;
    p.few = {0, 1, 0, INT32_MAX, 0, 0, 1};
    p.many = {0, 1, 0, INT32_MAX, 0, 0, 1};
    const long long most_tokens = b->max_kv ? b->max_kv : (long long)b->table_pages * c->page_size;
    const long long short_units = (rows / rm + seqs) * c->kv_heads * ((most_tokens + kUnit - 1) / kUnit);
    if (longest <= limit || (tree && short_units <= 4 * device_cus())) {
        /* Trees over few tokens too: tiles of 128 rows would leave most of the CUs without any, and take longer to begin. One sequence of
         * 1500 tokens, 8 key heads of 128, BF16: 36, 64, 128 rows 14.6, 14.1, 17.2 us, with the chunk kernel 18.1, 18.8,
         * 23.6; of 20000: 31.5, 32.7, 44.8 and 30.0, 31.1, 40.9. */
        p.few.items = (int)(rows / rm + seqs);
    } else if ((long long)b->seqs * max_new == b->rows || group > limit || (tree && rows > 32 * seqs)) {
        /* all alike (whatever the bound says, this launch takes every sequence), or of trees that have more rows on average: two
         * launches more cost more than a few idle waves */
        p.many.items = (int)(rows / kChunkRows + seqs);
    } else {
        p.few.items = (int)seqs;
        p.few.upto = p.many.over = rm;
        p.many.items = (int)(rows / kChunkRows + (rows / (rm + 1) < seqs ? rows / (rm + 1) : seqs));
    }
    const long long tokens = most_tokens;
    if (p.few.items) {
        /* One round of blocks, and no more than there are units. Two rounds are better for batches of many
         * sequences and worse for few or short ones; the host knows bounds, not lengths, and one round loses least
         * where it loses. One, one and a half, two rounds, the join included, us: 48 ragged sequences of up to 8192
         * tokens, D = 128, INT8 100.7 / 106.4 / 95.5, BF16 142 / 152 / 138; 32 of 8192, BF16, D = 128 201 / 210 / 206,
         * D = 256 217 / 245 / 203; 16 of up to 4096 with five rows, FP8 31.0 / 35.5 / 33.5; 100003 tokens, one
         * sequence, BF16 91.7 / 99.8 / 96.0, two, D = 256, FP8 93.7 / 99.4 / 100.6. */
        const long long blocks = (long long)rows_blocks(dim, c->format, p.rt) * device_cus();
        const long long pairs = (long long)p.few.items * c->kv_heads, units = pairs * ((tokens + kUnit - 1) / kUnit);
        p.few.splits = (int)(units < 1 ? 1 : units < blocks ? units : blocks);
        /* Short sequences are not cut at all: no partial results and no second launch. One sequence,
         * 8 key heads of 128, BF16, cut and whole, in a graph: 512 tokens 10.5 and 9.2 us, 768 10.6 and 11.6;
         * sixteen sequences: 768 16.9 and 14.9, 1024 18.6 and 18.1, 1536 22.9 and 24.8. */
        if (tokens <= (pairs >= device_cus() / 2 ? 1024 : 512)) p.few.splits = 0;
        if (!tree && pairs > 65536) p.few.splits = 0; /* places for their parts would take gigabytes */
        p.few.blocks = p.few.splits + pairs;
        if (p.few.splits) p.ws_bytes = (size_t)(tree ? tree_places(p.few) : p.few.blocks) * rm * (dim + 2) * 4;
    }
    if (p.many.items && tree) {
        /* A tree's rows see all of what stands before them, and sequences are as long as they are: parts of equal size, one round
         * of blocks. */
        const long long blocks = (long long)chunk_blocks(dim, dim == 256) * device_cus();
        const long long pairs = (long long)p.many.items * c->kv_heads, units = pairs * ((tokens + kUnit - 1) / kUnit);
        p.many.splits = (int)(units < 1 ? 1 : units < blocks ? units : blocks);
        p.many.least = 2;
        p.many.blocks = p.many.splits + pairs;
        p.many.ws_at = p.ws_bytes;
        p.ws_bytes += (size_t)tree_places(p.many) * kChunkRows * (dim + 2) * 4;
    } else if (p.many.items) {
        /* Two blocks a CU, by the tiles there are if max_new holds (`items` can be up to twice as many);
         * one, or parts of `least` tokens, where two would make those shorter, since a part's results
         * are 66 KB at 128 values a head. 16 sequences of 4096 tokens with 32 new ones, FP8: 1024 tokens
         * 80 us, 1536 91; one of 32768 with 64, BF16: 85 and 69. */
        const int least = c->format == W4A16_KV_BF16 ? 1536 : 1024;
        const long long blocks = (long long)p.many.items * c->kv_heads, cus = device_cus();
        const long long likely = seqs * ((longest + kChunkRows - 1) / kChunkRows);
        const long long tiles = (likely < p.many.items ? likely : p.many.items) * c->kv_heads;
        const long long most = (tokens + kFewestTokens - 1) / kFewestTokens;
        long long splits = (2 * cus + tiles - 1) / tiles;
        if (tokens < least * splits) {
            const long long one = (cus + tiles - 1) / tiles, parts = (tokens + least - 1) / least;
            splits = one > parts ? one : parts;
        }
        if (splits > most) splits = most;
        if (splits > 256) splits = 256;
        p.many.splits = splits < 1 ? 1 : (int)splits;
        p.many.ws_at = p.ws_bytes;
        if (p.many.splits > 1) p.ws_bytes += (size_t)blocks * p.many.splits * kChunkRows * (dim + 2) * 4;
    }
    return p;
}

template <int D, int RM, bool EVEN, bool TREE>
void launch_join(int parts, const AttnArgs &a, hipStream_t s) {
    unsigned x = a.kv.heads * a.items;
    if (TREE && x > (unsigned)a.splits) x = a.splits; /* pairs that are cut */
    if constexpr (TREE && RM == kChunkRows) {
        /* Side by side only where there are fewer blocks than CUs else, however many parts there are. FP8, 128 values, 60 nodes, one part after
         * another and four at a time: 16 sequences of 2048 tokens 63 and 77 us, four of 8192 62 and 63, one of 100000 166 and 154 (16
         * at a time 144, 77, 153). */
        if (x * (RM / 16) < (unsigned)device_cus()) launch_k(attn_join_kernel<D, RM, 4, EVEN, TREE>, dim3(x, RM / 4), dim3(256), 0, s, a);
        else launch_k(attn_join_kernel<D, RM, 1, EVEN, TREE>, dim3(x, RM / 16), dim3(256), 0, s, a);
    } else {
        if (parts > 16) launch_k(attn_join_kernel<D, RM, 16, EVEN, TREE>, dim3(x, RM), dim3(256), 0, s, a);
        else if (parts > 4) launch_k(attn_join_kernel<D, RM, 4, EVEN, TREE>, dim3(x, RM / 4), dim3(256), 0, s, a);
        else if (parts > 1) launch_k(attn_join_kernel<D, RM, 1, EVEN, TREE>, dim3(x, RM / 16), dim3(256), 0, s, a);
    }
}

/* Parts of a (tile, head), about. */
int parts_of(const AttnArgs &a) { return (a.splits + a.items * a.kv.heads - 1) / (a.items * a.kv.heads) + 1; }

AttnArgs part_args(const AttnArgs &all, const Part &p) {
    AttnArgs a = all;
    a.items = p.items;
    a.splits = p.splits;
    a.blocks = (int)p.blocks;
    a.over = p.over;
    a.upto = p.upto;
    a.least = p.least;
    a.ws += p.ws_at / 4;
    return a;
}

template <int D, int FMT, bool TREE>
void launch_format(const Plan &p, const AttnArgs &all, hipStream_t s) {
    if (p.many.items) {
        const AttnArgs a = part_args(all, p.many);
        auto kernel = attn_chunk_kernel<D, FMT, D == 256, TREE>;
        size_t lds = Chunk<D, FMT, D == 256, TREE>::kBytes;
        if constexpr (D == 64 && FMT != W4A16_KV_BF16 && !TREE) /* with trees it would spill */
            if ((long long)a.kv.heads * a.items * a.splits > chunk_blocks(D, false) * device_cus()) {
                kernel = attn_chunk_kernel<D, FMT, true, TREE>;
                lds = Chunk<D, FMT, true, TREE>::kBytes;
            }
        if constexpr (TREE) {
            launch_k(kernel, dim3((unsigned)p.many.blocks), dim3(256), lds, s, a);
            launch_join<D, kChunkRows, true, TREE>(parts_of(a), a, s);
        } else {
            launch_k(kernel, dim3(a.kv.heads * a.items, a.splits), dim3(256), lds, s, a);
            launch_join<D, kChunkRows, false, TREE>(a.splits, a, s);
        }
    }
    if (p.few.items) {
        const AttnArgs a = part_args(all, p.few);
        if constexpr (D <= 128 || TREE)
            if (p.rt == 2) {
                launch_k(attn_rows_kernel<D, FMT, 2, TREE>, dim3((unsigned)p.few.blocks), dim3(256), 0, s, a);
                if (a.splits) launch_join<D, 32, true, TREE>(parts_of(a), a, s);
                return;
            }
        launch_k(attn_rows_kernel<D, FMT, 1, TREE>, dim3((unsigned)p.few.blocks), dim3(256), 0, s, a);
        if (a.splits) launch_join<D, 16, true, TREE>(parts_of(a), a, s);
    }
}

template <int D, bool TREE>
void launch_dim(int format, const Plan &p, const AttnArgs &a, hipStream_t s) {
    if (format == W4A16_KV_BF16) launch_format<D, W4A16_KV_BF16, TREE>(p, a, s);
    else if (format == W4A16_KV_INT8) launch_format<D, W4A16_KV_INT8, TREE>(p, a, s);
    else launch_format<D, W4A16_KV_FP8, TREE>(p, a, s);
}

template <bool TREE>
void launch_all(int dim, int format, const Plan &p, const AttnArgs &a, hipStream_t s) {
    if (dim == 64) launch_dim<64, TREE>(format, p, a, s);
    else if (dim == 128) launch_dim<128, TREE>(format, p, a, s);
    else launch_dim<256, TREE>(format, p, a, s);
}

int check_heads(const KvView &kv, int q_heads, const char *what) {
    if (q_heads < 1 || q_heads % kv.heads || (long long)q_heads * kv.rows > INT32_MAX / 2)
        return set_error(W4A16_ERR_CONFIG, "%s: q_heads=%d is no multiple of the cache's %d heads, or %d rows of them "
                         "are too many", what, q_heads, kv.heads, kv.rows);
    return W4A16_OK;
}

} // namespace

namespace {

int workspace(const char *what, const W4A16KvCache *cache, const W4A16KvBatch *batch, int q_heads, bool tree, size_t *bytes) {
    if (!bytes) return set_error(W4A16_ERR_CONFIG, "%s: null result", what);
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (!st) st = check_heads(kv, q_heads, what);
    if (st) return st;
    *bytes = kv.rows && kv.seqs ? plan_of(cache, batch, q_heads, tree).ws_bytes : 0;
    return W4A16_OK;
}

} // namespace

extern "C" int w4a16_paged_attention_workspace(const W4A16KvCache *cache, const W4A16KvBatch *batch, int q_heads,
                                               size_t *bytes) {
    return workspace("w4a16_paged_attention_workspace", cache, batch, q_heads, false, bytes);
}

extern "C" int w4a16_paged_tree_attention_workspace(const W4A16KvCache *cache, const W4A16KvBatch *batch, int q_heads,
                                                    size_t *bytes) {
    return workspace("w4a16_paged_tree_attention_workspace", cache, batch, q_heads, true, bytes);
}

namespace {

int attend(const char *what, const W4A16KvCache *cache, const W4A16KvBatch *batch, const W4A16KvTree *tree, const uint16_t *q,
           long long q_row_stride, long long q_head_stride, int q_heads, float scale, int causal, int window, uint16_t *out,
           long long out_row_stride, long long out_head_stride, float *lse, void *ws, size_t ws_bytes, void *stream) {
    KvView kv;
    int st = kv_check(cache, batch, what, &kv);
    if (!st) st = check_heads(kv, q_heads, what);
    if (st) return st;
    if (!(scale - scale == 0.0f)) return set_error(W4A16_ERR_CONFIG, "%s: the scale is not finite", what);
    if (window < 0) return set_error(W4A16_ERR_CONFIG, "%s: window=%d is negative", what, window);
    if (tree) {
        if (tree->nodes < 1 || tree->nodes > 256)
            return set_error(W4A16_ERR_CONFIG, "%s: trees of nodes=%d are not of 1 to 256", what, tree->nodes);
        if (window && window < tree->nodes) /* a row's window would end inside its tree, by depths that the bits do not have */
            return set_error(W4A16_ERR_CONFIG, "%s: window=%d is smaller than trees of %d nodes", what, window, tree->nodes);
    }
    if (kv.rows == 0 || kv.seqs == 0) return W4A16_OK;
    if (!q || !out) return set_error(W4A16_ERR_CONFIG, "%s: null buffer", what);
    if (misaligned(q) || misaligned(out) || misaligned(ws) || ((uintptr_t)lse & 3))
        return set_error(W4A16_ERR_CONFIG, "%s: buffers must be 16-byte aligned (lse: 4)", what);
    const int dim = cache->head_dim;
    drop_strides_of_one(kv.rows, &q_row_stride, q_heads, &q_head_stride);
    drop_strides_of_one(kv.rows, &out_row_stride, q_heads, &out_head_stride);
    const size_t qb = strided_bytes(kv.rows, q_row_stride, q_heads, q_head_stride, dim);
    const size_t ob = strided_bytes(kv.rows, out_row_stride, q_heads, out_head_stride, dim);
    if (!qb || !ob) return set_error(W4A16_ERR_CONFIG, "%s: strides must be multiples of 8 elements from 0", what);
    const RowsView qr = {q, qb, q_row_stride, q_head_stride, q_heads}, outs = {out, ob, out_row_stride, out_head_stride, q_heads};
    if (!rows_apart(kv.rows, outs, dim)) return set_error(W4A16_ERR_CONFIG, "%s: output rows overlap each other", what);
    const Plan p = plan_of(cache, batch, q_heads, tree != nullptr);
    if (p.ws_bytes > 0 && (!ws || ws_bytes < p.ws_bytes))
        return set_error(W4A16_ERR_CONFIG, "%s: a workspace of %zu bytes, the call needs %zu", what, ws ? ws_bytes : 0,
                         p.ws_bytes);
    /* q and out may be the same tensor, or heads of the same rows side by side */
    bool clash = !rows_same(qr, outs) && !rows_beside(kv.rows, outs, qr, dim);
    size_t tb = 0, pb = 0, nb = 0;
    if (tree) {
        if (!tree->seen || !tree->positions) return set_error(W4A16_ERR_CONFIG, "%s: null tree", what);
        if (((uintptr_t)tree->seen & 7) || (((uintptr_t)tree->positions | (uintptr_t)tree->sizes) & 3))
            return set_error(W4A16_ERR_CONFIG, "%s: the tree's bits must be 8-byte aligned, positions and sizes 4-byte", what);
        tb = (size_t)kv.rows * ((tree->nodes + 63) / 64) * 8;
        pb = (size_t)kv.rows * 4;
        nb = tree->sizes ? (size_t)kv.seqs * 4 : 0;
    }
    const size_t lb = lse ? (size_t)kv.rows * q_heads * 4 : 0, cb = kv_bytes(cache), sb = kv_scale_bytes(cache);
    const struct { const void *p; size_t n; } writes[] = {{out, ob}, {lse, lb}, {ws, p.ws_bytes}};
    const struct { const void *p; size_t n; } reads[] = {{cache->k, cb}, {cache->v, cb}, {kv.k_scale, sb}, {kv.v_scale, sb},
                                                         {tree ? tree->seen : nullptr, tb}, {tree ? tree->positions : nullptr, pb},
                                                         {tree ? tree->sizes : nullptr, nb}};
    for (int i = 0; i < 3; ++i) {
        for (const auto &r : reads) clash = clash || overlap(writes[i].p, writes[i].n, r.p, r.n);
        if (i) clash = clash || overlap(writes[i].p, writes[i].n, q, qb);
        for (int j = 0; j < i; ++j) clash = clash || overlap(writes[i].p, writes[i].n, writes[j].p, writes[j].n);
    }
    if (clash) return set_error(W4A16_ERR_CONFIG, "%s: an output or the workspace overlaps another buffer", what);
    const long long tiles = (long long)(p.few.items > p.many.items ? p.few.items : p.many.items) * kv.heads;
    if (tiles > 1 << 23)
        return set_error(W4A16_ERR_CONFIG, "%s: %lld tiles of rows: at most 2^23 a call", what, tiles);
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
    a.splits = a.items = a.blocks = a.over = a.upto = a.least = 0; /* part_args */
    a.scale = fabsf(scale) * 1.4426950408889634f;
    a.flip = scale < 0.0f ? 0x80008000u : 0u;
    a.tree = tree ? *tree : W4A16KvTree{};
    hipStream_t s = static_cast<hipStream_t>(stream);
    (tree ? launch_all<true> : launch_all<false>)(dim, cache->format, p, a, s);
    return hip_status(hipGetLastError(), "paged attention launch");
}

} // namespace

extern "C" int w4a16_paged_attention_bf16(const W4A16KvCache *cache, const W4A16KvBatch *batch, const uint16_t *q,
                                          long long q_row_stride, long long q_head_stride, int q_heads, float scale,
                                          int causal, int window, uint16_t *out, long long out_row_stride,
                                          long long out_head_stride, float *lse, void *ws, size_t ws_bytes,
                                          void *stream) {
    return attend("w4a16_paged_attention_bf16", cache, batch, nullptr, q, q_row_stride, q_head_stride, q_heads, scale, causal,
                  window, out, out_row_stride, out_head_stride, lse, ws, ws_bytes, stream);
}

extern "C" int w4a16_paged_tree_attention_bf16(const W4A16KvCache *cache, const W4A16KvBatch *batch, const W4A16KvTree *tree,
                                               const uint16_t *q, long long q_row_stride, long long q_head_stride,
                                               int q_heads, float scale, int window, uint16_t *out,
                                               long long out_row_stride, long long out_head_stride, float *lse, void *ws,
                                               size_t ws_bytes, void *stream) {
    const char *what = "w4a16_paged_tree_attention_bf16";
    if (!tree) return set_error(W4A16_ERR_CONFIG, "%s: null tree", what);
    return attend(what, cache, batch, tree, q, q_row_stride, q_head_stride, q_heads, scale, 1, window, out, out_row_stride,
                  out_head_stride, lse, ws, ws_bytes, stream);
}
