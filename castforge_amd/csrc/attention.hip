// Attention over the paged cache of 4-bit keys and values:
//   o[i] = sum_t p[i, t] v[t],  p = softmax over the visible t of scale * <q[i], k[t]>,
//   k[t], v[t] = (codes - z) * s a group of channels.
//
// Query i of the n of a sequence with L cached tokens sees the tokens t < L, and with `causal` only those
// with t <= L - n + i (its own place, counted from the end).  A query that sees no token gives zeros, and
// -inf as the logarithm of its sum.
//
// The softmax's maximum and sum, the scores and the output sums are f32.
#include <algorithm>
#include <atomic>

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"
#include "kv4.hpp"

namespace cfh {
namespace {

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -3.402823466e38f;  // below every score, finite: exp2(-inf - kNoMax) is 0, not NaN

struct AttnArgs {
    const uint16_t *q;
    int64_t q_stride;
    const uint32_t *k_codes, *k_groups, *v_codes, *v_groups;
    const int32_t *cu_q;  // NULL: one query a sequence
    const int32_t *table, *kv_lens;
    uint16_t *out;
    float *lse;
    float *part;  // splits > 1: [tokens * q heads][splits][D + 4], output sums, reference, sum, two unused
    float scale;
    int tokens, batch, heads, ratio, page_shift, table_cols, num_pages, causal, splits;
    int first_tile;  // of a launch's row tiles, where one launch cannot hold them all
};

// A uniform word through the scalar cache: no vector load, whose wait would take in the tile loads before it.
__device__ __forceinline__ int32_t scalar_load(const int32_t *p, int64_t i) {
    return ((const __attribute__((address_space(4))) int32_t *)(p))[i];
}

__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Codes as they stand in a word are f16 denormals: pairs 16 bits apart, code times 2^-24, or 2^-20 where it lies 4 bits
// higher; a zero point held the same way is subtracted from them exactly.  (Subtracting the zero points'
// share of a sum instead leaves the f32 rounding of sums of up to 15 times a weight, 2^-22 of them each (measured): up to 2^-18 of
// a heavy token's weight where its codes equal its zero point.)
__device__ __forceinline__ uint32_t minus(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(halfx2, a) - __builtin_bit_cast(halfx2, b));
}

__device__ __forceinline__ halfx8 eight(uint32_t p0, uint32_t p1, uint32_t p2, uint32_t p3) {
    return __builtin_bit_cast(halfx8, uintx4{p0, p1, p2, p3});
}

// A word's eight codes without their zero point zz (both halves), in the order 0 4 1 5 2 6 3 7; those of positions
// 1, 3, 5, 7 are 16 times the others.
__device__ __forceinline__ halfx8 codes_f16(uint32_t w, uint32_t zz) {
    const uint32_t v = w >> 8, z16 = zz << 4;
    return eight(minus(w & 0x000F000Fu, zz), minus(w & 0x00F000F0u, z16), minus(v & 0x000F000Fu, zz), minus(v & 0x00F000F0u, z16));
}

__device__ __forceinline__ float sum_over_g(float v) { v += __shfl_xor(v, 16); return v + __shfl_xor(v, 32); }
__device__ __forceinline__ float max_over_g(float v) { v = fmaxf(v, __shfl_xor(v, 16)); return fmaxf(v, __shfl_xor(v, 32)); }
__device__ __forceinline__ int max_over_wave(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o));
    return __builtin_amdgcn_readfirstlane(v);
}

// The instruction itself: fmaxf() quiets each operand first, ten instructions more for a row's eight scores.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// One sequence's share of a workgroup.
struct Seq {
    int seq, first, n, len, tile;  // first token of its n queries; cached tokens; row tile
};

// Tokens that a sequence's table holds: so far below 2^31 (check_counts) that a round of a workgroup's tokens past a length does not
// wrap.
__device__ __forceinline__ int token_cap(const AttnArgs &a) { return a.table_cols << a.page_shift; }

// Splits that share a sequence of len tokens: at least 128 tokens each.
__device__ __forceinline__ int splits_of(int len, int splits) { return max(1, min(splits, (len + 127) / 128)); }

// Which sequence's row tile a workgroup has: tiles are dealt to the sequences in order, rows_per_tile rows each.
// The lanes of a wave look at 64 sequences at once.  Returns seq -1 past the last tile.
__device__ __forceinline__ Seq find_tile(const AttnArgs &a, int tile, int rows_per_tile) {
    const int lane = threadIdx.x & 63;
    const int cap = token_cap(a);
    if (!a.cu_q) {
        const int per = (a.ratio + rows_per_tile - 1) / rows_per_tile, s = tile / per;
        if (s >= a.batch) return Seq{-1, 0, 0, 0, 0};
        return Seq{s, s, 1, a.num_pages > 0 ? min(max(scalar_load(a.kv_lens, s), 0), cap) : 0, tile - s * per};
    }
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        int first = 0, n = 0;
        if (b < a.batch) {  // clamped: a malformed list stays inside the rows
            first = min(max(a.cu_q[b], 0), a.tokens);
            n = min(max(a.cu_q[b + 1], first), a.tokens) - first;
        }
        const int tiles = static_cast<int>((static_cast<int64_t>(n) * a.ratio + rows_per_tile - 1) / rows_per_tile);
        int upto = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        const uint64_t hit = __ballot(before + upto > tile);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            Seq s;
            s.seq = b0 + l;
            s.first = __builtin_amdgcn_readlane(first, l);
            s.n = __builtin_amdgcn_readlane(n, l);
            s.tile = tile - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(tiles, l));
            s.len = a.num_pages > 0 ? min(max(scalar_load(a.kv_lens, s.seq), 0), cap) : 0;
            return s;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return Seq{-1, 0, 0, 0, 0};
}

// Registers of 32 tokens' keys and values of a head, in halves of 16.  n = lane % 16, g = lane / 16.
template <int D, int G>
struct KvTile {
    static constexpr int GR = D / G, W = G / 32;
    uint32_t kc[2][GR][W];  // token n: words g W .. of each group
    // tokens 4 g + r: word n % (G / 8) of each group; where a row has 16 words in several groups word n alone, from which
    // attend() deals the groups' out through LDS (a lane would load each word GR times over)
    static constexpr bool kDeal = D == 128 && GR > 1;
    static constexpr int VW = kDeal ? 1 : GR;
    uint32_t vc[2][4][VW];
    uint32_t words[GR];     // group words of one token: lanes 0 .. 31 of the keys, 32 .. 63 of the values
    bool live[2];           // uniform: the half's page is one of the cache's
};

// What the group words of N tokens say, in LDS: worked out once, each lane for one token's keys or values, and read four tokens
// at a time.
template <int GR, int N>
struct Tokens {
    float keys[N][GR];   // scale times what turns a product into a score
    float exponent[N];   // of the values' largest scale, by magnitude; -inf where there is no token
    float back[N];       // 2^-exponent
};

// What a wave keeps to itself of N tokens: zero points, the values' scales, and its deal of their words.
template <int D, int G, int N, class C>
struct Own {
    static constexpr int GR = D / G, kRow = N + 4;   // tokens a row of `v`, padded for the banks
    uint32_t v[KvTile<D, G>::kDeal ? 16 * kRow : 4];  // the values' codes: word by word, a token each
    uint32_t k[N][GR];  // zero point in both halves, as f16 denormals
    uint16_t z[GR][N];  // of the values
    // the values' scales without the exponent: f32 ones a token's together, f16 ones, times 2^11, in pairs of tokens
    static constexpr bool kPairs = sizeof(C) == 2;
    C c[kPairs ? GR : N][kPairs ? N : GR];
};

template <int D, int G>
__device__ __forceinline__ void load_tile(const AttnArgs &a, KvTile<D, G> &t, int head, const int (&page)[2], int at, int end) {
    constexpr int GR = D / G, W = G / 32, kWords = D / 8;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    int64_t rows[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        t.live[h] = at + 16 * h < end && page[h] >= 0 && page[h] < a.num_pages;
        rows[h] = kv4_row(t.live[h] ? page[h] : 0, head, (at + 16 * h) & ((1 << a.page_shift) - 1), a.heads, a.page_shift);
        const uint32_t *kc = a.k_codes + rows[h] * kWords + n * kWords + g * W;
        const uint32_t *vc = a.v_codes + rows[h] * kWords + 4 * g * kWords + (KvTile<D, G>::kDeal ? n : n % (G / 8));
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
            if constexpr (W == 4) {
                // whole cache lines in one instruction, past the caches: 48 sequences of up to 8000 tokens 65 -> 60 us.  (Not so the
                // values' or smaller groups' words, whose lines several instructions share: up to a fifth slower.)
                const uint4 v = load_once(kc + gr * (G / 8));
                t.kc[h][gr][0] = v.x, t.kc[h][gr][1] = v.y, t.kc[h][gr][2] = v.z, t.kc[h][gr][3] = v.w;
            } else if constexpr (W == 2) {
                const uint2 v = *reinterpret_cast<const uint2 *>(kc + gr * (G / 8));
                t.kc[h][gr][0] = v.x, t.kc[h][gr][1] = v.y;
            } else {
                t.kc[h][gr][0] = kc[gr * (G / 8)];
            }
        }
#pragma unroll
        for (int i = 0; i < KvTile<D, G>::VW; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) t.vc[h][r][i] = vc[r * kWords + i * (G / 8)];
    }
    const uint32_t *w = (lane < 32 ? a.k_groups : a.v_groups) + ((lane & 16 ? rows[1] : rows[0]) + n) * GR;
    if constexpr (GR == 4) {
        const uint4 v = *reinterpret_cast<const uint4 *>(w);
        t.words[0] = v.x, t.words[1] = v.y, t.words[2] = v.z, t.words[3] = v.w;
    } else if constexpr (GR == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(w);
        t.words[0] = v.x, t.words[1] = v.y;
    } else {
        t.words[0] = *w;
    }
}

// LDS accesses of one wave keep their order; the compiler must not move them past each other either.
__device__ __forceinline__ void wave_order() { asm volatile("" ::: "memory"); }

// The lane's token (`token` of the table; value: its values' words, else its keys') into the tables.  off: there is no such token,
// and its words may be anything.
template <int D, int G, int N, int M, class C>
__device__ __forceinline__ void fill_token(const uint32_t (&words)[D / G], bool value, int token, bool off, float qk, Tokens<D / G, N> &tokens, Own<D, G, M, C> &own, int at) {
    constexpr int GR = D / G;
    float v[GR], top = 0.f;
    uint32_t z[GR];
#pragma unroll
    for (int gr = 0; gr < GR; ++gr) {
        const uint32_t w = off ? 0u : words[gr];
        v[gr] = kv4_scale(w);
        top = fmaxf(top, fabsf(v[gr]));  // a caller's own cache may hold negative ones
        z[gr] = kv4_zero(w);
    }
    const int ex = __builtin_amdgcn_frexp_expf(top);
    if (value) {
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
            own.z[gr][at] = static_cast<uint16_t>(z[gr]);
            v[gr] = __builtin_ldexpf(v[gr], (sizeof(C) == 2 ? 11 : 0) - ex);
            if constexpr (Own<D, G, M, C>::kPairs) own.c[gr][at] = static_cast<C>(v[gr]);  // exact down to 2^-25
        }
        if constexpr (!Own<D, G, M, C>::kPairs) __builtin_memcpy(__builtin_assume_aligned(own.c[at], 4 * GR), v, 4 * GR);
    } else {
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) v[gr] *= qk, z[gr] *= 0x00010001u;
        __builtin_memcpy(__builtin_assume_aligned(tokens.keys[token], 4 * GR), v, 4 * GR);
        __builtin_memcpy(__builtin_assume_aligned(own.k[at], 4 * GR), z, 4 * GR);
    }
    if (value) tokens.exponent[token] = off ? -INFINITY : static_cast<float>(ex), tokens.back[token] = __builtin_ldexpf(1.0f, -ex);
}

// Four tokens' words of a row of V^T as pairs of tokens, codes 0 .. 3 and 4 .. 7: the row is word n % (G / 8) of the group, and its
// codes are those from n / (G / 8) on in steps of R = 128 / G.
struct Pairs {
    uint32_t lo[2], hi[2];
};
template <int G>
__device__ __forceinline__ Pairs pairs_of(uint4 w, int n) {
    if constexpr (G < 128) {
        const int sh = 4 * (n / (G / 8));
        w.x >>= sh, w.y >>= sh, w.z >>= sh, w.w >>= sh;
    }
    return Pairs{{low_halves(w.x, w.y), low_halves(w.z, w.w)}, {high_halves(w.x, w.y), high_halves(w.z, w.w)}};
}

// Code `code` of pair i without its zero points.
__device__ __forceinline__ uint32_t pair_code(const Pairs &p, int i, int code, uint32_t z) {
    const uint32_t x = code < 4 ? p.lo[i] : p.hi[i], y = code % 4 < 2 ? x : x >> 8;
    return code % 2 == 0 ? minus(y & 0x000F000Fu, z) : minus(y & 0x00F000F0u, z << 4);
}

// The same with the scales c (f16, times 2^11) taken in, rounded once to f16: codes in the mantissas of 1024 or 64, from which the
// zero points are subtracted exactly.
__device__ __forceinline__ uint32_t pair_value(const Pairs &p, int i, int code, uint32_t z, uint32_t c) {
    const uint32_t x = code < 4 ? p.lo[i] : p.hi[i], y = code % 4 < 2 ? x : x >> 8;
    const uint32_t v = code % 2 == 0 ? minus((y & 0x000F000Fu) | 0x64006400u, z | 0x64006400u) : minus((y & 0x00F000F0u) | 0x54005400u, (z << 4) | 0x54005400u);
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(halfx2, v) * __builtin_bit_cast(halfx2, c));
}

// Rows of a wave: 16 MT of the n * ratio (query, head of the group) pairs of a sequence and a head of keys, row = query *
// ratio + head; the MFMAs' columns.  With S^T = K Q^T a lane holds the scores of one row and four tokens a
// half, which is the layout that O^T = V^T P^T takes its second operand in: the weights stay in registers.
template <int D, int G, int MT>
struct Rows {
    static constexpr int GR = D / G, W = G / 32, R = 128 / G, NT = 8 / R;  // NT output tiles of 16 channels a group
    halfx8 q[MT][GR][W];     // the row by a power of two, in the order and by the factors of codes_f16
    float rel[MT];           // what undoes the power of two; in the tile kernel, what the tables' share of it leaves
    bool uneven;             // tile kernel, uniform: rel is not 1 everywhere
    int limit[MT];           // tokens that the lane's row sees
    floatx4 o[MT][GR][NT];   // sum of weight * (code - zero point), by code position times 2^-24 or 2^-20
    float m[MT], l[MT];      // reference and this lane's part of the sum
};

// Loads the rows.  A row's power of two takes its largest element below 2^14, so that a sixteenth of it keeps bf16's bits down to
// 2^-24 of the largest.  kShared: all rows take the greatest one's, whose exponent is returned for the tables to hold: a row
// 2^10 smaller keeps its bits down to 2^-16 of its largest and loses 2^-25 of that below.  Rows smaller still have their own, as
// have rows above 2^64, whose exponent would take the tables out of f32's range; `uneven` is set then.  most(v): the greatest v of
// those who read the tables.
template <bool kShared, int D, int G, int MT, class Most>
__device__ __forceinline__ int load_rows(const AttnArgs &a, Rows<D, G, MT> &s, const Seq &sq, int head, int row0, const Most &most) {
    constexpr int GR = D / G, W = G / 32, kNone = -1000;
    const int n = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    uint4 raw[MT][GR][W];
    int ex[MT], greatest = kNone;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int row = row0 + 16 * mt + n, i = row / a.ratio;
        const bool in = i < sq.n;
        // rows past the sequence's see all: they are not stored, and do not make a tile an edge
        s.limit[mt] = in ? (a.causal ? min(sq.len, sq.len - sq.n + i + 1) : sq.len) : 0x7fffffff;
        const uint16_t *p = a.q + (sq.first + (in ? i : 0)) * a.q_stride + (head * a.ratio + (in ? row - i * a.ratio : 0)) * D;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int u = 0; u < W; ++u) raw[mt][gr][u] = *reinterpret_cast<const uint4 *>(p + gr * G + (g * W + u) * 8);
    }
    const auto element = [&](int mt, int gr, int u, int e) {
        const uint4 v = raw[mt][gr][u];
        const uint32_t b = e / 2 == 0 ? v.x : e / 2 == 1 ? v.y : e / 2 == 2 ? v.z : v.w;
        return __uint_as_float(e % 2 ? b & 0xffff0000u : b << 16);
    };
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float top = 0.f;
#pragma unroll
        for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int u = 0; u < W; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(element(mt, gr, u, e)));
        top = max_over_g(top);
        ex[mt] = top > 0.f ? __builtin_amdgcn_frexp_expf(top) - 14 : kNone;
        greatest = max(greatest, ex[mt]);
    }
    int all = kShared ? most(max_over_wave(greatest)) : 0;
    all = all == kNone ? 0 : min(all, 50);  // kNone: rows of zeros
    bool apart = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const bool own = ex[mt] != kNone && (!kShared || ex[mt] < all - 10 || ex[mt] > all);
        const int at_ex = own ? ex[mt] : all;
        apart |= own;
        s.rel[mt] = __builtin_ldexpf(1.0f, at_ex - all);
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const auto at = [&](int e) { return static_cast<_Float16>(__builtin_ldexpf(element(mt, gr, u, e), -at_ex - (e % 2 ? 4 : 0))); };
                s.q[mt][gr][u] = halfx8{at(0), at(4), at(1), at(5), at(2), at(6), at(3), at(7)};
            }
#pragma unroll
            for (int t = 0; t < Rows<D, G, MT>::NT; ++t) s.o[mt][gr][t] = floatx4{0.f, 0.f, 0.f, 0.f};
        }
        s.m[mt] = kNoMax, s.l[mt] = 0.f;
    }
    s.uneven = __any(apart);
    return all;
}

// What turns a product of codes and a row (by 2^-ex) into a score, base 2; the codes' 2^-24 undone.
__device__ __forceinline__ float score_factor(const AttnArgs &a, int ex) { return __builtin_ldexpf(a.scale * 1.44269504088896341f, ex + 24); }

// 32 tokens at `at`.  A token's weight is held with the exponent of its values' scale: with s_t = c_t 2^e_t (the largest
// of its groups' magnitudes, c in [0.5, 1)), exp2(score + e_t - m) times c rounds to f16 as what the token adds to the output, whatever
// the scales are; the sum takes the 2^-e_t back.  m is 7 below the largest so far when it moves, and it moves only
// when something exceeds it by 15: weights stay below 2^15, the largest ones above 2^7 (f16 keeps its 11 bits
// down to 2^-21 of them), and the rescaling is rare.
// keys(h, gr, u): the MFMA operand of half h's 16 tokens and 32 channels; values(gr) prepares a group's rows of V^T and gives what
// turns u into the operand of 16 channels and 32 tokens.  first: the tokens' place in the table.  kShared: the values hold c
// already, rounded to f16 with it, and the weights are rounded alone; many rows share that work then.
template <bool kShared, int D, int G, int MT, int N, class Keys, class Values>
__device__ __forceinline__ void attend(const Tokens<D / G, N> &tokens, const float (*scales)[D / G], int first, Rows<D, G, MT> &s, int at, int sure, const Keys &keys, const Values &values) {
    constexpr int GR = D / G, W = G / 32, NT = G / 16;
    const int g = (threadIdx.x >> 4) & 3;
    const bool edge = at + 32 > sure;  // uniform: some row does not see some token
    const auto four = [&](const float *p, int h) { return *reinterpret_cast<const floatx4 *>(p + first + 16 * h + 4 * g); };
    struct Four {
        float v[4][GR];
    };
    const auto four_by = [&](const float (*p)[GR], int h) {  // of tokens with GR numbers each
        Four f;
        __builtin_memcpy(&f, __builtin_assume_aligned(p[first + 16 * h + 4 * g], 16), sizeof f);
        return f;
    };
    float y[MT][2][4];  // scores and their tokens' exponents, base 2
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const floatx4 e = four(tokens.exponent, h);
        const Four ks = four_by(tokens.keys, h);
        const auto product = [&](int gr, floatx4 (&dot)[MT]) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < W; ++u) {
                const halfx8 k = keys(h, gr, u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                    dot[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, s.q[mt][gr][u], u ? dot[mt] : floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
            }
        };
        if constexpr (kShared || (MT > 1 && GR == 4)) {
            // group by group: two row tiles of four groups fit the registers only so (all products first: one tile, and 267 us instead of
            // 198 for a prompt of 4096 tokens in groups of 32, 264 instead of 170 for 512 after 8192)
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) {
                floatx4 dot[MT];
                product(gr, dot);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[mt][h][r] = gr || kShared ? __builtin_fmaf(dot[mt][r], ks.v[r][gr], gr ? y[mt][h][r] : e[r]) : dot[mt][r] * ks.v[r][gr];
            }
            if constexpr (!kShared)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[mt][h][r] = __builtin_fmaf(y[mt][h][r], s.rel[mt], e[r]);
        } else {
            floatx4 dot[GR][MT];
#pragma unroll
            for (int gr = 0; gr < GR; ++gr) product(gr, dot[gr]);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float v = dot[0][mt][r] * ks.v[r][0];
#pragma unroll
                    for (int gr = 1; gr < GR; ++gr) v = __builtin_fmaf(dot[gr][mt][r], ks.v[r][gr], v);
                    y[mt][h][r] = __builtin_fmaf(v, s.rel[mt], e[r]);
                }
        }
    }
    if (edge || (kShared && s.uneven)) {
        asm volatile("");  // a branch: as selects on a uniform condition these were a quarter of the loop
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (kShared) {
                    const float e = tokens.exponent[first + 16 * (i / 4) + 4 * g + i % 4];
                    y[mt][i / 4][i % 4] = e > -INFINITY ? __builtin_fmaf(y[mt][i / 4][i % 4] - e, s.rel[mt], e) : -INFINITY;
                }
                if (at + 16 * (i / 4) + 4 * g + i % 4 >= s.limit[mt]) y[mt][i / 4][i % 4] = -INFINITY;
            }
    }
    constexpr int PG = kShared ? 1 : GR;
    uint32_t p[MT][PG][4];  // weights, times c, as f16 pairs: tokens (0, 1), (2, 3) of both halves
    {
        floatx4 back[2];
        Four c[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            back[h] = four(tokens.back, h);
            if constexpr (!kShared) c[h] = four_by(scales, h);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float (&v)[2][4] = y[mt];
            const float top = max3(max3(v[0][0], v[0][1], v[0][2]), max3(v[0][3], v[1][0], v[1][1]), max3(v[1][2], v[1][3], v[1][3]));
            if (__any(top > s.m[mt] + 15.f)) {
                const float m = fmaxf(s.m[mt], max_over_g(top) - 7.f), f = __builtin_amdgcn_exp2f(s.m[mt] - m);
                s.m[mt] = m;
                s.l[mt] *= f;
#pragma unroll
                for (int gr = 0; gr < GR; ++gr)
#pragma unroll
                    for (int u = 0; u < NT; ++u) s.o[mt][gr][u] *= f;
            }
            float w[2][4];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i / 4][i % 4] = __builtin_amdgcn_exp2f(y[mt][i / 4][i % 4] - s.m[mt]);
                s.l[mt] = __builtin_fmaf(w[i / 4][i % 4], back[i / 4][i % 4], s.l[mt]);
            }
#pragma unroll
            for (int gr = 0; gr < PG; ++gr)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int h = i / 2, r = i % 2 * 2;
                    const float c0 = kShared ? 1.f : c[h].v[r][gr], c1 = kShared ? 1.f : c[h].v[r + 1][gr];
                    const halfx2 v = {static_cast<_Float16>(w[h][r] * c0), static_cast<_Float16>(w[h][r + 1] * c1)};
                    p[mt][gr][i] = __builtin_bit_cast(uint32_t, v);
                }
        }
    }
#pragma unroll
    for (int gr = 0; gr < GR; ++gr) {
        halfx8 pw[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const uint32_t(&w)[4] = p[mt][kShared ? 0 : gr];
            pw[mt] = eight(w[0], w[1], w[2], w[3]);
        }
        const auto operand = values(gr);
        static_for<NT>([&](auto u) __attribute__((always_inline)) {
            const halfx8 v = operand(u);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s.o[mt][gr][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, pw[mt], s.o[mt][gr][u], 0, 0, 0);
        });
    }
}

// The least of the rows' limits: tokens below it are seen by every row of the wave.
template <int D, int G, int MT>
__device__ __forceinline__ int seen_by_all(const Rows<D, G, MT> &s, int len) {
    int sure = len;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) sure = min(sure, s.limit[mt]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sure = min(sure, __shfl_xor(sure, o));
    return __builtin_amdgcn_readfirstlane(sure);
}


// A wave's walk over tokens first, first + step, .. (of 32) below end, the next tile's loads in flight.
template <int D, int G, int MT>
__device__ __forceinline__ void walk(const AttnArgs &a, Tokens<D / G, 32> &tokens, Own<D, G, 32, float> &own, Rows<D, G, MT> &s, const Seq &sq, int head,
                                     int first, int step, int end) {
    constexpr int R = 128 / G;
    if (first >= end) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int sure = seen_by_all(s, sq.len);
    const float qk = score_factor(a, 0);
    const int32_t *table = a.table + static_cast<int64_t>(sq.seq) * a.table_cols;
    const auto pages = [&](int at, int (&p)[2]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) p[h] = at + 16 * h < end ? scalar_load(table, (at + 16 * h) >> a.page_shift) : -1;
    };
    KvTile<D, G> cur;
    int page[2];
    pages(first, page);
    load_tile<D, G>(a, cur, head, page, first, end);
    pages(first + step, page);
    for (int at = first; at < end; at += step) {
        KvTile<D, G> next;
        if (at + step < end) {
            load_tile<D, G>(a, next, head, page, at + step, end);
            pages(at + 2 * step, page);
        } else {
            next = cur;
        }
        const int token = lane & 31;
        wave_order();
        fill_token(cur.words, lane >= 32, token, !(token < 16 ? cur.live[0] : cur.live[1]) || at + token >= sq.len, qk, tokens, own, token);
        if constexpr (KvTile<D, G>::kDeal) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<uint4 *>(&own.v[n * Own<D, G, 32, float>::kRow + 16 * h + 4 * g]) = make_uint4(cur.vc[h][0][0], cur.vc[h][1][0], cur.vc[h][2][0], cur.vc[h][3][0]);
        }
        wave_order();
        attend<false, D, G, MT>(
            tokens, own.c, 0, s, at, sure, [&](int h, int gr, int u) { return codes_f16(cur.kc[h][gr][u], own.k[16 * h + n][gr]); },
            [&](int gr) {
                Pairs p[2];
                uint2 z[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (KvTile<D, G>::kDeal)
                        p[h] = pairs_of<G>(*reinterpret_cast<const uint4 *>(&own.v[(gr * (G / 8) + n % (G / 8)) * Own<D, G, 32, float>::kRow + 16 * h + 4 * g]), n);
                    else
                        p[h] = pairs_of<G>(make_uint4(cur.vc[h][0][gr], cur.vc[h][1][gr], cur.vc[h][2][gr], cur.vc[h][3][gr]), n);
                    z[h] = *reinterpret_cast<const uint2 *>(&own.z[gr][16 * h + 4 * g]);
                }
                return [=](int u) {
                    return eight(pair_code(p[0], 0, R * u, z[0].x), pair_code(p[0], 1, R * u, z[0].y), pair_code(p[1], 0, R * u, z[1].x),
                                 pair_code(p[1], 1, R * u, z[1].y));
                };
            });
        cur = next;
    }
}

// Channel of element (r of a lane's four, group gr, tile u) of O^T.
template <int G>
__device__ __forceinline__ int channel(int g, int r, int gr, int u) {
    constexpr int R = 128 / G;
    const int n = 4 * g + r;
    return gr * G + 8 * (n % (G / 8)) + R * u + n / (G / 8);
}

// The whole sum, and the outputs without the codes' factors.
template <bool kShared, int D, int G, int MT>
__device__ __forceinline__ void settle(Rows<D, G, MT> &s) {
    typedef Rows<D, G, MT> S;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        s.l[mt] = sum_over_g(s.l[mt]);
#pragma unroll
        for (int gr = 0; gr < S::GR; ++gr)
#pragma unroll
            for (int u = 0; u < S::NT; ++u) s.o[mt][gr][u] *= kShared ? 0x1p-11f : (S::R * u) % 2 ? 0x1p20f : 0x1p24f;
    }
}

// One workgroup's NW waves take the same rows and every NW-th 32 tokens of a split's share, and are joined through LDS;
// splits are joined by kv4_attention_join_kernel.  For few rows a sequence: bound by the cache's bytes where they are many (48
// sequences of up to 8000 tokens, 8 heads: 235 MB in 60 us with the join), by latency where they are few.
template <int D, int G, int NW>
struct SplitLds {
    float sums[NW][16][D + 4];
    Tokens<D / G, 32> tokens[NW];
    Own<D, G, 32, float> own[NW];
    float m[NW][16], l[NW][16];
};

// Waves a SIMD at least, by the registers they take without spilling.  (Fewer registers, for one wave more with several group words in
// 128 channels, and loads two tiles ahead were no faster: 33 us for a sequence of 131072, 4 heads in groups of 32, against 36 and 36.)
constexpr int split_waves(int d, int g, int mt) { return (d == 128 && g < 128) || mt > 1 ? 2 : g == 32 ? 3 : 4; }

template <int D, int G, int MT, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW > 4 ? NW / 4 : split_waves(D, G, MT)))) void kv4_attention_split_kernel(AttnArgs a) {
    typedef Rows<D, G, MT> S;
    extern __shared__ __align__(16) uint8_t lds[];
    SplitLds<D, G, NW> &sh = *reinterpret_cast<SplitLds<D, G, NW> *>(lds);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    const int split = blockIdx.x % a.splits, head = blockIdx.x / a.splits % a.heads;
    const Seq sq = find_tile(a, a.first_tile + blockIdx.x / a.splits / a.heads, 16 * MT);
    if (sq.seq < 0) return;
    const int row0 = sq.tile * 16 * MT;
    // the last row of the tile sees the most
    const int rows = min(16 * MT, sq.n * a.ratio - row0);
    const int seen = a.causal ? max(0, min(sq.len, sq.len - sq.n + (row0 + rows - 1) / a.ratio + 1)) : sq.len;
    const int used = splits_of(sq.len, a.splits);
    if (split >= used) return;
    const int share = (sq.len / used + 32 * NW) / (32 * NW) * (32 * NW);  // used * share >= len; whole rounds of the waves
    // shares are rounded up, each of up to 2 a CU: the end of one may lie past 2^31, so it is not a sum
    const int first = split * share, end = seen - first > share ? first + share : seen;
    S s;
    load_rows<false>(a, s, sq, head, row0, [](int v) { return v; });
    walk<D, G, MT>(a, sh.tokens[wave], sh.own[wave], s, sq, head, first + 32 * wave, 32 * NW, end);
    settle<false>(s);
    const int hq = a.heads * a.ratio;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (16 * mt >= rows) break;
        __syncthreads();
        if (g == 0) sh.m[wave][n] = s.m[mt], sh.l[wave][n] = s.l[mt];
        __syncthreads();
        const auto top = [&](int row) {
            float m = sh.m[0][row];
#pragma unroll
            for (int w = 1; w < NW; ++w) m = fmaxf(m, sh.m[w][row]);
            return m;
        };
        const float f = __builtin_amdgcn_exp2f(s.m[mt] - top(n));
#pragma unroll
        for (int gr = 0; gr < S::GR; ++gr)
#pragma unroll
            for (int u = 0; u < S::NT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) sh.sums[wave][n][channel<G>(g, r, gr, u)] = s.o[mt][gr][u][r] * f;
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (D / 8); i += 64 * NW) {
            const int rl = i / (D / 8), ch = i % (D / 8) * 8, row = row0 + 16 * mt + rl;
            if (row >= sq.n * a.ratio) continue;
            const int64_t at = static_cast<int64_t>(sq.first + row / a.ratio) * hq + head * a.ratio + row % a.ratio;
            const float mm = top(rl);
            float l = 0.f, v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = 0.f;
#pragma unroll 4
            for (int w = 0; w < NW; ++w) {
                l = __builtin_fmaf(sh.l[w][rl], __builtin_amdgcn_exp2f(sh.m[w][rl] - mm), l);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] += sh.sums[w][rl][ch + e];
            }
            if (a.splits > 1) {
                float *p = a.part + (at * a.splits + split) * (D + 4);
                *reinterpret_cast<float4 *>(p + ch) = make_float4(v[0], v[1], v[2], v[3]);
                *reinterpret_cast<float4 *>(p + ch + 4) = make_float4(v[4], v[5], v[6], v[7]);
                if (ch == 0) p[D] = mm, p[D + 1] = l;
            } else {
                const float inv = l == 0.f ? 0.f : 1.0f / l;  // 0: no token was seen
                uint4 o;
                o.x = f32x2_to_bf16x2_rne(v[0] * inv, v[1] * inv), o.y = f32x2_to_bf16x2_rne(v[2] * inv, v[3] * inv);
                o.z = f32x2_to_bf16x2_rne(v[4] * inv, v[5] * inv), o.w = f32x2_to_bf16x2_rne(v[6] * inv, v[7] * inv);
                *reinterpret_cast<uint4 *>(a.out + at * D + ch) = o;
                if (a.lse && ch == 0) a.lse[at] = l == 0.f ? -INFINITY : (mm + log2f(l)) * 0.693147180559945309f;
            }
        }
    }
}

// Joins the splits: a workgroup a (token, query head), D / 8 lanes of eight channels by 2048 / D lanes of splits, each with a
// reference of its own until the end: one pass, whose first loads wait for nothing, not even for the number of splits (0.5 us less
// than a pass for the references first).  By latency: 4.8 us for 1536 rows of two splits, 5.3 us for 28 rows of 128, and the host's
// second launch.
template <int D>
__global__ __launch_bounds__(256) void kv4_attention_join_kernel(AttnArgs a) {
    constexpr int kCh = D / 8, kSp = 256 / kCh;
    __shared__ __align__(16) float sums[kSp][D + 4];
    __shared__ float ms[kSp], ls[kSp];
    const int hq = a.heads * a.ratio, token = blockIdx.x / hq;
    const int64_t at = blockIdx.x;
    const int ch = threadIdx.x % kCh * 8, sl = threadIdx.x / kCh;
    struct Part {
        float4 x, y;
        float2 ml;
    };
    const float *part = a.part + at * a.splits * (D + 4);
    const auto load = [&](int s) {
        const float *p = part + static_cast<int64_t>(s) * (D + 4);
        return Part{*reinterpret_cast<const float4 *>(p + ch), *reinterpret_cast<const float4 *>(p + ch + 4), *reinterpret_cast<const float2 *>(p + D)};
    };
    Part next = load(min(sl, a.splits - 1));
    int seq = token;
    if (a.cu_q) {
        seq = -1;
        for (int b0 = 0; b0 < a.batch && seq < 0; b0 += 64) {
            const int b = b0 + (threadIdx.x & 63);
            const uint64_t hit = __ballot(b < a.batch && a.cu_q[min(b, a.batch)] <= token && token < a.cu_q[min(b, a.batch - 1) + 1]);
            if (hit) seq = b0 + __builtin_ctzll(hit);
        }
        if (seq < 0) return;
    }
    const int used = splits_of(a.num_pages > 0 ? min(max(a.kv_lens[seq], 0), token_cap(a)) : 0, a.splits);
    float m = kNoMax, l = 0.f, v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int s = sl; s < used; s += kSp) {
        const Part p = next;
        if (s + kSp < used) next = load(s + kSp);
        const float top = fmaxf(m, p.ml.x), f = __builtin_amdgcn_exp2f(m - top), g = __builtin_amdgcn_exp2f(p.ml.x - top);
        const float o[8] = {p.x.x, p.x.y, p.x.z, p.x.w, p.y.x, p.y.y, p.y.z, p.y.w};
        m = top;
        l = __builtin_fmaf(p.ml.y, g, l * f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(o[e], g, v[e] * f);
    }
    if (ch == 0) ms[sl] = m;
    __syncthreads();
    float top = ms[0];
#pragma unroll
    for (int i = 1; i < kSp; ++i) top = fmaxf(top, ms[i]);
    const float f = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[sl][ch + e] = v[e] * f;
    if (ch == 0) ls[sl] = l * f;
    __syncthreads();
    if (threadIdx.x < D) {
        float t = 0.f, o = 0.f;
#pragma unroll
        for (int i = 0; i < kSp; ++i) t += ls[i], o += sums[i][threadIdx.x];
        a.out[at * D + threadIdx.x] = f32_to_bf16_rne(t == 0.f ? 0.f : o / t);
        if (a.lse && threadIdx.x == 0) a.lse[at] = t == 0.f ? -INFINITY : (top + log2f(t)) * 0.693147180559945309f;
    }
}

// Many rows: each wave takes 32 rows of its own, and the NW of a workgroup share the work on the codes.  Of every 16 NW tokens a
// wave turns 16 into MFMA operands in LDS (f16: of the keys codes less zero points, exactly; of the values that times c) and all
// read them back; two stages, one barrier a stage: the operands of the next tokens are made while the present ones are used, and
// the words of those after that are on their way.
// A prompt of 4096 tokens, 32 query heads on 8 of 128 channels: 160 us, 137 GFLOP at 860 TFLOP/s.  VALU work and MFMAs hardly overlap on a
// SIMD (an MFMA of 16 cycles hides one or two instructions), so it is bound by their sum: 38% of the busy cycles are MFMAs, 47% the softmax
// and the making of operands; without the latter it takes 145 us, without LDS reads 7 us less, and the products of
// the next tokens issued among the present ones' exponentials change nothing.
// Two or three waves a SIMD: with 64 channels three take 110 us for 4096 tokens, two 140 and four 121.
// Heads are dealt out first (one head's keys and values stay with one XCD where there are eight heads), and row tiles from the
// last, which see the most tokens.
template <int D, int G, int NW>
struct Stage {
    static constexpr int GR = D / G, kSteps = D / 32, kTiles = D / 16;
    uint4 keys[NW][kSteps][64];     // 16 tokens, 32 channels: a lane's operand
    uint4 values[NW / 2][kTiles][64];   // 32 tokens, 16 channels
    Tokens<GR, 16 * NW> tokens;
};

template <int D, int G, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 3))) void kv4_attention_tile_kernel(AttnArgs a, int tiles) {
    constexpr int MT = 2;
    typedef Rows<D, G, MT> S;
    constexpr int GR = D / G, W = G / 32, R = 128 / G, NT = G / 16, kWords = D / 8, VW = KvTile<D, G>::VW, kRow = D + 4, kTokens = 16 * NW;
    extern __shared__ __align__(16) uint8_t lds[];
    Stage<D, G, NW> *stages = reinterpret_cast<Stage<D, G, NW> *>(lds);
    __shared__ __align__(16) Own<D, G, 16, _Float16> all[NW];
    __shared__ int greatest[NW];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.heads;
    const Seq sq = find_tile(a, tiles - 1 - (a.first_tile + blockIdx.x / a.heads), 16 * NW * MT);
    if (sq.seq < 0) return;
    const int total = sq.n * a.ratio, row_of_all = sq.tile * 16 * NW * MT, row0 = row_of_all + wave * 16 * MT;
    const auto seen = [&](int last_row) { return a.causal ? max(0, min(sq.len, sq.len - sq.n + last_row / a.ratio + 1)) : sq.len; };
    const int end = seen(min(row_of_all + 16 * NW * MT, total) - 1);  // of the workgroup
    const int mine = row0 < total ? seen(min(row0 + 16 * MT, total) - 1) : 0;
    S s;
    const float qk = score_factor(a, load_rows<true>(a, s, sq, head, row0, [&](int v) {
        if (lane == 0) greatest[wave] = v;
        __syncthreads();
        for (int w = 0; w < NW; ++w) v = max(v, greatest[w]);
        return __builtin_amdgcn_readfirstlane(v);
    }));
    const int sure = seen_by_all(s, sq.len);
    const int32_t *table = a.table + static_cast<int64_t>(sq.seq) * a.table_cols;
    Own<D, G, 16, _Float16> &own = all[wave];

    // this wave's 16 tokens of a stage
    struct Part {
        uint32_t kc[GR][W], vc[4][VW], words[GR];
        bool live;
    };
    const auto page_of = [&](int at) { return at < end ? scalar_load(table, at >> a.page_shift) : -1; };
    const auto load = [&](Part &t, int page, int at) {
        t.live = at < end && page >= 0 && page < a.num_pages;
        const int64_t row = kv4_row(t.live ? page : 0, head, at & ((1 << a.page_shift) - 1), a.heads, a.page_shift);
        const uint32_t *kc = a.k_codes + row * kWords + n * kWords + g * W;
        const uint32_t *vc = a.v_codes + row * kWords + 4 * g * kWords + (KvTile<D, G>::kDeal ? n : n % (G / 8));
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) __builtin_memcpy(t.kc[gr], __builtin_assume_aligned(kc + gr * (G / 8), 4 * W), 4 * W);
#pragma unroll
        for (int i = 0; i < VW; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) t.vc[r][i] = vc[r * kWords + i * (G / 8)];
        __builtin_memcpy(t.words, __builtin_assume_aligned((lane & 16 ? a.v_groups : a.k_groups) + (row + n) * GR, 4 * GR), 4 * GR);
    };
    const auto make = [&](const Part &t, Stage<D, G, NW> &st, int at) {
        wave_order();
        if (lane < 32) fill_token(t.words, lane >= 16, 16 * wave + n, !t.live || at + n >= sq.len, qk, st.tokens, own, n);
        if constexpr (KvTile<D, G>::kDeal) *reinterpret_cast<uint4 *>(&own.v[n * own.kRow + 4 * g]) = make_uint4(t.vc[0][0], t.vc[1][0], t.vc[2][0], t.vc[3][0]);
        wave_order();
#pragma unroll
        for (int gr = 0; gr < GR; ++gr) {
            const uint32_t zz = own.k[n][gr];
#pragma unroll
            for (int u = 0; u < W; ++u) st.keys[wave][gr * W + u][lane] = __builtin_bit_cast(uint4, codes_f16(t.kc[gr][u], zz));
            uint4 w;
            if constexpr (KvTile<D, G>::kDeal) w = *reinterpret_cast<const uint4 *>(&own.v[(gr * (G / 8) + n % (G / 8)) * own.kRow + 4 * g]);
            else w = make_uint4(t.vc[0][gr], t.vc[1][gr], t.vc[2][gr], t.vc[3][gr]);
            const Pairs p = pairs_of<G>(w, n);
            const uint2 z = *reinterpret_cast<const uint2 *>(&own.z[gr][4 * g]), c = *reinterpret_cast<const uint2 *>(&own.c[gr][4 * g]);
            static_for<NT>([&](auto u) __attribute__((always_inline)) {
                reinterpret_cast<uint2 *>(&st.values[wave / 2][gr * NT + u][lane])[wave % 2] = make_uint2(pair_value(p, 0, R * u, z.x, c.x), pair_value(p, 1, R * u, z.y, c.y));
            });
        }
    };
    Part part;
    if (end > 0) {
        load(part, page_of(16 * wave), 16 * wave);
        make(part, stages[0], 16 * wave);
        load(part, page_of(kTokens + 16 * wave), kTokens + 16 * wave);
    }
    int page = page_of(2 * kTokens + 16 * wave);
    for (int at = 0, i = 0; at < end; at += kTokens, i ^= 1) {
        __syncthreads();  // stage i is made, and the other one no longer read
        if (at + kTokens < end) {
            make(part, stages[i ^ 1], at + kTokens + 16 * wave);
            load(part, page, at + 2 * kTokens + 16 * wave);
            page = page_of(at + 3 * kTokens + 16 * wave);
        }
        const Stage<D, G, NW> &st = stages[i];
#pragma unroll
        for (int sub = 0; sub < NW / 2; ++sub) {
            if (at + 32 * sub >= mine) break;
            attend<true, D, G, MT>(
                st.tokens, nullptr, 32 * sub, s, at + 32 * sub, sure, [&](int h, int gr, int u) { return __builtin_bit_cast(halfx8, st.keys[2 * sub + h][gr * W + u][lane]); },
                [&](int gr) { return [&st, gr, sub, lane](int u) { return __builtin_bit_cast(halfx8, st.values[sub][gr * NT + u][lane]); }; });
        }
    }
    settle<true>(s);
    __syncthreads();  // the stages' LDS now holds outputs, each wave's own part
    if (row0 >= total) return;
    float (*sums)[kRow] = reinterpret_cast<float (*)[kRow]>(lds) + 16 * wave;
    const int hq = a.heads * a.ratio, rows = min(16 * MT, total - row0);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (16 * mt >= rows) break;
        const float l = s.l[mt], inv = l == 0.f ? 0.f : 1.0f / l;  // 0: no token was seen
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int gr = 0; gr < GR; ++gr)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) sums[n][channel<G>(g, r, gr, u)] = s.o[mt][gr][u][r] * inv;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const int row = row0 + 16 * mt + n;
        if (a.lse && g == 0 && row < total)
            a.lse[static_cast<int64_t>(sq.first + row / a.ratio) * hq + head * a.ratio + row % a.ratio] = l == 0.f ? -INFINITY : (s.m[mt] + log2f(l)) * 0.693147180559945309f;
#pragma unroll
        for (int k = lane; k < 16 * (D / 8); k += 64) {
            const int rl = k / (D / 8), ch = k % (D / 8) * 8, to = row0 + 16 * mt + rl;
            if (to >= total) continue;
            const int64_t out = static_cast<int64_t>(sq.first + to / a.ratio) * hq + head * a.ratio + to % a.ratio;
            const float *v = &sums[rl][ch];
            *reinterpret_cast<uint4 *>(a.out + out * D + ch) =
                make_uint4(f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]), f32x2_to_bf16x2_rne(v[4], v[5]), f32x2_to_bf16x2_rne(v[6], v[7]));
        }
    }
}

// How a call is laid out: rows a wave (16 mt), whether waves share rows (splits of the tokens) or have their own, row
// tiles at most, splits.
struct Plan {
    int mt, waves;
    bool rows, wide;  // wide: more waves a workgroup in place of splits
    int64_t tiles, splits, bytes;
};

// Waves of a wide workgroup: as many as its registers allow.
constexpr int wide_waves(int64_t d, int64_t g) { return d / g == 1 ? 16 : 8; }

Plan plan_of(const cfh_kv4_cache_t *c, int64_t tokens, int64_t q_heads, int64_t batch, int64_t table_cols, bool varlen) {
    Plan p{1, 4, false, false, 0, 1, 0};
    if (tokens == 0 || batch == 0) return p;
    const int64_t ratio = q_heads / c->kv_heads, cus = cu_count(), rows = tokens * ratio;
    const auto tiles = [&](int64_t per) { return varlen ? rows / per + batch : batch * ((ratio + per - 1) / per); };
    // Enough rows for six waves a CU of 32 rows: every wave its own rows.  8 heads of 128, 4 queries each: prompts of 1024 (four
    // waves a CU), 1536 and 2048 tokens 39, 57 and 74 us; as splits 32, 56 and 85.  The rule is for the call: single queries in it walk
    // their tokens in one workgroup (2048 rows of a prompt beside 47 queries over 8000 tokens 253 us, in two calls 71 and 88).
    p.rows = varlen && rows / 32 * c->kv_heads >= 6 * cus;
    if (p.rows) {
        p.mt = 2;
        // Eight waves share the making of operands where there are two workgroups of them a CU, the heavy ones to be evened out by the
        // light ones.  Prompts of 4096 and of 2048 tokens, 8 heads of 128 channels, 4 queries each: 158 and 78 us, with four waves
        // 186 and 73.  With 64 channels four of them take 110 us and eight 120: three waves a SIMD of different workgroups then wait at
        // different times.
        if (c->head_dim == 128 && rows / (128 * p.mt) * c->kv_heads >= 2 * cus) p.waves = 8;
        p.tiles = tiles(16 * p.waves * p.mt);
        return p;
    }
    const int64_t each = (rows + batch - 1) / batch;
    // Two row tiles a wave (three spill) halve the work on the codes; with few rows a sequence they leave tiles half empty and
    // sequences of unlike lengths unevenly dealt.  8 heads of 128, 4 queries each: 16 sequences of up to 33 tokens (86 rows on
    // average) 42 us with one tile and 58 with two, 4 of 16 tokens 30 and 29, 8 of 64 tokens 81 and 64.
    p.mt = each <= 96 ? 1 : 2;
    p.tiles = tiles(16 * p.mt);
    const int64_t tasks = p.tiles * c->kv_heads, len = table_cols * c->page_size;
    // A short table and few workgroups: one launch of wide workgroups, two rounds of 32 tokens a wave at most, no partial sums.
    // One sequence of 777 tokens, 8 heads of 128: 11.5 us a call against 15.9 with splits and their join, whose second launch
    // costs the host more than the longer walk costs the GPU (10.5 against 8.4 us on the GPU); 32 sequences of 1000: 13.9
    // against 16.3 on the GPU.  At 2000 tokens, four rounds, one sequence takes 16.1 against 8.5 there.
    p.wide = p.mt == 1 && tasks <= cus && len > 128 && len <= 64 * wide_waves(c->head_dim, c->group);
    if (p.wide) return p;
    // Two workgroups a CU.  With three or four: 512 tokens after 8192 (8 heads of 128, 4 queries each) 118, 148 and 148 us; one sequence
    // of 32768 18.2, 18.5 and 20.6.
    p.splits = std::max<int64_t>(1, std::min((2 * cus + tasks - 1) / tasks, (len + 127) / 128));
    const int64_t row = (c->head_dim + 4) * 4;
    p.splits = std::max<int64_t>(1, std::min(p.splits, (int64_t{256} << 20) / (tokens * q_heads * row)));
    if (p.splits > 1) p.bytes = tokens * q_heads * p.splits * row;
    return p;
}

// Raises a kernel's dynamic-LDS limit once per device (bit = device ordinal < 64).
void raise_lds_limit(const void *kern, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    check_hip(hipGetDevice(&dev), "hipGetDevice");
    const uint64_t bit = dev < 64 ? (uint64_t{1} << dev) : 0;
    if (bit == 0 || !(done.load(std::memory_order_acquire) & bit)) {
        check_hip(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "hipFuncSetAttribute(attention)");
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
}

// launch(workgroups) of as many row tiles as one launch holds, `each` workgroups a tile, until all have run.
template <class F>
void for_tiles(AttnArgs &a, const Plan &p, int64_t each, int threads, const F &launch) {
    require(p.tiles <= 0x7fffffff, "too many rows and sequences for one call");
    const int64_t most = most_workgroups(threads) / each;
    for (int64_t t = 0; t < p.tiles; t += most) {
        a.first_tile = static_cast<int>(t);
        launch(static_cast<unsigned>(std::min(p.tiles - t, most) * each));
    }
}

template <int D, int G, int NW>
void launch_tile(AttnArgs a, const Plan &p, hipStream_t st) {
    constexpr int sums = 16 * NW * (D + 4) * 4, stages = 2 * sizeof(Stage<D, G, NW>), lds = stages > sums ? stages : sums;
    static_assert(lds + NW * sizeof(Own<D, G, 16, _Float16>) <= NW * 20 * 1024, "two workgroups a CU");
    static std::atomic<uint64_t> attr_devices{0};
    const auto kern = kv4_attention_tile_kernel<D, G, NW>;
    raise_lds_limit(reinterpret_cast<const void *>(kern), lds, attr_devices);
    for_tiles(a, p, a.heads, 64 * NW, [&](unsigned grid) {
        kern<<<dim3(grid), dim3(64 * NW), lds, st>>>(a, static_cast<int>(p.tiles));
        check_launch("kv4_attention_tile");
    });
}

template <int D, int G, int MT, int NW>
void launch_split(AttnArgs a, const Plan &p, hipStream_t st) {
    constexpr int lds = sizeof(SplitLds<D, G, NW>);
    static_assert(lds <= 160 * 1024, "LDS budget");
    const auto kern = kv4_attention_split_kernel<D, G, MT, NW>;
    static std::atomic<uint64_t> attr_devices{0};
    if (lds > 64 * 1024) raise_lds_limit(reinterpret_cast<const void *>(kern), lds, attr_devices);
    for_tiles(a, p, a.heads * p.splits, 64 * NW, [&](unsigned grid) {
        kern<<<dim3(grid), dim3(64 * NW), lds, st>>>(a);
        check_launch("kv4_attention_split");
    });
    if (p.splits > 1) {
        kv4_attention_join_kernel<D><<<dim3(static_cast<unsigned>(a.tokens * a.heads * a.ratio)), dim3(256), 0, st>>>(a);
        check_launch("kv4_attention_join");
    }
}

void check_counts(const cfh_kv4_cache_t *c, int64_t tokens, int64_t q_heads, int64_t batch, int64_t table_cols) {
    require(tokens >= 0 && tokens <= 0x7fffffff && batch >= 0 && batch <= 0x7fffffff, "tokens and batch must be in [0, 2^31)");
    require(q_heads >= 1 && q_heads % c->kv_heads == 0 && q_heads / c->kv_heads <= 64,
            "q_heads must be a multiple of kv_heads, at most 64 of them a head of keys");
    require(table_cols >= 0 && table_cols <= 0x7ffff000 / c->page_size, "a sequence's table must hold at most 2^31 - 4096 tokens");
    require(tokens * q_heads <= 0x7fffffff, "tokens * q_heads must be below 2^31");
}

}  // namespace
}  // namespace cfh

using namespace cfh;

extern "C" {

int32_t castforge_hip_kv4_attention_workspace(const cfh_kv4_cache_t *cache, int64_t tokens, int64_t q_heads, int64_t batch,
                                              int64_t table_cols, int32_t varlen, int64_t *out_bytes, char **out_error) {
    if (out_bytes) *out_bytes = 0;
    return guarded(out_error, [&] {
        check_kv4(cache);
        require(out_bytes != nullptr, "out_bytes must not be NULL");
        check_counts(cache, tokens, q_heads, batch, table_cols);
        *out_bytes = plan_of(cache, tokens, q_heads, batch, table_cols, varlen != 0).bytes;
    });
}

int32_t castforge_hip_kv4_attention(const cfh_kv4_cache_t *cache, const uint16_t *q, int64_t q_stride, int64_t tokens,
                                    int64_t q_heads, int64_t batch, const int32_t *cu_q, const int32_t *page_table,
                                    int64_t table_cols, const int32_t *kv_lens, int32_t causal, float scale, uint16_t *out,
                                    float *lse, void *workspace, int64_t workspace_bytes, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_kv4(cache);
        check_counts(cache, tokens, q_heads, batch, table_cols);
        require(causal == 0 || causal == 1, "causal must be 0 or 1");
        require(cu_q != nullptr || tokens == batch, "without cu_q every sequence has one query: tokens must equal batch");
        if (tokens == 0) return;
        require(q && out && (batch == 0 || kv_lens) && (batch == 0 || table_cols == 0 || page_table), "buffers must not be NULL");
        require(aligned(q, 16) && aligned(out, 16), "q and out must be 16-byte aligned");
        require(tokens <= 1 || (q_stride >= q_heads * cache->head_dim && q_stride % 8 == 0),
                "q's token stride must be a multiple of 8 and at least q_heads * head_dim");
        if (batch == 0) return;
        const Plan p = plan_of(cache, tokens, q_heads, batch, table_cols, cu_q != nullptr);
        require(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 16)),
                "workspace must be 16-byte aligned and hold the bytes that castforge_hip_kv4_attention_workspace gives");
        AttnArgs a{q, q_stride, cache->k_codes, cache->k_groups, cache->v_codes, cache->v_groups, cu_q, page_table, kv_lens, out, lse,
                   static_cast<float *>(workspace), scale, static_cast<int>(tokens), static_cast<int>(batch),
                   static_cast<int>(cache->kv_heads), static_cast<int>(q_heads / cache->kv_heads), log2_of(cache->page_size),
                   static_cast<int>(table_cols), static_cast<int>(cache->num_pages), causal, static_cast<int>(p.splits), 0};
        hipStream_t st = static_cast<hipStream_t>(stream);
        kv4_by_shape(cache, [&](auto d, auto gr) {
            constexpr int D = decltype(d)::value, G = decltype(gr)::value;
            if (p.rows && p.waves == 4) {
                launch_tile<D, G, 4>(a, p, st);
            } else if (p.rows) {
                if constexpr (D == 128) launch_tile<D, G, 8>(a, p, st);
            } else if (p.wide) {
                launch_split<D, G, 1, wide_waves(D, G)>(a, p, st);
            } else if (p.mt == 1) {
                launch_split<D, G, 1, 4>(a, p, st);
            } else {
                launch_split<D, G, 2, 4>(a, p, st);
            }
        });
    });
}

}  // extern "C"
