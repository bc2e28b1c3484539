// Attention over the paged cache of 8-bit keys and values:
//   o[i] = sum_t p[i, t] v[t],  p = softmax over the visible t of scale * <q[i], k[t]>,
//   k[t], v[t] = codes * the scale of their page and head.
//
// Query i of the n of a sequence with L cached tokens has the place L - n + i.  It sees the tokens t < L, with `causal` only
// those with t <= its place, and with a window only those of t > place - window and the first `sinks` of the sequence.  A
// query that sees no token gives zeros, and -inf as the logarithm of its sum.
//
// The softmax's maximum and sum, the scores and the output sums are f32.  Codes reach the MFMAs exactly, keys as bf16 (as the
// queries are) and values as f16; weights are rounded to f16, 2^-11 of themselves (bf16 would be 2^-8).
//
// Three kernels and what bounds them (8 heads of keys, 32 of queries, 128 channels): few rows a sequence read the cache at HBM's rate (48
// single queries over up to 8000 tokens 98 us, 4.8 TB/s; a large copy runs at 5.1); many rows are bound by the sum of MFMAs and vector
// instructions (prompt of 4096 tokens 141 to 152 us by the card, 0.9 to 0.97 PFLOP/s); the weights that tokens got are the keys' half of
// that again, or a pass over scores that the first kernel left.
#include <algorithm>
#include <atomic>

#include "../../include/castforge_hip.h"
#include "attention_rows.hpp"
#include "cfh_common.hpp"
#include "kv8.hpp"

namespace cfh {
namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct AttnArgs8 {
    const uint16_t *q;
    int64_t q_stride;
    const uint8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int32_t *cu_q;  // NULL: one query a sequence
    const int32_t *table, *kv_lens;
    uint16_t *out;
    float *lse;
    float *part;  // splits > 1: [tokens * q heads][splits][D + 4], output sums, reference, sum, how many splits there are (of the first), unused
    float scale;  // of scores, base 2
    int tokens, batch, heads, ratio, page_shift, table_cols, num_pages, causal, splits;
    int window, sinks;  // window 0x7fffffff: none
    uint32_t ratio_mul;  // query_of's
    int ratio_shift;
    float *scores;      // NULL, or where the kernel of few rows leaves its scores: [tokens * q heads][score_cols], base 2
    int score_cols;
    int first_tile;     // of a launch's row tiles, where one launch cannot hold them all
};

// row / ratio of a row below 2^31: by ceil(2^(31 + l) / ratio), l = ceil(log2 ratio), which is exact there (a division takes ten times as
// long, and tiles begin with several).
__device__ __forceinline__ int query_of(const AttnArgs8 &a, int row) {
    return static_cast<int>(static_cast<uint64_t>(static_cast<uint32_t>(row)) * a.ratio_mul >> a.ratio_shift);
}

// What a query at a place sees: t < limit, and t >= low or t < sinks.
__device__ __forceinline__ int limit_of(const AttnArgs8 &a, const Seq &sq, int i) { return a.causal ? min(sq.len, sq.len - sq.n + i + 1) : sq.len; }
__device__ __forceinline__ int low_of(const AttnArgs8 &a, const Seq &sq, int i) {
    const int place = sq.len - sq.n + i;
    return place >= a.window ? place - a.window + 1 : 0;
}

// The tokens that the queries i0 .. i1 of a sequence see, in steps of 32: those below `gap`, and from gap + skip to end.  Walks count
// steps: token_of() gives a step's first token.
struct Span {
    int gap, skip, end;  // gap and skip multiples of 32
    __device__ __forceinline__ int steps() const { return (end - skip + 31) >> 5; }
    __device__ __forceinline__ int token_of(int step) const { return 32 * step + (32 * step >= gap ? skip : 0); }
};
__device__ __forceinline__ Span span_of(const AttnArgs8 &a, const Seq &sq, int i0, int i1) {
    Span s;
    s.end = max(limit_of(a, sq, i1), 0);
    s.gap = (a.sinks + 31) & ~31;
    s.skip = max((low_of(a, sq, i0) & ~31) - s.gap, 0);
    return s;
}
// Splits that share a sequence: by the tokens that its queries see, at least 128 each.
__device__ __forceinline__ int splits_of_seq(const AttnArgs8 &a, const Seq &sq) {
    const Span s = span_of(a, sq, 0, sq.n - 1);
    return splits_of(32 * s.steps(), a.splits);
}

// The exponent of a page's scale of values.  Held to append's range, within which a sum of weights by 2^-exponent neither overflows
// nor loses a weight of 2^-23 of the largest: scales differ by 2^100 there, and f32 has 2^126.
__device__ __forceinline__ float exponent_of(float scale) {
    const float e = static_cast<float>(__builtin_amdgcn_frexp_expf(scale)) + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(scale));
    return fminf(fmaxf(e, static_cast<float>(kKv8LeastExponent)), static_cast<float>(kKv8GreatestExponent));
}

// Registers of 32 tokens' keys and values of a head, in halves of 16.  n = lane % 16, g = lane / 16.
template <int D>
struct Tile8 {
    static constexpr int W = D / 64;
    uint4 k[2][W];        // token n: codes 64 i + 16 g ..
    uint32_t v[2][4][W];  // tokens 4 g + r: codes 4 W n ..
    float ks[2], vs[2];   // uniform
    bool live[2];         // uniform: the half's page is one of the cache's
};

template <int D>
__device__ __forceinline__ void load_tile(const AttnArgs8 &a, Tile8<D> &t, int head, const int (&page)[2], int at, int end) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        t.live[h] = at + 16 * h < end && page[h] >= 0 && page[h] < a.num_pages;
        const int p = t.live[h] ? page[h] : 0;
        const int64_t row = kv8_row(p, head, (at + 16 * h) & ((1 << a.page_shift) - 1), a.heads, a.page_shift);
        const uint8_t *k = a.k_codes + (row + n) * D + 16 * g, *v = a.v_codes + (row + 4 * g) * D + n * (D / 16);
#pragma unroll
        for (int i = 0; i < Tile8<D>::W; ++i) t.k[h][i] = *reinterpret_cast<const uint4 *>(k + 64 * i);
#pragma unroll
        for (int r = 0; r < 4; ++r) __builtin_memcpy(t.v[h][r], __builtin_assume_aligned(v + r * D, D / 16), D / 16);
        const int64_t at_scale = static_cast<int64_t>(p) * a.heads + head;
        t.ks[h] = scalar_load(a.k_scales, at_scale), t.vs[h] = scalar_load(a.v_scales, at_scale);
    }
}

__device__ __forceinline__ uint32_t bf16_pair(uint32_t codes, bool high) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.0f, false));
}
__device__ __forceinline__ uint32_t f16_pair(uint32_t codes, bool high) {
    return __builtin_bit_cast(uint32_t, high ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes, 1.0f, false));
}

// Eight keys' codes as an MFMA operand.
__device__ __forceinline__ bf16x8 keys_bf16(uint32_t a, uint32_t b) {
    return __builtin_bit_cast(bf16x8, uintx4{bf16_pair(a, false), bf16_pair(a, true), bf16_pair(b, false), bf16_pair(b, true)});
}

// Four codes a token of two tokens as pairs of tokens: codes 0 and 1, and codes 2 and 3.
__device__ __forceinline__ uint32_t low_codes(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05010400u); }
__device__ __forceinline__ uint32_t high_codes(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07030602u); }

// Code u of four tokens, W words each, as f16.
template <int u, int W>
__device__ __forceinline__ uint2 values_f16(const uint32_t (&v)[4][W]) {
    constexpr int i = u / 4, c = u % 4;
    const auto pair = [&](int r) { return f16_pair(c < 2 ? low_codes(v[r][i], v[r + 1][i]) : high_codes(v[r][i], v[r + 1][i]), c % 2); };
    return make_uint2(pair(0), pair(2));
}

// Rows of a wave: 16 MT of the n * ratio (query, head of the group) pairs of a sequence and a head of keys, row = query *
// ratio + head; the MFMAs' columns.  With S^T = K Q^T a lane holds the scores of one row and four tokens a
// half, which is the layout that O^T = V^T P^T takes its second operand in: the weights stay in registers.
// Channel of element r of tile u of O^T: (4 g + r) D / 16 + u, so that a lane's outputs lie behind one another.
template <int D, int MT>
struct Rows8 {
    static constexpr int KS = D / 32, NT = D / 16;
    uint4 q[MT][KS];       // channels 64 (i / 2) + 16 g + 8 (i % 2) ..
    int limit[MT], low[MT];
    floatx4 o[MT][NT];
    float m[MT], l[MT];    // reference and this lane's part of the sum
};

template <int D, int MT>
__device__ __forceinline__ void load_rows(const AttnArgs8 &a, Rows8<D, MT> &s, const Seq &sq, int head, int row0) {
    const int n = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int row = row0 + 16 * mt + n, i = query_of(a, row);
        const bool in = i < sq.n;
        // rows past the sequence's see all: they are not stored, and do not make a tile an edge
        s.limit[mt] = in ? limit_of(a, sq, i) : 0x7fffffff;
        s.low[mt] = in ? low_of(a, sq, i) : 0;
        const uint16_t *p = a.q + (sq.first + (in ? i : 0)) * a.q_stride + (head * a.ratio + (in ? row - i * a.ratio : 0)) * D;
#pragma unroll
        for (int i8 = 0; i8 < D / 32; ++i8) s.q[mt][i8] = *reinterpret_cast<const uint4 *>(p + 64 * (i8 / 2) + 16 * g + 8 * (i8 % 2));
#pragma unroll
        for (int u = 0; u < D / 16; ++u) s.o[mt][u] = floatx4{0.f, 0.f, 0.f, 0.f};
        s.m[mt] = kNoMax, s.l[mt] = 0.f;
    }
}

// Tokens that every row of the wave sees: [low, limit).
struct Sure {
    int low, limit;
};
template <int D, int MT>
__device__ __forceinline__ Sure seen_by_all(const Rows8<D, MT> &s, int len) {
    int limit = len, low = 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) limit = min(limit, s.limit[mt]), low = max(low, s.low[mt]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) limit = min(limit, __shfl_xor(limit, o)), low = max(low, __shfl_xor(low, o));
    return Sure{__builtin_amdgcn_readfirstlane(low), __builtin_amdgcn_readfirstlane(limit)};
}

// What the tokens of a half's page share: what turns a product into a score, base 2, the exponent e of their values' scale, and 2^-e.
struct Page {
    float kf, e, back;
};
__device__ __forceinline__ Page page_of(float scale, float ks, float vs) {
    const float e = exponent_of(vs);
    return Page{scale * ks, e, __builtin_amdgcn_exp2f(-e)};
}

// 32 tokens at `at`.  A token's weight is held with the exponent e of its values' scale: exp2(score + e - m) rounds to f16 as what
// the token adds to the output, whatever the scales are; the sum takes the 2^-e back.  m is 7 below the largest so far when it
// moves, and it moves only when something exceeds it by 15: weights stay below 2^15, the largest ones above 2^7 (f16 keeps its
// 11 bits down to 2^-21 of them), and the rescaling is rare.
// keys(h, i): the MFMA operand of half h's 16 tokens and 32 channels; values(u): that of 16 channels and 32 tokens.  gone: a half's
// page is none of the cache's; edge, uniform: so, or some row does not see some token.
template <bool kScored, int D, int MT, class Keys, class Values>
__device__ __forceinline__ void attend(const AttnArgs8 &a, Rows8<D, MT> &s, int at, bool edge, const bool (&gone)[2], const Page (&pages)[2], float *const (&score_rows)[MT], const Keys &keys, const Values &values) {
    constexpr int KS = D / 32, NT = D / 16;
    const int g = (threadIdx.x >> 4) & 3;
    floatx4 dot[MT][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            const bf16x8 k = keys(h, i);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
                dot[mt][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, __builtin_bit_cast(bf16x8, s.q[mt][i]), i ? dot[mt][h] : floatx4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
        }
    float y[MT][2][4];  // scores and their values' exponents, base 2
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[mt][h][r] = __builtin_fmaf(dot[mt][h][r], pages[h].kf, pages[h].e);
    if (edge) {
        int first = at + 4 * g;
        asm volatile("" : "+v"(first));  // a branch: the comparisons stay in it
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int t = first + 16 * (i / 4) + i % 4;
            const bool behind = t >= a.sinks;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const bool hidden = gone[i / 4] | (t >= s.limit[mt]) | ((t < s.low[mt]) & behind);
                y[mt][i / 4][i % 4] = hidden ? -INFINITY : y[mt][i / 4][i % 4];
            }
        }
    }
    if constexpr (kScored) {  // scores of what a row does not see, and of no page, are not read
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                floatx4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = dot[mt][h][r] * pages[h].kf;
                if (score_rows[mt] && at + 16 * h < a.score_cols) *reinterpret_cast<floatx4 *>(score_rows[mt] + at + 16 * h) = v;  // a table may end with a half
            }
    }
    uint32_t p[MT][4];  // weights as f16 pairs: tokens (0, 1), (2, 3) of both halves
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const float (&v)[2][4] = y[mt];
        const float most = max3(max3(v[0][0], v[0][1], v[0][2]), max3(v[0][3], v[1][0], v[1][1]), max3(v[1][2], v[1][3], v[1][3]));
        if (__any(most > s.m[mt] + 15.f)) {
            const float m = fmaxf(s.m[mt], max_over_g(most) - 7.f), f = __builtin_amdgcn_exp2f(s.m[mt] - m);
            s.m[mt] = m;
            s.l[mt] *= f;
#pragma unroll
            for (int u = 0; u < NT; ++u) s.o[mt][u] *= f;
        }
        float w[2][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i / 4][i % 4] = __builtin_amdgcn_exp2f(v[i / 4][i % 4] - s.m[mt]);
            s.l[mt] = __builtin_fmaf(w[i / 4][i % 4], pages[i / 4].back, s.l[mt]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            p[mt][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{w[i / 2][i % 2 * 2], w[i / 2][i % 2 * 2 + 1]}), halfx2));
    }
    static_for<NT>([&](auto u) __attribute__((always_inline)) {
        const halfx8 v = values(u);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
            s.o[mt][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, __builtin_bit_cast(halfx8, uintx4{p[mt][0], p[mt][1], p[mt][2], p[mt][3]}), s.o[mt][u], 0, 0, 0);
    });
}

// Where a row's output goes, of the sequence's row tile.
__device__ __forceinline__ int64_t out_row(const AttnArgs8 &a, const Seq &sq, int head, int row) {
    const int i = query_of(a, row);
    return static_cast<int64_t>(sq.first + i) * (a.heads * a.ratio) + head * a.ratio + row - i * a.ratio;
}

// A wave's walk over steps first, first + by, .. below last of a span, the next tile's loads in flight.
template <bool kScored, int D, int MT>
__device__ __forceinline__ void walk(const AttnArgs8 &a, Rows8<D, MT> &s, const Seq &sq, int head, const Span &span, int row0, int first, int by, int last) {
    if (first >= last) return;
    constexpr int W = Tile8<D>::W;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const Sure sure = seen_by_all(s, sq.len);
    const int32_t *table = a.table + static_cast<int64_t>(sq.seq) * a.table_cols;
    float *score_rows[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int row = row0 + 16 * mt + (lane & 15);
        score_rows[mt] = kScored && row < sq.n * a.ratio ? a.scores + out_row(a, sq, head, row) * a.score_cols + 4 * g : nullptr;
    }
    const auto pages = [&](int step, int (&p)[2]) {
        const int at = span.token_of(step);
#pragma unroll
        for (int h = 0; h < 2; ++h) p[h] = step < last && at + 16 * h < span.end ? scalar_load(table, (at + 16 * h) >> a.page_shift) : -1;
    };
    Tile8<D> cur;
    int page[2];
    pages(first, page);
    load_tile<D>(a, cur, head, page, span.token_of(first), span.end);
    pages(first + by, page);
    for (int step = first; step < last; step += by) {
        Tile8<D> next;
        if (step + by < last) {
            load_tile<D>(a, next, head, page, span.token_of(step + by), span.end);
            pages(step + 2 * by, page);
        } else {
            next = cur;
        }
        const int at = span.token_of(step);
        const bool apart = !(cur.live[0] && cur.live[1]);
        if (apart || at + 32 > sq.len) {  // uniform: bytes that are no token's may be NaN, which a weight of 0 does not take away
            asm volatile("");
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        if (!cur.live[h] || at + 16 * h + 4 * g + r >= sq.len) cur.v[h][r][i] = 0;
        }
        const Page pages_of[2] = {page_of(a.scale, cur.ks[0], cur.vs[0]), page_of(a.scale, cur.ks[1], cur.vs[1])};
        const bool gone[2] = {!cur.live[0], !cur.live[1]}, edge = apart || at + 32 > sure.limit || (at < sure.low && at + 32 > a.sinks);
        attend<kScored, D, MT>(
            a, s, at, edge, gone, pages_of, score_rows,
            [&](int h, int i) {
                const uint4 w = cur.k[h][i / 2];
                return i % 2 ? keys_bf16(w.z, w.w) : keys_bf16(w.x, w.y);
            },
            [&](auto u) {
                const uint2 x = values_f16<u>(cur.v[0]), y = values_f16<u>(cur.v[1]);
                return __builtin_bit_cast(halfx8, uintx4{x.x, x.y, y.x, y.y});
            });
        cur = next;
    }
}

// A sequence's queries and length, as find_tile gives them.
__device__ __forceinline__ Seq seq_of(const AttnArgs8 &a, int seq) {
    Seq sq{seq, seq, 1, 0, 0};
    if (a.cu_q) {
        sq.first = min(max(scalar_load(a.cu_q, seq), 0), a.tokens);
        sq.n = min(max(scalar_load(a.cu_q, seq + 1), sq.first), a.tokens) - sq.first;
    }
    sq.len = a.num_pages > 0 ? min(max(scalar_load(a.kv_lens, seq), 0), token_cap(a)) : 0;
    return sq;
}

__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f; }

// One workgroup's NW waves take the same rows and every NW-th 32 tokens of a split's share, and are joined through LDS;
// splits are joined by kv8_attention_join_kernel.  Codes go from memory to registers, without LDS: each is used once, and a wave has the next
// 32 tokens' on their way while it works on these.  Three waves a SIMD for 16 rows (48 sequences of up to 8000 tokens 106 -> 100 us; with
// 32 rows they would spill).
template <int D, int NW>
struct SplitLds8 {
    float sums[NW][16][D + 4];
    float m[NW][16], l[NW][16];
};

template <bool kScored, int D, int MT, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(NW > 4 ? NW / 4 : MT == 1 ? 3 : 2))) void kv8_attention_split_kernel(AttnArgs8 a) {
    extern __shared__ __align__(16) uint8_t lds[];
    SplitLds8<D, NW> &sh = *reinterpret_cast<SplitLds8<D, NW> *>(lds);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
    const int split = blockIdx.x % a.splits, head = blockIdx.x / a.splits % a.heads;
    const Seq sq = find_tile(a, a.first_tile + blockIdx.x / a.splits / a.heads, 16 * MT);
    if (sq.seq < 0) return;
    const int row0 = sq.tile * 16 * MT, rows = min(16 * MT, sq.n * a.ratio - row0);
    const int used = splits_of_seq(a, sq);
    if (split >= used) return;
    const Span span = span_of(a, sq, query_of(a, row0), query_of(a, row0 + rows - 1));
    const int steps = span.steps(), share = (steps + used * NW - 1) / (used * NW) * NW;  // whole rounds of the waves
    Rows8<D, MT> s;
    load_rows(a, s, sq, head, row0);
    // shares are rounded up: the last ones may be empty
    walk<kScored, D, MT>(a, s, sq, head, span, row0, split * share + wave, NW, min(steps, (split + 1) * share));
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (16 * mt >= rows) break;
        s.l[mt] = sum_over_g(s.l[mt]);
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
        for (int u = 0; u < D / 16; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) sh.sums[wave][n][(4 * g + r) * (D / 16) + u] = s.o[mt][u][r] * f;
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * (D / 8); i += 64 * NW) {
            const int rl = i / (D / 8), ch = i % (D / 8) * 8, row = row0 + 16 * mt + rl;
            if (row >= sq.n * a.ratio) continue;
            const int64_t at = out_row(a, sq, head, row);
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
                if (ch == 0) *reinterpret_cast<float4 *>(p + D) = make_float4(mm, l, __int_as_float(used), 0.f);
            } else {
                const float inv = l == 0.f ? 0.f : 1.0f / l;  // 0: no token was seen
                *reinterpret_cast<uint4 *>(a.out + at * D + ch) =
                    make_uint4(f32x2_to_bf16x2_rne(v[0] * inv, v[1] * inv), f32x2_to_bf16x2_rne(v[2] * inv, v[3] * inv),
                               f32x2_to_bf16x2_rne(v[4] * inv, v[5] * inv), f32x2_to_bf16x2_rne(v[6] * inv, v[7] * inv));
                if (a.lse && ch == 0) a.lse[at] = lse_of(mm, l);
            }
        }
    }
}

// Joins the splits of many rows: D / 4 lanes of four channels a row, which take four splits at a time: 32768 rows of two splits cost a
// prompt 6 us, by the kernel below 34.
template <int D>
__global__ __launch_bounds__(256) void kv8_attention_join_rows_kernel(AttnArgs8 a) {
    constexpr int kLanes = D / 4, kRows = 256 / kLanes;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / kLanes, hq = a.heads * a.ratio;
    const int ch = threadIdx.x % kLanes * 4;
    if (at >= (a.cu_q ? min(a.cu_q[a.batch], a.tokens) : a.tokens) * hq) return;  // of no sequence
    const float *part = a.part + at * a.splits * (D + 4);
    const int used = min(max(__float_as_int(part[D + 2]), 1), a.splits);
    float m = kNoMax, l = 0.f;
    floatx4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < used; s += 4) {
        floatx4 o[4];
        floatx2 ml[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float *p = part + static_cast<int64_t>(min(s + i, used - 1)) * (D + 4);
            o[i] = *reinterpret_cast<const floatx4 *>(p + ch), ml[i] = *reinterpret_cast<const floatx2 *>(p + D);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, ml[i].x);
        const float f = __builtin_amdgcn_exp2f(m - top);
        m = top, l *= f, v *= f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float g = s + i < used ? __builtin_amdgcn_exp2f(ml[i].x - m) : 0.f;
            l = __builtin_fmaf(ml[i].y, g, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = __builtin_fmaf(o[i][e], g, v[e]);
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // 0: no token was seen
    *reinterpret_cast<uint2 *>(a.out + at * D + ch) = make_uint2(f32x2_to_bf16x2_rne(v[0] * inv, v[1] * inv), f32x2_to_bf16x2_rne(v[2] * inv, v[3] * inv));
    if (a.lse && ch == 0) a.lse[at] = lse_of(m, l);
}

// Joins the many splits of few rows: a workgroup a (token, query head), D / 8 lanes of eight channels by 2048 / D lanes of splits, each
// with a reference of its own until the end.
template <int D>
__global__ __launch_bounds__(256) void kv8_attention_join_kernel(AttnArgs8 a) {
    constexpr int kCh = D / 8, kSp = 256 / kCh;
    __shared__ __align__(16) float sums[kSp][D + 4];
    __shared__ float ms[kSp], ls[kSp];
    const int hq = a.heads * a.ratio;
    const int64_t at = blockIdx.x;
    const int token = static_cast<int>(at / hq), ch = threadIdx.x % kCh * 8, sl = threadIdx.x / kCh;
    struct Part {
        floatx4 x, y;
        floatx2 ml;
    };
    const float *part = a.part + at * a.splits * (D + 4);
    const auto load = [&](int s) {
        const float *p = part + static_cast<int64_t>(s) * (D + 4);
        return Part{*reinterpret_cast<const floatx4 *>(p + ch), *reinterpret_cast<const floatx4 *>(p + ch + 4), *reinterpret_cast<const floatx2 *>(p + D)};
    };
    Part next = load(min(sl, a.splits - 1));
    const int used = min(max(__float_as_int(part[D + 2]), 1), a.splits);
    if (a.cu_q && token >= a.cu_q[a.batch]) return;  // of no sequence
    float m = kNoMax, l = 0.f, v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int s = sl; s < used; s += kSp) {
        const Part p = next;
        if (s + kSp < used) next = load(s + kSp);
        const float top = fmaxf(m, p.ml.x), f = __builtin_amdgcn_exp2f(m - top), g = __builtin_amdgcn_exp2f(p.ml.x - top);
        m = top;
        l = __builtin_fmaf(p.ml.y, g, l * f);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(e < 4 ? p.x[e % 4] : p.y[e % 4], g, v[e] * f);
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
        if (a.lse && threadIdx.x == 0) a.lse[at] = lse_of(top, t);
    }
}

// Many rows: each wave takes 32 rows of its own, and the eight of a workgroup share the making of the MFMA operands: of every 128
// tokens a wave turns 32 tokens' half rows of keys and 16 tokens' values into operands in LDS, and all read them back; two stages, one
// barrier a stage: the operands of the next tokens are made while the present ones are used, and the codes of those after that are on
// their way.  Eight waves, one workgroup a CU: a prompt of 4096 tokens takes 147 us, by four waves a workgroup, two a CU, which make every
// operand twice as often, 171.  Each wave for itself (the kernel above) 384.
// Of the busy cycles MFMAs are 44% and vector instructions 41%, hardly beside each other: 32 x 32 x 16 MFMAs alone, on registers with
// random numbers, run at 1.5 to 1.65 PFLOP/s here (power), with six fmas each at 1.3, which would be 105 us, and a score costs more than
// that (an fma, an exponential of 16 cycles, an addition, half a conversion and half a maximum).  The operands' making costs 15 us, the
// exponentials 7, the reading of keys 9.  16 x 16 x 32 MFMAs: 153 us.  Keys read a step ahead, raised wave priority, other orders of the
// instructions: no faster.  A workgroup's start (lists, table, first codes, first operands) takes 12000 cycles, a stage 8200: four rounds
// of workgroups in a prompt of 8192 tokens through a window of 1024 (168 us).  Queries fetched into L2 for the workgroup that follows: no faster.
// One workgroup a CU that goes through several tiles, the next one's codes on their way under the last one's stores, needs all 256
// registers, and reads LDS no longer ahead: 177.
// 32 x 32 x 16 MFMAs: of S^T = K Q^T lane (n = lane % 32, h = lane / 32) holds row n's scores of the tokens 8 j + 4 h + r of 32 (j, r < 4),
// which is what O^T = V^T P^T takes of 16 tokens (j < 2, then j >= 2) as its second operand.  Row i of a tile of V^T is channel
// i D / 32 + u.
template <int D, int NW>
struct Stage8 {
    static constexpr int KS = D / 16, NT = D / 32;
    uint4 keys[NW / 2][KS][64];       // 32 tokens, 16 channels: a lane's operand
    uint4 values[NW / 2][2][NT][64];  // 16 tokens, 32 channels
    Page pages[NW / 2][2];
};

typedef float floatx16 __attribute__((ext_vector_type(16)));

// A wave's rows, one a lane and a half of the tokens.
template <int D>
struct TileRows {
    static constexpr int KS = D / 16, NT = D / 32;
    bf16x8 q[KS];    // channels 32 (i / 2) + 16 h + 8 (i % 2) ..
    int limit, low;
    floatx16 o[NT];
    float m, l;
};

// Scores of 32 tokens and rows, unscaled.
template <int D, int NW>
__device__ __forceinline__ floatx16 tile_scores(const TileRows<D> &s, const Stage8<D, NW> &st, int sub, int lane) {
    floatx16 dot;
#pragma unroll
    for (int i = 0; i < 16; ++i) dot[i] = 0.f;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) dot = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, st.keys[sub][i][lane]), s.q[i], dot, 0, 0, 0);
    return dot;
}

// attend()'s steps: exponents less m by one fma each, which are made from the products again where m moves.
struct Exponents {
    float z[16], most;
};
__device__ __forceinline__ float most_of(const float (&z)[16]) {
    const float a = max3(max3(z[0], z[1], z[2]), z[3], z[4]), b = max3(max3(z[5], z[6], z[7]), z[8], z[9]);
    return max3(max3(a, b, z[10]), max3(z[11], z[12], z[13]), max3(z[14], z[15], z[15]));
}
__device__ __forceinline__ Exponents exponents_of(const floatx16 &dot, const Page (&pages)[2], float m) {
    Exponents e;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float em = pages[h].e - m;
#pragma unroll
        for (int i = 8 * h; i < 8 * h + 8; ++i) e.z[i] = __builtin_fmaf(dot[i], pages[h].kf, em);
    }
    e.most = most_of(e.z);
    return e;
}

// What lies in branches: masks, and moves of m.
template <int D>
__device__ __forceinline__ void settle(const AttnArgs8 &a, TileRows<D> &s, Exponents &e, const floatx16 &dot, const Page (&pages)[2], int at, bool edge) {
    if (edge) {
        int first = at + 4 * ((threadIdx.x >> 5) & 1);
        asm volatile("" : "+v"(first));  // a branch: the comparisons stay in it
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int t = first + 8 * (i / 4) + i % 4;
            e.z[i] = (t >= s.limit) | ((t < s.low) & (t >= a.sinks)) ? -INFINITY : e.z[i];
        }
        e.most = most_of(e.z);
    }
    if (__any(e.most > 15.f)) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = __builtin_fmaf(dot[i], pages[i / 8].kf, pages[i / 8].e);
            e.z[i] = e.z[i] == -INFINITY ? -INFINITY : y;
            top = fmaxf(top, e.z[i]);
        }
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m = fmaxf(s.m, top - 7.f), f = __builtin_amdgcn_exp2f(s.m - m);
        s.m = m;
        s.l *= f;
#pragma unroll
        for (int u = 0; u < D / 32; ++u) s.o[u] *= f;
#pragma unroll
        for (int i = 0; i < 16; ++i) e.z[i] -= m;
    }
}

// Weights as f16 pairs, and their sum.
template <int D>
__device__ __forceinline__ void tile_weights(TileRows<D> &s, const Exponents &e, const Page (&pages)[2], uint32_t (&p)[8]) {
    float w[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(e.z[i]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const float *v = w + 8 * h;
        s.l = __builtin_fmaf(((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])), pages[h].back, s.l);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector((floatx2{w[2 * i], w[2 * i + 1]}), halfx2));
}

template <int D, int NW>
__device__ __forceinline__ void tile_outputs(TileRows<D> &s, const Stage8<D, NW> &st, int sub, int lane, const uint32_t (&p)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int u = 0; u < D / 32; ++u)
            s.o[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, st.values[sub][h][u][lane]),
                                                            __builtin_bit_cast(halfx8, uintx4{p[4 * h], p[4 * h + 1], p[4 * h + 2], p[4 * h + 3]}), s.o[u], 0, 0, 0);
}

template <int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) void kv8_attention_tile_kernel(AttnArgs8 a, int tiles) {
    constexpr int kRows = 32, KS = D / 16, NT = D / 32, W = D / 64, kSteps = NW / 2;  // steps of 32 tokens a stage
    extern __shared__ __align__(16) uint8_t lds[];
    Stage8<D, NW> *stages = reinterpret_cast<Stage8<D, NW> *>(lds);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.heads, split = blockIdx.x / a.heads % a.splits;
    const Seq sq = find_tile(a, tiles - 1 - (a.first_tile + static_cast<int>(blockIdx.x / a.heads / a.splits)), kRows * NW);
    if (sq.seq < 0) return;
    const int used = splits_of_seq(a, sq);
    if (split >= used) return;
    const int total = sq.n * a.ratio, row_of_all = sq.tile * kRows * NW, row0 = row_of_all + wave * kRows, row = row0 + n;
    const Span span = span_of(a, sq, query_of(a, row_of_all), query_of(a, min(row_of_all + kRows * NW, total) - 1));
    // the split's steps: whole stages; shares are rounded up, the last ones may be empty
    const int share = (span.steps() + used * kSteps - 1) / (used * kSteps) * kSteps;
    const int begin = split * share, steps = min(span.steps(), begin + share);
    // the wave's own rows see tokens below `mine`, and from `from` on or sinks
    const int mine = row0 < total ? limit_of(a, sq, query_of(a, min(row0 + kRows, total) - 1)) : 0;
    const int from = row0 < total ? low_of(a, sq, query_of(a, row0)) : 0;
    TileRows<D> s;
    {
        const int i = query_of(a, row);
        const bool in = i < sq.n;
        // rows past the sequence's see all: they are not stored, and do not make a tile an edge
        s.limit = in ? limit_of(a, sq, i) : 0x7fffffff;
        s.low = in ? low_of(a, sq, i) : 0;
        const uint16_t *p = a.q + (sq.first + (in ? i : 0)) * a.q_stride + (head * a.ratio + (in ? row - i * a.ratio : 0)) * D + 16 * h;
#pragma unroll
        for (int k = 0; k < KS; ++k) s.q[k] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(p + 32 * (k / 2) + 8 * (k % 2)));
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int i16 = 0; i16 < 16; ++i16) s.o[u][i16] = 0.f;
        s.m = kNoMax, s.l = 0.f;
    }
    int sure_limit = min(sq.len, s.limit), sure_low = s.low;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sure_limit = min(sure_limit, __shfl_xor(sure_limit, o)), sure_low = max(sure_low, __shfl_xor(sure_low, o));
    sure_limit = __builtin_amdgcn_readfirstlane(sure_limit), sure_low = __builtin_amdgcn_readfirstlane(sure_low);
    const int32_t *table = a.table + static_cast<int64_t>(sq.seq) * a.table_cols;

    // This wave's 16 tokens of a stage: half wave % 2 of step wave / 2.  n16 = lane % 16, g = lane / 16.
    const int sub_of = wave / 2, half = wave & 1, n16 = lane & 15, g = lane >> 4;
    struct Part {
        uint4 k[W];     // token n16: codes 16 (W g + i) ..
        uint32_t v[8];  // tokens 8 j + 4 h + r: codes n D / 32 ..
        float ks, vs;
        int at;         // its first token
        bool live;      // its page is one of the cache's
    };
    const uint32_t page_bytes = (static_cast<uint32_t>(a.heads) << a.page_shift) * D;  // below 2^26
    const int page_mask = (1 << a.page_shift) - 1;
    const uint32_t head_bytes = (static_cast<uint32_t>(head) << a.page_shift) * D;
    const auto token_at = [&](int step) { return span.token_of(step + sub_of) + 16 * half; };
    const auto page_at = [&](int step) {
        const int at = token_at(step);
        return step + sub_of < steps && at < span.end ? scalar_load(table, at >> a.page_shift) : -1;
    };
    const auto load = [&](Part &t, int page, int step) {
        t.at = token_at(step);
        t.live = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages);
        const uint32_t p = t.live ? page : 0;
        const uint64_t from_codes = static_cast<uint64_t>(p) * page_bytes + head_bytes + static_cast<uint32_t>(t.at & page_mask) * D;
        const uint8_t *k = a.k_codes + from_codes, *v = a.v_codes + from_codes;
#pragma unroll
        for (int i = 0; i < W; ++i) t.k[i] = *reinterpret_cast<const uint4 *>(k + n16 * D + 16 * (W * g + i));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint8_t *q = v + 4 * h * D + n * NT + (8 * (i / 4) + i % 4) * D;
            if constexpr (D == 128) t.v[i] = *reinterpret_cast<const uint32_t *>(q);
            else t.v[i] = *reinterpret_cast<const uint16_t *>(q);
        }
        const int64_t at_scale = static_cast<int64_t>(static_cast<uint64_t>(p) * static_cast<uint32_t>(a.heads) + static_cast<uint32_t>(head));
        t.ks = scalar_load(a.k_scales, at_scale), t.vs = scalar_load(a.v_scales, at_scale);
    };
    const auto make = [&](Part &t, Stage8<D, NW> &st) {
        if (!t.live || t.at + 16 > sq.len) {  // uniform: bytes that are no token's may be NaN, which a weight of 0 does not take away
            int at = t.at;
            asm volatile("" : "+v"(at));
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (!t.live) t.k[i] = uint4{};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!t.live || at + 8 * (i / 4) + 4 * h + i % 4 >= sq.len) t.v[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const int piece = W * g + i;  // of the MFMAs' 32 channels piece / 2, half piece % 2
            uint4 *to = &st.keys[sub_of][piece & ~1][32 * (piece & 1) + 16 * half + n16];
            to[0] = __builtin_bit_cast(uint4, keys_bf16(t.k[i].x, t.k[i].y));
            to[64] = __builtin_bit_cast(uint4, keys_bf16(t.k[i].z, t.k[i].w));
        }
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) lo[i] = low_codes(t.v[2 * i], t.v[2 * i + 1]), hi[i] = high_codes(t.v[2 * i], t.v[2 * i + 1]);
        static_for<NT>([&](auto u) __attribute__((always_inline)) {
            const auto pair = [&](int i) { return f16_pair(u < 2 ? lo[i] : hi[i], u % 2); };
            st.values[sub_of][half][u][lane] = make_uint4(pair(0), pair(1), pair(2), pair(3));
        });
        // no page of the cache: scores of -inf, by products of zeros
        if (lane == 0) st.pages[sub_of][half] = t.live ? page_of(a.scale, t.ks, t.vs) : Page{0.f, -INFINITY, 0.f};
    };
    // a stage's tokens for the wave's rows
    const auto walk_stage = [&](int step, int i) {
        const Stage8<D, NW> &st = stages[i];
        // the wave's steps of the stage: those below the window of all its rows are left out where no sink is among them
        const auto at_of = [&](int sub) { return span.token_of(step + sub); };
        int sub = 0, last = kSteps;
        if (at_of(0) >= a.sinks)
            while (sub < kSteps && at_of(sub) + 32 <= from) ++sub;
        while (last > sub && (step + last > steps || at_of(last - 1) >= mine)) --last;
        if (sub >= last) return;
        const auto is_edge = [&](int at) { return at + 32 > sure_limit || (at < sure_low && at + 32 > a.sinks); };
        // The next step's products are issued among this one's weights: vector work and MFMAs then have each other to run beside.
        floatx16 dot = tile_scores<D, NW>(s, st, sub, lane);
        Exponents e;
        Page pg[2];
        uint32_t p[8];
        const auto exponents = [&](int at) {
            pg[0] = st.pages[sub][0], pg[1] = st.pages[sub][1];
            e = exponents_of(dot, pg, s.m);
            settle<D>(a, s, e, dot, pg, at, is_edge(at));
        };
        exponents(at_of(sub));
        for (; sub + 1 < last;) {
            dot = tile_scores<D, NW>(s, st, sub + 1, lane);
            tile_weights<D>(s, e, pg, p);
            tile_outputs<D, NW>(s, st, sub, lane, p);
            ++sub;
            exponents(at_of(sub));
        }
        tile_weights<D>(s, e, pg, p);
        tile_outputs<D, NW>(s, st, sub, lane, p);
    };
    int i = 0;
    if (steps > begin) {
        Part part;
        int page = page_at(begin + kSteps);
        load(part, page_at(begin), begin);
        make(part, stages[0]);
        // the queries have come too: else the compiler waits for them in every stage, and with them for the codes on their way (as it would
        // with the loop behind this branch, not in it)
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
        load(part, page, begin + kSteps);
        page = page_at(begin + 2 * kSteps);
        for (int step = begin; step < steps; step += kSteps, i ^= 1) {
            __syncthreads();  // stage i is made, and the other one no longer read
            walk_stage(step, i);
            if (step + kSteps < steps) {
                make(part, stages[i ^ 1]);
                load(part, page, step + 2 * kSteps);
                page = page_at(step + 3 * kSteps);
            }
        }
    }
    float l = s.l + __shfl_xor(s.l, 32);
    // The zeros that stand for a missing page's keys make NaN with a query of NaN or infinity.  A row that sees missing pages alone gives nothing
    // all the same; asked here, for such rows only (masked in the loop: 0.6% of a prompt of 128 channels, 3% of one of 64).
    if (__any(l != l && row < total)) {
        bool seen = false;
        for (int step = begin; step < steps; ++step)
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const int at = span.token_of(step) + 16 * part, page = at < span.end ? scalar_load(table, at >> a.page_shift) : -1;
                seen |= static_cast<uint32_t>(page) < static_cast<uint32_t>(a.num_pages) && at < s.limit && (at + 16 > s.low || at < a.sinks);
            }
        if (!seen) {
            l = 0.f, s.m = kNoMax;
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) s.o[u][e] = 0.f;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;  // 0: no token was seen
    const int to = static_cast<int>(out_row(a, sq, head, row));
    // Rows are stored by D / 8 lanes each, through LDS (stage i is no longer read): by the lanes that hold them each store touches 64 lines
    // (64 queries of 7 heads after 16384 tokens, whose splits leave 30 MB: 60.9 -> 54.2 us).  A lane has D / 8 channels behind one another for
    // each j; piece p of row r lies at p ^ r: in order, a piece of all rows would lie in the same banks.
    constexpr int kLanes = D / 8, kPer = 64 / kLanes, kStores = kRows / kPer;  // lanes a row, rows a store, stores
    const int of_row = lane / kLanes, piece = lane % kLanes;
    uintx4 *rows = reinterpret_cast<uintx4 *>(stages + i) + wave * kRows * kLanes;
    const auto put = [&](int at, const uintx4 &v) { rows[n * kLanes + (at ^ (n & (kLanes - 1)))] = v; };
    const auto for_rows = [&](const auto &store) {
        wave_order();
#pragma unroll
        for (int c = 0; c < kStores; ++c) {
            const int r = kPer * c + of_row, to_row = __shfl(to, r);
            const uintx4 v = rows[r * kLanes + (piece ^ (r & (kLanes - 1)))];
            if (row0 + r < total) store(static_cast<int64_t>(to_row), v);
        }
        wave_order();
    };
    if (a.splits > 1) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {  // of the channels
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < D / 8; c += 4) {
                    const auto v = [&](int e) { return __float_as_uint(s.o[(c + e) % NT][4 * (2 * half + j) + (c + e) / NT]); };
                    put(((8 * j + 4 * h) * NT + c) / 4, uintx4{v(0), v(1), v(2), v(3)});
                }
            for_rows([&](int64_t at, const uintx4 &v) {
                *reinterpret_cast<uintx4 *>(a.part + (at * a.splits + split) * (D + 4) + half * (D / 2) + 4 * piece) = v;
            });
        }
        if (h == 0 && row < total) *reinterpret_cast<float4 *>(a.part + (static_cast<int64_t>(to) * a.splits + split) * (D + 4) + D) = make_float4(s.m, l, __int_as_float(used), 0.f);
        return;
    }
    if (a.lse && h == 0 && row < total) a.lse[to] = lse_of(s.m, l);
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < D / 8; c += 8) {
            const auto v = [&](int e) { return s.o[(c + e) % NT][4 * j + (c + e) / NT] * inv; };
            put(((8 * j + 4 * h) * NT + c) / 8,
                uintx4{f32x2_to_bf16x2_rne(v(0), v(1)), f32x2_to_bf16x2_rne(v(2), v(3)), f32x2_to_bf16x2_rne(v(4), v(5)), f32x2_to_bf16x2_rne(v(6), v(7))});
        }
    for_rows([&](int64_t at, const uintx4 &v) { *reinterpret_cast<uintx4 *>(a.out + at * D + 8 * piece) = v; });
}

// Weights that the cached tokens got, from the logarithms of the rows' sums: weights[seq, head, t] += sum over the head's rows of
// exp(score - lse).  Each sum has one writer.
struct WeightArgs8 {
    float *weights;
    int cols;             // tokens of a row of weights
    int blocks;           // workgroups a sequence and head
    int64_t first_block;  // of a launch's workgroups, where one launch cannot hold them all
};

// The queries of a sequence that see some of the tokens t0 .. t1 - 1.
struct Queries {
    int first, end;
};
__device__ __forceinline__ Queries queries_that_see(const AttnArgs8 &a, const Seq &sq, int t0, int t1) {
    const int64_t before = static_cast<int64_t>(sq.len) - sq.n;  // place of the first query
    const int64_t i0 = a.causal ? max(t0 - before, int64_t{0}) : 0;
    const int64_t i1 = t0 < a.sinks ? sq.n : min(static_cast<int64_t>(sq.n), static_cast<int64_t>(t1) + a.window - 1 - before);
    return i0 < i1 ? Queries{static_cast<int>(i0), static_cast<int>(i1)} : Queries{0, 0};
}

// A workgroup has 64 tokens of a sequence and head, whose keys each wave holds as MFMA operands; its one to eight waves take the row tiles of
// 32 in turn, each through LDS of its own, the next one's queries on their way: no barrier until the end, where the waves' sums are joined.
// With S^T = K Q^T a lane has one row's 16 of 32 scores: -lse is one number a lane, what turns products into scores one a half of 16
// tokens, and a score costs an fma, an exponential and an addition.
// kByHead: a tile is 32 queries of one query head (the last one of a head reaches back over queries that it leaves out), whose rows lie a
// stride apart; else 32 rows in order, each with a query and a head to be told apart (as many instructions again, but full tiles where
// a sequence has few queries: below 32 a sequence).
// 64 queries of 28 heads after 16384 tokens: 20 us of that call's 55; a prompt's of 4096 tokens 113, and 418 when each lane read its rows itself.
// Bound by its vector instructions (an exponential of 16 cycles a score), and by a workgroup's start, from table to operands; 240 registers
// leave two waves a SIMD.
// Queries are read by rows, 16 lanes each, and stored for operand c and half h of lanes at row r ^ (2 c + h): in order, all 16 pieces of a
// row would lie in the same banks.
template <int D, bool kByHead>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2))) void kv8_attention_weights_kernel(AttnArgs8 a, WeightArgs8 wa) {
    constexpr int KS = D / 16, W = D / 64, kLanes = D / 8, kPer = 64 / kLanes, kLoads = 32 / kPer;  // lanes a row, rows a load, loads a tile
    extern __shared__ __align__(16) uint8_t lds[];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6, lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    uintx4(*staged)[64] = reinterpret_cast<uintx4(*)[64]>(lds) + wave * KS;
    const auto sums_of = [&](int w) { return reinterpret_cast<float *>(lds + w * KS * sizeof(*staged)); };  // 64, once its rows are done with
    const int64_t block = wa.first_block + blockIdx.x;
    const int seq = static_cast<int>(block / a.heads / wa.blocks), head = static_cast<int>(block % a.heads);
    // the first tokens are seen by the most rows: they come first, and the last ones beside them (one head after another: a prompt of 4096
    // tokens took 240 us instead of 174 before rows were staged in LDS, 113 since)
    const int k = static_cast<int>(block / a.heads % wa.blocks), most_heavy = (wa.blocks + 1) / 2;
    const int t0 = 64 * (k < most_heavy ? k : wa.blocks - 1 - (k - most_heavy));
    const Seq sq = seq_of(a, seq);
    const int most = min(sq.len, wa.cols);
    if (t0 >= most || sq.n == 0) return;
    const Queries who = queries_that_see(a, sq, t0, min(t0 + 64, most));
    if (who.first >= who.end) return;
    uintx4 keys[2][KS];
    float kf[2][2];
    bool live[2][2];  // of 16 tokens
    {
        const int32_t *table = a.table + static_cast<int64_t>(seq) * a.table_cols;
        uintx4 codes[2][2 * W];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            int64_t row[2];
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int t = t0 + 32 * m + 16 * s, page = t < most ? scalar_load(table, t >> a.page_shift) : -1;
                live[m][s] = page >= 0 && page < a.num_pages;
                const int p = live[m][s] ? page : 0;
                row[s] = kv8_row(p, head, t & ((1 << a.page_shift) - 1), a.heads, a.page_shift);
                kf[m][s] = a.scale * scalar_load(a.k_scales, static_cast<int64_t>(p) * a.heads + head);
            }
            const uint8_t *from = a.k_codes + ((n & 16 ? row[1] : row[0]) + (n & 15)) * D + 16 * h;
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) codes[m][i] = *reinterpret_cast<const uintx4 *>(from + 32 * i);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 2 * W; ++i) {
                keys[m][2 * i] = __builtin_bit_cast(uintx4, keys_bf16(codes[m][i][0], codes[m][i][1]));
                keys[m][2 * i + 1] = __builtin_bit_cast(uintx4, keys_bf16(codes[m][i][2], codes[m][i][3]));
            }
    }
    const int hq = a.heads * a.ratio, of_row = lane / kLanes, piece = lane % kLanes;
    struct RowTile {
        uintx4 q[kLoads];
        float lse;
        int i;      // the lane's row's query
        bool in;    // the row is one of the tile's
        int i0, i1; // uniform: queries of the tile's first and last row
    };
    // by heads: tile `tile` of head `x`
    const int per_head = (who.end - who.first + 31) / 32;
    int x = 0, tile = wave;
    int64_t at[kLoads], lse_at;
    if constexpr (kByHead) {
        // a sequence of fewer than 32 queries has one tile a head, from its first query on: rows past the last one are that one again
#pragma unroll
        for (int c = 0; c < kLoads; ++c) at[c] = min(kPer * c + of_row, sq.n - 1) * a.q_stride + 8 * piece;
        lse_at = static_cast<int64_t>(min(n, sq.n - 1)) * hq;
    }
    // in order: rows that go on by `step`, each a query and a head of the group
    struct Row {
        int i, x;
    };
    const int step = 32 * waves, queries = query_of(a, step), rest = step - queries * a.ratio;
    const int first_row = who.first * a.ratio + 32 * wave;
    const Row last{who.end - 1, a.ratio - 1};
    Row mine, its[kLoads];
    const auto row_at = [&](int row) {
        const int i = query_of(a, row);
        return Row{i, row - i * a.ratio};
    };
    const auto advance = [&](Row &r) {
        r.i += queries, r.x += rest;
        const bool over = r.x >= a.ratio;
        r.x -= over ? a.ratio : 0, r.i += over;
    };
    if constexpr (!kByHead) {
        mine = row_at(first_row + n);
#pragma unroll
        for (int c = 0; c < kLoads; ++c) its[c] = row_at(first_row + kPer * c + of_row);
    }
    const auto load = [&](int row0) {  // past the end: the last rows again
        RowTile p;
        if constexpr (kByHead) {
            while (tile >= per_head && x < a.ratio) tile -= per_head, ++x;
            const int from = who.first + 32 * (x < a.ratio ? tile : 0), i0 = max(min(from, who.end - 32), 0), head_x = head * a.ratio + min(x, a.ratio - 1);
            const uint16_t *q = a.q + (sq.first + i0) * a.q_stride + head_x * D;
#pragma unroll
            for (int c = 0; c < kLoads; ++c) p.q[c] = *reinterpret_cast<const uintx4 *>(q + at[c]);
            p.lse = a.lse[static_cast<int64_t>(sq.first + i0) * hq + head_x + lse_at];
            p.i = i0 + n, p.in = p.i >= from && p.i < who.end;
            p.i0 = i0, p.i1 = min(i0 + 31, sq.n - 1);
            tile += waves;
        } else {
#pragma unroll
            for (int c = 0; c < kLoads; ++c) {
                const Row r = its[c].i < who.end ? its[c] : last;
                p.q[c] = *reinterpret_cast<const uintx4 *>(a.q + (sq.first + r.i) * a.q_stride + (head * a.ratio + r.x) * D + 8 * piece);
                advance(its[c]);
            }
            p.in = mine.i < who.end;
            const Row r = p.in ? mine : last;
            p.lse = a.lse[static_cast<int64_t>(sq.first + r.i) * hq + head * a.ratio + r.x];
            p.i = r.i;
            p.i0 = query_of(a, row0), p.i1 = min(query_of(a, row0 + 31), who.end - 1);
            advance(mine);
        }
        return p;
    };
    // this wave's tiles
    const int tiles = kByHead ? per_head * a.ratio : ((who.end - who.first) * a.ratio + 31) / 32;
    float sum[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) sum[i] = 0.f;
    RowTile next = load(first_row);
    for (int done = wave, row0 = first_row; done < tiles; done += waves) {
        wave_order();
        // channels 8 e ..: of the MFMAs' 32 channels e / 4, half e / 2 % 2, the first or second of two
        const int c_of = piece / 4 * 2 + piece % 2, h_of = piece / 2 % 2;
#pragma unroll
        for (int c = 0; c < kLoads; ++c) staged[c_of][32 * h_of + ((kPer * c + of_row) ^ (2 * c_of + h_of))] = next.q[c];
        // no weight for rows past the end, and for those whose scores are all -inf: less their logarithm, which is -inf too, NaN
        const float minus_lse = next.in && next.lse != -INFINITY ? next.lse * -1.44269504088896341f : -INFINITY;
        const int limit = limit_of(a, sq, next.i), low = low_of(a, sq, next.i);
        // uniform: every row of the tile sees every token
        const bool all = t0 + 64 <= limit_of(a, sq, next.i0) && (t0 >= low_of(a, sq, next.i1) || t0 + 64 <= a.sinks);
        row0 += step;
        next = load(row0);
        wave_order();
        uintx4 q[KS];
#pragma unroll
        for (int c = 0; c < KS; ++c) q[c] = staged[c][32 * h + (n ^ (2 * c + h))];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            floatx16 dot;
#pragma unroll
            for (int i = 0; i < 16; ++i) dot[i] = 0.f;
#pragma unroll
            for (int c = 0; c < KS; ++c) dot = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, keys[m][c]), __builtin_bit_cast(bf16x8, q[c]), dot, 0, 0, 0);
            float w[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(dot[i], kf[m][i / 8], minus_lse));
            if (!all) {
                int first = t0 + 32 * m + 4 * h;
                asm volatile("" : "+v"(first));  // a branch: the comparisons stay in it
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int t = first + 8 * (i / 4) + i % 4;
                    w[i] = (t >= limit) | ((t < low) & (t >= a.sinks)) ? 0.f : w[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[16 * m + i] += w[i];
        }
    }
    // over the 32 lanes of a half: each step halves the sums a lane has; lane n keeps number n
    static_for<5>([&](auto s) __attribute__((always_inline)) {
        constexpr int o = 16 >> s;
        const bool up = n & o;
        static_for<o>([&](auto i) __attribute__((always_inline)) {
            const float kept = up ? sum[i + o] : sum[i], given = up ? sum[i] : sum[i + o];
            sum[i] = kept + __shfl_xor(given, o);
        });
    });
    const int of = 32 * (n / 16) + 8 * (n / 4 % 4) + 4 * h + n % 4;  // its token
    wave_order();
    sums_of(wave)[of] = sum[0];
    __syncthreads();
    const int t = t0 + static_cast<int>(threadIdx.x);
    if (threadIdx.x < 64 && t < most && (threadIdx.x < 32 ? threadIdx.x < 16 ? live[0][0] : live[0][1] : threadIdx.x < 48 ? live[1][0] : live[1][1])) {
        float v = 0.f;
        for (int w = 0; w < waves; ++w) v += sums_of(w)[threadIdx.x];
        float *p = wa.weights + (static_cast<int64_t>(seq) * a.heads + head) * wa.cols + t;
        *p += v;
    }
}

// The same where the kernel of few rows has left its scores (base 2), [rows][score_cols] from the first row of the sequence and head on:
// four tokens a lane.  Up to eight rows a sequence and head on average, where the scores' 4 bytes a row and token are read back in less time than the
// keys are multiplied again (32 sequences of up to 8000 tokens, 4 query heads a head of keys: 104 us in all against 140; more rows have
// more scores than keys), and up to 256 MB of them, by the table's width (behind one of 131072 tokens those sequences take 122 us, not 99).
__global__ __launch_bounds__(256) void kv8_attention_scored_kernel(AttnArgs8 a, WeightArgs8 wa) {
    const int64_t block = wa.first_block + blockIdx.x;
    const int seq = static_cast<int>(block / wa.blocks / a.heads), head = static_cast<int>(block / wa.blocks % a.heads);
    const Seq sq = seq_of(a, seq);
    const int most = min(sq.len, wa.cols), t = 1024 * static_cast<int>(block % wa.blocks) + 4 * static_cast<int>(threadIdx.x), hq = a.heads * a.ratio;
    if (t >= most || sq.n == 0) return;
    // Tokens of no page are left out as such, not by their scores of -inf: a row that sees no others has -inf as its logarithm too, and their
    // difference is NaN.  The lane's four lie in one page.
    const int page = a.table[static_cast<int64_t>(seq) * a.table_cols + (t >> a.page_shift)];
    if (page < 0 || page >= a.num_pages) return;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    bool seen = false;
    for (int i = 0; i < sq.n; ++i) {
        const int limit = limit_of(a, sq, i), low = low_of(a, sq, i);
        if (t >= limit || (t + 4 <= low && t >= a.sinks)) continue;
        seen = true;
        for (int x = 0; x < a.ratio; ++x) {
            const int64_t row = static_cast<int64_t>(sq.first + i) * hq + head * a.ratio + x;
            const float lse = a.lse[row] * 1.44269504088896341f;
            if (lse == -INFINITY) continue;  // all scores are -inf, and their difference is NaN
            const floatx4 y = *reinterpret_cast<const floatx4 *>(a.scores + row * a.score_cols + t);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sum[r] += (t + r >= limit) | ((t + r < low) & (t + r >= a.sinks)) ? 0.f : __builtin_amdgcn_exp2f(y[r] - lse);
        }
    }
    float *p = wa.weights + (static_cast<int64_t>(seq) * a.heads + head) * wa.cols + t;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (seen && t + r < most) p[r] += sum[r];
}

// How a call is laid out: rows a wave (16 mt), whether waves share rows (splits of the tokens) or have their own, row
// tiles at most, splits, workspace.
struct Plan {
    int mt, waves;
    bool rows, wide;       // wide: more waves a workgroup in place of splits
    int64_t tiles, splits, bytes;
    bool scored;           // weights: the kernel of few rows leaves its scores in the workspace, behind the splits' sums
    int64_t score_cols, scores_at;  // scores_at: bytes before them
};

Plan plan_of(const cfh_kv8_cache_t *c, int64_t tokens, int64_t q_heads, int64_t batch, int64_t table_cols, bool varlen, int64_t window, int64_t sinks, bool weights) {
    Plan p{1, 4, false, false, 0, 1, 0, false, 0, 0};
    if (tokens == 0 || batch == 0) return p;
    const int64_t ratio = q_heads / c->kv_heads, cus = cu_count(), rows = tokens * ratio, each = (rows + batch - 1) / batch;
    const auto tiles = [&](int64_t per) { return varlen ? rows / per + batch : batch * ((ratio + per - 1) / per); };
    const int64_t row = (c->head_dim + 4) * 4;
    // tokens that the queries of a row tile see: a window's, and one more a query that a tile may have
    const auto len_of = [&](int64_t per) { return std::min(table_cols * c->page_size, window + sinks + 64 + std::min(tokens, per / ratio + 1)); };
    const int64_t most_splits = std::max<int64_t>(1, (int64_t{256} << 20) / (tokens * q_heads * row));
    const auto splits_for = [&](int64_t splits, int64_t len, int64_t least) { return std::max<int64_t>(1, std::min({splits, len / least, most_splits})); };
    // Several queries a sequence: the form and its splits by their cost in us.  A workgroup takes `start`, and `token` for each token that its
    // rows see, of which causal rows see fewer; `slots` of them run at once; splits cost a launch, and the writing and reading of their
    // sums at 4 TB/s.  The numbers are fits to 69 shapes a head size (1 to 64 sequences of 16 to 2400 queries after 0 to 16000 tokens, in
    // every form): over them the choice takes 3% (128 channels) and 1% (64) longer than the best form does, 24% at most.  (128 channels, us, tile
    // kernel and split kernel: prompt of 512 tokens 22 and 14, of 1600 52 and 57, of 2400 77 and 100; 16 prompts of 100 tokens 14 and 27; 64 queries
    // of 32 heads after 4000 tokens 31 and 23, 128 after 16000 54 and 63, 512 after 16000 147 and 186.  By rows a sequence alone: up to 1.9 times
    // the better one's.)
    // The host does not know the lengths: the table's width stands for them, here and below, and those shapes' tables were as wide as their
    // lengths.  Behind one of 16384 tokens a prompt of 512 takes 28 us (14), of 1600 77 (52); behind one of 131072 64 queries after 4000 tokens
    // 29 (21), and a call of one query over 1009, which loses the one launch below, 13.8 (10.5).
    const auto cost = [&](double token, double start, int64_t slots, int64_t tasks, int64_t splits, int64_t len) {
        const double seen = std::min(len, std::max(table_cols * c->page_size - tokens / batch / 2, int64_t{1})), rounds = static_cast<double>((tasks * splits + slots - 1) / slots);
        return std::max(len * token / splits + start, rounds * (seen * token / splits + start)) + (splits > 1 ? 5 + 2e-6 * tokens * q_heads * splits * row / 4 : 0);
    };
    const bool large = c->head_dim == 128;
    const auto tasks_of = [&](int64_t per) { return batch * c->kv_heads * ((each + per - 1) / per); };
    p.mt = each <= 96 ? 1 : 2;
    const int64_t len = len_of(16 * p.mt);
    p.tiles = tiles(16 * p.mt);
    // Two workgroups of four waves a CU, or one of eight, which needs no partial sums and no second launch.  The latter for short tables: one
    // sequence of 1009 tokens, 8 heads of 128, takes 11.7 us a call against 15.7 with splits and their join, whose launch costs the host more
    // than the longer walk costs the GPU (10.3 against 7.4 us there; of 2000 tokens 16.1 against 8.0; 64 channels 1500 tokens 10.2 against 7.8
    // there and 11.7 against 14.8 a call; sixteen waves 11.0).  And where it fills half the card with walks that are short or, through a
    // window, alike: on the GPU 24 sequences of 2000 tokens 20.4 us against 25.3, of 500 to 2000 18.0 against 19.1, 32 through a window of 4096
    // 55.3 against 58.1.  (Of up to 8000 tokens the longest one is waited for: 24 sequences 59.2 against 56.4.)
    const int64_t tasks = p.tiles * c->kv_heads;
    p.wide = p.mt == 1 && tasks <= cus && (len <= (large ? 1024 : 1536) || (2 * tasks > cus && (len <= 2048 || 2 * len <= table_cols * c->page_size)));
    if (!p.wide) p.splits = splits_for((2 * cus + tasks - 1) / tasks, len, 128);
    if (varlen && each > 16) {
        const double token = p.wide ? (large ? .0065 : .005) : p.mt == 1 ? (large ? .0155 : .0095) : large ? .0115 : .0085;
        const int64_t slots = p.wide ? cus : (p.mt == 1 ? 3 : 2) * cus;
        const auto split_cost = [&](int64_t s) { return cost(token, large ? 6 : 4.5, slots, tasks_of(16 * p.mt), s, len); };
        const int64_t fewer = splits_for(p.splits, len, 256);  // from 97 rows on a join has many
        if (p.mt == 2) p.splits = fewer;
        double best = split_cost(p.splits);
        const auto take = [&](double us, bool rows, int waves, int64_t splits) {
            if (us < best) best = us, p.rows = rows, p.waves = waves, p.splits = splits, p.wide = p.wide && !rows;
        };
        take(split_cost(1), false, 4, 1);
        const int64_t half = tasks_of(128), seen = len_of(256);
        take(half <= cus ? cost(large ? .0255 : .0205, large ? 6 : 5.5, cus, half, 1, seen) : cost(large ? .037 : .027, large ? 10 : 7, 2 * cus, half, 1, seen), true, 4, 1);
        for (int64_t s = 1; s <= splits_for(32, seen, 256); ++s) take(cost(large ? .027 : .0205, large ? 9 : 6.5, cus, tasks_of(256), s, seen), true, 8, s);
    }
    if (p.splits > 1) p.bytes = tokens * q_heads * p.splits * row;
    if (p.rows) {
        p.tiles = tiles(32 * p.waves);
        return p;
    }
    p.score_cols = table_cols * c->page_size;
    p.scored = weights && each <= 8 && tokens * q_heads * p.score_cols <= int64_t{64} << 20;
    p.scores_at = p.bytes;
    if (p.scored) p.bytes += 4 * tokens * q_heads * p.score_cols;
    return p;
}

// launch(workgroups) of as many row tiles as one launch holds, `each` workgroups a tile, until all have run.
template <class F>
void for_tiles(AttnArgs8 &a, const Plan &p, int64_t each, int threads, const F &launch) {
    require(p.tiles <= 0x7fffffff, "too many rows and sequences for one call");
    const int64_t most = most_workgroups(threads) / each;
    for (int64_t t = 0; t < p.tiles; t += most) {
        a.first_tile = static_cast<int>(t);
        launch(static_cast<unsigned>(std::min(p.tiles - t, most) * each));
    }
}

template <bool kScored, int D, int MT, int NW>
void launch_split(AttnArgs8 a, const Plan &p, hipStream_t st) {
    constexpr int lds = sizeof(SplitLds8<D, NW>);
    static_assert(lds <= 160 * 1024, "LDS budget");
    static std::atomic<uint64_t> attr_devices{0};
    if (lds > 64 * 1024) raise_lds_limit(reinterpret_cast<const void *>(kv8_attention_split_kernel<kScored, D, MT, NW>), lds, attr_devices);
    for_tiles(a, p, a.heads * p.splits, 64 * NW, [&](unsigned grid) {
        kv8_attention_split_kernel<kScored, D, MT, NW><<<dim3(grid), dim3(64 * NW), lds, st>>>(a);
        check_launch("kv8_attention_split");
    });
}

template <int D>
void launch_join(const AttnArgs8 &a, hipStream_t st) {
    const int64_t rows = static_cast<int64_t>(a.tokens) * a.heads * a.ratio;
    if (rows >= 1024) {
        constexpr int per = 1024 / D;
        kv8_attention_join_rows_kernel<D><<<dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), 0, st>>>(a);
    } else {
        kv8_attention_join_kernel<D><<<dim3(static_cast<unsigned>(rows)), dim3(256), 0, st>>>(a);
    }
    check_launch("kv8_attention_join");
}

template <int D, int NW>
void launch_tile(AttnArgs8 a, const Plan &p, hipStream_t st) {
    constexpr int lds = 2 * sizeof(Stage8<D, NW>);
    static_assert(lds <= NW * 20 * 1024, "eight waves a CU");
    static std::atomic<uint64_t> attr_devices{0};
    const auto kern = kv8_attention_tile_kernel<D, NW>;
    raise_lds_limit(reinterpret_cast<const void *>(kern), lds, attr_devices);
    for_tiles(a, p, a.heads * p.splits, 64 * NW, [&](unsigned grid) {
        kern<<<dim3(grid), dim3(64 * NW), lds, st>>>(a, static_cast<int>(p.tiles));
        check_launch("kv8_attention_tile");
    });
}

// window 0 (none) as one that no place reaches.
int64_t window_of(int64_t window) { return window > 0 ? window : 0x7fffffff; }

void check_attention(const cfh_kv8_cache_t *c, int64_t tokens, int64_t q_heads, int64_t batch, int64_t table_cols, int64_t window, int64_t sinks) {
    check_kv8(c);
    check_kv8_table(c, batch, table_cols);
    require(tokens >= 0 && tokens <= 0x7fffffff, "tokens must be in [0, 2^31)");
    require(q_heads >= 1 && q_heads % c->kv_heads == 0 && q_heads / c->kv_heads <= 64,
            "q_heads must be a multiple of kv_heads, at most 64 of them a head of keys");
    require(tokens * q_heads <= 0x7fffffff, "tokens * q_heads must be below 2^31");
    require(window >= 0 && window <= 0x7fffffff, "window must be in [0, 2^31): 0 for none");
    require(sinks >= 0 && sinks <= 0x7ffff000, "sinks must be in [0, 2^31 - 4096]");
}

}  // namespace
}  // namespace cfh

using namespace cfh;

extern "C" {

int32_t castforge_hip_kv8_attention_workspace(const cfh_kv8_cache_t *cache, int64_t tokens, int64_t q_heads, int64_t batch, int64_t table_cols,
                                              int32_t varlen, int64_t window, int64_t sinks, int32_t weights,
                                              int64_t *out_bytes, char **out_error) {
    if (out_bytes) *out_bytes = 0;
    return guarded(out_error, [&] {
        check_attention(cache, tokens, q_heads, batch, table_cols, window, sinks);
        require(out_bytes != nullptr, "out_bytes must not be NULL");
        *out_bytes = plan_of(cache, tokens, q_heads, batch, table_cols, varlen != 0, window_of(window), sinks, weights != 0).bytes;
    });
}

int32_t castforge_hip_kv8_attention(const cfh_kv8_cache_t *cache, const uint16_t *q, int64_t q_stride, int64_t tokens, int64_t q_heads,
                                    int64_t batch, const int32_t *cu_q, const int32_t *page_table, int64_t table_cols, const int32_t *kv_lens,
                                    int32_t causal, int64_t window, int64_t sinks, float scale, uint16_t *out, float *lse, float *weights,
                                    int64_t weights_cols, void *workspace, int64_t workspace_bytes, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_attention(cache, tokens, q_heads, batch, table_cols, window, sinks);
        require(causal == 0 || causal == 1, "causal must be 0 or 1");
        require(causal == 1 || window == 0, "a window needs causal");
        require(cu_q != nullptr || tokens == batch, "without cu_q every sequence has one query: tokens must equal batch");
        require(weights == nullptr || (weights_cols >= 0 && weights_cols <= 0x7fffffff), "weights_cols must be in [0, 2^31)");
        if (tokens == 0) return;
        require(q && out && (batch == 0 || kv_lens) && (batch == 0 || table_cols == 0 || page_table), "buffers must not be NULL");
        require(weights == nullptr || lse != nullptr, "weights need lse");
        require(aligned(q, 16) && aligned(out, 16), "q and out must be 16-byte aligned");
        require(tokens <= 1 || (q_stride >= q_heads * cache->head_dim && q_stride % 8 == 0),
                "q's token stride must be a multiple of 8 and at least q_heads * head_dim");
        if (batch == 0) return;
        const Plan p = plan_of(cache, tokens, q_heads, batch, table_cols, cu_q != nullptr, window_of(window), sinks, weights != nullptr);
        require(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 16)),
                "workspace must be 16-byte aligned and hold the bytes that castforge_hip_kv8_attention_workspace gives");
        AttnArgs8 a{q, q_stride, cache->k_codes, cache->v_codes, cache->k_scales, cache->v_scales, cu_q, page_table, kv_lens, out, lse,
                    static_cast<float *>(workspace), scale * 1.44269504088896341f, static_cast<int>(tokens), static_cast<int>(batch),
                    static_cast<int>(cache->kv_heads), static_cast<int>(q_heads / cache->kv_heads), kv8_log2(cache->page_size),
                    static_cast<int>(table_cols), static_cast<int>(cache->num_pages), causal, static_cast<int>(p.splits),
                    static_cast<int>(window_of(window)), static_cast<int>(sinks), 0, 0,
                    p.scored ? static_cast<float *>(workspace) + p.scores_at / 4 : nullptr, static_cast<int>(p.score_cols), 0};
        const int l = a.ratio > 1 ? kv8_log2(a.ratio - 1) + 1 : 0;  // ceil(log2 ratio)
        a.ratio_shift = 31 + l, a.ratio_mul = static_cast<uint32_t>(((uint64_t{1} << a.ratio_shift) + a.ratio - 1) / a.ratio);
        const hipStream_t st = static_cast<hipStream_t>(stream);
        const auto launch = [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (p.rows) p.waves == 8 ? launch_tile<D, 8>(a, p, st) : launch_tile<D, 4>(a, p, st);
            else if (p.wide) p.scored ? launch_split<true, D, 1, 8>(a, p, st) : launch_split<false, D, 1, 8>(a, p, st);
            else if (p.scored) launch_split<true, D, 1, 4>(a, p, st);  // 8 rows a sequence and head on average: tiles of 16
            else p.mt == 1 ? launch_split<false, D, 1, 4>(a, p, st) : launch_split<false, D, 2, 4>(a, p, st);
            if (p.splits > 1) launch_join<D>(a, st);
        };
        cache->head_dim == 64 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 128>{});
        if (weights) {
            const int64_t each = p.scored ? 1024 : 64, blocks = (std::min(weights_cols, table_cols * cache->page_size) + each - 1) / each;
            WeightArgs8 wa{weights, static_cast<int>(weights_cols), static_cast<int>(blocks), 0};
            // Waves a workgroup, which share its rows: as many as fill the card once, two a SIMD, for a workgroup's start costs as much as
            // several tiles of rows.  A call with its weights, us: 64 queries of 32 heads after 4000 tokens, four sequences: one wave 60, two
            // 63, four 70; of 28 heads after 16384 tokens two 55, one 61, four 57; prompt of 512 tokens eight 31, four 35, two 47.
            const int64_t rows = (tokens * a.ratio + batch - 1) / batch;
            int64_t waves = 1;
            while (waves < 8 && 32 * waves < rows && 2 * waves * blocks * batch * cache->kv_heads <= 8 * cu_count()) waves *= 2;
            const int64_t threads = p.scored ? 256 : 64 * waves, lds = p.scored ? 0 : waves * 64 * cache->head_dim;
            const int64_t all = blocks * batch * cache->kv_heads, most = most_workgroups(threads);
            for (; wa.first_block < all; wa.first_block += most) {
                const dim3 grid(static_cast<unsigned>(std::min(all - wa.first_block, most)));
                const bool by_head = tokens >= 32 * batch;
                const auto kern = p.scored ? kv8_attention_scored_kernel
                    : cache->head_dim == 64 ? by_head ? kv8_attention_weights_kernel<64, true> : kv8_attention_weights_kernel<64, false>
                    : by_head ? kv8_attention_weights_kernel<128, true> : kv8_attention_weights_kernel<128, false>;
                kern<<<grid, dim3(static_cast<unsigned>(threads)), static_cast<size_t>(lds), st>>>(a, wa);
                check_launch("kv8_attention_weights");
            }
        }
    });
}

}  // extern "C"
