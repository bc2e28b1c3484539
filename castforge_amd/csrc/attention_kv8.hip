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
    float *part;  // splits > 1: [tokens * q heads][splits][D + 4], output sums, reference, sum, two unused
    float scale;  // of scores, base 2
    int tokens, batch, heads, ratio, page_shift, table_cols, num_pages, causal, splits;
    int window, sinks;  // window 0x7fffffff: none
    int first_tile;     // of a launch's row tiles, where one launch cannot hold them all
};

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
        const int row = row0 + 16 * mt + n, i = row / a.ratio;
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
// kFold: one fma takes a product to an exponent less m; where m moves, they are made from the products again, which stay until then
// (a register a score: the kernel of few rows has none left).
template <bool kFold, int D, int MT, class Keys, class Values>
__device__ __forceinline__ void attend(const AttnArgs8 &a, Rows8<D, MT> &s, int at, bool edge, const bool (&gone)[2], const Page (&pages)[2], const Keys &keys, const Values &values) {
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
    float z[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float em = kFold ? pages[h].e - s.m[mt] : pages[h].e;
#pragma unroll
            for (int r = 0; r < 4; ++r) z[mt][h][r] = __builtin_fmaf(dot[mt][h][r], pages[h].kf, em);
        }
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
                z[mt][i / 4][i % 4] = hidden ? -INFINITY : z[mt][i / 4][i % 4];
            }
        }
    }
    uint32_t p[MT][4];  // weights as f16 pairs: tokens (0, 1), (2, 3) of both halves
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float (&v)[2][4] = z[mt];
        const float most = max3(max3(v[0][0], v[0][1], v[0][2]), max3(v[0][3], v[1][0], v[1][1]), max3(v[1][2], v[1][3], v[1][3]));
        if (__any(most > (kFold ? 15.f : s.m[mt] + 15.f))) {
            float top = most;
            if constexpr (kFold) {
                top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float y = __builtin_fmaf(dot[mt][i / 4][i % 4], pages[i / 4].kf, pages[i / 4].e);
                    v[i / 4][i % 4] = v[i / 4][i % 4] == -INFINITY ? -INFINITY : y;
                    top = fmaxf(top, v[i / 4][i % 4]);
                }
            }
            const float m = fmaxf(s.m[mt], max_over_g(top) - 7.f), f = __builtin_amdgcn_exp2f(s.m[mt] - m);
            s.m[mt] = m;
            s.l[mt] *= f;
#pragma unroll
            for (int u = 0; u < NT; ++u) s.o[mt][u] *= f;
            if constexpr (kFold)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i / 4][i % 4] -= m;
        }
        float w[2][4];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i / 4][i % 4] = __builtin_amdgcn_exp2f(kFold ? v[i / 4][i % 4] : v[i / 4][i % 4] - s.m[mt]);
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

// A wave's walk over steps first, first + by, .. below last of a span, the next tile's loads in flight.
template <int D, int MT>
__device__ __forceinline__ void walk(const AttnArgs8 &a, Rows8<D, MT> &s, const Seq &sq, int head, const Span &span, int first, int by, int last) {
    if (first >= last) return;
    constexpr int W = Tile8<D>::W;
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const Sure sure = seen_by_all(s, sq.len);
    const int32_t *table = a.table + static_cast<int64_t>(sq.seq) * a.table_cols;
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
        attend<false, D, MT>(
            a, s, at, edge, gone, pages_of,
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

// Where a row's output goes, of the sequence's row tile.
__device__ __forceinline__ int64_t out_row(const AttnArgs8 &a, const Seq &sq, int head, int row) {
    return static_cast<int64_t>(sq.first + row / a.ratio) * (a.heads * a.ratio) + head * a.ratio + row % a.ratio;
}

__device__ __forceinline__ float lse_of(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.693147180559945309f; }

// One workgroup's NW waves take the same rows and every NW-th 32 tokens of a split's share, and are joined through LDS;
// splits are joined by kv8_attention_join_kernel.
template <int D, int NW>
struct SplitLds8 {
    float sums[NW][16][D + 4];
    float m[NW][16], l[NW][16];
};

template <int D, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void kv8_attention_split_kernel(AttnArgs8 a) {
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
    const Span span = span_of(a, sq, row0 / a.ratio, (row0 + rows - 1) / a.ratio);
    const int steps = span.steps(), share = (steps + used * NW - 1) / (used * NW) * NW;  // whole rounds of the waves
    Rows8<D, MT> s;
    load_rows(a, s, sq, head, row0);
    // shares are rounded up: the last ones may be empty
    walk<D, MT>(a, s, sq, head, span, split * share + wave, NW, min(steps, (split + 1) * share));
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
                if (ch == 0) p[D] = mm, p[D + 1] = l;
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

// Joins the splits: a workgroup a (token, query head), D / 8 lanes of eight channels by 2048 / D lanes of splits, each with a
// reference of its own until the end.
template <int D>
__global__ __launch_bounds__(256) void kv8_attention_join_kernel(AttnArgs8 a) {
    constexpr int kCh = D / 8, kSp = 256 / kCh;
    __shared__ __align__(16) float sums[kSp][D + 4];
    __shared__ float ms[kSp], ls[kSp];
    const int hq = a.heads * a.ratio;
    const int64_t at = blockIdx.x;
    const int token = static_cast<int>(at / hq), ch = threadIdx.x % kCh * 8, sl = threadIdx.x / kCh;
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
            if (hit) seq = __builtin_amdgcn_readfirstlane(b0 + __builtin_ctzll(hit));
        }
        if (seq < 0) return;
    }
    const int used = splits_of_seq(a, seq_of(a, seq));
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
        if (a.lse && threadIdx.x == 0) a.lse[at] = lse_of(top, t);
    }
}

// Many rows: each wave takes 32 rows of its own, and the NW of a workgroup share the making of the MFMA operands.  Of every 16 NW
// tokens a wave turns 16 into operands in LDS and all read them back; two stages, one barrier a stage: the operands of the next tokens
// are made while the present ones are used, and the codes of those after that are on their way.
// Heads are dealt out first (one head's keys and values stay with one XCD where there are eight heads), and row tiles from the
// last, which see the most tokens.
template <int D, int NW>
struct Stage8 {
    static constexpr int KS = D / 32, NT = D / 16;
    uint4 keys[NW][KS][64];        // 16 tokens, 32 channels: a lane's operand
    uint4 values[NW / 2][NT][64];  // 32 tokens, 16 channels
    Page pages[NW];
};

template <int D, int NW>
__global__ __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 3))) void kv8_attention_tile_kernel(AttnArgs8 a, int tiles) {
    constexpr int MT = 2, KS = D / 32, NT = D / 16, W = D / 64, kSteps = NW / 2;  // steps of 32 tokens a stage
    extern __shared__ __align__(16) uint8_t lds[];
    Stage8<D, NW> *stages = reinterpret_cast<Stage8<D, NW> *>(lds);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int n = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.heads;
    const Seq sq = find_tile(a, tiles - 1 - (a.first_tile + blockIdx.x / a.heads), 16 * NW * MT);
    if (sq.seq < 0) return;
    const int total = sq.n * a.ratio, row_of_all = sq.tile * 16 * NW * MT, row0 = row_of_all + wave * 16 * MT;
    const Span span = span_of(a, sq, row_of_all / a.ratio, (min(row_of_all + 16 * NW * MT, total) - 1) / a.ratio);
    const int steps = span.steps();
    // the wave's own rows see tokens below `mine`, and from `from` on or sinks
    const int mine = row0 < total ? limit_of(a, sq, (min(row0 + 16 * MT, total) - 1) / a.ratio) : 0;
    const int from = row0 < total ? low_of(a, sq, row0 / a.ratio) : 0;
    Rows8<D, MT> s;
    load_rows(a, s, sq, head, row0);
    const Sure sure = seen_by_all(s, sq.len);
    const int32_t *table = a.table + static_cast<int64_t>(sq.seq) * a.table_cols;

    // this wave's 16 tokens of a stage
    struct Part {
        uint4 k[W];
        uint32_t v[4][W];
        float ks, vs;
        int at;
        bool live;
    };
    const auto token_at = [&](int step) { return span.token_of(step + wave / 2) + 16 * (wave & 1); };
    const auto page_at = [&](int step) {
        const int at = token_at(step);
        return step + wave / 2 < steps && at < span.end ? scalar_load(table, at >> a.page_shift) : -1;
    };
    const auto load = [&](Part &t, int page, int step) {
        t.at = token_at(step);
        t.live = page >= 0 && page < a.num_pages;
        const int p = t.live ? page : 0;
        const int64_t row = kv8_row(p, head, t.at & ((1 << a.page_shift) - 1), a.heads, a.page_shift), at_scale = static_cast<int64_t>(p) * a.heads + head;
        const uint8_t *k = a.k_codes + (row + n) * D + 16 * g, *v = a.v_codes + (row + 4 * g) * D + n * (D / 16);
#pragma unroll
        for (int i = 0; i < W; ++i) t.k[i] = *reinterpret_cast<const uint4 *>(k + 64 * i);
#pragma unroll
        for (int r = 0; r < 4; ++r) __builtin_memcpy(t.v[r], __builtin_assume_aligned(v + r * D, D / 16), D / 16);
        t.ks = scalar_load(a.k_scales, at_scale), t.vs = scalar_load(a.v_scales, at_scale);
    };
    const auto make = [&](Part &t, Stage8<D, NW> &st) {
        if (!t.live || t.at + 16 > sq.len) {  // uniform: bytes that are no token's may be NaN, which a weight of 0 does not take away
            asm volatile("");
#pragma unroll
            for (int i = 0; i < W; ++i) {
                if (!t.live) t.k[i] = uint4{};
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!t.live || t.at + 4 * g + r >= sq.len) t.v[r][i] = 0;
            }
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            st.keys[wave][2 * i][lane] = __builtin_bit_cast(uint4, keys_bf16(t.k[i].x, t.k[i].y));
            st.keys[wave][2 * i + 1][lane] = __builtin_bit_cast(uint4, keys_bf16(t.k[i].z, t.k[i].w));
        }
        static_for<NT>([&](auto u) __attribute__((always_inline)) { reinterpret_cast<uint2 *>(&st.values[wave / 2][u][lane])[wave & 1] = values_f16<u>(t.v); });
        // no page of the cache: scores of -inf, by products of zeros
        if (lane == 0) st.pages[wave] = t.live ? page_of(a.scale, t.ks, t.vs) : Page{0.f, -INFINITY, 0.f};
    };
    Part part;
    if (steps > 0) {
        load(part, page_at(0), 0);
        make(part, stages[0]);
        load(part, page_at(kSteps), kSteps);
    }
    int page = page_at(2 * kSteps);
    // the queries have come: else the compiler waits for them in every stage, and with them for the codes on their way
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    for (int step = 0, i = 0; step < steps; step += kSteps, i ^= 1) {
        __syncthreads();  // stage i is made, and the other one no longer read
        if (step + kSteps < steps) {
            make(part, stages[i ^ 1]);
            load(part, page, step + 2 * kSteps);
            page = page_at(step + 3 * kSteps);
        }
        const Stage8<D, NW> &st = stages[i];
#pragma unroll
        for (int sub = 0; sub < kSteps; ++sub) {
            const int at = span.token_of(step + sub);
            if (at >= mine) break;
            if (at + 32 <= from && at >= a.sinks) continue;
            const Page pages_of[2] = {st.pages[2 * sub], st.pages[2 * sub + 1]};
            attend<true, D, MT>(
                a, s, at, at + 32 > sure.limit || (at < sure.low && at + 32 > a.sinks), {false, false}, pages_of,
                [&](int h, int k) { return __builtin_bit_cast(bf16x8, st.keys[2 * sub + h][k][lane]); },
                [&](auto u) { return __builtin_bit_cast(halfx8, st.values[sub][u][lane]); });
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const int row = row0 + 16 * mt + n;
        const float l = sum_over_g(s.l[mt]), inv = l == 0.f ? 0.f : 1.0f / l;  // 0: no token was seen
        if (row >= total) continue;
        const int64_t to = out_row(a, sq, head, row);
        if (a.lse && g == 0) a.lse[to] = lse_of(s.m[mt], l);
        // a lane's D / 4 channels lie behind one another
        uint16_t *out = a.out + to * D + g * (D / 4);
#pragma unroll
        for (int c = 0; c < D / 4; c += 8) {
            const auto v = [&](int e) { return s.o[mt][(c + e) % NT][(c + e) / NT] * inv; };
            *reinterpret_cast<uint4 *>(out + c) = make_uint4(f32x2_to_bf16x2_rne(v(0), v(1)), f32x2_to_bf16x2_rne(v(2), v(3)), f32x2_to_bf16x2_rne(v(4), v(5)), f32x2_to_bf16x2_rne(v(6), v(7)));
        }
    }
}

// Weights that the cached tokens got, from the logarithms of the rows' sums: weights[seq, head, t] += sum over the head's rows of
// exp(score - lse).  A wave has 16 tokens' keys, as MFMA operands, and walks over the rows that see some of them; S^T = K Q^T leaves
// each lane four tokens' sums over its rows, joined over the 16 lanes at the end.  Every sum has one writer.
template <int D>
__global__ __launch_bounds__(256) void kv8_attention_weights_kernel(AttnArgs8 a, float *weights, int cols, int blocks, int64_t first_block) {
    constexpr int KS = D / 32, W = D / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int64_t block = first_block + blockIdx.x;
    const int seq = static_cast<int>(block / blocks / a.heads), head = static_cast<int>(block / blocks % a.heads);
    const int t0 = 64 * static_cast<int>(block % blocks) + 16 * wave;
    const Seq sq = seq_of(a, seq);
    const int most = min(sq.len, cols);
    if (t0 >= most || sq.n == 0) return;
    const int page = scalar_load(a.table, static_cast<int64_t>(seq) * a.table_cols + (t0 >> a.page_shift));
    if (page < 0 || page >= a.num_pages) return;
    const uint8_t *k = a.k_codes + (kv8_row(page, head, t0 & ((1 << a.page_shift) - 1), a.heads, a.page_shift) + n) * D + 16 * g;
    bf16x8 keys[KS];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const uint4 w = *reinterpret_cast<const uint4 *>(k + 64 * i);
        keys[2 * i] = keys_bf16(w.x, w.y), keys[2 * i + 1] = keys_bf16(w.z, w.w);
    }
    const float kf = a.scale * scalar_load(a.k_scales, static_cast<int64_t>(page) * a.heads + head);
    const int before = sq.len - sq.n;  // place of the first query
    const int i0 = a.causal ? max(t0 - before, 0) : 0;
    const int64_t last_place = static_cast<int64_t>(t0) + 15 + a.window - 1;
    const int i1 = t0 < a.sinks ? sq.n - 1 : static_cast<int>(min<int64_t>(sq.n - 1, last_place - before));
    const int end = (i1 + 1) * a.ratio, hq = a.heads * a.ratio;
    float sums[4] = {0.f, 0.f, 0.f, 0.f};
    for (int row = i0 * a.ratio + n; row - n < end; row += 16) {
        const bool in = row < end;
        const int i = in ? row / a.ratio : i1, h = head * a.ratio + (in ? row - i * a.ratio : 0);
        const uint16_t *q = a.q + (sq.first + i) * a.q_stride + h * D;
        const float lse = a.lse[static_cast<int64_t>(sq.first + i) * hq + h] * 1.44269504088896341f;
        const int limit = in ? limit_of(a, sq, i) : 0, low = low_of(a, sq, i);
        floatx4 dot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s)
            dot = __builtin_amdgcn_mfma_f32_16x16x32_bf16(keys[s], __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(q + 64 * (s / 2) + 16 * g + 8 * (s % 2))), dot, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int t = t0 + 4 * g + r;
            const bool seen = t < limit && (t >= low || t < a.sinks);
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(dot[r], kf, -lse));
            sums[r] += seen ? w : 0.f;
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float v = sums[r];
        v += lane_xor<1>(v);
        v += lane_xor<2>(v);
        v += lane_xor<4>(v);
        v += lane_xor<8>(v);
        const int t = t0 + 4 * g + r;
        if (n == 0 && t < most) {
            float *p = weights + (static_cast<int64_t>(seq) * a.heads + head) * cols + t;
            *p += v;
        }
    }
}

// How a call is laid out: rows a wave (16 mt), whether waves share rows (splits of the tokens) or have their own, row
// tiles at most, splits, workspace.
struct Plan {
    int mt, waves;
    bool rows;
    int64_t tiles, splits, bytes;
};

Plan plan_of(const cfh_kv8_cache_t *c, int64_t tokens, int64_t q_heads, int64_t batch, int64_t table_cols, bool varlen, int64_t window, int64_t sinks) {
    Plan p{1, 4, false, 0, 1, 0};
    if (tokens == 0 || batch == 0) return p;
    const int64_t ratio = q_heads / c->kv_heads, cus = cu_count(), rows = tokens * ratio, each = (rows + batch - 1) / batch;
    const auto tiles = [&](int64_t per) { return varlen ? rows / per + batch : batch * ((ratio + per - 1) / per); };
    p.rows = varlen && rows / 32 * c->kv_heads >= 6 * cus;
    if (p.rows) {
        p.mt = 2;
        if (rows / (128 * p.mt) * c->kv_heads >= 2 * cus) p.waves = 8;
        p.tiles = tiles(16 * p.waves * p.mt);
        return p;
    }
    p.mt = each <= 96 ? 1 : 2;
    p.tiles = tiles(16 * p.mt);
    const int64_t tasks = p.tiles * c->kv_heads, len = std::min(table_cols * c->page_size, window + sinks + 64 + tokens);
    p.splits = std::max<int64_t>(1, std::min((2 * cus + tasks - 1) / tasks, (len + 127) / 128));
    const int64_t row = (c->head_dim + 4) * 4;
    p.splits = std::max<int64_t>(1, std::min(p.splits, (int64_t{256} << 20) / (tokens * q_heads * row)));
    if (p.splits > 1) p.bytes = tokens * q_heads * p.splits * row;
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

template <int D, int MT, int NW>
void launch_split(AttnArgs8 a, const Plan &p, hipStream_t st) {
    constexpr int lds = sizeof(SplitLds8<D, NW>);
    static_assert(lds <= 64 * 1024, "LDS budget");
    for_tiles(a, p, a.heads * p.splits, 64 * NW, [&](unsigned grid) {
        kv8_attention_split_kernel<D, MT, NW><<<dim3(grid), dim3(64 * NW), lds, st>>>(a);
        check_launch("kv8_attention_split");
    });
    if (p.splits > 1) {
        kv8_attention_join_kernel<D><<<dim3(static_cast<unsigned>(static_cast<int64_t>(a.tokens) * a.heads * a.ratio)), dim3(256), 0, st>>>(a);
        check_launch("kv8_attention_join");
    }
}

template <int D, int NW>
void launch_tile(AttnArgs8 a, const Plan &p, hipStream_t st) {
    constexpr int lds = 2 * sizeof(Stage8<D, NW>);
    static_assert(lds <= NW * 20 * 1024, "eight waves a CU");
    static std::atomic<uint64_t> attr_devices{0};
    const auto kern = kv8_attention_tile_kernel<D, NW>;
    raise_lds_limit(reinterpret_cast<const void *>(kern), lds, attr_devices);
    for_tiles(a, p, a.heads, 64 * NW, [&](unsigned grid) {
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
                                              int32_t varlen, int64_t window, int64_t sinks, int64_t *out_bytes, char **out_error) {
    if (out_bytes) *out_bytes = 0;
    return guarded(out_error, [&] {
        check_attention(cache, tokens, q_heads, batch, table_cols, window, sinks);
        require(out_bytes != nullptr, "out_bytes must not be NULL");
        *out_bytes = plan_of(cache, tokens, q_heads, batch, table_cols, varlen != 0, window_of(window), sinks).bytes;
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
        const Plan p = plan_of(cache, tokens, q_heads, batch, table_cols, cu_q != nullptr, window_of(window), sinks);
        require(p.bytes == 0 || (workspace && workspace_bytes >= p.bytes && aligned(workspace, 16)),
                "workspace must be 16-byte aligned and hold the bytes that castforge_hip_kv8_attention_workspace gives");
        AttnArgs8 a{q, q_stride, cache->k_codes, cache->v_codes, cache->k_scales, cache->v_scales, cu_q, page_table, kv_lens, out, lse,
                    static_cast<float *>(workspace), scale * 1.44269504088896341f, static_cast<int>(tokens), static_cast<int>(batch),
                    static_cast<int>(cache->kv_heads), static_cast<int>(q_heads / cache->kv_heads), kv8_log2(cache->page_size),
                    static_cast<int>(table_cols), static_cast<int>(cache->num_pages), causal, static_cast<int>(p.splits),
                    static_cast<int>(window_of(window)), static_cast<int>(sinks), 0};
        const hipStream_t st = static_cast<hipStream_t>(stream);
        const auto launch = [&](auto d) {
            constexpr int D = decltype(d)::value;
            if (p.rows) p.waves == 8 ? launch_tile<D, 8>(a, p, st) : launch_tile<D, 4>(a, p, st);
            else p.mt == 1 ? launch_split<D, 1, 4>(a, p, st) : launch_split<D, 2, 4>(a, p, st);
        };
        cache->head_dim == 64 ? launch(std::integral_constant<int, 64>{}) : launch(std::integral_constant<int, 128>{});
        const int64_t reach = std::min(weights ? weights_cols : 0, table_cols * cache->page_size), blocks = (reach + 63) / 64;
        const int64_t all = blocks * batch * cache->kv_heads;
        for (int64_t b = 0, most = most_workgroups(256); b < all; b += most) {
            const dim3 grid(static_cast<unsigned>(std::min(all - b, most)));
            const auto kern = cache->head_dim == 64 ? kv8_attention_weights_kernel<64> : kv8_attention_weights_kernel<128>;
            kern<<<grid, dim3(256), 0, st>>>(a, weights, static_cast<int>(weights_cols), static_cast<int>(blocks), b);
            check_launch("kv8_attention_weights");
        }
    });
}

}  // extern "C"
