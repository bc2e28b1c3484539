// Appending keys and values to the paged 8-bit cache, with the position rotation on the way, reading rows back, and
// moving the tokens that are worth most to new pages.
//
// Rotation of a head's first `rot` channels by the angles of the token's position: pairs (i, i + rot / 2),
// or (2 i, 2 i + 1) where interleaved; (a, b) -> (a c - b s, b c + a s), each product and the difference
// rounded to f32 where it stands.  Keys go from the rotated f32 straight into codes; queries, rotated in the
// same launch, are rounded once to bf16.
//
// Codes of a page and head: s' = max(s, 2^e), e the least with absmax <= 448 * 2^e over the call's tokens there, s the
// page's scale, or 0 where its first place is among them (the page starts anew); code = E4M3(x / s'), NaN -> 0.
// Codes of tokens before the call's go over to s', rounded from the codes.
#include <algorithm>

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"
#include "kv8.hpp"

namespace cfh {
namespace {

struct AppendArgs8 {
    const uint16_t *k, *v, *q;
    int64_t k_stride, v_stride, q_stride;  // elements from a token's row to the next one's
    const int32_t *cu_q, *table, *kv_lens;
    const int64_t *positions;
    const float *cos, *sin;
    uint16_t *q_out;
    int64_t max_pos;
    int tokens, batch, heads, q_heads, page_shift, table_cols, num_pages, rot, interleaved;
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    int64_t first_block;  // of a launch's workgroups, where one launch cannot hold them all
    int64_t kv_blocks;    // workgroups with keys or values; one a token of the queries follows
};

// A page's new tokens: places lo .. hi - 1 of the page in column `col` of sequence seq's table; `row` the first one's row.
struct Unit {
    int seq, col, lo, hi, row;
};

// New tokens of a sequence with n rows and a length: those at places first .. end - 1, pages' columns from first >> shift on.
__device__ __forceinline__ void new_tokens(const AppendArgs8 &a, int n, int len, int &first, int &end) {
    first = max(len - n, 0);
    end = n > 0 ? min(len, a.table_cols << a.page_shift) : 0;
}

// The unit of a number: the pages that get tokens, sequence by sequence.  The lanes of a wave look at 64 sequences at once.
__device__ __forceinline__ Unit find_unit(const AppendArgs8 &a, int unit) {
    const int lane = threadIdx.x & 63, page = 1 << a.page_shift;
    const auto made = [&](int seq, int begin, int n, int len, int k) {
        int first, end;
        new_tokens(a, n, len, first, end);
        Unit u;
        u.seq = seq, u.col = (first >> a.page_shift) + k;
        const int base = u.col << a.page_shift;
        u.lo = max(first - base, 0), u.hi = min(end - base, page);
        u.row = begin + (base + u.lo - (len - n));
        return u;
    };
    if (!a.cu_q) {
        if (unit >= a.batch) return Unit{-1, 0, 0, 0, 0};
        const int len = a.kv_lens[unit];
        int first, end;
        new_tokens(a, 1, len, first, end);
        return first < end ? made(unit, unit, 1, len, 0) : Unit{-1, 0, 0, 0, 0};
    }
    int before = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int b = b0 + lane;
        int begin = 0, n = 0, len = 0, pages = 0;
        if (b < a.batch) {  // clamped: a malformed list stays inside the rows
            begin = min(max(a.cu_q[b], 0), a.tokens);
            n = min(max(a.cu_q[b + 1], begin), a.tokens) - begin;
            len = a.kv_lens[b];
            int first, end;
            new_tokens(a, n, len, first, end);
            if (first < end) pages = ((end - 1) >> a.page_shift) - (first >> a.page_shift) + 1;
        }
        int upto = pages;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(upto, o);
            if (lane >= o) upto += v;
        }
        const uint64_t hit = __ballot(before + upto > unit);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            return made(b0 + l, __builtin_amdgcn_readlane(begin, l), __builtin_amdgcn_readlane(n, l), __builtin_amdgcn_readlane(len, l),
                        unit - before - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(pages, l)));
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return Unit{-1, 0, 0, 0, 0};
}

__device__ __forceinline__ void unpack8(const uint4 &w, float (&x)[8]) {
    const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(b[i] << 16), x[2 * i + 1] = __uint_as_float(b[i] & 0xffff0000u);
}

typedef uint32_t uintx2 __attribute__((ext_vector_type(2)));

// Four elements and four more.  Read through the caches, for a row's halves share no lines with their loads: past them 52.3 us, not 49.6,
// where 4096 tokens of 32 heads are appended and read back.
__device__ __forceinline__ uint4 load8(const uint16_t *lo, const uint16_t *hi) {
    const uint2 a = *reinterpret_cast<const uint2 *>(lo), b = *reinterpret_cast<const uint2 *>(hi);
    return make_uint4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4_past(uint16_t *p, uint32_t a, uint32_t b) { __builtin_nontemporal_store(uintx2{a, b}, reinterpret_cast<uintx2 *>(p)); }

// A lane's eight channels of a row, lo .. lo + 3 and hi .. hi + 3: both of each pair that is turned together, so that a lane reads an angle
// once and no channel twice (by eight channels in a row a lane: 96 bytes for eight, not 48).
struct Channels {
    int lo, hi;
    bool turned;
    __device__ __forceinline__ Channels(const AppendArgs8 &a, int piece) : lo(8 * piece), hi(8 * piece + 4), turned(8 * piece < a.rot) {
        if (turned && !a.interleaved) lo = 4 * piece, hi = a.rot / 2 + 4 * piece;
    }
};

// The angles of a lane's four pairs, of a token at a position.
struct Turn {
    float c[4], s[4];
    __device__ __forceinline__ void load(const AppendArgs8 &a, int64_t position, int piece) {
        // a position outside the table takes its nearest row
        const int64_t at = min(max(position, int64_t{0}), a.max_pos - 1) * (a.rot / 2) + 4 * piece;
        const float4 cc = *reinterpret_cast<const float4 *>(a.cos + at), ss = *reinterpret_cast<const float4 *>(a.sin + at);
        c[0] = cc.x, c[1] = cc.y, c[2] = cc.z, c[3] = cc.w;
        s[0] = ss.x, s[1] = ss.y, s[2] = ss.z, s[3] = ss.w;
    }
    __device__ __forceinline__ void apply(const AppendArgs8 &a, float (&x)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = a.interleaved ? x[2 * i] : x[i], q = a.interleaved ? x[2 * i + 1] : x[4 + i];
            const float u = p * c[i] - q * s[i], v = q * c[i] + p * s[i];
            (a.interleaved ? x[2 * i] : x[i]) = u, (a.interleaved ? x[2 * i + 1] : x[4 + i]) = v;
        }
    }
};

// A workgroup has the keys, or the values, of one head in one page: eight channels a lane, D / 8 lanes a token, NP rounds of
// 2048 / D tokens whose numbers stay in registers between the absmax and the codes.  The workgroups after those have a token's
// queries each.  HBM: 4096 tokens of 32 heads of each kind, 128 channels, with their read-back 49 us a call, 5.5 TB/s (a large copy runs at
// 5.1: part of this stays in the last-level cache).  16 tokens of as many sequences 6 us on the GPU and 22 a call, the host's for two calls.
template <int D, int NP>
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendArgs8 a) {
    constexpr int kLanes = D / 8, kRows = 256 / kLanes;
    __shared__ float tops[4];
    const int piece = threadIdx.x % kLanes, local = threadIdx.x / kLanes;
    const int64_t block = a.first_block + blockIdx.x;
    const Channels ch(a, piece);
    if (block >= a.kv_blocks) {
        const int token = static_cast<int>(block - a.kv_blocks);
        if (token >= (a.cu_q ? a.cu_q[a.batch] : a.tokens)) return;  // of no sequence
        Turn turn;
        if (ch.turned) turn.load(a, a.positions[token], piece);
        for (int h = local; h < a.q_heads; h += kRows) {
            const uint16_t *src = a.q + token * a.q_stride + h * D;
            float x[8];
            unpack8(load8(src + ch.lo, src + ch.hi), x);
            if (ch.turned) turn.apply(a, x);
            uint16_t *to = a.q_out + (static_cast<int64_t>(token) * a.q_heads + h) * D;
            store4_past(to + ch.lo, f32x2_to_bf16x2_rne(x[0], x[1]), f32x2_to_bf16x2_rne(x[2], x[3]));
            store4_past(to + ch.hi, f32x2_to_bf16x2_rne(x[4], x[5]), f32x2_to_bf16x2_rne(x[6], x[7]));
        }
        return;
    }
    const int which = static_cast<int>(block % (2 * a.heads));
    const bool is_v = which >= a.heads;
    const int head = is_v ? which - a.heads : which;
    const Unit u = find_unit(a, static_cast<int>(block / (2 * a.heads)));
    if (u.seq < 0) return;
    const int page = a.table[static_cast<int64_t>(u.seq) * a.table_cols + u.col];
    if (page < 0 || page >= a.num_pages) return;
    const int64_t row0 = kv8_row(page, head, 0, a.heads, a.page_shift);
    uint8_t *codes = (is_v ? a.v_codes : a.k_codes) + row0 * D;
    float *scale_at = (is_v ? a.v_scales : a.k_scales) + static_cast<int64_t>(page) * a.heads + head;
    const float old = u.lo > 0 ? *scale_at : 0.f;
    const int count = u.hi - u.lo;
    float x[NP][8], top = 0.f;
    const uint16_t *rows = is_v ? a.v + head * D : a.k + head * D;
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        // rows past the last one are that one again: under a branch each load would wait for itself (4096 tokens 64 -> 57 us with their
        // read-back when it was done; four rounds' loads at once: 73, three waves a SIMD instead of seven)
        const int r = j * kRows + local, at = u.row + min(r, count - 1);
        if (j * kRows >= count) break;
        const uint16_t *row = rows + at * stride;
        if (is_v) {
            unpack8(load_once(row + 8 * piece), x[j]);
        } else {
            unpack8(load8(row + ch.lo, row + ch.hi), x[j]);
            if (ch.turned) {
                Turn turn;
                turn.load(a, a.positions[at], piece);
                turn.apply(a, x[j]);
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = __builtin_elementwise_maximum(top, fabsf(x[j][i]));  // NaN stays
    }
    const auto most = [&](float lane_top, bool nan) {
        lane_top = wave_max<64>(lane_top);
        if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = nan ? __builtin_nanf("") : lane_top;
        __syncthreads();  // also: every lane has read the old scale
        return __builtin_elementwise_maximum(__builtin_elementwise_maximum(tops[0], tops[1]), __builtin_elementwise_maximum(tops[2], tops[3]));
    };
    top = most(top, __any(top != top));
    const bool nan = top != top;
    if (nan) {  // uniform: once more, NaN left out
        __syncthreads();
        top = 0.f;
#pragma unroll
        for (int j = 0; j < NP; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) top = j * kRows < count ? fmaxf(top, fabsf(x[j][i])) : top;
        top = most(top, false);
    }
    const float scale = fmaxf(old, kv8_scale_of(top));
    if (scale > old) {
        if (threadIdx.x == 0) *scale_at = scale;
        const float ratio = old / scale;
        for (int r = local; r < u.lo; r += kRows) {
            uint2 *p = reinterpret_cast<uint2 *>(codes + r * D + 8 * piece);
            *p = make_uint2(e4m3x4_by(p->x, ratio), e4m3x4_by(p->y, ratio));
        }
    }
    const auto store = [&](const auto &code_of) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = j * kRows + local;
            if (r < count) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = code_of(x[j][i]);
                uint8_t *to = codes + (u.lo + r) * D;
                const uint32_t one = f32_to_e4m3x4(y), two = f32_to_e4m3x4(y + 4);
                if (is_v) *reinterpret_cast<uint2 *>(to + 8 * piece) = make_uint2(one, two);
                else *reinterpret_cast<uint32_t *>(to + ch.lo) = one, *reinterpret_cast<uint32_t *>(to + ch.hi) = two;
            }
        }
    };
    // Where the scale is a power of two, whose reciprocal is exact, and all quotients are numbers of at most 448, a product is the quotient
    // and nothing is to be cut (1% of 4096 tokens' time).
    const float inv = 1.0f / scale;
    if (!nan && top <= 448.f * scale && (__float_as_uint(scale) & 0x7fffffu) == 0) store([&](float v) { return v * inv; });
    else store([&](float v) { return v != v ? 0.f : __builtin_amdgcn_fmed3f(v / scale, -448.f, 448.f); });
}

// Rows of the cache as numbers, a workgroup a token, eight elements a lane; a slot outside the cache gives zeros.
template <int D>
__global__ __launch_bounds__(256) void kv8_gather_kernel(const uint8_t *__restrict__ k_codes, const float *__restrict__ k_scales,
                                                         const uint8_t *__restrict__ v_codes, const float *__restrict__ v_scales,
                                                         const int64_t *__restrict__ slots, int64_t capacity, int heads, int page_shift,
                                                         void *__restrict__ k_out, void *__restrict__ v_out, int bf16, int share) {
    constexpr int kLanes = D / 8, kUnits = 256 / kLanes;
    const int64_t token = blockIdx.x, slot = slots[token];
    const bool kept = slot >= 0 && slot < capacity;
    const int64_t page = kept ? slot >> page_shift : 0;
    const int at = static_cast<int>(slot & ((1 << page_shift) - 1));
    const int piece = threadIdx.x % kLanes, end = min(2 * heads, static_cast<int>(blockIdx.y + 1) * share);
#pragma unroll 2
    for (int u = static_cast<int>(blockIdx.y) * share + static_cast<int>(threadIdx.x) / kLanes; u < end; u += kUnits) {
        const bool is_v = u >= heads;
        const int head = is_v ? u - heads : u;
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (kept) {
            // past the caches, which hold what is written: 61006 tokens of 8 heads after their move 155 -> 125 us together
            const uintx2 w = __builtin_nontemporal_load(reinterpret_cast<const uintx2 *>((is_v ? v_codes : k_codes) + kv8_row(page, head, at, heads, page_shift) * D + 8 * piece));
            const float scale = (is_v ? v_scales : k_scales)[page * heads + head];
            e4m3x4_to_f32(w.x, x), e4m3x4_to_f32(w.y, x + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= scale;
        }
        const int64_t out = (token * heads + head) * D + 8 * piece;
        if (bf16) {
            store_past(static_cast<uint16_t *>(is_v ? v_out : k_out) + out,
                       make_uint4(f32x2_to_bf16x2_rne(x[0], x[1]), f32x2_to_bf16x2_rne(x[2], x[3]), f32x2_to_bf16x2_rne(x[4], x[5]), f32x2_to_bf16x2_rne(x[6], x[7])));
        } else {
            float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(is_v ? v_out : k_out) + out);
            o[0] = make_float4(x[0], x[1], x[2], x[3]);
            o[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
    }
}

struct EvictArgs8 {
    uint8_t *k_codes, *v_codes;
    float *k_scales, *v_scales;
    const int32_t *table, *kv_lens, *new_table;
    const float *weights;
    int32_t *kept, *new_lens;
    float *new_weights;
    int heads, page_shift, table_cols, new_cols, num_pages, weights_cols, keep, sinks, recent;
    int used_cols;        // of new_table: those that keep tokens take
    int64_t first_block;  // of a launch's workgroups, where one launch cannot hold them all
};

__device__ __forceinline__ int evict_len(const EvictArgs8 &a, int seq) { return min(max(a.kv_lens[seq], 0), a.table_cols << a.page_shift); }

// A weight as a number that orders alike: greater ones first, -0 as 0, NaN last.
__device__ __forceinline__ uint32_t rank_of(float w) {
    const uint32_t b = __float_as_uint(w + 0.f);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0;
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The sums of the lanes before this one, over a workgroup of kWaves waves: of a and b apart.
template <int kWaves>
__device__ __forceinline__ uint2 sums_before(uint32_t a, uint32_t b, uint2 *waves, uint2 &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint2 v = make_uint2(a, b);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(v.x, o), y = __shfl_up(v.y, o);
        if (lane >= o) v.x += x, v.y += y;
    }
    __syncthreads();  // the last call's are read
    if (lane == 63) waves[wave] = v;
    __syncthreads();
    uint2 before = make_uint2(v.x - a, v.y - b);
    all = make_uint2(0, 0);
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave) before.x += waves[w].x, before.y += waves[w].y;
        all.x += waves[w].x, all.y += waves[w].y;
    }
    return before;
}

// Which tokens of a sequence and head are kept: a workgroup each.  The rank of the last one that is comes from its bits, 11, 11 and 10
// at a time: a histogram in LDS of the ranks that agree so far, and the bin in which the count is reached.  Then one pass in the
// tokens' order gives each kept one its place: those of higher rank, and the first of the last rank's.
// kEach: tokens a lane whose weights stay in registers, where the table holds no more (one sequence of 4001 tokens 11.7 -> 9.9 us); 0:
// they are read in every pass, from the caches (16 in registers took as long for sequences of 8192: 18 us).
// Bound by one CU's vector instructions: 131072 tokens take 150 us, half of it the last pass, whatever the number of sequences up to one a CU.
// Batches of eight loads, a ballot for the histogram's additions, other runs of tokens a lane: slower.  Several workgroups a sequence would
// take four to seven launches.
constexpr int kSelectThreads = 1024;
template <int kEach>
__global__ __launch_bounds__(kSelectThreads) void kv8_select_kernel(EvictArgs8 a) {
    constexpr int kWaves = kSelectThreads / 64, kRound = kEach ? kEach : 4;  // tokens a lane of a round in their order
    __shared__ uint32_t bins[2048];
    __shared__ uint2 waves[kWaves];
    __shared__ uint32_t found[2];
    const int64_t block = a.first_block + blockIdx.x;
    const int seq = static_cast<int>(block / a.heads), head = static_cast<int>(block % a.heads), tid = threadIdx.x;
    const int len = evict_len(a, seq), keep = min(len, a.keep);
    const float *weights = a.weights + block * a.weights_cols;
    int32_t *kept = a.kept + block * a.keep;
    float *new_weights = a.new_weights ? a.new_weights + block * a.keep : nullptr;
    const auto weight = [&](int t) { return t < a.weights_cols ? weights[t] : 0.f; };
    float held[kRound];
    const auto hold = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kRound; ++i) {
            const int t = t0 + tid * kRound + i;
            held[i] = t < len ? weight(t) : 0.f;
        }
    };
    if constexpr (kEach > 0) hold(0);
    if (head == 0 && tid == 0) a.new_lens[seq] = keep;
    for (int i = keep + tid; i < a.keep; i += kSelectThreads) {
        kept[i] = -1;
        if (new_weights) new_weights[i] = 0.f;
    }
    // candidates: tokens first .. last - 1, of which `want` stay; fewer than all of them, but where all tokens stay
    const bool all = len <= a.keep;
    const int first = all ? len : a.sinks, last = all ? len : len - a.recent;
    const uint32_t want = all ? 0 : static_cast<uint32_t>(a.keep - a.sinks - a.recent);
    const auto for_candidates = [&](const auto &f) {
        if constexpr (kEach > 0) {
#pragma unroll
            for (int i = 0; i < kRound; ++i) {
                const int t = tid * kRound + i;
                if (t >= first && t < last) f(rank_of(held[i]));
            }
        } else {
            for (int t = first + tid; t < last; t += kSelectThreads) f(rank_of(weight(t)));
        }
    };
    uint32_t prefix = 0, mask = 0, left = want;  // of the last kept one's rank: its bits so far; candidates still to come with them
    for (int shift = 21, step = 0; step < 3 && want > 0; ++step) {
        const int bits = step < 2 ? 11 : 10;
        for (int i = tid; i < 2048; i += kSelectThreads) bins[i] = 0;
        __syncthreads();
        for_candidates([&](uint32_t r) {
            if ((r & mask) == prefix) atomicAdd(&bins[(r >> shift) & ((1u << bits) - 1)], 1u);
        });
        __syncthreads();
        // bins from the top: lane tid has two of them
        const uint32_t hi = bins[2047 - 2 * tid], lo = bins[2046 - 2 * tid];
        uint2 total;
        const uint32_t before = sums_before<kWaves>(hi + lo, 0, waves, total).x;
        if (before < left && before + hi + lo >= left) {
            const bool in_hi = before + hi >= left;
            found[0] = static_cast<uint32_t>(2047 - 2 * tid - (in_hi ? 0 : 1));
            found[1] = left - before - (in_hi ? 0 : hi);
        }
        __syncthreads();
        prefix |= found[0] << shift, mask |= ((1u << bits) - 1) << shift, left = found[1];
        shift -= step == 0 ? 11 : 10;
    }
    // in order, kRound tokens a lane
    uint32_t above = 0, equal = 0;  // kept before these tokens, those of the last rank apart
    for (int t0 = 0; t0 < len; t0 += kSelectThreads * kRound) {
        if constexpr (kEach == 0) hold(t0);
        uint32_t sure = 0, tie = 0;  // bit masks
#pragma unroll
        for (int i = 0; i < kRound; ++i) {
            const int t = t0 + tid * kRound + i;
            const uint32_t r = rank_of(held[i]);
            const bool always = t < first || t >= last;
            if (t < len && (always || (want > 0 && r > prefix))) sure |= 1u << i;
            if (t < len && !always && want > 0 && r == prefix) tie |= 1u << i;
        }
        uint2 total;
        const uint2 before = sums_before<kWaves>(__popc(sure), __popc(tie), waves, total);
        uint32_t s = above + before.x, e = equal + before.y;
#pragma unroll
        for (int i = 0; i < kRound; ++i) {
            const bool is_tie = tie >> i & 1u, in = (sure >> i & 1u) || (is_tie && e < left);
            if (in) {
                const uint32_t to = s + min(e, left);
                kept[to] = t0 + tid * kRound + i;
                if (new_weights) new_weights[to] = held[i];
            }
            s += sure >> i & 1u, e += is_tie;
        }
        above += total.x, equal += total.y;
    }
}

// Moves the kept tokens: a workgroup the keys, or the values, of one head in one new page; 16 codes a lane.  The new page takes the
// greatest of its tokens' scales: their codes move as they are, others are rounded to it.  HBM: 32 sequences of up to 8000 tokens to 2048, with
// the selection and the read-back, 125 us, 5 TB/s.
template <int D>
__global__ __launch_bounds__(256) void kv8_move_kernel(EvictArgs8 a) {
    constexpr int kLanes = D / 16, kRows = 256 / kLanes, kMost = 256 / kRows;  // rounds of the largest page
    __shared__ float tops[4];
    const int64_t block = a.first_block + blockIdx.x;
    const int which = static_cast<int>(block % (2 * a.heads)), col = static_cast<int>(block / (2 * a.heads) % a.used_cols);
    const int seq = static_cast<int>(block / (2 * a.heads) / a.used_cols);
    const bool is_v = which >= a.heads;
    const int head = is_v ? which - a.heads : which, page = 1 << a.page_shift;
    const int count = min(min(evict_len(a, seq), a.keep) - col * page, page);
    if (count <= 0) return;
    const int to = a.new_table[static_cast<int64_t>(seq) * a.new_cols + col];
    if (to < 0 || to >= a.num_pages) return;
    uint8_t *codes = is_v ? a.v_codes : a.k_codes;
    float *scales = is_v ? a.v_scales : a.k_scales;
    const int32_t *kept = a.kept + (static_cast<int64_t>(seq) * a.heads + head) * a.keep + col * page;
    const int32_t *table = a.table + static_cast<int64_t>(seq) * a.table_cols;
    const int piece = threadIdx.x % kLanes, local = threadIdx.x / kLanes;
    uint4 w[kMost];
    float s[kMost], top = 0.f;
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int r = j * kRows + local;
        w[j] = uint4{}, s[j] = 0.f;
        if (r < count) {
            const int t = kept[r], p = table[t >> a.page_shift];
            if (p >= 0 && p < a.num_pages) {  // else zeros
                w[j] = load_once(codes + kv8_row(p, head, t & (page - 1), a.heads, a.page_shift) * D + 16 * piece);
                s[j] = scales[static_cast<int64_t>(p) * a.heads + head];
            }
            top = fmaxf(top, s[j]);
        }
    }
    top = wave_max<64>(top);
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (!(top > 0.f)) top = 1.f;  // no token's page is one of the cache's
    if (threadIdx.x == 0) scales[static_cast<int64_t>(to) * a.heads + head] = top;
    uint8_t *out = codes + kv8_row(to, head, 0, a.heads, a.page_shift) * D + 16 * piece;
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
        const int r = j * kRows + local;
        if (r < count) {
            if (s[j] != top) {
                const float ratio = s[j] / top;
                w[j] = make_uint4(e4m3x4_by(w[j].x, ratio), e4m3x4_by(w[j].y, ratio), e4m3x4_by(w[j].z, ratio), e4m3x4_by(w[j].w, ratio));
            }
            *reinterpret_cast<uint4 *>(out + r * D) = w[j];
        }
    }
}

// Heads a workgroup of the gather takes of a token: one round of its lanes where that leaves the card with less than four
// workgroups a CU, else more of them, for whom the slot is read once.
int share_of(int64_t tokens, int units, int lanes) {
    const int round = 256 / lanes, rounds = (units + round - 1) / round;
    const int64_t wanted = (4 * cu_count() + tokens - 1) / tokens;  // workgroups a token
    const int ways = static_cast<int>(std::min<int64_t>(rounds, wanted));
    return (rounds + ways - 1) / ways * round;
}

void check_rows8(const void *p, int64_t stride, int64_t heads, int64_t d, int64_t tokens, const char *what) {
    require(aligned(p, 16), std::string(what) + " must be 16-byte aligned");
    require(tokens <= 1 || (stride >= heads * d && stride % 8 == 0),
            std::string(what) + "'s token stride must be a multiple of 8 and at least heads * head_dim");
}

template <int D, int NP>
void launch_append(const AppendArgs8 &a, unsigned grid, hipStream_t st) {
    kv8_append_kernel<D, NP><<<dim3(grid), dim3(256), 0, st>>>(a);
}

}  // namespace
}  // namespace cfh

using namespace cfh;

extern "C" {

int32_t castforge_hip_kv8_append(const cfh_kv8_cache_t *cache, const uint16_t *k, int64_t k_stride, const uint16_t *v, int64_t v_stride,
                                 int64_t tokens, int64_t batch, const int32_t *cu_q, const int32_t *page_table, int64_t table_cols,
                                 const int32_t *kv_lens, const int64_t *positions, const float *cos, const float *sin, int64_t max_pos,
                                 int64_t rot, int32_t interleaved, const uint16_t *q, int64_t q_stride, int64_t q_heads, uint16_t *q_out,
                                 void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_kv8(cache);
        check_kv8_table(cache, batch, table_cols);
        require(tokens >= 0 && tokens <= 0x7fffffff, "tokens must be in [0, 2^31)");
        require(rot >= 0 && rot <= cache->head_dim && rot % 16 == 0, "rot must be a multiple of 16 and at most head_dim");
        require(interleaved == 0 || interleaved == 1, "interleaved must be 0 or 1");
        require((q != nullptr) == (q_out != nullptr), "q and q_out go together: both NULL or neither");
        require(q == nullptr || (q_heads >= 1 && q_heads <= 65536), "q_heads must be in [1, 65536]");
        require(cu_q != nullptr || tokens == batch, "without cu_q every sequence has one token: tokens must equal batch");
        if (tokens == 0 || batch == 0) return;
        require(k && v && kv_lens && (table_cols == 0 || page_table), "buffers must not be NULL");
        check_rows8(k, k_stride, cache->kv_heads, cache->head_dim, tokens, "k");
        check_rows8(v, v_stride, cache->kv_heads, cache->head_dim, tokens, "v");
        if (q) {
            check_rows8(q, q_stride, q_heads, cache->head_dim, tokens, "q");
            require(aligned(q_out, 16), "q_out must be 16-byte aligned");
        }
        require(rot == 0 || (positions && cos && sin && max_pos >= 1), "positions, cos and sin must be given for a rotation");
        require(rot == 0 || (aligned(cos, 16) && aligned(sin, 16)), "cos and sin must be 16-byte aligned");
        // pages that n tokens lie in: n at most, and n / page_size + 2
        const int64_t units = cu_q ? std::min(tokens, tokens / cache->page_size + 2 * batch) : batch;
        AppendArgs8 a{k, v, q, k_stride, v_stride, q_stride, cu_q, page_table, kv_lens, positions, cos, sin, q_out, max_pos,
                      static_cast<int>(tokens), static_cast<int>(batch), static_cast<int>(cache->kv_heads), q ? static_cast<int>(q_heads) : 0,
                      kv8_log2(cache->page_size), static_cast<int>(table_cols), static_cast<int>(cache->num_pages), static_cast<int>(rot),
                      interleaved, cache->k_codes, cache->v_codes, cache->k_scales, cache->v_scales, 0, units * 2 * cache->kv_heads};
        const int64_t blocks = a.kv_blocks + (q ? tokens : 0);
        const int rounds = static_cast<int>(std::max<int64_t>(1, cache->page_size * cache->head_dim / 2048));
        for (int64_t most = most_workgroups(256); a.first_block < blocks; a.first_block += most) {
            const unsigned grid = static_cast<unsigned>(std::min(blocks - a.first_block, most));
            const hipStream_t st = static_cast<hipStream_t>(stream);
            if (cache->head_dim == 64) {
                if (rounds == 1) launch_append<64, 1>(a, grid, st);
                else if (rounds == 2) launch_append<64, 2>(a, grid, st);
                else if (rounds == 4) launch_append<64, 4>(a, grid, st);
                else launch_append<64, 8>(a, grid, st);
            } else {
                if (rounds == 1) launch_append<128, 1>(a, grid, st);
                else if (rounds == 2) launch_append<128, 2>(a, grid, st);
                else if (rounds == 4) launch_append<128, 4>(a, grid, st);
                else if (rounds == 8) launch_append<128, 8>(a, grid, st);
                else launch_append<128, 16>(a, grid, st);
            }
            check_launch("kv8_append");
        }
    });
}

int32_t castforge_hip_kv8_gather(const cfh_kv8_cache_t *cache, const int64_t *slots, int64_t tokens, void *k_out, void *v_out,
                                 int32_t out_dtype, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_kv8(cache);
        require(tokens >= 0 && tokens <= 0x7fffffff, "tokens must be in [0, 2^31)");
        require(out_dtype == CFH_DTYPE_F32 || out_dtype == CFH_DTYPE_BF16, "out_dtype must be F32 or BF16");
        if (tokens == 0) return;
        require(slots && k_out && v_out, "buffers must not be NULL");
        require(aligned(k_out, 16) && aligned(v_out, 16), "k_out and v_out must be 16-byte aligned");
        const int units = static_cast<int>(2 * cache->kv_heads), share = share_of(tokens, units, static_cast<int>(cache->head_dim / 8));
        const int shares = (units + share - 1) / share;  // workgroups a token
        const int64_t row = cache->kv_heads * cache->head_dim * (out_dtype == CFH_DTYPE_BF16 ? 2 : 4);
        for (int64_t t = 0, most = most_workgroups(256) / shares; t < tokens; t += most) {
            const dim3 grid(static_cast<unsigned>(std::min(tokens - t, most)), shares);
            const auto launch = [&](auto kern) {
                kern<<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    cache->k_codes, cache->k_scales, cache->v_codes, cache->v_scales, slots + t, cache->num_pages * cache->page_size,
                    static_cast<int>(cache->kv_heads), kv8_log2(cache->page_size), static_cast<char *>(k_out) + t * row,
                    static_cast<char *>(v_out) + t * row, out_dtype == CFH_DTYPE_BF16, share);
            };
            cache->head_dim == 64 ? launch(kv8_gather_kernel<64>) : launch(kv8_gather_kernel<128>);
            check_launch("kv8_gather");
        }
    });
}

int32_t castforge_hip_kv8_evict(const cfh_kv8_cache_t *cache, const int32_t *page_table, int64_t table_cols, const int32_t *kv_lens, int64_t batch,
                                const float *weights, int64_t weights_cols, int64_t keep, int64_t sinks, int64_t recent, const int32_t *new_table,
                                int64_t new_cols, int32_t *kept, int32_t *new_lens, float *new_weights, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_kv8(cache);
        check_kv8_table(cache, batch, table_cols);
        require(weights_cols >= 0 && weights_cols <= 0x7fffffff, "weights_cols must be in [0, 2^31)");
        require(keep >= 1 && keep <= 0x7ffff000, "keep must be in [1, 2^31 - 4096]");
        require(sinks >= 0 && recent >= 0 && sinks <= keep && recent <= keep - sinks, "sinks and recent must not be negative, and at most keep together");
        require(new_cols >= 0 && new_cols <= 0x7ffff000 / cache->page_size && new_cols * cache->page_size >= keep, "new_table must have room for keep tokens");
        if (batch == 0) return;
        require(kv_lens && (table_cols == 0 || page_table) && (weights_cols == 0 || weights) && new_table && kept && new_lens, "buffers must not be NULL");
        EvictArgs8 a{cache->k_codes, cache->v_codes, cache->k_scales, cache->v_scales, page_table, kv_lens, new_table, weights, kept, new_lens, new_weights,
                     static_cast<int>(cache->kv_heads), kv8_log2(cache->page_size), static_cast<int>(table_cols), static_cast<int>(new_cols),
                     static_cast<int>(cache->num_pages), static_cast<int>(weights_cols), static_cast<int>(keep), static_cast<int>(sinks), static_cast<int>(recent),
                     static_cast<int>((keep + cache->page_size - 1) / cache->page_size), 0};
        const hipStream_t st = static_cast<hipStream_t>(stream);
        const auto launches = [&](int64_t blocks, int threads, const char *what, const auto &launch) {
            for (a.first_block = 0; a.first_block < blocks; a.first_block += most_workgroups(threads)) {
                launch(dim3(static_cast<unsigned>(std::min(blocks - a.first_block, most_workgroups(threads)))));
                check_launch(what);
            }
        };
        const int64_t most = table_cols * cache->page_size;  // tokens a sequence
        launches(batch * cache->kv_heads, kSelectThreads, "kv8_select", [&](dim3 grid) {
            const auto kern = most <= 4 * kSelectThreads ? kv8_select_kernel<4> : kv8_select_kernel<0>;
            kern<<<grid, dim3(kSelectThreads), 0, st>>>(a);
        });
        launches(batch * a.used_cols * 2 * cache->kv_heads, 256, "kv8_move", [&](dim3 grid) {
            const auto kern = cache->head_dim == 64 ? kv8_move_kernel<64> : kv8_move_kernel<128>;
            kern<<<grid, dim3(256), 0, st>>>(a);
        });
    });
}

}  // extern "C"
