// Appending keys and values to the paged 4-bit cache, with the position rotation on the way, and reading
// rows back.
//
// Rotation of a head's first `rot` channels by the angles of the token's position: pairs (i, i + rot / 2),
// or (2 i, 2 i + 1) where interleaved; (a, b) -> (a c - b s, b c + a s), each product and the difference
// rounded to f32 where it stands.  Keys go from the rotated f32 straight into codes; queries, rotated in the
// same launch, are rounded once to bf16.
//
// Codes of a group: lo = min(x, 0), hi = max(x, 0) (the range holds zero, so a group of one sign keeps its
// spread), scale = f16 of (hi - lo) * (1 / 15), z = clamp(rne(-lo / scale), 0, 15), q = clamp(rne(x / scale) + z,
// 0, 15), NaN -> z.
#include <algorithm>

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"
#include "kv4.hpp"

namespace cfh {
namespace {

// f16 bits of a group's scale: 1 for a range of (nearly) nothing, kept above zero and finite.
__device__ __forceinline__ uint16_t group_scale_bits(float hi, float lo) {
    const float range = hi - lo;
    float step = range * (1.0f / 15.0f);
    asm("" : "+v"(step));  // rounded to f32 before f16: one mixed-precision instruction would round once
    uint16_t h = range >= 1e-12f ? f32_to_f16_rne(step) : static_cast<uint16_t>(0x3C00);
    if (h == 0) h = 0x0001;
    if (h == 0x7C00) h = 0x7BFF;
    return h;
}

struct AppendArgs {
    const uint16_t *k, *v, *q;
    int64_t k_stride, v_stride, q_stride;  // elements from a token's row to the next one's
    const int64_t *slots, *positions;
    const float *cos, *sin;
    uint16_t *q_out;
    int64_t capacity, max_pos;
    int heads, q_heads, page_shift, rot, interleaved;
    uint32_t *k_codes, *k_groups, *v_codes, *v_groups;
};

// Least and greatest over G / 8 lanes of a DPP row.
template <int G>
__device__ __forceinline__ void range_of(float &lo, float &hi) {
    lo = fminf(lo, lane_xor<1>(lo)), hi = fmaxf(hi, lane_xor<1>(hi));
    lo = fminf(lo, lane_xor<2>(lo)), hi = fmaxf(hi, lane_xor<2>(hi));
    if constexpr (G >= 64) lo = fminf(lo, lane_xor<4>(lo)), hi = fmaxf(hi, lane_xor<4>(hi));
    if constexpr (G >= 128) lo = fminf(lo, lane_xor<8>(lo)), hi = fmaxf(hi, lane_xor<8>(hi));
}

// Eight codes of finite numbers whose range and scale are finite.  The quotient is RN(x / scale) from the reciprocal by two
// fmas; adding 1.5 * 2^23 rounds it to the nearest even integer and med3 clamps it to [-z, 15 - z]; four codes at a time
// become a 16-bit number in f32, exactly.  A tenth of a division and rint each.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float scale, float y, float z) {
    constexpr float kMagic = 12582912.f;
    const float lo = kMagic - z, hi = kMagic + 15.f - z;
    const auto code = [&](float v) {
        const float q0 = v * y;
        const float q = __builtin_fmaf(__builtin_fmaf(-q0, scale, v), y, q0);
        return __builtin_amdgcn_fmed3f(q + kMagic, lo, hi) - lo;
    };
    uint32_t half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
        half[h] = static_cast<uint32_t>(__builtin_fmaf(code(x[4 * h + 3]), 4096.f, __builtin_fmaf(code(x[4 * h + 2]), 256.f, __builtin_fmaf(code(x[4 * h + 1]), 16.f, code(x[4 * h])))));
    return half[0] | (half[1] << 16);
}

// Any numbers: NaN takes the zero point.
__device__ __forceinline__ uint32_t codes_of_any(const float (&x)[8], float scale, float z) {
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float t = rintf(x[i] / scale);
        if (t != t) t = 0.f;
        word |= static_cast<uint32_t>(fminf(fmaxf(t + z, 0.f), 15.f)) << (4 * i);
    }
    return word;
}

// A workgroup has one token (its slot, position and angles are read once) and up to `share` of its heads, in the order K, V, Q:
// eight elements a lane, D / 8 lanes a head.  HBM-bound where the tokens are many, its vector instructions about as busy: 4096 tokens of 32 heads
// of each kind, all in places of their own, move 152 MB, more with the cache's partial lines, in 32 to 34 us (4.5 to 4.7 TB/s);
// 16 tokens of 8 heads and 32 of the queries take 3.4 us.  Rows are read and queries written past the caches, which keep the cache's
// partial lines then: 68 -> 56 us with the read-back where outputs are new memory, 56 -> 54 where they are not.
template <int D, int G>
__global__ __launch_bounds__(256) void kv4_append_kernel(AppendArgs a, int share) {
    constexpr int kLanes = D / 8, kUnits = 256 / kLanes;
    const int64_t token = blockIdx.x;
    const int piece = threadIdx.x % kLanes, local = threadIdx.x / kLanes;
    const int64_t slot = a.slots[token];
    const bool kept = slot >= 0 && slot < a.capacity;
    const int64_t row0 = kv4_row(kept ? slot >> a.page_shift : 0, 0, static_cast<int>(slot & ((1 << a.page_shift) - 1)), a.heads, a.page_shift);
    const uint16_t *k = a.k + token * a.k_stride, *v = a.v + token * a.v_stride, *q = a.q_heads ? a.q + token * a.q_stride : nullptr;
    const int half = a.rot / 2;
    const bool turns = 8 * piece < a.rot, low = 8 * piece < half;
    const int other = a.interleaved ? piece : low ? piece + half / 8 : piece - half / 8;
    float c[8], t[8];  // cosines and sines of the lane's channels, the sine's sign taken in
    if (turns) {
        // a position outside the table takes its nearest row
        const int64_t pos = min(max(a.positions[token], int64_t{0}), a.max_pos - 1);
        const float *cp = a.cos + pos * half, *sp = a.sin + pos * half;
        if (a.interleaved) {
            const float4 cc = *reinterpret_cast<const float4 *>(cp + 4 * piece), ss = *reinterpret_cast<const float4 *>(sp + 4 * piece);
            c[0] = c[1] = cc.x, c[2] = c[3] = cc.y, c[4] = c[5] = cc.z, c[6] = c[7] = cc.w;
            t[0] = -ss.x, t[1] = ss.x, t[2] = -ss.y, t[3] = ss.y, t[4] = -ss.z, t[5] = ss.z, t[6] = -ss.w, t[7] = ss.w;
        } else {
            const int at = low ? 8 * piece : 8 * piece - half;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const float4 cc = reinterpret_cast<const float4 *>(cp + at)[h], ss = reinterpret_cast<const float4 *>(sp + at)[h];
                c[4 * h] = cc.x, c[4 * h + 1] = cc.y, c[4 * h + 2] = cc.z, c[4 * h + 3] = cc.w;
                t[4 * h] = low ? -ss.x : ss.x, t[4 * h + 1] = low ? -ss.y : ss.y, t[4 * h + 2] = low ? -ss.z : ss.z, t[4 * h + 3] = low ? -ss.w : ss.w;
            }
        }
    }
    const auto unpack = [](const uint4 &w, float (&x)[8]) {
        const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(b[i] << 16), x[2 * i + 1] = __uint_as_float(b[i] & 0xffff0000u);
    };
    const int units = 2 * a.heads + a.q_heads, end = min(units, static_cast<int>(blockIdx.y + 1) * share);
    const auto source = [&](int u) { return (u < a.heads ? k + u * D : u < 2 * a.heads ? v + (u - a.heads) * D : q + (u - 2 * a.heads) * D); };
    const auto load = [&](int u, uint4 (&w)[2]) {
        const uint16_t *src = source(u);
        w[0] = load_once(src + 8 * piece);
        if (turns && !a.interleaved && (u < a.heads || u >= 2 * a.heads)) w[1] = *reinterpret_cast<const uint4 *>(src + 8 * other);
    };
    int u = static_cast<int>(blockIdx.y) * share + local;
    uint4 w[2], ahead[2];
    if (u < end) load(u, ahead);
    for (; u < end; u += kUnits) {
        w[0] = ahead[0], w[1] = ahead[1];
        if (u + kUnits < end) load(u + kUnits, ahead);
        const bool is_v = u >= a.heads && u < 2 * a.heads;
        float x[8];
        unpack(w[0], x);
        if (turns && !is_v) {
            // (a, b) -> (a c - b s, b c + a s): x c + partner * (+- s), which rounds as the difference does
            float y[8];
            if (a.interleaved) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = x[i ^ 1];
            } else {
                unpack(w[1], y);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * c[i] + y[i] * t[i];
        }
        if (u >= 2 * a.heads) {
            uint4 o;
            o.x = f32x2_to_bf16x2_rne(x[0], x[1]), o.y = f32x2_to_bf16x2_rne(x[2], x[3]);
            o.z = f32x2_to_bf16x2_rne(x[4], x[5]), o.w = f32x2_to_bf16x2_rne(x[6], x[7]);
            store_past(a.q_out + (token * a.q_heads + u - 2 * a.heads) * D + 8 * piece, o);
            continue;
        }
        if (!kept) continue;
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
        // in a group's lanes alike: a NaN leaves the range, an infinity makes it infinite
        bool odd = __builtin_isunordered(x[0], x[1]) | __builtin_isunordered(x[2], x[3]) | __builtin_isunordered(x[4], x[5]) | __builtin_isunordered(x[6], x[7]);
        range_of<G>(lo, hi);
        odd |= !(hi - lo < INFINITY);
        const uint16_t h = group_scale_bits(hi, lo);
        const float scale = f16_to_f32(h), inv = 1.0f / scale;
        uint32_t word, zero;
        if (odd) {
            float z = rintf(-lo / scale);
            z = z != z ? 0.f : fminf(fmaxf(z, 0.f), 15.f);
            word = codes_of_any(x, scale, z), zero = static_cast<uint32_t>(z);
        } else {
            const float z0 = -lo * inv;
            const float z = __builtin_amdgcn_fmed3f(rintf(__builtin_fmaf(__builtin_fmaf(-z0, scale, -lo), inv, z0)), 0.f, 15.f);
            word = codes_of(x, scale, inv, z), zero = static_cast<uint32_t>(z);
        }
        const int head = is_v ? u - a.heads : u;
        const int64_t row = row0 + (static_cast<int64_t>(head) << a.page_shift);
        (is_v ? a.v_codes : a.k_codes)[row * kLanes + piece] = word;
        if (piece % (G / 8) == 0) (is_v ? a.v_groups : a.k_groups)[row * (D / G) + piece / (G / 8)] = static_cast<uint32_t>(h) | (zero << 16);
    }
}

// Rows of the cache as numbers, a workgroup a token, eight elements a lane; a slot outside the cache gives zeros.  HBM-bound: 4096
// tokens of 32 heads, 85 MB, in 21 us (4.1 TB/s).
template <int D, int G>
__global__ __launch_bounds__(256) void kv4_gather_kernel(const uint32_t *__restrict__ k_codes, const uint32_t *__restrict__ k_groups,
                                                         const uint32_t *__restrict__ v_codes, const uint32_t *__restrict__ v_groups,
                                                         const int64_t *__restrict__ slots, int64_t capacity, int heads, int page_shift,
                                                         void *__restrict__ k_out, void *__restrict__ v_out, int bf16, int share) {
    constexpr int kLanes = D / 8, kUnits = 256 / kLanes;
    const int64_t token = blockIdx.x, slot = slots[token];
    const bool kept = slot >= 0 && slot < capacity;
    const int piece = threadIdx.x % kLanes, end = min(2 * heads, static_cast<int>(blockIdx.y + 1) * share);
    const int64_t row0 = kv4_row(kept ? slot >> page_shift : 0, 0, static_cast<int>(slot & ((1 << page_shift) - 1)), heads, page_shift);
#pragma unroll 2
    for (int u = static_cast<int>(blockIdx.y) * share + static_cast<int>(threadIdx.x) / kLanes; u < end; u += kUnits) {
        const bool is_v = u >= heads;
        const int head = is_v ? u - heads : u;
        float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (kept) {
            const int64_t row = row0 + (static_cast<int64_t>(head) << page_shift);
            const uint32_t w = (is_v ? v_codes : k_codes)[row * kLanes + piece];
            const uint32_t g = (is_v ? v_groups : k_groups)[row * (D / G) + piece / (G / 8)];
            const float scale = kv4_scale(g);
            const int z = static_cast<int>(kv4_zero(g));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(static_cast<int>((w >> (4 * i)) & 15u) - z) * scale;
        }
        const int64_t at = (token * heads + head) * D + 8 * piece;
        if (bf16) {
            uint4 w;
            w.x = f32x2_to_bf16x2_rne(x[0], x[1]), w.y = f32x2_to_bf16x2_rne(x[2], x[3]);
            w.z = f32x2_to_bf16x2_rne(x[4], x[5]), w.w = f32x2_to_bf16x2_rne(x[6], x[7]);
            store_past(static_cast<uint16_t *>(is_v ? v_out : k_out) + at, w);
        } else {
            float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(is_v ? v_out : k_out) + at);
            o[0] = make_float4(x[0], x[1], x[2], x[3]);
            o[1] = make_float4(x[4], x[5], x[6], x[7]);
        }
    }
}

// Heads a workgroup takes of a token: one round of its lanes where that leaves the card with less than four workgroups a CU, else
// more of them, for whom the angles and the slot are read once.  16 tokens of 96 heads: 3.3 us, as one workgroup a token 6.2; 4096
// of them: 32 us, by one round a workgroup 42.
int share_of(int64_t tokens, int units, int lanes) {
    const int round = 256 / lanes, rounds = (units + round - 1) / round;
    const int64_t wanted = (4 * cu_count() + tokens - 1) / tokens;  // workgroups a token
    const int ways = static_cast<int>(std::min<int64_t>(rounds, wanted));
    return (rounds + ways - 1) / ways * round;
}

void check_rows(const void *p, int64_t stride, int64_t heads, int64_t d, int64_t tokens, const char *what) {
    require(aligned(p, 16), std::string(what) + " must be 16-byte aligned");
    require(tokens <= 1 || (stride >= heads * d && stride % 8 == 0),
            std::string(what) + "'s token stride must be a multiple of 8 and at least heads * head_dim");
}

}  // namespace
}  // namespace cfh

using namespace cfh;

extern "C" {

int32_t castforge_hip_kv4_append(const cfh_kv4_cache_t *cache, const uint16_t *k, int64_t k_stride, const uint16_t *v,
                                 int64_t v_stride, int64_t tokens, const int64_t *slots, const int64_t *positions,
                                 const float *cos, const float *sin, int64_t max_pos, int64_t rot, int32_t interleaved,
                                 const uint16_t *q, int64_t q_stride, int64_t q_heads, uint16_t *q_out, void *stream,
                                 char **out_error) {
    return guarded(out_error, [&] {
        check_kv4(cache);
        require(tokens >= 0 && tokens <= 0x7fffffff, "tokens must be in [0, 2^31)");
        require(rot >= 0 && rot <= cache->head_dim && rot % 16 == 0, "rot must be a multiple of 16 and at most head_dim");
        require(interleaved == 0 || interleaved == 1, "interleaved must be 0 or 1");
        require((q != nullptr) == (q_out != nullptr), "q and q_out go together: both NULL or neither");
        require(q == nullptr || (q_heads >= 1 && q_heads <= 65536), "q_heads must be in [1, 65536]");
        if (tokens == 0) return;
        require(k && v && slots, "buffers must not be NULL");
        check_rows(k, k_stride, cache->kv_heads, cache->head_dim, tokens, "k");
        check_rows(v, v_stride, cache->kv_heads, cache->head_dim, tokens, "v");
        if (q) {
            check_rows(q, q_stride, q_heads, cache->head_dim, tokens, "q");
            require(aligned(q_out, 16), "q_out must be 16-byte aligned");
        }
        require(rot == 0 || (positions && cos && sin && max_pos >= 1), "positions, cos and sin must be given for a rotation");
        require(rot == 0 || (aligned(cos, 16) && aligned(sin, 16)), "cos and sin must be 16-byte aligned");
        const int units = static_cast<int>(2 * cache->kv_heads + (q ? q_heads : 0)), share = share_of(tokens, units, static_cast<int>(cache->head_dim / 8));
        const int shares = (units + share - 1) / share;  // workgroups a token
        for (int64_t t = 0, most = most_workgroups(256) / shares; t < tokens; t += most) {
            const AppendArgs a{k + t * k_stride, v + t * v_stride, q ? q + t * q_stride : nullptr, k_stride, v_stride, q_stride, slots + t,
                               rot ? positions + t : nullptr, cos, sin, q ? q_out + t * q_heads * cache->head_dim : nullptr,
                               cache->num_pages * cache->page_size, max_pos, static_cast<int>(cache->kv_heads),
                               q ? static_cast<int>(q_heads) : 0, log2_of(cache->page_size), static_cast<int>(rot), interleaved,
                               cache->k_codes, cache->k_groups, cache->v_codes, cache->v_groups};
            const dim3 grid(static_cast<unsigned>(std::min(tokens - t, most)), shares);
            kv4_by_shape(cache, [&](auto d, auto g) {
                kv4_append_kernel<decltype(d)::value, decltype(g)::value><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a, share);
            });
            check_launch("kv4_append");
        }
    });
}

int32_t castforge_hip_kv4_gather(const cfh_kv4_cache_t *cache, const int64_t *slots, int64_t tokens, void *k_out, void *v_out,
                                 int32_t out_dtype, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_kv4(cache);
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
            kv4_by_shape(cache, [&](auto d, auto g) {
                kv4_gather_kernel<decltype(d)::value, decltype(g)::value><<<grid, dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                    cache->k_codes, cache->k_groups, cache->v_codes, cache->v_groups, slots + t, cache->num_pages * cache->page_size,
                    static_cast<int>(cache->kv_heads), log2_of(cache->page_size), static_cast<char *>(k_out) + t * row,
                    static_cast<char *>(v_out) + t * row, out_dtype == CFH_DTYPE_BF16, share);
            });
            check_launch("kv4_gather");
        }
    });
}

}  // extern "C"
