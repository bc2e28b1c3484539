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
    int64_t tokens, capacity, max_pos;
    int heads, q_heads, page_shift, rot, interleaved;
    uint32_t *k_codes, *k_groups, *v_codes, *v_groups;
};

// Eight elements a lane, D / 8 lanes a head of a token; the heads of a token in the order K, V, Q.
template <int D, int G>
__global__ __launch_bounds__(256) void kv4_append_kernel(AppendArgs a) {
    constexpr int kLanes = D / 8;
    const int64_t per_token = 2 * a.heads + a.q_heads;
    const int64_t unit = (blockIdx.x * 256ll + threadIdx.x) / kLanes;
    const int piece = threadIdx.x % kLanes;  // 256 % kLanes == 0
    if (unit >= a.tokens * per_token) return;  // whole groups of kLanes lanes
    const int64_t token = unit / per_token;
    const int u = static_cast<int>(unit % per_token);
    const int kind = u < a.heads ? 0 : u < 2 * a.heads ? 1 : 2;  // K, V, Q
    const int head = u - (kind == 0 ? 0 : kind == 1 ? a.heads : 2 * a.heads);
    const uint16_t *src = kind == 0 ? a.k + token * a.k_stride : kind == 1 ? a.v + token * a.v_stride : a.q + token * a.q_stride;
    src += head * D;
    const auto load8 = [&](int p, float (&x)[8]) {
        const uint4 w = *reinterpret_cast<const uint4 *>(src + 8 * p);
        const uint32_t b[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(b[i] << 16), x[2 * i + 1] = __uint_as_float(b[i] & 0xffff0000u);
    };
    float x[8];
    load8(piece, x);
    if (kind != 1 && 8 * piece < a.rot) {
        // a position outside the table takes its nearest row
        const int64_t pos = min(max(a.positions[token], int64_t{0}), a.max_pos - 1);
        const int half = a.rot / 2;
        const float *c = a.cos + pos * half, *s = a.sin + pos * half;
        if (a.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float cc = c[4 * piece + i], ss = s[4 * piece + i], p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = p * cc - q * ss;
                x[2 * i + 1] = q * cc + p * ss;
            }
        } else {
            const bool low = 8 * piece < half;
            const int other = low ? piece + half / 8 : piece - half / 8;
            const int at = low ? 8 * piece : 8 * piece - half;
            float y[8];
            load8(other, y);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float cc = c[at + i], ss = s[at + i];
                x[i] = low ? x[i] * cc - y[i] * ss : x[i] * cc + y[i] * ss;
            }
        }
    }
    if (kind == 2) {
        uint4 w;
        w.x = f32x2_to_bf16x2_rne(x[0], x[1]), w.y = f32x2_to_bf16x2_rne(x[2], x[3]);
        w.z = f32x2_to_bf16x2_rne(x[4], x[5]), w.w = f32x2_to_bf16x2_rne(x[6], x[7]);
        *reinterpret_cast<uint4 *>(a.q_out + (token * a.q_heads + head) * D + 8 * piece) = w;
        return;
    }
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= a.capacity) return;  // whole groups of lanes: not appended
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
    lo = wave_min<G / 8>(lo);
    hi = wave_max<G / 8>(hi);
    const uint16_t h = group_scale_bits(hi, lo);
    const float scale = f16_to_f32(h);
    float z = rintf(-lo / scale);
    z = z != z ? 0.f : fminf(fmaxf(z, 0.f), 15.f);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float t = rintf(x[i] / scale);
        if (t != t) t = 0.f;
        word |= static_cast<uint32_t>(fminf(fmaxf(t + z, 0.f), 15.f)) << (4 * i);
    }
    const int64_t row = kv4_row(slot >> a.page_shift, head, static_cast<int>(slot & ((1 << a.page_shift) - 1)), a.heads, a.page_shift);
    (kind == 0 ? a.k_codes : a.v_codes)[row * kLanes + piece] = word;
    if (piece % (G / 8) == 0)
        (kind == 0 ? a.k_groups : a.v_groups)[row * (D / G) + piece / (G / 8)] = static_cast<uint32_t>(h) | (static_cast<uint32_t>(z) << 16);
}

// Rows of the cache as numbers, eight elements a lane; a slot outside the cache gives zeros.
template <int D, int G>
__global__ __launch_bounds__(256) void kv4_gather_kernel(const uint32_t *__restrict__ k_codes, const uint32_t *__restrict__ k_groups,
                                                         const uint32_t *__restrict__ v_codes, const uint32_t *__restrict__ v_groups,
                                                         const int64_t *__restrict__ slots, int64_t tokens, int64_t capacity, int heads,
                                                         int page_shift, void *__restrict__ k_out, void *__restrict__ v_out, int bf16) {
    constexpr int kLanes = D / 8;
    const int64_t unit = (blockIdx.x * 256ll + threadIdx.x) / kLanes;
    const int piece = threadIdx.x % kLanes;
    if (unit >= 2 * heads * tokens) return;
    const int64_t token = unit / (2 * heads);
    const int u = static_cast<int>(unit % (2 * heads)), head = u % heads;
    const bool is_v = u >= heads;
    const int64_t slot = slots[token];
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (slot >= 0 && slot < capacity) {
        const int64_t row = kv4_row(slot >> page_shift, head, static_cast<int>(slot & ((1 << page_shift) - 1)), heads, page_shift);
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
        *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(is_v ? v_out : k_out) + at) = w;
    } else {
        float4 *o = reinterpret_cast<float4 *>(static_cast<float *>(is_v ? v_out : k_out) + at);
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
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
        AppendArgs a{k, v, q, k_stride, v_stride, q_stride, slots, positions, cos, sin, q_out, tokens,
                     cache->num_pages * cache->page_size, max_pos, static_cast<int>(cache->kv_heads),
                     q ? static_cast<int>(q_heads) : 0, log2_of(cache->page_size), static_cast<int>(rot), interleaved,
                     cache->k_codes, cache->k_groups, cache->v_codes, cache->v_groups};
        const int64_t threads = tokens * (2 * a.heads + a.q_heads) * (cache->head_dim / 8), grid = (threads + 255) / 256;
        require(grid <= 0x7fffffff, "too many tokens for one launch");
        kv4_by_shape(cache, [&](auto d, auto g) {
            kv4_append_kernel<decltype(d)::value, decltype(g)::value><<<dim3(static_cast<unsigned>(grid)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(a);
        });
        check_launch("kv4_append");
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
        const int64_t grid = (tokens * 2 * cache->kv_heads * (cache->head_dim / 8) + 255) / 256;
        require(grid <= 0x7fffffff, "too many tokens for one launch");
        kv4_by_shape(cache, [&](auto d, auto g) {
            kv4_gather_kernel<decltype(d)::value, decltype(g)::value><<<dim3(static_cast<unsigned>(grid)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
                cache->k_codes, cache->k_groups, cache->v_codes, cache->v_groups, slots, tokens, cache->num_pages * cache->page_size,
                static_cast<int>(cache->kv_heads), log2_of(cache->page_size), k_out, v_out, out_dtype == CFH_DTYPE_BF16);
        });
        check_launch("kv4_gather");
    });
}

}  // extern "C"
