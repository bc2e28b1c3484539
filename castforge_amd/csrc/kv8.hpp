// The paged cache of 8-bit keys and values: what its kernels share.
//
// codes u8 [pages, heads, page, D], E4M3FN; scales f32 [pages, heads], one a page and head.  An element stands for
// code * scale.  Append makes scales powers of two, 2^-70 to 2^30: an element then takes a new scale without a
// second rounding (but below 2^-6 of the codes' unit), and products with it are exact.
#pragma once

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"

namespace cfh {

typedef float floatx2 __attribute__((ext_vector_type(2)));

constexpr int kKv8LeastExponent = -70, kKv8GreatestExponent = 30;

// A row's index (of D-element rows, over all pages and heads) from its page, head and place in the page.
__device__ __forceinline__ int64_t kv8_row(int64_t page, int head, int at, int heads, int page_shift) {
    return ((page * heads + head) << page_shift) + at;
}

// The least power of two, within the bounds above, that brings amax (not negative, not NaN) to 448 or less:
// 448 = 1.75 * 2^8, so a mantissa above 1.75 takes the next one.
__device__ __forceinline__ float kv8_scale_of(float amax) {
    const int e = static_cast<int>((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
    return __builtin_ldexpf(1.0f, min(max(e, kKv8LeastExponent), kKv8GreatestExponent));
}

// Four codes as numbers.
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t w, float *x) {
    const floatx2 a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}

// Four numbers of at most 448 as codes, to the nearest even one.
__device__ __forceinline__ uint32_t f32_to_e4m3x4(const float *x) {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true));
}

// Four codes of one scale as those of another, ratio (at most 1) the one by the other.
__device__ __forceinline__ uint32_t e4m3x4_by(uint32_t w, float ratio) {
    float x[4];
    e4m3x4_to_f32(w, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] *= ratio;
    return f32_to_e4m3x4(x);
}

inline int kv8_log2(int64_t v) { return 63 - __builtin_clzll(static_cast<uint64_t>(v)); }

inline void check_kv8(const cfh_kv8_cache_t *c) {
    require(c != nullptr, "cache must not be NULL");
    require(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
    require(c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0,
            "page_size must be a power of two in [16, 256]");
    require(c->kv_heads >= 1 && c->kv_heads <= 1024, "kv_heads must be in [1, 1024]");
    require(c->num_pages >= 0 && c->num_pages <= 0x7fffffff, "num_pages must be in [0, 2^31)");
    require(c->num_pages == 0 || (c->k_codes && c->k_scales && c->v_codes && c->v_scales), "cache buffers must not be NULL");
    require(aligned(c->k_codes, 16) && aligned(c->v_codes, 16), "codes must be 16-byte aligned");
    require(aligned(c->k_scales, 4) && aligned(c->v_scales, 4), "scales must be 4-byte aligned");
}

// A batch's table: 2^31 - 4096 tokens a sequence at most, so that a round of a workgroup's tokens past a length does not wrap.
inline void check_kv8_table(const cfh_kv8_cache_t *c, int64_t batch, int64_t table_cols) {
    require(batch >= 0 && batch <= 0x7fffffff, "batch must be in [0, 2^31)");
    require(table_cols >= 0 && table_cols <= 0x7ffff000 / c->page_size, "a sequence's table must hold at most 2^31 - 4096 tokens");
}

}  // namespace cfh
