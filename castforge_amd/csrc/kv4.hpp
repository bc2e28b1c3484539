// The paged cache of 4-bit keys and values: what its kernels share.
//
// codes u32 [pages, heads, page, D / 8], element i of a row in bits 4 (i % 8) of word i / 8; one word a
// group of `group` elements, u32 [pages, heads, page, D / group]: the f16 scale in bits 0..15, the zero
// point in bits 16..19.  An element stands for (q - z) * scale.
#pragma once

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"

namespace cfh {

// A row's index (of D-element rows, over all pages and heads) from its page, head and place in the page.
__device__ __forceinline__ int64_t kv4_row(int64_t page, int head, int at, int heads, int page_shift) {
    return ((page * heads + head) << page_shift) + at;
}

__device__ __forceinline__ float kv4_scale(uint32_t word) { return f16_to_f32(static_cast<uint16_t>(word)); }
__device__ __forceinline__ uint32_t kv4_zero(uint32_t word) { return (word >> 16) & 15u; }

inline int log2_of(int64_t v) { return 63 - __builtin_clzll(static_cast<uint64_t>(v)); }

inline void check_kv4(const cfh_kv4_cache_t *c) {
    require(c != nullptr, "cache must not be NULL");
    require(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
    require((c->group == 32 || c->group == 64 || c->group == 128) && c->group <= c->head_dim,
            "group must be 32, 64 or 128 and at most head_dim");
    require(c->page_size >= 16 && c->page_size <= 4096 && (c->page_size & (c->page_size - 1)) == 0,
            "page_size must be a power of two in [16, 4096]");
    require(c->kv_heads >= 1 && c->kv_heads <= 1024, "kv_heads must be in [1, 1024]");
    require(c->num_pages >= 0 && c->num_pages <= 0x7fffffff, "num_pages must be in [0, 2^31)");
    require(c->num_pages == 0 || (c->k_codes && c->k_groups && c->v_codes && c->v_groups), "cache buffers must not be NULL");
    require(aligned(c->k_codes, 16) && aligned(c->v_codes, 16) && aligned(c->k_groups, 16) && aligned(c->v_groups, 16),
            "cache buffers must be 16-byte aligned");
}

// Calls f(D, G) with the head's channels and the group as compile-time constants.
template <class F>
void kv4_by_shape(const cfh_kv4_cache_t *c, F &&f) {
    const auto of = [&](auto d, auto g) { f(d, g); };
    if (c->head_dim == 64) {
        if (c->group == 32) of(std::integral_constant<int, 64>{}, std::integral_constant<int, 32>{});
        else of(std::integral_constant<int, 64>{}, std::integral_constant<int, 64>{});
    } else {
        if (c->group == 32) of(std::integral_constant<int, 128>{}, std::integral_constant<int, 32>{});
        else if (c->group == 64) of(std::integral_constant<int, 128>{}, std::integral_constant<int, 64>{});
        else of(std::integral_constant<int, 128>{}, std::integral_constant<int, 128>{});
    }
}

}  // namespace cfh
