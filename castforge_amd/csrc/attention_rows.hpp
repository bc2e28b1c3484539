// What the attention kernels over paged caches share: which rows a workgroup has, and small steps across a wave.
//
// Args of a kernel: tokens, batch, ratio (query heads a head of keys), page_shift, table_cols, num_pages, cu_q (NULL: one query a
// sequence) and kv_lens.
#pragma once

#include <atomic>

#include "cfh_common.hpp"

namespace cfh {

typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uintx4 __attribute__((ext_vector_type(4)));

constexpr float kNoMax = -3.402823466e38f;  // below every score, finite: exp2(-inf - kNoMax) is 0, not NaN

// A uniform word through the scalar cache: no vector load, whose wait would take in the tile loads before it.
template <class T>
__device__ __forceinline__ T scalar_load(const T *p, int64_t i) {
    return ((const __attribute__((address_space(4))) T *)(p))[i];
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
template <class Args>
__device__ __forceinline__ int token_cap(const Args &a) { return a.table_cols << a.page_shift; }

// Splits that share a sequence of len tokens: at least 128 tokens each.
__device__ __forceinline__ int splits_of(int len, int splits) { return max(1, min(splits, (len + 127) / 128)); }

// Which sequence's row tile a workgroup has: tiles are dealt to the sequences in order, rows_per_tile rows each.
// The lanes of a wave look at 64 sequences at once.  Returns seq -1 past the last tile.
template <class Args>
__device__ __forceinline__ Seq find_tile(const Args &a, int tile, int rows_per_tile) {
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

// LDS accesses of one wave keep their order; the compiler must not move them past each other either.
__device__ __forceinline__ void wave_order() { asm volatile("" ::: "memory"); }

// Raises a kernel's dynamic-LDS limit once per device (bit = device ordinal < 64).
inline void raise_lds_limit(const void *kern, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    check_hip(hipGetDevice(&dev), "hipGetDevice");
    const uint64_t bit = dev < 64 ? (uint64_t{1} << dev) : 0;
    if (bit == 0 || !(done.load(std::memory_order_acquire) & bit)) {
        check_hip(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "hipFuncSetAttribute(attention)");
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
}

}  // namespace cfh
