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

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"
#include "kv4.hpp"

namespace cfh {
namespace {

struct AttnArgs {
    const uint16_t *q;
    int64_t q_stride;
    const uint32_t *k_codes, *k_groups, *v_codes, *v_groups;
    const int32_t *cu_q;  // NULL: one query a sequence
    const int32_t *table, *kv_lens;
    uint16_t *out;
    float *lse;
    float scale;
    int tokens, batch, heads, ratio, page_shift, table_cols, num_pages, causal;
};

// One wave a (query, head): the plain order of the formula.
template <int D, int G>
__global__ __launch_bounds__(64) void kv4_attention_simple_kernel(AttnArgs a) {
    constexpr int E = D / 64;  // channels a lane
    const int lane = threadIdx.x, hq = a.heads * a.ratio;
    const int token = blockIdx.x / hq, head = blockIdx.x % hq, kvh = head / a.ratio;
    int seq = token, first = token, last = token + 1;
    if (a.cu_q) {
        seq = -1;
        for (int b = 0; b < a.batch; ++b) {
            const int s0 = a.cu_q[b], s1 = a.cu_q[b + 1];
            if (token >= s0 && token < s1) {
                seq = b, first = s0, last = s1;
                break;
            }
        }
        if (seq < 0) return;
    }
    const int len = min(max(a.kv_lens[seq], 0), a.table_cols << a.page_shift);
    const int seen = a.causal ? min(len, len - (last - first) + (token - first) + 1) : len;
    float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        q[e] = bf16_to_f32(a.q[token * a.q_stride + head * D + E * lane + e]) * a.scale;
        o[e] = 0.f;
    }
    for (int t = 0; t < seen; ++t) {
        const int page = a.table[static_cast<int64_t>(seq) * a.table_cols + (t >> a.page_shift)];
        if (page < 0 || page >= a.num_pages) continue;
        const int64_t row = kv4_row(page, kvh, t & ((1 << a.page_shift) - 1), a.heads, a.page_shift);
        const int at = E * lane;
        const auto value = [&](const uint32_t *codes, const uint32_t *groups, int e) {
            const uint32_t w = codes[row * (D / 8) + at / 8], g = groups[row * (D / G) + at / G];
            return static_cast<float>(static_cast<int>((w >> (4 * ((at + e) % 8))) & 15u) - static_cast<int>(kv4_zero(g))) * kv4_scale(g);
        };
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += q[e] * value(a.k_codes, a.k_groups, e);
        s = wave_sum<64>(s);
        const float mn = fmaxf(m, s), f = __expf(m - mn), p = __expf(s - mn);
        l = l * f + p;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * value(a.v_codes, a.v_groups, e);
        m = mn;
    }
    const int64_t at = (static_cast<int64_t>(token) * hq + head) * D + E * lane;
#pragma unroll
    for (int e = 0; e < E; ++e) a.out[at + e] = f32_to_bf16_rne(m > -INFINITY ? o[e] / l : 0.f);
    if (a.lse && lane == 0) a.lse[static_cast<int64_t>(token) * hq + head] = m > -INFINITY ? m + logf(l) : -INFINITY;
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
    });
}

int32_t castforge_hip_kv4_attention(const cfh_kv4_cache_t *cache, const uint16_t *q, int64_t q_stride, int64_t tokens,
                                    int64_t q_heads, int64_t batch, const int32_t *cu_q, const int32_t *page_table,
                                    int64_t table_cols, const int32_t *kv_lens, int32_t causal, float scale, uint16_t *out,
                                    float *lse, void *workspace, int64_t workspace_bytes, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_kv4(cache);
        require(tokens >= 0 && tokens <= 0x7fffffff && batch >= 0 && batch <= 0x7fffffff, "tokens and batch must be in [0, 2^31)");
        require(q_heads >= 1 && q_heads % cache->kv_heads == 0 && q_heads / cache->kv_heads <= 64,
                "q_heads must be a multiple of kv_heads, at most 64 of them a head of keys");
        require(table_cols >= 0 && table_cols <= 0x7fffffff / cache->page_size, "a sequence must be shorter than 2^31 tokens");
        require(causal == 0 || causal == 1, "causal must be 0 or 1");
        require(cu_q != nullptr || tokens == batch, "without cu_q every sequence has one query: tokens must equal batch");
        if (tokens == 0) return;
        require(q && out && (batch == 0 || kv_lens) && (batch == 0 || table_cols == 0 || page_table), "buffers must not be NULL");
        require(aligned(q, 16) && aligned(out, 16), "q and out must be 16-byte aligned");
        require(tokens <= 1 || (q_stride >= q_heads * cache->head_dim && q_stride % 8 == 0),
                "q's token stride must be a multiple of 8 and at least q_heads * head_dim");
        AttnArgs a{q, q_stride, cache->k_codes, cache->k_groups, cache->v_codes, cache->v_groups, cu_q, page_table, kv_lens, out, lse,
                   scale, static_cast<int>(tokens), static_cast<int>(batch), static_cast<int>(cache->kv_heads),
                   static_cast<int>(q_heads / cache->kv_heads), log2_of(cache->page_size), static_cast<int>(table_cols),
                   static_cast<int>(cache->num_pages), causal};
        require(tokens * q_heads <= 0x7fffffff, "too many queries for one launch");
        kv4_by_shape(cache, [&](auto d, auto g) {
            kv4_attention_simple_kernel<decltype(d)::value, decltype(g)::value><<<dim3(static_cast<unsigned>(tokens * q_heads)), dim3(64), 0, static_cast<hipStream_t>(stream)>>>(a);
        });
        check_launch("kv4_attention");
    });
}

}  // extern "C"
