// 8-bit product with a scale per block of 128 for gfx950:
//   Y[m, n] = sum_b sa[m, b] sw[n / 128, b] sum_{k in block b} A[m, k] W[n, k]
//
// A: E4M3 [M, K], a scale per row and run of 128 columns (sa [M, ceil(K / 128)]); W: E4M3 [N, K], a
// scale per 128 x 128 (sw [ceil(N / 128), ceil(K / 128)]); both K-contiguous.
#include <algorithm>
#include <atomic>

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"

namespace cfh {
namespace {

constexpr int kRun = 128;

// Any shape: one thread per output, exact E4M3 decode, f32 sums.
__global__ __launch_bounds__(256) void fp8_block_gemm_generic_kernel(const uint8_t *__restrict__ A, const float *__restrict__ sa,
                                                                     const uint8_t *__restrict__ W, const float *__restrict__ sw,
                                                                     void *__restrict__ Y, int y_bf16, int64_t M, int64_t N, int64_t K) {
    const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (idx >= M * N) return;
    const int64_t m = idx / N, n = idx - m * N, runs = (K + kRun - 1) / kRun;
    float acc = 0.f;
    for (int64_t b = 0; b < runs; ++b) {
        const int64_t end = min(K, (b + 1) * kRun);
        float part = 0.f;
        for (int64_t k = b * kRun; k < end; ++k) part += e4m3fn_to_f32(A[m * K + k]) * e4m3fn_to_f32(W[n * K + k]);
        acc += part * (sa[m * runs + b] * sw[n / kRun * runs + b]);
    }
    if (y_bf16) static_cast<uint16_t *>(Y)[idx] = f32_to_bf16_rne(acc);
    else static_cast<float *>(Y)[idx] = acc;
}

}  // namespace
}  // namespace cfh

using namespace cfh;

extern "C" int32_t castforge_hip_gemm_fp8_block(const uint8_t *qa, const float *sa, int64_t m, const uint8_t *qw, const float *sw,
                                                int64_t n, int64_t k, void *y, int32_t y_dtype, int32_t exact, void *stream,
                                                char **out_error) {
    return guarded(out_error, [&] {
        require(m >= 0 && n >= 0 && k >= 0, "m, n, k must be non-negative");
        require(y_dtype == CFH_DTYPE_F32 || y_dtype == CFH_DTYPE_BF16, "y_dtype must be F32 or BF16");
        require(exact == 0 || exact == 1, "exact must be 0 or 1");
        if (m == 0 || n == 0) return;
        require(y != nullptr && (k == 0 || (qa && sa && qw && sw)), "buffers must not be NULL");
        require(m <= 0x7fffffff && n <= 0x7fffffff && k <= 0x7fffffff, "dimensions must fit in int32");
        hipStream_t st = static_cast<hipStream_t>(stream);
        const int yb = y_dtype == CFH_DTYPE_BF16;
        const int64_t tot = m * n;
        require((tot + 255) / 256 <= 0x7fffffff, "shape too large for the generic FP8 kernel");
        fp8_block_gemm_generic_kernel<<<dim3(static_cast<unsigned>((tot + 255) / 256)), dim3(256), 0, st>>>(qa, sa, qw, sw, y, yb, m, n, k);
        check_launch("fp8_block_gemm_generic");
    });
}
