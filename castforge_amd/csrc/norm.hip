// RMS norm with the residual's addition and an E4M3 output, and E4M3 quantization in blocks of 128:
// what makes the left operand of the 8-bit products.
//
//   h = x + r, rounded once to x's type (the new residual stream);
//   y = h / sqrt(mean(h^2) + eps) * w, in f32;
//   codes = E4M3(y / s), to the nearest even; s = absmax(y) < 1e-12 ? 1 : absmax(y) * (1 / 448) over the
//   row (block 0) or over each run of 128 columns.
//
// The codec is v_cvt_pk_fp8_f32 as it is: |y / s| <= 448.0001, inside the range that it rounds to +-448.  (The
// reference's codec, which castforge_hip_quantize_fp8 keeps bit for bit, gives the code after the right one
// for 32 numbers just below powers of two.  With bf16 inputs and this scale such quotients are common: 4 / 7 of
// an absmax is one.)
//
// The sum of squares and y stay in f32; h alone is rounded to 16 bits, because later layers read it
// so, and the norm is of the rounded h.
#include <algorithm>

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"

namespace cfh {
namespace {

constexpr int kRun = 128;  // columns that share a scale

// The scale of a block: one product with the rounded reciprocal (within an ulp of the quotient).
__device__ __forceinline__ float scale_of(float amax) { return amax < 1e-12f ? 1.0f : amax * (1.0f / 448.0f); }

// What a block's values are divided by: the quotient RN(v / s) from y = RN(1 / s) by two fmas (q0 is
// within an ulp of v / s and the remainder exact).  An infinite s (a block that holds an infinity) becomes
// 0 and 0, which gives v / inf = 0 and NaN for the infinity itself.
struct Quot {
    float s, y;
    __device__ __forceinline__ explicit Quot(float scale) : s(scale < INFINITY ? scale : 0.f), y(scale < INFINITY ? 1.0f / scale : 0.f) {}
    __device__ __forceinline__ float operator()(float v) const {
        const float q0 = v * y;
        return __builtin_fmaf(-__builtin_fmaf(q0, s, -v), y, q0);
    }
};

// E4M3 codes of four quotients (byte i = value i).
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true));
}

__device__ __forceinline__ float load_elem(const void *p, int bf16, int64_t i) {
    return bf16 ? bf16_to_f32(static_cast<const uint16_t *>(p)[i]) : static_cast<const float *>(p)[i];
}

// Any row length and alignment: one workgroup a row, three passes over it.
__global__ __launch_bounds__(256) void rms_norm_fp8_generic_kernel(const void *x, const void *r, int x_bf16,
                                                                   const void *__restrict__ w, int w_bf16, float eps,
                                                                   int64_t cols, int block, void *h, uint8_t *__restrict__ codes,
                                                                   float *__restrict__ scales) {
    __shared__ float red[4];
    const int64_t row = blockIdx.x, base = row * cols;
    const int tid = threadIdx.x;
    const auto elem = [&](int64_t i) {  // h of one column
        float v = load_elem(x, x_bf16, base + i);
        if (r) {
            v += load_elem(r, x_bf16, base + i);
            if (x_bf16) v = bf16_to_f32(f32_to_bf16_rne(v));
        }
        return v;
    };
    const auto over_block = [&](float v, bool sum) {
        v = sum ? wave_sum<64>(v) : wave_max<64>(v);
        __syncthreads();
        if ((tid & 63) == 0) red[tid >> 6] = v;
        __syncthreads();
        return sum ? red[0] + red[1] + red[2] + red[3] : fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    };
    float ss = 0.f;
    for (int64_t i = tid; i < cols; i += 256) {
        const float v = elem(i);
        ss += v * v;
    }
    const float rstd = 1.0f / sqrtf(over_block(ss, true) / static_cast<float>(cols) + eps);
    const auto y = [&](int64_t i) { return elem(i) * rstd * load_elem(w, w_bf16, i); };
    const int64_t run = block ? block : cols, runs = (cols + run - 1) / run;
    for (int64_t g = 0; g < runs; ++g) {
        const int64_t end = min(cols, (g + 1) * run);
        float am = 0.f;
        for (int64_t i = g * run + tid; i < end; i += 256) am = fmaxf(am, fabsf(y(i)));
        const float scale = scale_of(over_block(am, false));
        const Quot quot(scale);
        for (int64_t i = g * run + tid; i < end; i += 256) codes[base + i] = static_cast<uint8_t>(e4m3x4(quot(y(i)), 0.f, 0.f, 0.f));
        if (tid == 0) scales[row * runs + g] = scale;
    }
    if (!r) return;
    __syncthreads();  // h may be x or r: written after the last read
    for (int64_t i = tid; i < cols; i += 256) {
        const float v = elem(i);
        if (x_bf16) static_cast<uint16_t *>(h)[base + i] = f32_to_bf16_rne(v);
        else static_cast<float *>(h)[base + i] = v;
    }
}

// E4M3 codes and scales of blocks of block_rows x 128: one workgroup a block, two passes.
__global__ __launch_bounds__(256) void quant_fp8_block_generic_kernel(const void *__restrict__ src, int bf16, int64_t rows,
                                                                      int64_t cols, int block_rows, uint8_t *__restrict__ codes,
                                                                      float *__restrict__ scales) {
    __shared__ float red[4];
    const int64_t runs = (cols + kRun - 1) / kRun;
    const int64_t br = blockIdx.x / runs, g = blockIdx.x % runs;
    const int64_t r0 = br * block_rows, c0 = g * kRun;
    const int n_rows = static_cast<int>(min(static_cast<int64_t>(block_rows), rows - r0));
    const int n_cols = static_cast<int>(min(static_cast<int64_t>(kRun), cols - c0));
    const int c = threadIdx.x % kRun;
    float am = 0.f;
    for (int i = threadIdx.x / kRun; i < n_rows; i += 256 / kRun)
        if (c < n_cols) am = fmaxf(am, fabsf(load_elem(src, bf16, (r0 + i) * cols + c0 + c)));
    am = wave_max<64>(am);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = am;
    __syncthreads();
    const float scale = scale_of(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const Quot quot(scale);
    for (int i = threadIdx.x / kRun; i < n_rows; i += 256 / kRun)
        if (c < n_cols) codes[(r0 + i) * cols + c0 + c] = static_cast<uint8_t>(e4m3x4(quot(load_elem(src, bf16, (r0 + i) * cols + c0 + c)), 0.f, 0.f, 0.f));
    if (threadIdx.x == 0) scales[blockIdx.x] = scale;
}

__global__ __launch_bounds__(256) void dequant_fp8_block_kernel(const uint8_t *__restrict__ codes, const float *__restrict__ scales,
                                                                int64_t rows, int64_t cols, int block_rows, float *__restrict__ out) {
    const int64_t n = rows * cols, runs = (cols + kRun - 1) / kRun;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
        out[i] = e4m3fn_to_f32(codes[i]) * scales[i / cols / block_rows * runs + i % cols / kRun];
}

void check_dtype(int32_t d, const char *what) {
    require(d == CFH_DTYPE_F32 || d == CFH_DTYPE_BF16, std::string(what) + " must be CFH_DTYPE_F32 or CFH_DTYPE_BF16");
}

void check_rows_cols(int64_t rows, int64_t cols) {
    require(rows >= 0 && cols >= 0, "rows and cols must be non-negative");
    require(cols == 0 || rows <= INT64_MAX / 8 / cols, "rows * cols must fit in int64");
}

}  // namespace
}  // namespace cfh

using namespace cfh;

extern "C" {

int32_t castforge_hip_rms_norm_fp8(const void *x, int32_t x_dtype, const void *residual, const void *weight,
                                   int32_t weight_dtype, float eps, int64_t rows, int64_t cols, int32_t block, void *h,
                                   uint8_t *codes, float *scales, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_rows_cols(rows, cols);
        check_dtype(x_dtype, "x_dtype");
        check_dtype(weight_dtype, "weight_dtype");
        require(block == 0 || block == kRun, "block must be 0 (a scale per row) or 128");
        require(eps >= 0.f, "eps must be non-negative");
        require((residual != nullptr) == (h != nullptr), "residual and h go together: both NULL or neither");
        if (rows == 0 || cols == 0) return;
        require(x && weight && codes && scales, "buffers must not be NULL");
        require(rows <= 0x7fffffff, "too many rows for one launch");
        hipStream_t st = static_cast<hipStream_t>(stream);
        rms_norm_fp8_generic_kernel<<<dim3(static_cast<unsigned>(rows)), dim3(256), 0, st>>>(
            x, residual, x_dtype == CFH_DTYPE_BF16, weight, weight_dtype == CFH_DTYPE_BF16, eps, cols, block, h, codes, scales);
        check_launch("rms_norm_fp8");
    });
}

int32_t castforge_hip_quantize_fp8_block(const void *src, int32_t src_dtype, int64_t rows, int64_t cols, int32_t block_rows,
                                         uint8_t *codes, float *scales, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_rows_cols(rows, cols);
        check_dtype(src_dtype, "src_dtype");
        require(block_rows == 1 || block_rows == kRun, "block_rows must be 1 or 128");
        if (rows == 0 || cols == 0) return;
        require(src && codes && scales, "buffers must not be NULL");
        const int64_t blocks = ((rows + block_rows - 1) / block_rows) * ((cols + kRun - 1) / kRun);
        require(blocks <= 0x7fffffff, "too many blocks for one launch");
        quant_fp8_block_generic_kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
            src, src_dtype == CFH_DTYPE_BF16, rows, cols, block_rows, codes, scales);
        check_launch("quant_fp8_block");
    });
}

int32_t castforge_hip_dequantize_fp8_block(const uint8_t *codes, const float *scales, int64_t rows, int64_t cols,
                                           int32_t block_rows, float *out, void *stream, char **out_error) {
    return guarded(out_error, [&] {
        check_rows_cols(rows, cols);
        require(block_rows == 1 || block_rows == kRun, "block_rows must be 1 or 128");
        if (rows == 0 || cols == 0) return;
        require(codes && scales && out, "buffers must not be NULL");
        const unsigned grid = static_cast<unsigned>(std::min<int64_t>((rows * cols + 255) / 256, 16 * cu_count()));
        dequant_fp8_block_kernel<<<dim3(grid), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(codes, scales, rows, cols,
                                                                                               block_rows, out);
        check_launch("dequant_fp8_block");
    });
}

}  // extern "C"
