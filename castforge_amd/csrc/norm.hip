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

// Eight consecutive elements, kept as they are stored.  `at`: the first one's index; rows of any length start at any element, so
// the addresses are only as aligned as an element (global accesses of up to 16 bytes may be).
template <bool kBf16>
struct Piece {
    typedef typename std::conditional<kBf16, uint16_t, float>::type elem;
    elem e[8];
    __device__ __forceinline__ void load(const void *p, int64_t at) { __builtin_memcpy(e, static_cast<const elem *>(p) + at, sizeof e); }
    // past the caches
    __device__ __forceinline__ void load_once(const void *p, int64_t at) {
        typedef nt_uint4 any __attribute__((aligned(2)));
        const any *src = reinterpret_cast<const any *>(static_cast<const elem *>(p) + at);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof e) / 16; ++i) {
            const nt_uint4 v = __builtin_nontemporal_load(src + i);
            __builtin_memcpy(reinterpret_cast<char *>(e) + 16 * i, &v, 16);
        }
    }
    __device__ __forceinline__ void store(void *p, int64_t at) const { __builtin_memcpy(static_cast<elem *>(p) + at, e, sizeof e); }
    // the first n elements alone, zeros behind them
    __device__ __forceinline__ void load_first(const void *p, int64_t at, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = i < n ? static_cast<const elem *>(p)[at + i] : elem(0);
    }
    __device__ __forceinline__ void store_first(void *p, int64_t at, int n) const {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) static_cast<elem *>(p)[at + i] = e[i];
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
        if constexpr (kBf16) {
            uint32_t b[4];
            __builtin_memcpy(b, e, 16);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(b[i] << 16), v[2 * i + 1] = __uint_as_float(b[i] & 0xffff0000u);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = e[i];
        }
    }
    __device__ __forceinline__ void set(const float (&v)[8]) {
        if constexpr (kBf16) {
            uint32_t b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = f32x2_to_bf16x2_rne(v[2 * i], v[2 * i + 1]);
            __builtin_memcpy(e, b, 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e[i] = v[i];
        }
    }
};

// Piece p of a row of `cols` that starts at element `base`: pieces past the end repeat the last whole one (an index clamp, not a
// branch: a load under a divergent branch waits for itself); a last, cut piece is read element by element.  cols >= 8.
template <bool kCut, bool kOnce = false, class P>
__device__ __forceinline__ void load_piece(P &x, const void *src, int64_t base, int p, int cols) {
    const int whole = cols / 8;
    if constexpr (kOnce) x.load_once(src, base + 8 * min(p, whole - 1));
    else x.load(src, base + 8 * min(p, whole - 1));
    if (kCut && p == whole && cols % 8) x.load_first(src, base + 8 * p, cols % 8);
}
template <bool kCut, class P>
__device__ __forceinline__ void store_piece(const P &x, void *dst, int64_t base, int p, int cols) {
    if (8 * p + 8 <= cols) x.store(dst, base + 8 * p);
    else if (kCut && 8 * p < cols) x.store_first(dst, base + 8 * p, cols - 8 * p);
}
template <bool kCut>
__device__ __forceinline__ void store_codes(uint2 c, uint8_t *dst, int64_t base, int p, int cols) {
    if (8 * p + 8 <= cols) {
        __builtin_memcpy(dst + base + 8 * p, &c, 8);
    } else if (kCut && 8 * p < cols) {
        for (int i = 0; i < cols - 8 * p; ++i) dst[base + 8 * p + i] = static_cast<uint8_t>((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    }
}

__device__ __forceinline__ float amax8(const float (&v)[8]) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
    return m;
}

__device__ __forceinline__ uint2 codes8(const Quot &quot, const float (&v)[8]) {
    return make_uint2(e4m3x4(quot(v[0]), quot(v[1]), quot(v[2]), quot(v[3])), e4m3x4(quot(v[4]), quot(v[5]), quot(v[6]), quot(v[7])));
}

// Maximum over the 16 lanes of a DPP row: what holds a run of 128 at eight elements a lane.
__device__ __forceinline__ float max16(float v) {
    v = fmaxf(v, lane_xor<1>(v));
    v = fmaxf(v, lane_xor<2>(v));
    v = fmaxf(v, lane_xor<4>(v));
    return fmaxf(v, lane_xor<8>(v));
}

// The norm with a row in registers, so that HBM sees each byte once: TPR threads a row (64: four rows a
// workgroup and no barrier), VPT pieces of eight elements a thread.  Threads past the row's end stay out of the sum and the
// maximum (where h is x, the piece that they repeat may have been written by then) and store nothing.
// HBM-bound: 7 bytes an element with a bf16 residual, 4096 x 4096 in 20.0 us (5.9 TB/s).
// kCut: rows that are no multiple of eight; their pieces are not aligned either.
template <bool kXBf16, bool kWBf16, bool kCut, int VPT, int TPR>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_fp8_kernel(const void *x, const void *r, const void *__restrict__ w, float eps,
                                                                             int64_t rows, int cols, int block, void *h, uint8_t *__restrict__ codes,
                                                                             float *__restrict__ scales) {
    constexpr int kWaves = TPR / 64;
    __shared__ float red[2][kWaves];
    const int t = threadIdx.x % TPR;
    const int64_t row = TPR == 64 ? blockIdx.x * 4ll + threadIdx.x / 64 : blockIdx.x;
    if (TPR == 64 && row >= rows) return;  // whole waves, which share nothing
    const int64_t base = row * cols;
    const auto over_row = [&](float v, bool sum, int which) {
        v = sum ? wave_sum<64>(v) : wave_max<64>(v);
        if constexpr (kWaves > 1) {
            if ((threadIdx.x & 63) == 0) red[which][threadIdx.x >> 6] = v;
            __syncthreads();
            v = red[which][0];
#pragma unroll
            for (int i = 1; i < kWaves; ++i) v = sum ? v + red[which][i] : fmaxf(v, red[which][i]);
        }
        return v;
    };
    Piece<kXBf16> px[VPT], pr[VPT];
    Piece<kWBf16> pw[VPT];
    static_for<VPT>([&](auto i) __attribute__((always_inline)) { load_piece<kCut>(px[i], x, base, t + i * TPR, cols); });
    if (r) static_for<VPT>([&](auto i) __attribute__((always_inline)) { load_piece<kCut>(pr[i], r, base, t + i * TPR, cols); });
    static_for<VPT>([&](auto i) __attribute__((always_inline)) { load_piece<kCut>(pw[i], w, 0, t + i * TPR, cols); });
    float ss = 0.f;
    float v[VPT][8];
    static_for<VPT>([&](auto i) __attribute__((always_inline)) {
        px[i].get(v[i]);
        if (r) {
            float q[8];
            pr[i].get(q);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] += q[e];
            px[i].set(v[i]);
            store_piece<kCut>(px[i], h, base, t + i * TPR, cols);
            px[i].get(v[i]);
        }
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[i][e] * v[i][e];
        ss += 8 * (t + i * TPR) < cols ? s : 0.f;
    });
    const float rstd = 1.0f / sqrtf(over_row(ss, true, 0) / static_cast<float>(cols) + eps);
    float am[VPT], top = 0.f;
    static_for<VPT>([&](auto i) __attribute__((always_inline)) {
        float g[8];
        pw[i].get(g);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = v[i][e] * rstd * g[e];
        am[i] = 8 * (t + i * TPR) < cols ? amax8(v[i]) : 0.f;
        top = fmaxf(top, am[i]);
    });
    if (!block) top = over_row(top, false, 1);
    const int runs = block ? (cols + kRun - 1) / kRun : 1;
    if (!block && t == 0) scales[row] = scale_of(top);
    static_for<VPT>([&](auto i) __attribute__((always_inline)) {
        const int p = t + i * TPR;
        const float scale = scale_of(block ? max16(am[i]) : top);
        const uint2 c = codes8(Quot(scale), v[i]);
        store_codes<kCut>(c, codes, base, p, cols);
        if (block && (t & 15) == 0 && 8 * p < cols) scales[row * runs + p / 16] = scale;
    });
}

// Runs of 128 of any rows, without the norm: 16 lanes a run, eight elements a lane.  HBM-bound, 3 bytes an
// element of bf16: 4096 x 4096 in 12.5 us (4.0 TB/s).  The source is read past the caches: between two products of 1024 x 11008 x 4096
// 152 us for all instead of 167 (4096 rows: 424 either way).
template <bool kBf16, bool kCut>
__global__ __launch_bounds__(256) void quant_fp8_run_kernel(const void *__restrict__ src, int64_t tasks, int cols, int runs,
                                                            uint8_t *__restrict__ codes, float *__restrict__ scales) {
    const int sub = threadIdx.x & 15;
    const int64_t stride = gridDim.x * 16ll;
    for (int64_t task = blockIdx.x * 16ll + (threadIdx.x >> 4); task < tasks; task += stride) {
        const int64_t row = task / runs;
        const int p = static_cast<int>(task - row * runs) * 16 + sub;  // piece of the row
        Piece<kBf16> x;
        load_piece<kCut, true>(x, src, row * cols, p, cols);
        float v[8];
        x.get(v);
        const float scale = scale_of(max16(8 * p < cols ? amax8(v) : 0.f));
        store_codes<kCut>(codes8(Quot(scale), v), codes, row * cols, p, cols);
        if (sub == 0) scales[task] = scale;
    }
}

// Rows shorter than eight elements or longer than the registers hold: one workgroup a row, three passes over it.
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
    const int64_t run = block ? block : cols, runs = block ? (cols + run - 1) / run : 1;
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

// E4M3 codes and scales of blocks of block_rows x 128, from block `first` on: one workgroup a block, two passes, an element a load.
// A weight is quantized once, at load: 11008 x 4096 of bf16 by 128 x 128 in 114 us (1.2 TB/s), by its loads' number.
__global__ __launch_bounds__(256) void quant_fp8_block_generic_kernel(const void *__restrict__ src, int bf16, int64_t rows,
                                                                      int64_t cols, int block_rows, int64_t first, uint8_t *__restrict__ codes,
                                                                      float *__restrict__ scales) {
    __shared__ float red[4];
    const int64_t runs = (cols + kRun - 1) / kRun, block = first + blockIdx.x;
    const int64_t br = block / runs, g = block % runs;
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
    if (threadIdx.x == 0) scales[block] = scale;
}

// A code a lane: 11008 x 4096 by 128 x 128 in 123 us (1.8 TB/s).
__global__ __launch_bounds__(256) void dequant_fp8_block_kernel(const uint8_t *__restrict__ codes, const float *__restrict__ scales,
                                                                int64_t rows, int64_t cols, int block_rows, float *__restrict__ out) {
    const int64_t n = rows * cols, runs = (cols + kRun - 1) / kRun;
    for (int64_t i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll)
        out[i] = e4m3fn_to_f32(codes[i]) * scales[i / cols / block_rows * runs + i % cols / kRun];
}

// The register kernel's shape by the row's length; false: the generic kernel.  Few lanes a row, and so no barrier and several rows a
// workgroup, as long as a lane holds few pieces: 4096 rows of 512 5.1 us by waves and 7.9 by 256 threads, of 1024 8.2 and 9.5; one
// row of 2048 2.9 us by 256 threads and 3.7 by a wave of four pieces a lane; 4096 rows of 8192 39.4 us by 256 and 43.6 by 1024
// threads.
template <bool kXBf16, bool kWBf16, bool kCut>
bool launch_norm(const void *x, const void *r, const void *w, float eps, int64_t rows, int64_t cols, int block, void *h, uint8_t *codes,
                 float *scales, hipStream_t st) {
    const auto go = [&](auto vpt, auto tpr) {
        constexpr int V = decltype(vpt)::value, T = decltype(tpr)::value;
        const int64_t grid = T == 64 ? (rows + 3) / 4 : rows;
        rms_norm_fp8_kernel<kXBf16, kWBf16, kCut, V, T><<<dim3(static_cast<unsigned>(grid)), dim3(T < 256 ? 256 : T), 0, st>>>(
            x, r, w, eps, rows, static_cast<int>(cols), block, h, codes, scales);
        return true;
    };
    typedef std::integral_constant<int, 1> one;
    typedef std::integral_constant<int, 2> two;
    typedef std::integral_constant<int, 4> four;
    typedef std::integral_constant<int, 64> wave;
    typedef std::integral_constant<int, 256> wg;
    typedef std::integral_constant<int, 1024> big;
    const int64_t nv = (cols + 7) / 8;
    if (nv <= 64) return go(one{}, wave{});
    if (nv <= 128) return go(two{}, wave{});
    if (nv <= 256) return go(one{}, wg{});
    if (nv <= 512) return go(two{}, wg{});
    if (nv <= 1024) return go(four{}, wg{});
    if (nv <= 2048) return go(two{}, big{});
    if (nv <= 4096) return go(four{}, big{});
    return false;
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
        if (rows == 0 || (cols == 0 && block)) return;
        // a row without elements still has its scale, 1
        require(scales && (cols == 0 || (x && weight && codes)), "buffers must not be NULL");
        hipStream_t st = static_cast<hipStream_t>(stream);
        const bool xb = x_dtype == CFH_DTYPE_BF16, wb = weight_dtype == CFH_DTYPE_BF16;
        const int64_t runs = block ? (cols + kRun - 1) / kRun : 1;
        const auto norm = [&](const void *x, const void *residual, int64_t rows, void *h, uint8_t *codes, float *scales) {
            if (cols >= 8) {
                const bool cut = cols % 8 != 0;
                const auto go = [&](auto x_bf16, auto w_bf16) {
                    constexpr bool X = decltype(x_bf16)::value, W = decltype(w_bf16)::value;
                    return cut ? launch_norm<X, W, true>(x, residual, weight, eps, rows, cols, block, h, codes, scales, st)
                               : launch_norm<X, W, false>(x, residual, weight, eps, rows, cols, block, h, codes, scales, st);
                };
                if (xb ? (wb ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{}))
                       : (wb ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{}))) {
                    check_launch("rms_norm_fp8");
                    return;
                }
            }
            rms_norm_fp8_generic_kernel<<<dim3(static_cast<unsigned>(rows)), dim3(256), 0, st>>>(
                x, residual, xb, weight, wb, eps, cols, block, h, codes, scales);
            check_launch("rms_norm_fp8");
        };
        // a workgroup a row, of up to 1024
        for (int64_t row = 0; row < rows; row += most_workgroups(1024)) {
            const auto from = [&](auto *p) { return p ? reinterpret_cast<decltype(p)>(reinterpret_cast<uintptr_t>(p) + row * cols * (xb ? 2 : 4)) : p; };
            norm(from(x), from(residual), std::min(rows - row, most_workgroups(1024)), from(h), codes + row * cols, scales + row * runs);
        }
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
        hipStream_t st = static_cast<hipStream_t>(stream);
        if (block_rows == 1 && cols >= 8 && cols <= 0x7fffff00) {
            const int runs = static_cast<int>((cols + kRun - 1) / kRun);
            const unsigned grid = static_cast<unsigned>(std::min<int64_t>((blocks + 15) / 16, 32 * cu_count()));
            const auto go = [&](auto bf16, auto cut) {
                quant_fp8_run_kernel<decltype(bf16)::value, decltype(cut)::value><<<dim3(grid), dim3(256), 0, st>>>(src, blocks, static_cast<int>(cols), runs, codes, scales);
            };
            if (src_dtype == CFH_DTYPE_BF16) cols % 8 ? go(std::true_type{}, std::true_type{}) : go(std::true_type{}, std::false_type{});
            else cols % 8 ? go(std::false_type{}, std::true_type{}) : go(std::false_type{}, std::false_type{});
            check_launch("quant_fp8_block");
            return;
        }
        for (int64_t first = 0; first < blocks; first += most_workgroups(256)) {
            const unsigned grid = static_cast<unsigned>(std::min(blocks - first, most_workgroups(256)));
            quant_fp8_block_generic_kernel<<<dim3(grid), dim3(256), 0, st>>>(src, src_dtype == CFH_DTYPE_BF16, rows, cols, block_rows, first, codes, scales);
            check_launch("quant_fp8_block");
        }
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
