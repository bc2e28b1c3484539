// 8-bit product with a scale per block of 128 for gfx950:
//   Y[m, n] = sum_b sa[m, b] sw[n / 128, b] sum_{k in run b} A[m, k] W[n, k]
//
// A: E4M3 [M, K], a scale per row and run of 128 columns (sa [M, ceil(K / 128)]); W: E4M3 [N, K], a
// scale per 128 x 128 (sw [ceil(N / 128), ceil(K / 128)]); both K-contiguous.
//
// All kernels walk K in runs of 128: a run's products are summed by MFMAs that start from zero, and the
// f32 partial is folded into the total with one fma by sa * sw.  W is the MFMAs' row operand: a lane then
// holds several n of one m, and since sw is one number for 128 n, the fold's factor is one register a tile.
//   kExact false: the codes on the fp8 MFMAs, whose adder aligns each block of eight products to the
//     largest one and keeps about 13 bits below it.  kExact true: the codes widened to f16 (every E4M3
//     value is an f16 normal), exact products and f32 sums (beside a product of 1 one of 2^-23 counts) at half the MFMA rate.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "../../include/castforge_hip.h"
#include "cfh_common.hpp"

namespace cfh {
namespace {

typedef int int32x8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));

constexpr int kRun = 128;
constexpr int kXcds = 8;

// Eight E4M3 codes (bytes 8 c .. 8 c + 7 of a lane's 32) as exact f16.
__device__ __forceinline__ half8_t e4m3x8_to_f16(const int32x8 &v, int c) {
    const uint32_t lo = static_cast<uint32_t>(v[2 * c]), hi = static_cast<uint32_t>(v[2 * c + 1]);
    const half2_t p0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    const half2_t p1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const half2_t p2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    const half2_t p3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return half8_t{p0[0], p0[1], p1[0], p1[1], p2[0], p2[1], p3[0], p3[1]};
}

__device__ __forceinline__ int32x8 join(const uint4 &lo, const uint4 &hi) {
    return int32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// LDS panels of 128-byte rows: 16-byte chunk c of row r sits at c ^ ((r >> 1) & 7), so that sixteen rows read at one chunk
// cover the 256-byte bank window.
__device__ __forceinline__ int swz(int r, int c) { return c ^ ((r >> 1) & 7); }

// Chunks c and c + 1 of row r; `rows` starts at a multiple of 16 rows of its panel.
__device__ __forceinline__ int32x8 frag(const uint8_t *rows, int r, int c) {
    return join(*reinterpret_cast<const uint4 *>(rows + r * kRun + swz(r, c) * 16), *reinterpret_cast<const uint4 *>(rows + r * kRun + swz(r, c + 1) * 16));
}

// A workgroup's panels of W and A and the scales of A's rows as buffers: what lies past a panel's last row reads 0.
struct Panels {
    __amdgpu_buffer_rsrc_t w, a, s;
    // lane i of a load brings 16 bytes of row i / 8 of its eight: their offsets in the panel at K = 0 and in the run, for loads
    // whose rows start at an even, or odd, multiple of eight (the swizzle repeats every 16 rows)
    int at[2], in_run[2];
};

struct GemmArgs {
    const uint8_t *A, *W;
    const float *sa, *sw;
    void *Y;
    int y_bf16, y_vec;  // y_vec: N % 4 == 0 and Y 16-byte aligned
    int M, N, K, runs;
    int tiles_m, tiles_n;
};

__device__ __forceinline__ Panels panels_of(const GemmArgs &g, int n0, int rows_n, int m0, int rows_m, int lane) {
    Panels p;
    p.w = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(g.W + static_cast<int64_t>(n0) * g.K), 0, rows_n * g.K, 0x00020000);
    p.a = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t *>(g.A + static_cast<int64_t>(m0) * g.K), 0, rows_m * g.K, 0x00020000);
    p.s = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(g.sa + static_cast<int64_t>(m0) * g.runs), 0, rows_m * g.runs * 4, 0x00020000);
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        p.in_run[o] = swz(8 * o + (lane >> 3), lane & 7) * 16;
        p.at[o] = (lane >> 3) * g.K + p.in_run[o];
    }
    return p;
}

// One load of eight rows (8 block, ..) of run r into 1 KB of LDS.  kTail: the run's chunks past K read 0 too, sent past the panel.
template <bool kTail>
__device__ __forceinline__ void panel_load(__amdgpu_buffer_rsrc_t panel, const Panels &p, uint8_t *dst, int block, int odd, int K, int r) {
    int at = p.at[odd] + (block * 8 * K + r * kRun);
    if (kTail) at = r * kRun + p.in_run[odd] < K ? at : 0x7fffffff;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(panel, (__attribute__((address_space(3))) void *)dst, 16, at, 0, 0, 0);
}

__device__ __forceinline__ void store4(const GemmArgs &g, int m, int n, const float (&v)[4]) {
    if (m >= g.M || n >= g.N) return;
    const int64_t o = static_cast<int64_t>(m) * g.N + n;
    if (g.y_vec) {
        if (g.y_bf16)
            *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(g.Y) + o) = make_uint2(f32x2_to_bf16x2_rne(v[0], v[1]), f32x2_to_bf16x2_rne(v[2], v[3]));
        else
            *reinterpret_cast<float4 *>(static_cast<float *>(g.Y) + o) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (n + q < g.N) {
            if (g.y_bf16) static_cast<uint16_t *>(g.Y)[o + q] = f32_to_bf16_rne(v[q]);
            else static_cast<float *>(g.Y)[o + q] = v[q];
        }
}

// ---- many rows: tiles through LDS ------------------------------------------------------------------------
//
// Workgroup tile 32 I WN (n) x 32 J WM (m), WN x WM waves of 32 I x 32 J.  A stage is one run of 128 of both
// panels and the A rows' scales, brought by buffer loads straight into LDS; two stages, one barrier a stage:
// a stage is loaded while the other one is computed.  4096 x 11008 x 4096: 188 to 193 us, 1.9 PFLOP/s, up to 220 in long runs of them,
// as the clock falls; a third of a CU's last round of tiles is idle, the clock is 2.05 GHz under the load, and of the busy cycles 47% are MFMAs and 31%
// the folds and addresses, which hardly overlap on a SIMD.  No faster: a run's first fragments read ahead of its barrier; 128 x
// 128 a wave at one wave a SIMD, whose sums lie where vector instructions cannot reach them (73 -> 90 us for 4096 x 4096 x 4096).
template <int I, int J, int WN, int WM>
struct Tile {
    static constexpr int NW = WN * WM, BN = 32 * I * WN, BM = 32 * J * WM;
    static constexpr int kLoads = (BN + BM) / 8 / NW;  // 1 KB loads (8 rows) a wave and stage
    static constexpr int kStage = (BN + BM) * kRun + BM * 4;
    static constexpr int kEpiRow = 64 * I;             // a wave's bf16 output row of 32 I
    static constexpr int kEpi = NW * 32 * J * kEpiRow;
    static constexpr int kLds = 2 * kStage > kEpi ? 2 * kStage : kEpi;
    static_assert((BN + BM) / 8 % NW == 0 && BN % 8 == 0 && kLds <= 160 * 1024, "tile shape");
    static_assert(kRun % (32 * I) == 0, "a wave's n share one scale of W");
};

// This wave's loads of run r of both panels and of the A rows' scales into the stage `dst`.
template <class T>
__device__ __forceinline__ void tile_issue(const Panels &p, uint8_t *__restrict__ dst, int wave, int lane, int K, int runs, int r) {
    const auto load = [&](auto tail) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < T::kLoads; ++t) {
            const int first = wave * T::kLoads + t;  // of the stage's loads of eight rows
            const bool is_w = first * 8 < T::BN;     // uniform
            panel_load<decltype(tail)::value>(is_w ? p.w : p.a, p, dst + first * 1024, is_w ? first : first - T::BN / 8, t & 1, K, r);
        }
    };
    if ((r + 1) * kRun > K) {
        asm volatile("");  // a branch: selects would cost every run
        load(std::true_type{});
    } else {
        load(std::false_type{});
    }
    static_assert(T::kLoads % 2 == 0 && T::BN % 16 == 0, "the parity of a load is that of its rows");
    static_assert(T::BM <= 64 * T::NW, "one load of scales a wave");
    if (wave * 64 < T::BM)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(p.s, (__attribute__((address_space(3))) void *)(dst + (T::BN + T::BM) * kRun + wave * 256), 4,
                                                 ((wave * 64 + lane) * runs + r) * 4, 0, 0, 0);
}

// One run: loads the next one into `nxt`, computes `cur`.  The pointers are restrict-qualified: the reads of `cur`
// do not wait for the loads into `nxt`.
template <bool kExact, int I, int J, int WN, int WM>
__device__ __forceinline__ void tile_stage(const uint8_t *__restrict__ cur, uint8_t *__restrict__ nxt, const Panels &panels, int wave, int lane, int K, int runs, int r,
                                           float sw, int wn, int wm, floatx16 (&acc)[I][J]) {
    typedef Tile<I, J, WN, WM> T;
    if (r + 1 < runs) tile_issue<T>(panels, nxt, wave, lane, K, runs, r + 1);
    const int fr = lane & 31, fc = (lane >> 5) * 2;
    const float *scales = reinterpret_cast<const float *>(cur + (T::BN + T::BM) * kRun) + wm + fr;
    int32x8 w[I][2];
    float f[J];
    const auto read_a = [&](int j, int32x8 (&a)[2]) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) a[kk] = frag(cur + (T::BN + wm + 32 * j) * kRun, fr, 4 * kk + fc);
    };
    const auto fold = [&](floatx16 &sum, const floatx16 &part, float by) {
#pragma unroll
        for (int q = 0; q < 16; ++q) sum[q] = __builtin_fmaf(part[q], by, sum[q]);
    };
    floatx16 zero;
#pragma unroll
    for (int q = 0; q < 16; ++q) zero[q] = 0.f;
    if constexpr (!kExact && J >= 4) {
        // Tile by tile: the MFMAs of a tile run while the tile before is folded, and the A fragments of the next 32 rows are
        // read meanwhile.  One wave alone can so keep the matrix unit busy (two MFMAs take 128 cycles, a fold 64): 222 -> 208 us
        // for 4096 x 11008 x 4096.  Left to itself the scheduler waits for each tile to fold it.
        int32x8 a[2][2];
        floatx16 part[2];
        read_a(0, a[0]);
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) w[i][kk] = frag(cur + (wn + 32 * i) * kRun, fr, 4 * kk + fc);
#pragma unroll
        for (int j = 0; j < J; ++j) f[j] = scales[32 * j] * sw;
        static_for<I * J + 1>([&](auto TT) {
            constexpr int t = decltype(TT)::value;
            if constexpr (t < I * J) {
                constexpr int i = t % I, j = t / I;
                if constexpr (i == 0 && j + 1 < J) read_a(j + 1, a[(j + 1) & 1]);
                part[t & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i][0], a[j & 1][0], zero, 0, 0, 0, 0, 0, 0);
                part[t & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i][1], a[j & 1][1], part[t & 1], 0, 0, 0, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (t > 0) fold(acc[(t - 1) % I][(t - 1) / I], part[(t - 1) & 1], f[(t - 1) / I]);
            __builtin_amdgcn_sched_barrier(0);
        });
        return;
    }
    // two workgroups a CU, which fill each other's gaps
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) w[i][kk] = frag(cur + (wn + 32 * i) * kRun, fr, 4 * kk + fc);
    static_for<J>([&](auto JJ) {
        constexpr int j = decltype(JJ)::value;
        f[j] = scales[32 * j] * sw;
        int32x8 a[2];
        read_a(j, a);
        floatx16 part[I];
#pragma unroll
        for (int i = 0; i < I; ++i) part[i] = zero;
        if constexpr (kExact) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const half8_t ah = e4m3x8_to_f16(a[c / 4], c % 4);
#pragma unroll
                for (int i = 0; i < I; ++i)
                    part[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(e4m3x8_to_f16(w[i][c / 4], c % 4), ah, part[i], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < I; ++i)
                    part[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i][kk], a[kk], part[i], 0, 0, 0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < I; ++i) fold(acc[i][j], part[i], f[j]);
    });
}

template <bool kExact, int I, int J, int WN, int WM>
__global__ __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(2, 2)))
void fp8_block_tile_kernel(GemmArgs g) {
    typedef Tile<I, J, WN, WM> T;
    extern __shared__ __align__(16) uint8_t lds[];
    // workgroups are dealt round-robin to the XCDs: each owns a contiguous run of tiles, in groups of 4 m
    // tiles of one W panel (their rows stay in the XCD's L2)
    int pid = blockIdx.x;
    {
        const int per_xcd = g.tiles_m * g.tiles_n / kXcds, full = per_xcd * kXcds;
        if (pid < full) pid = (pid % kXcds) * per_xcd + pid / kXcds;
    }
    const int span = 4 * g.tiles_n, first_m = pid / span * 4, gm = min(4, g.tiles_m - first_m);
    const int m0 = (first_m + pid % span % gm) * T::BM, n0 = pid % span / gm * T::BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Panels panels = panels_of(g, n0, min(T::BN, g.N - n0), m0, min(T::BM, g.M - m0), lane);
    const int wn = (wave / WM) * 32 * I, wm = (wave % WM) * 32 * J;
    const int fr = lane & 31;
    floatx16 acc[I][J];
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
    // in the constant address space: scalar loads (a vector load here would wait for the stage's loads)
    const auto *swp = (const __attribute__((address_space(4))) float *)(g.sw + static_cast<int64_t>(min(n0 + wn, g.N - 1) / kRun) * g.runs);

    float sw = swp[0];
    tile_issue<T>(panels, lds, wave, lane, g.K, g.runs, 0);
    for (int r = 0; r < g.runs; ++r) {
        const uint8_t *cur = lds + (r & 1) * T::kStage;
        // this wave's loads of the stage have landed, and its reads of the other stage returned; then everyone's
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(0) & ~(15 << 8));
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        const float sw_next = swp[min(r + 1, g.runs - 1)];
        tile_stage<kExact, I, J, WN, WM>(cur, lds + ((r + 1) & 1) * T::kStage, panels, wave, lane, g.K, g.runs, r, sw, wn, wm, acc);
        sw = sw_next;
    }

    // acc[i][j] reg 4 t + q holds n = 32 i + 8 t + 4 (lane / 32) + q, m = 32 j + lane % 32
    if (g.y_bf16 && g.N % 8 == 0 && g.y_vec) {
        // through LDS, so that every global store is a run of 64 I bytes of a row; past the caches, which hold the panels that other
        // tiles read (4096 x 11008 x 4096 with its quantizer: 218 -> 202 us)
        constexpr int kChunks = 4 * I, kRows = 64 / kChunks;
        __syncthreads();  // every wave is done with the stages
        uint8_t *eb = lds + wave * 32 * J * T::kEpiRow;
        static_for<J>([&](auto JJ) {
            constexpr int j = decltype(JJ)::value;
            const int ml = 32 * j + fr;
            static_for<I>([&](auto II) {
                constexpr int i = decltype(II)::value;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const uint2 p = make_uint2(f32x2_to_bf16x2_rne(acc[i][j][4 * t], acc[i][j][4 * t + 1]), f32x2_to_bf16x2_rne(acc[i][j][4 * t + 2], acc[i][j][4 * t + 3]));
                    *reinterpret_cast<uint2 *>(eb + ml * T::kEpiRow + (((4 * i + t) ^ (ml & (kChunks - 1))) * 16) + (lane >> 5) * 8) = p;
                }
            });
        });
        __builtin_amdgcn_s_waitcnt(vmcnt_imm(63) & ~(15 << 8));  // this wave's writes; it reads its own block
        asm volatile("" ::: "memory");
        const int cl = lane % kChunks;
#pragma unroll 4
        for (int rb = 0; rb < 32 * J; rb += kRows) {
            const int ml = rb + lane / kChunks;
            const uint4 v = *reinterpret_cast<const uint4 *>(eb + ml * T::kEpiRow + ((cl ^ (ml & (kChunks - 1))) * 16));
            const int m = m0 + wm + ml, n = n0 + wn + cl * 8;
            if (m < g.M && n < g.N) store_past(static_cast<uint16_t *>(g.Y) + static_cast<int64_t>(m) * g.N + n, v);
        }
        return;
    }
    static_for<J>([&](auto JJ) {
        constexpr int j = decltype(JJ)::value;
        static_for<I>([&](auto II) {
            constexpr int i = decltype(II)::value;
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const float v[4] = {acc[i][j][4 * t], acc[i][j][4 * t + 1], acc[i][j][4 * t + 2], acc[i][j][4 * t + 3]};
                store4(g, m0 + wm + 32 * j + fr, n0 + wn + 32 * i + 8 * t + 4 * (lane >> 5), v);
            }
        });
    });
}

// ---- few tiles: K split over the waves --------------------------------------------------------------------
//
// Workgroup tile 32 I (n) x 32 J (m).  Each of NW waves computes the whole tile over its own runs (w, w + NW, ..), with an LDS ring
// of its own (S stages of both panels' rows of 128 bytes and the A rows' scales), so the loop has no barrier and up to NW S
// runs a workgroup are in flight; the tiles are summed through LDS in wave order.  Bound by the latency of the few runs that
// each wave walks, and by HBM where N K is large: one row, 4096 x 4096, 5.9 us; one row, 11008 x 4096, 9.3 us (4.9 TB/s).
template <int I, int J, int NW, int S>
struct Split {
    static constexpr int kPanels = 32 * (I + J) * kRun, kStage = kPanels + 256;
    static constexpr int kLoads = 4 * (I + J) + 1;  // a run: 1 KB each, and the scales
    static constexpr int kRow = 32 * I + 4;
    static constexpr int kSums = NW * 32 * J * kRow * 4, kLds = NW * S * kStage > kSums ? NW * S * kStage : kSums;
    static_assert(kLds <= 160 * 1024 && S * kLoads <= 63 && J <= 2, "LDS budget, vmcnt range, one load of scales");
};

// Waits until at most N vector-memory loads are outstanding and every LDS read has returned, and keeps memory accesses on
// their side of the wait.
template <int N>
__device__ __forceinline__ void wait_vm_fence() {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(N) & ~(15 << 8));
    asm volatile("" ::: "memory");
}

template <int I, int J>
__device__ __forceinline__ void split_issue(const Panels &p, uint8_t *__restrict__ dst, int lane, int K, int runs, int r) {
    const auto load = [&](auto tail) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < 4 * (I + J); ++t) panel_load<decltype(tail)::value>(t < 4 * I ? p.w : p.a, p, dst + t * 1024, t < 4 * I ? t : t - 4 * I, t & 1, K, r);
    };
    if ((r + 1) * kRun > K) {
        asm volatile("");  // a branch
        load(std::true_type{});
    } else {
        load(std::false_type{});
    }
    __builtin_amdgcn_raw_ptr_buffer_load_lds(p.s, (__attribute__((address_space(3))) void *)(dst + 32 * (I + J) * kRun), 4, (lane * runs + r) * 4, 0, 0, 0);
}

// One run: refill `nxt` (read a step ago) with run r_next if there is one, wait for `cur`, compute it.  The slots differ and are
// restrict-qualified: the reads of `cur` need not wait for the refill.
template <bool kExact, int I, int J, int NW, int S>
__device__ __forceinline__ void split_step(const uint8_t *__restrict__ cur, uint8_t *__restrict__ nxt, bool refill, const Panels &panels, int lane,
                                           int K, int runs, int r_next, float sw, floatx16 (&acc)[I][J]) {
    typedef Split<I, J, NW, S> P;
    wait_vm_fence<63>();
    if (refill) split_issue<I, J>(panels, nxt, lane, K, runs, r_next);
    if (refill) wait_vm_fence<(S - 1) * P::kLoads>();
    else wait_vm_fence<0>();
    const int fr = lane & 31, fc = (lane >> 5) * 2;
    int32x8 w[I][2], a[J][2];
    float f[J];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int i = 0; i < I; ++i) w[i][kk] = frag(cur + 32 * i * kRun, fr, 4 * kk + fc);
#pragma unroll
        for (int j = 0; j < J; ++j) a[j][kk] = frag(cur + 32 * (I + j) * kRun, fr, 4 * kk + fc);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) f[j] = reinterpret_cast<const float *>(cur + P::kPanels)[32 * j + fr] * sw;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        floatx16 part[I];
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) part[i][q] = 0.f;
        if constexpr (kExact) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const half8_t ah = e4m3x8_to_f16(a[j][c / 4], c % 4);
#pragma unroll
                for (int i = 0; i < I; ++i)
                    part[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(e4m3x8_to_f16(w[i][c / 4], c % 4), ah, part[i], 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < I; ++i)
                    part[i] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[i][kk], a[j][kk], part[i], 0, 0, 0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = __builtin_fmaf(part[i][q], f[j], acc[i][j][q]);
    }
}

template <bool kExact, int I, int J, int NW, int S>
__global__ __launch_bounds__(64 * NW) void fp8_block_split_kernel(GemmArgs g) {
    typedef Split<I, J, NW, S> P;
    constexpr int BN = 32 * I, BM = 32 * J;
    extern __shared__ __align__(16) uint8_t lds[];
    // each XCD owns a contiguous run of tiles, in groups of up to 8 m tiles of one W panel
    int pid = blockIdx.x;
    {
        const int per_xcd = g.tiles_m * g.tiles_n / kXcds, full = per_xcd * kXcds;
        if (pid < full) pid = (pid % kXcds) * per_xcd + pid / kXcds;
    }
    const int span = 8 * g.tiles_n, first_m = pid / span * 8, gm = min(8, g.tiles_m - first_m);
    const int m0 = (first_m + pid % span % gm) * BM, n0 = pid % span / gm * BN;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Panels panels = panels_of(g, n0, min(BN, g.N - n0), m0, min(BM, g.M - m0), lane);
    const auto *swp = (const __attribute__((address_space(4))) float *)(g.sw + static_cast<int64_t>(n0 / kRun) * g.runs);
    floatx16 acc[I][J];
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
    const int own = g.runs > wave ? (g.runs - wave + NW - 1) / NW : 0;
    uint8_t *ring = lds + wave * S * P::kStage;
#pragma unroll
    for (int t = 0; t < S - 1; ++t)
        if (t < own) {
            asm volatile("" ::: "memory");  // the waits count whole runs
            split_issue<I, J>(panels, ring + t * P::kStage, lane, g.K, g.runs, wave + NW * t);
        }
    for (int t0 = 0; t0 < own; t0 += S)
        static_for<S>([&](auto SI) {
            constexpr int s = decltype(SI)::value;
            const int t = t0 + s;
            if (t < own)
                split_step<kExact, I, J, NW, S>(ring + s * P::kStage, ring + (s + S - 1) % S * P::kStage, t + S - 1 < own, panels, lane, g.K, g.runs,
                                                wave + NW * (t + S - 1), swp[wave + NW * t], acc);
        });

    __syncthreads();  // every wave is done with its ring (all of its loads were waited for)
    float *sums = reinterpret_cast<float *>(lds);
    const int fr = lane & 31, fc = (lane >> 5) * 2;
    static_for<I * J>([&](auto II) {
        constexpr int i = decltype(II)::value / J, j = decltype(II)::value % J;
#pragma unroll
        for (int t = 0; t < 4; ++t)
            *reinterpret_cast<floatx4 *>(sums + (wave * BM + 32 * j + fr) * P::kRow + 32 * i + 8 * t + 2 * fc) =
                floatx4{acc[i][j][4 * t], acc[i][j][4 * t + 1], acc[i][j][4 * t + 2], acc[i][j][4 * t + 3]};
    });
    __syncthreads();
#pragma unroll
    for (int o = threadIdx.x; o < BM * BN / 4; o += 64 * NW) {
        const int ml = o / (BN / 4), nl = o % (BN / 4) * 4;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const floatx4 p = *reinterpret_cast<const floatx4 *>(sums + (w * BM + ml) * P::kRow + nl);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] += p[q];
        }
        store4(g, m0 + ml, n0 + nl, v);
    }
}

// Any shape and alignment: one thread per output, from output `first` on; exact E4M3 decode, f32 sums.  By its scalar decode: 64 rows,
// N = 4096, K = 4100 take 3.4 ms, where K = 4096 takes 7 us on the tiles.
__global__ __launch_bounds__(256) void fp8_block_gemm_generic_kernel(GemmArgs g, int64_t first) {
    const int64_t idx = first + static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    if (idx >= static_cast<int64_t>(g.M) * g.N) return;
    const int64_t m = idx / g.N, n = idx - m * g.N;
    const uint8_t *a = g.A + m * g.K, *w = g.W + n * g.K;
    float acc = 0.f;
    for (int b = 0; b < g.runs; ++b) {
        const int end = min(g.K - b * kRun, kRun);
        float part = 0.f;
        for (int k = 0; k < end; ++k) part += e4m3fn_to_f32(a[b * kRun + k]) * e4m3fn_to_f32(w[b * kRun + k]);
        acc = __builtin_fmaf(part, g.sa[m * g.runs + b] * g.sw[n / kRun * g.runs + b], acc);
    }
    if (g.y_bf16) static_cast<uint16_t *>(g.Y)[idx] = f32_to_bf16_rne(acc);
    else static_cast<float *>(g.Y)[idx] = acc;
}

// Raises a kernel's dynamic-LDS limit once per device (bit = device ordinal < 64).
void raise_lds_limit(const void *kern, int bytes, std::atomic<uint64_t> &done) {
    int dev = 0;
    check_hip(hipGetDevice(&dev), "hipGetDevice");
    const uint64_t bit = dev < 64 ? (uint64_t{1} << dev) : 0;
    if (bit == 0 || !(done.load(std::memory_order_acquire) & bit)) {
        check_hip(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, bytes), "hipFuncSetAttribute(fp8 block)");
        done.fetch_or(bit, std::memory_order_acq_rel);
    }
}

template <bool kExact, int I, int J, int NW, int S>
void launch_split(GemmArgs g, hipStream_t st) {
    typedef Split<I, J, NW, S> P;
    static std::atomic<uint64_t> attr_devices{0};
    const auto kern = fp8_block_split_kernel<kExact, I, J, NW, S>;
    raise_lds_limit(reinterpret_cast<const void *>(kern), P::kLds, attr_devices);
    g.tiles_m = (g.M + 32 * J - 1) / (32 * J), g.tiles_n = (g.N + 32 * I - 1) / (32 * I);
    require(static_cast<int64_t>(g.tiles_m) * g.tiles_n <= most_workgroups(64 * NW), "too many tiles for one launch");
    kern<<<dim3(g.tiles_m * g.tiles_n), dim3(64 * NW), P::kLds, st>>>(g);
    check_launch("fp8_block_split");
}

template <bool kExact, int I, int J, int WN, int WM>
void launch_tile(GemmArgs g, hipStream_t st) {
    typedef Tile<I, J, WN, WM> T;
    static std::atomic<uint64_t> attr_devices{0};
    const auto kern = fp8_block_tile_kernel<kExact, I, J, WN, WM>;
    raise_lds_limit(reinterpret_cast<const void *>(kern), T::kLds, attr_devices);
    g.tiles_m = (g.M + T::BM - 1) / T::BM, g.tiles_n = (g.N + T::BN - 1) / T::BN;
    require(static_cast<int64_t>(g.tiles_m) * g.tiles_n <= most_workgroups(64 * T::NW), "too many tiles for one launch");
    kern<<<dim3(g.tiles_m * g.tiles_n), dim3(64 * T::NW), T::kLds, st>>>(g);
    check_launch("fp8_block_tile");
}

// The cheapest kernel by the rounds of its workgroups over the CUs, in us at K = 4096 (all grow with K alike; fp8 and exact form),
// beside what it takes and what the next candidate takes, measured:
//   32 x 32, K over 8 waves      6.5 (7.0) and 4.5 (4.8) for each further round
//                                                    M = 64, N = 4096: 7.1 (64 n x 32 m: 8.6)
//   64 n x 32 m, K over 6 waves  8.8 (10.4) and 6.2 (7.6)
//                                                    M = 1, N = 11008: 9.7 (32 x 32: 11.2); M = 45, N = 5001, exact: 9.8 (11.9)
//   64 x 64, K over 4 waves      12 (15) and 10.3 (12.7)
//                                                    M = 256, N = 4096: 11.8 (64 n x 32 m: 14.8); M = 64, N = 11008: 12.5 (15.9)
//   128 x 128, two a CU          20.5 (35) times tiles over CUs, at least 24.5 (33)
//                                                    M = 1024, N = 4096: 28.4 (64 x 64: 38); M = 256, N = 11008: 27.1 (29.4)
//   256 x 256, fp8 form          70 a round, 54 for one that leaves CUs idle
//                                                    M = 4096, N = 11008: 189 (128 x 128: 212); M = 1024, N = 11008: 58 (64.5)
template <bool kExact>
void launch_by_cost(const GemmArgs &g, hipStream_t st) {
    const double cus = static_cast<double>(cu_count());
    const auto tiles = [&](int tn, int tm) { return static_cast<double>((g.M + tm - 1) / tm) * ((g.N + tn - 1) / tn); };
    const auto cost = [&](int tn, int tm, double first, double further) { return first + further * (std::ceil(tiles(tn, tm) / cus) - 1); };
    const double c32 = kExact ? cost(32, 32, 7.0, 4.8) : cost(32, 32, 6.5, 4.5);
    const double c64n = kExact ? cost(64, 32, 10.4, 7.6) : cost(64, 32, 8.8, 6.2);
    const double c64 = kExact ? cost(64, 64, 15, 12.7) : cost(64, 64, 12, 10.3);
    const double c128 = kExact ? std::max(33.0, 35 * tiles(128, 128) / cus) : std::max(24.5, 20.5 * tiles(128, 128) / cus);
    const double c256 = kExact ? 1e30 : tiles(256, 256) < 0.9 * cus ? 54 : cost(256, 256, 70, 70);
    const double best = std::min({c32, c64n, c64, c128, c256});
    if (best == c32) launch_split<kExact, 1, 1, 8, 2>(g, st);
    else if (best == c64n) launch_split<kExact, 2, 1, 6, 2>(g, st);
    else if (best == c64) launch_split<kExact, 2, 2, 4, 2>(g, st);
    else if (kExact || best == c128) launch_tile<kExact, 2, 2, 2, 2>(g, st);
    else if constexpr (!kExact) launch_tile<false, 2, 4, 4, 2>(g, st);
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
        require(m <= 0x7fffff00 && n <= 0x7fffff00 && k <= 0x7fffff00, "dimensions must fit in int32");
        hipStream_t st = static_cast<hipStream_t>(stream);
        GemmArgs g{qa, qw, sa, sw, y, y_dtype == CFH_DTYPE_BF16, n % 4 == 0 && aligned(y, 16), static_cast<int>(m),
                   static_cast<int>(n), static_cast<int>(k), static_cast<int>((k + kRun - 1) / kRun), 0, 0};
        // buffer resources address a panel of 256 rows: 256 k bytes must fit in 31 bits
        const bool fast = k > 0 && k % 16 == 0 && k < (1 << 23) && aligned(qa, 16) && aligned(qw, 16);
        if (fast) {
            exact ? launch_by_cost<true>(g, st) : launch_by_cost<false>(g, st);
            return;
        }
        const int64_t tot = m * n;
        for (int64_t first = 0; first < tot; first += most_workgroups(256) * 256) {
            const int64_t blocks = std::min((tot - first + 255) / 256, most_workgroups(256));
            fp8_block_gemm_generic_kernel<<<dim3(static_cast<unsigned>(blocks)), dim3(256), 0, st>>>(g, first);
            check_launch("fp8_block_gemm_generic");
        }
    });
}
