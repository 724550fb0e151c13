// Matrix product with bias, activation and residual (s2_linear_act):
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n],
// x, w fp16 or bf16, the sum and everything after it in fp32, one rounding at the end.
//
// One row of x (a time embedding) is a product of a matrix and a vector, linear_vec_kernel. From two rows
// on, two kernels on the tensor cores (tcgen05, accumulators in TMEM, operands staged by TMA in
// 64-element K slices, 128-byte swizzle, out-of-range rows and K read as zeros):
//  * linear_tile_kernel, many rows: a pair of CTAs computes 256 x 256 tiles of y, persistent,
//    two accumulators, so that a tile's epilogue runs beside the next tile's products. A 256 x 256 tile
//    reads 1 byte of operands from L2 for 128 multiplications; smaller ones would be bound by L2.
//  * linear_rows_kernel, few rows: the operands change sides, 128 rows of w against 16 to 128
//    rows of x, one tile of y^T a CTA, and K split over the CTAs of a cluster, which join their
//    sums through distributed shared memory in order. The weights stream through at the rate of
//    the memory however few rows there are, and no workspace or second launch is needed.
// Operands whose base or pitch is no multiple of 16 bytes (TMA's rule) are first copied into the
// workspace with such a pitch (pack_rows_kernel).
// Every wait is bounded: on timeout the CTA records an error code, drains its copies and
// products, frees its TMEM and ends.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <atomic>
#include <cstdint>

#include "s2_act.cuh"
#include "s2_gemm.h"
#include "s2_internal.h"
#include "s2_launch.h"
#include "s2_operator_error.h"
#include "s2_overlap.h"
#include "s2_sm100.cuh"

namespace {

using namespace s2dev;

struct LinearArgs {
    const float *bias;
    const void *residual;
    void *y;
    long long M, ldr, ldy;
    int N, K, act;
    uint32_t fmt;     // operand format of the products: 0 fp16, 1 bf16
    int vec;          // residual and y rows start on 16 bytes
    int ks;           // linear_rows_kernel: CTAs that share a tile's K
    int packed;       // operands come from a pack_rows_kernel right before
    int32_t *err;
};

constexpr int kBK = 64;  // K elements a slice (one 128-byte swizzled row)

// device error codes of these kernels
enum : int { E_FULL = 80, E_EMPTY = 81, E_ACCF = 82, E_ACCE = 83, E_DRAIN = 84, E_RES = 85 };

__device__ __forceinline__ bool wait_drain(uint32_t bar, uint32_t parity, int *err)
{
    int dummy = 0;
    return mbar_wait(bar, parity, &dummy, err, E_DRAIN);
}

template <int N, int kAct>
__device__ __forceinline__ void activate_each(float (&v)[N])
{
    if constexpr (N == 1) {
        v[0] = activate<kAct>(v[0]);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const float2 f = floats_of(activate2<kAct>(pair(v[i], v[i + 1])));
            v[i] = f.x;
            v[i + 1] = f.y;
        }
    }
}

// act over N values; the branch is the same for every thread
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act)
{
    switch (act) {
    case S2_ACT_RELU: activate_each<N, S2_ACT_RELU>(v); break;
    case S2_ACT_SILU: activate_each<N, S2_ACT_SILU>(v); break;
    case S2_ACT_GELU: activate_each<N, S2_ACT_GELU>(v); break;
    case S2_ACT_GELU_TANH: activate_each<N, S2_ACT_GELU_TANH>(v); break;
    default: break;
    }
}

// ---- few rows ------------------------------------------------------------------

constexpr int kRowsThreads = 192;  // warp 0 TMA, warp 1 products, warps 2-5 epilogue
constexpr int kRowsN = 128;        // rows of w a tile

template <int MB>
struct Rows {
    static constexpr uint32_t kWBytes = kRowsN * kBK * 2, kXBytes = MB * kBK * 2;
    static constexpr uint32_t kStageBytes = kWBytes + kXBytes;
    // two CTAs an SM: up to 113 KB each
    static constexpr int kStages = MB <= 32 ? 5 : (MB == 64 ? 4 : 3);
    static constexpr uint32_t kOffBar = kStages * kStageBytes;
    static constexpr uint32_t kSmemBytes = kOffBar + 128 + 1024;
    static constexpr uint32_t kTmemCols = MB < 32 ? 32 : MB;
    static_assert(kSmemBytes <= 113 * 1024, "two CTAs an SM");
    static_assert(MB * kRowsN * 4 <= kOffBar, "the joined sums reuse the stages");
};

// Few rows are bound by the reading of w, which every block of x's rows repeats from L2: 58 x 2560 x 5120 takes 12.4 us
// (26 MB, 4.1 at the copy rate; the rest is the start, a first trip to memory and the join), 200 x 2560 x 5120 17.6 us.
template <int MB, typename TO>
__global__ void __launch_bounds__(kRowsThreads, 2)
    linear_rows_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                       const LinearArgs a)
{
    using R = Rows<MB>;
    constexpr int kStages = R::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (base - raw);
    const uint32_t bar_full = base + R::kOffBar, bar_empty = bar_full + 8 * kStages, bar_acc = bar_empty + 8 * kStages;
    volatile int *abort = reinterpret_cast<volatile int *>(gbase + R::kOffBar + 16 * kStages + 8);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(gbase + R::kOffBar + 16 * kStages + 12);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = static_cast<int>(blockIdx.x) % a.ks;
    const int n0 = static_cast<int>(blockIdx.x) / a.ks * kRowsN;
    const long long m0 = static_cast<long long>(blockIdx.y) * MB;
    const int n_k = (a.K + kBK - 1) / kBK;
    const int k_lo = static_cast<int>(1LL * n_k * rank / a.ks), k_hi = static_cast<int>(1LL * n_k * (rank + 1) / a.ks);

    if (threadIdx.x == 0) {
        for (int i = 0; i < 2 * kStages + 1; ++i) mbar_init(bar_full + 8 * i, 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(tmem_slot), R::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            wait_dependency();
            uint32_t p = 0;
            for (int kc = k_lo; kc < k_hi; ++kc, ++p) {
                const uint32_t s = p % kStages, u = p / kStages;
                if (!mbar_wait(bar_empty + 8 * s, (u & 1u) ^ 1u, abort, a.err, E_EMPTY)) break;
                const uint32_t sa = base + s * R::kStageBytes;
                mbar_arrive_expect_tx(bar_full + 8 * s, R::kStageBytes);
                tma_load_2d(sa, &tmW, bar_full + 8 * s, kc * kBK, n0);
                tma_load_2d(sa + R::kWBytes, &tmX, bar_full + 8 * s, kc * kBK, static_cast<int>(m0));
            }
            // no copy may still be landing when the stages are reused
            for (uint32_t s = 0; s < kStages; ++s)
                if (p > s) wait_drain(bar_full + 8 * s, ((p - 1 - s) / kStages) & 1u, a.err);
        }
        __syncwarp();
    } else if (warp == 1) {
        const bool leader = elect_one();
        const uint32_t idesc = idesc_f16(a.fmt, MB, 0);
        const uint64_t d0 = smem_desc_sw128(base, 16, 1024);
        uint32_t s = 0, phase = 0;
        for (int kc = k_lo; kc < k_hi; ++kc) {
            if (!__all_sync(0xffffffffu, mbar_wait(bar_full + 8 * s, phase, abort, a.err, E_FULL))) break;
            tc_fence_after();
            const uint64_t dw = d0 + static_cast<uint64_t>((s * R::kStageBytes) >> 4);
            if (leader) {
                mma_chunk_ss_k64(tmem, dw, dw + (R::kWBytes >> 4), idesc, kc > k_lo ? 1u : 0u);
                mma_commit(bar_empty + 8 * s);
            }
            __syncwarp();
            if (++s == kStages) {
                s = 0;
                phase ^= 1u;
            }
        }
        if (leader) mma_commit(bar_acc);
        wait_drain(bar_acc, 0, a.err);
        __syncwarp();
    } else {
        const bool ok = mbar_wait(bar_acc, 0, abort, a.err, E_ACCF);
        __all_sync(0xffffffffu, ok);
        tc_fence_after();
    }
    // CTA r joins and finishes rows [MB r / ks, MB (r + 1) / ks) of x: once no CTA reads its stages any
    // more, every CTA sends it its sums, [part][row][128] in place of the stages, and they are added in
    // the order of the parts. (Sent, not fetched: fetches would cost a round trip a row.)
    __syncwarp();
    if (a.ks > 1) cluster_sync();
    const int cols = static_cast<int>(min(static_cast<long long>(MB), a.M - m0));
    const int share = MB / a.ks, shift = 31 - __clz(share);
    const int quad = warp & 3, nl = quad * 32 + lane, n = n0 + nl;
    if (warp >= 2) {
        for (int c = 0; c < cols; c += 16) {
            uint32_t r[16];
            tmem_ld16(tmem + (static_cast<uint32_t>(quad * 32) << 16) + c, r);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t to = static_cast<uint32_t>(c + i) >> shift, row = (c + i) & (share - 1);
                const uint32_t at = base + static_cast<uint32_t>((rank * share + row) * kRowsN + nl) * 4;
                if (c + i < cols) st_cluster_b32(cluster_map(at, to), r[i]);
            }
        }
    }
    __syncwarp();
    if (a.ks > 1)
        cluster_sync();
    else
        __syncthreads();
    if (warp >= 2 && n < a.N) {
        const float *part = reinterpret_cast<const float *>(gbase) + nl;
        const float bias = a.bias ? __ldg(a.bias + n) : 0.f;
        const int c0 = rank * share, c1 = min(cols, c0 + share);
        const TO *res = static_cast<const TO *>(a.residual) + (m0 + c0) * a.ldr + n;
        TO *y = static_cast<TO *>(a.y) + (m0 + c0) * a.ldy + n;
        constexpr int kRun = 8;  // rows at a time: their residuals are all asked for first
        const int last = share - 1;
#pragma unroll 1
        for (int i = 0; c0 + i < c1; i += kRun) {
            float rv[kRun], v[kRun];
#pragma unroll
            for (int k = 0; k < kRun; ++k, res += a.ldr) rv[k] = a.residual && c0 + i + k < c1 ? to_float<TO>(*res) : 0.f;
            const float *q = part + i * kRowsN;
#pragma unroll
            for (int k = 0; k < kRun; ++k) v[k] = q[(i + k <= last ? k : 0) * kRowsN];
#pragma unroll 1
            for (int t = 1; t < a.ks; ++t) {
                q += share * kRowsN;
#pragma unroll
                for (int k = 0; k < kRun; ++k) v[k] += q[(i + k <= last ? k : 0) * kRowsN];
            }
#pragma unroll
            for (int k = 0; k < kRun; ++k) v[k] += bias;
            activate_all<kRun>(v, a.act);
#pragma unroll
            for (int k = 0; k < kRun; ++k, y += a.ldy)
                if (c0 + i + k < c1) *y = from_float<TO>(v[k] + rv[k]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, R::kTmemCols);
    }
}

// ---- one row ---------------------------------------------------------------

constexpr int kVecThreads = 256, kVecWarps = kVecThreads / 32;

// VEC 16-bit values as they are loaded
template <int VEC>
struct Raw;
template <>
struct Raw<8> {
    using type = uint4;
    static __device__ __forceinline__ uint4 zero() { return make_uint4(0, 0, 0, 0); }
    static __device__ __forceinline__ uint4 load(const void *p) { return __ldg(static_cast<const uint4 *>(p)); }
    // weights, read once: past L1
    static __device__ __forceinline__ uint4 stream(const void *p)
    {
        uint4 v;
        asm volatile("ld.global.nc.L1::no_allocate.L2::256B.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(p));
        return v;
    }
    template <typename T>
    static __device__ __forceinline__ void floats(const uint4 &v, float (&f)[8])
    {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 q = unpack2<T>(u[i]);
            f[2 * i] = q.x;
            f[2 * i + 1] = q.y;
        }
    }
};
template <>
struct Raw<1> {
    using type = uint16_t;
    static __device__ __forceinline__ uint16_t zero() { return 0; }
    static __device__ __forceinline__ uint16_t load(const void *p) { return __ldg(static_cast<const uint16_t *>(p)); }
    static __device__ __forceinline__ uint16_t stream(const void *p) { return load(p); }
    template <typename T>
    static __device__ __forceinline__ void floats(uint16_t v, float (&f)[1])
    {
        f[0] = to_float<T>(*reinterpret_cast<const T *>(&v));
    }
};

// One row of x, bound by the reading of w: 15360 x 2560 (79 MB) takes 16.4 us, 4.8 TB/s with start and end;
// 2560 x 2560 5.6 us, most of it two trips to memory and the start. The tensor cores would not read faster,
// and their tiles leave the GPU idle when N is small (2560 x 2560: 7.3 us in linear_rows_kernel).
// Every warp streams two rows of w, a.ks warps (1, 2, 4 or 8) share their K by pieces of 32
// vectors, kAhead pieces in flight. VEC = 8: w's rows and x start on 16 bytes; else values one by one.
template <typename T, typename TO, int VEC, int kAhead>
__global__ void __launch_bounds__(kVecThreads) linear_vec_kernel(const T *__restrict__ x, const T *__restrict__ w, long long ldw,
                                                                 const LinearArgs a)
{
    constexpr int kPiece = 32 * VEC;
    using R = Raw<VEC>;
    __shared__ float sums[kVecWarps][2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = warp % a.ks, n = 2 * ((static_cast<int>(blockIdx.x) * kVecWarps + warp) / a.ks);
    float acc0 = 0.f, acc1 = 0.f;
    if (n < a.N) {
        const T *w0 = w + n * ldw + lane * VEC;
        const T *w1 = w + min(n + 1, a.N - 1) * ldw + lane * VEC;
        const T *xl = x + lane * VEC;
        const int step = kPiece * a.ks, whole = a.K / VEC * VEC - (lane + 1) * VEC;
        for (int k = part * kPiece; k < a.K; k += kAhead * step) {
            typename R::type q0[kAhead], q1[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const bool in = k + u * step <= whole;
                q0[u] = in ? R::stream(w0 + k + u * step) : R::zero();
                q1[u] = in ? R::stream(w1 + k + u * step) : R::zero();
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (k + u * step <= whole) {
                    float f0[VEC], f1[VEC], f[VEC];
                    R::template floats<T>(q0[u], f0);
                    R::template floats<T>(q1[u], f1);
                    R::template floats<T>(R::load(xl + k + u * step), f);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        acc0 = fmaf(f0[e], f[e], acc0);
                        acc1 = fmaf(f1[e], f[e], acc1);
                    }
                }
        }
        // the values past the last whole vector, one a lane
        const int tail = a.K / VEC * VEC + lane;
        if (VEC > 1 && part == 0 && tail < a.K) {
            const float f = to_float<T>(x[tail]);
            acc0 = fmaf(to_float<T>(w[n * ldw + tail]), f, acc0);
            acc1 = fmaf(to_float<T>(w[min(n + 1, a.N - 1) * ldw + tail]), f, acc1);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            acc0 += __shfl_xor_sync(0xffffffffu, acc0, o);
            acc1 += __shfl_xor_sync(0xffffffffu, acc1, o);
        }
    }
    if (lane == 0) {
        sums[warp][0] = acc0;
        sums[warp][1] = acc1;
    }
    __syncthreads();
    // a thread a column of the block: the parts' sums in order, then the epilogue
    const int groups = kVecWarps / a.ks;
    if (threadIdx.x < groups * 2) {
        const int g = threadIdx.x >> 1, i = threadIdx.x & 1, col = 2 * (static_cast<int>(blockIdx.x) * groups + g) + i;
        if (col < a.N) {
            float v[1] = {sums[g * a.ks][i]};
            for (int t = 1; t < a.ks; ++t) v[0] += sums[g * a.ks + t][i];
            if (a.bias) v[0] += __ldg(a.bias + col);
            activate_all<1>(v, a.act);
            if (a.residual) v[0] += to_float<TO>(static_cast<const TO *>(a.residual)[col]);
            static_cast<TO *>(a.y)[col] = from_float<TO>(v[0]);
        }
    }
}

// ---- many rows -------------------------------------------------------------------

constexpr int kTileThreads = 320;  // warp 0 TMA, warp 1 products, warps 2-9 epilogue
constexpr int kTileN = 256, kTileHalf = 128;

struct Tile {
    static constexpr uint32_t kABytes = kTileHalf * kBK * 2, kBBytes = kTileHalf * kBK * 2;
    static constexpr uint32_t kStageBytes = kABytes + kBBytes;  // of each CTA of the pair
    static constexpr int kStages = 5;
    static constexpr uint32_t kSlabBytes = 32 * 128;  // 32 rows x 128 bytes of y; each epilogue warp has two
    static constexpr uint32_t kOffSlab = kStages * kStageBytes;
    static constexpr uint32_t kOffBias = kOffSlab + 16 * kSlabBytes;
    static constexpr uint32_t kOffBar = kOffBias + kTileN * 4;
    static constexpr uint32_t kSmemBytes = kOffBar + 384 + 1024;
    static_assert(kSmemBytes <= 232448, "shared memory budget");
};
enum TileBar {
    T_FULL = 0,
    T_EMPTY = T_FULL + Tile::kStages,
    T_ACCF = T_EMPTY + Tile::kStages,
    T_ACCE = T_ACCF + 2,
    T_DRAIN = T_ACCE + 2,
    T_RES = T_DRAIN + 1,  // [8 epilogue warps][2] a residual slab has landed
    T_COUNT = T_RES + 16
};
static_assert(8 * T_COUNT + 8 <= 384, "barrier area");

// Tiles in bands of kBand row blocks, column by column in a band: the CTA pairs that run at one
// time share few blocks of x and of w.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_of(int t, int m_blocks, int n_blocks, int &mb, int &nb)
{
    const int per = kBand * n_blocks, band = t / per, in = t - band * per;
    const int rows = min(kBand, m_blocks - band * kBand);
    nb = in / rows;
    mb = band * kBand + in - nb * rows;
}

// Large products run at the rate that the power limit leaves the tensor cores: 21600 x 10240 x 2560 bf16 takes 772 us
// without an activation, 1.47 PFLOP/s (1.40 measured for a library's plain product kept up for seconds), and 754 (cool)
// to 850 with gelu, whose arithmetic the epilogue warps do beside the products. With K short the tiles' operands bound
// it, 0.5 MB of them from L2 for each 128 KB of y at K = 512: 86400 x 512 x 512 fp16 takes 51 us
// with a residual (40.6 to read and write once), 43.5 without, and about 65 at the clocks of a long run.
template <typename TO>
__global__ void __launch_bounds__(kTileThreads, 1)
    linear_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                       const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmY,
                       const LinearArgs a)
{
    constexpr int kStages = Tile::kStages;
    constexpr int kE = 16 / sizeof(TO);   // values of 16 bytes
    constexpr int kSlab = 8 * kE;         // columns of a slab
    const uint32_t rank = cluster_rank();
    const int unit = static_cast<int>(blockIdx.x >> 1), n_units = static_cast<int>(gridDim.x >> 1);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *gbase = smem_raw + (base - raw);
    const uint32_t bar0 = base + Tile::kOffBar;
    volatile int *abort = reinterpret_cast<volatile int *>(gbase + Tile::kOffBar + 8 * T_COUNT);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(gbase + Tile::kOffBar + 8 * T_COUNT + 4);
    auto bar = [&](int i) { return bar0 + 8u * static_cast<uint32_t>(i); };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_blocks = (a.N + kTileN - 1) / kTileN, m_blocks = static_cast<int>((a.M + 255) / 256);
    const int n_tiles = m_blocks * n_blocks;
    const int n_k = (a.K + kBK - 1) / kBK;

    if (threadIdx.x == 0) {
        // the accumulator-empty barriers (rank 0's) count both CTAs' epilogue threads
        for (int i = 0; i < T_COUNT; ++i) mbar_init(bar(i), i >= T_ACCE && i < T_ACCE + 2 ? 512u : 1u);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(tmem_slot), 2 * kTileN);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // both CTAs' barriers exist before any signal between them
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        if (lane == 0) {
            tma_prefetch_desc(&tmX);
            tma_prefetch_desc(&tmW);
            wait_dependency();
            uint32_t p = 0;
            bool ok = true;
            for (int t = unit; ok && t < n_tiles; t += n_units) {
                int mb, nb;
                tile_of(t, m_blocks, n_blocks, mb, nb);
                const int m0 = mb * 256 + static_cast<int>(rank) * kTileHalf;
                const int n0 = nb * kTileN + static_cast<int>(rank) * kTileHalf;
                for (int kc = 0; kc < n_k; ++kc, ++p) {
                    const uint32_t s = p % kStages, u = p / kStages;
                    if (!(ok = mbar_wait(bar(T_EMPTY + s), (u & 1u) ^ 1u, abort, a.err, E_EMPTY))) break;
                    const uint32_t sa = base + s * Tile::kStageBytes;
                    // both CTAs' slices are counted on rank 0's barrier
                    if (rank == 0) mbar_arrive_expect_tx(bar(T_FULL + s), 2 * Tile::kStageBytes);
                    const uint32_t fb = cluster_map(bar(T_FULL + s), 0);
                    tma_load_2d_pair(sa, &tmX, fb, kc * kBK, m0);
                    tma_load_2d_pair(sa + Tile::kABytes, &tmW, fb, kc * kBK, n0);
                }
            }
            // No copy may still be landing when the CTA exits: rank 0 drains the full barriers, rank 1
            // waits for its last stages to be released by the products that read them.
            for (uint32_t s = 0; s < kStages; ++s)
                if (p > s) wait_drain(bar((rank == 0 ? T_FULL : T_EMPTY) + s), ((p - 1 - s) / kStages) & 1u, a.err);
        }
    } else if (warp == 1) {
        // The warp stays together and one lane issues: descriptors and barriers stay in uniform
        // registers, and the issue keeps ahead of the products (with a lone thread's loop they took
        // 570 to 650 cycles a slice where the tensor cores need 512).
        if (rank == 0) {
            const bool leader = elect_one();
            const uint32_t idesc = idesc_f16(a.fmt, kTileN, 0, 256u);
            const uint64_t d0 = smem_desc_sw128(base, 16, 1024);
            uint32_t lt = 0, s = 0, phase = 0;
            bool ok = true;
            for (int t = unit; ok && t < n_tiles; t += n_units, ++lt) {
                const uint32_t b = lt & 1u;
                ok = __all_sync(0xffffffffu, mbar_wait(bar(T_ACCE + b), ((lt >> 1) & 1u) ^ 1u, abort, a.err, E_ACCE));
                if (!ok) break;
                tc_fence_after();
                for (int kc = 0; kc < n_k; ++kc) {
                    ok = __all_sync(0xffffffffu, mbar_wait(bar(T_FULL + s), phase, abort, a.err, E_FULL));
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t da = d0 + static_cast<uint64_t>((s * Tile::kStageBytes) >> 4);
                    if (leader) {
                        mma_chunk_pair_k64(tmem + b * kTileN, da, da + (Tile::kABytes >> 4), idesc, kc > 0 ? 1u : 0u);
                        mma_commit_both(bar(T_EMPTY + s));
                    }
                    __syncwarp();
                    if (++s == kStages) {
                        s = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (leader) mma_commit_both(bar(T_ACCF + b));
                __syncwarp();
            }
            if (leader) mma_commit_pair(cluster_map(bar(T_DRAIN), 0));
            wait_drain(bar(T_DRAIN), 0, a.err);
        }
    } else {
        // Warp w holds TMEM lanes 32 (w % 4) .. +31, rows of the tile, and one half of its columns.
        // A slab is 32 rows x 128 bytes of y. With aligned rows (a.vec) its residual is brought in and
        // its values are stored by TMA, one slab ahead and one behind; 16-byte piece k of row r lies at
        // k ^ (r % 8), TMA's 128-byte swizzle, so that a thread's row is read without conflicts.
        // Otherwise the warp moves slabs value by value, whole rows at a time.
        const int quad = warp & 3, half = (warp - 2) >> 2, hw = warp - 2;
        const uint32_t lane_off = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t slab_s = base + Tile::kOffSlab + hw * 2 * Tile::kSlabBytes;
        uint8_t *slab_g = gbase + Tile::kOffSlab + hw * 2 * Tile::kSlabBytes;
        float *bias_g = reinterpret_cast<float *>(gbase + Tile::kOffBias) + hw * 32;  // of the warp's 32 columns
        const TO *res = static_cast<const TO *>(a.residual);
        TO *y = static_cast<TO *>(a.y);
        const bool ahead = res && a.vec;

        // asks for the residual of slab `js` (counted over the warp's tiles) at column n of row m
        auto ask = [&](uint32_t js, int n, int m) {
            if (lane == 0) {
                const uint32_t rb = bar(T_RES + 2 * hw + (js & 1u));
                mbar_arrive_expect_tx(rb, Tile::kSlabBytes);
                tma_load_2d(slab_s + (js & 1u) * Tile::kSlabBytes, &tmR, rb, n, m);
            }
        };
        auto ask_tile = [&](uint32_t js, int t) {
            int mb, nb;
            tile_of(t, m_blocks, n_blocks, mb, nb);
            ask(js, nb * kTileN + half * kTileHalf, mb * 256 + static_cast<int>(rank) * kTileHalf + quad * 32);
        };
        uint32_t lt = 0, js = 0, asked = 0;  // slabs begun, residual slabs asked for
        bool ok = true;
        if (ahead && unit < n_tiles) {
            ask_tile(0, unit);
            asked = 1;
        }
        for (int t = unit; ok && t < n_tiles; t += n_units, ++lt) {
            int mb, nb;
            tile_of(t, m_blocks, n_blocks, mb, nb);
            const int m0 = mb * 256 + static_cast<int>(rank) * kTileHalf + quad * 32;
            const int n_lo = nb * kTileN + half * kTileHalf;
            const uint32_t b = lt & 1u;
            ok = mbar_wait(bar(T_ACCF + b), (lt >> 1) & 1u, abort, a.err, E_ACCF);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int s = 0; ok && s < kTileHalf / kSlab; ++s, ++js) {
                const int n = n_lo + s * kSlab;
                float bias[kSlab / 32];
#pragma unroll
                for (int h = 0; h < kSlab / 32; ++h)
                    bias[h] = a.bias && n + 32 * h + lane < a.N ? __ldg(a.bias + n + 32 * h + lane) : 0.f;
                const uint32_t buf = js & 1u;
                uint4 *slab4 = reinterpret_cast<uint4 *>(slab_g + buf * Tile::kSlabBytes);
                TO *slab = reinterpret_cast<TO *>(slab4);
                if (ahead) {
                    // the other slab is free once its store has read it
                    const bool more = s + 1 < kTileHalf / kSlab;
                    if (more || t + n_units < n_tiles) {
                        if (lane == 0) bulk_wait_group_read<0>();
                        if (more)
                            ask(js + 1, n + kSlab, m0);
                        else
                            ask_tile(js + 1, t + n_units);
                        ++asked;
                    }
                    ok = mbar_wait(bar(T_RES + 2 * hw + buf), (js >> 1) & 1u, abort, a.err, E_RES);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                } else {
                    if (lane == 0) bulk_wait_group_read<1>();
                    __syncwarp();
                    if (res) {
                        constexpr int kRows = 8;  // rows whose values are asked for together
#pragma unroll 1
                        for (int r = 0; r < 32; r += kRows) {
                            TO t[kRows][kSlab / 32];
#pragma unroll
                            for (int k = 0; k < kRows; ++k)
#pragma unroll
                                for (int c = 0; c < kSlab / 32; ++c)
                                    t[k][c] = m0 + r + k < a.M && n + 32 * c + lane < a.N
                                                  ? res[(m0 + r + k) * a.ldr + n + 32 * c + lane]
                                                  : from_float<TO>(0.f);
#pragma unroll
                            for (int k = 0; k < kRows; ++k)
#pragma unroll
                                for (int c = 0; c < kSlab / 32; ++c) {
                                    const int col = 32 * c + lane;
                                    slab[((r + k) * 8 + ((col / kE) ^ ((r + k) & 7))) * kE + col % kE] = t[k][c];
                                }
                        }
                    }
                }
                __syncwarp();
#pragma unroll
                for (int h = 0; h < kSlab / 32; ++h) {
                    __syncwarp();
                    bias_g[lane] = bias[h];
                    __syncwarp();
                    uint32_t r32[32];
                    tmem_ld32(tmem + lane_off + b * kTileN + static_cast<uint32_t>(half * kTileHalf + s * kSlab + 32 * h), r32);
                    tmem_wait_ld();
                    float v[32];
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const float4 bv = *reinterpret_cast<const float4 *>(bias_g + 4 * q);
                        v[4 * q] = __uint_as_float(r32[4 * q]) + bv.x;
                        v[4 * q + 1] = __uint_as_float(r32[4 * q + 1]) + bv.y;
                        v[4 * q + 2] = __uint_as_float(r32[4 * q + 2]) + bv.z;
                        v[4 * q + 3] = __uint_as_float(r32[4 * q + 3]) + bv.w;
                    }
                    activate_all<32>(v, a.act);
                    uint4 *cell[32 / kE];
#pragma unroll
                    for (int k = 0; k < 32 / kE; ++k) cell[k] = slab4 + lane * 8 + ((h * (32 / kE) + k) ^ (lane & 7));
                    if (res) {
#pragma unroll
                        for (int k = 0; k < 32 / kE; ++k) {
                            const uint4 q = *cell[k];
                            const uint32_t u[4] = {q.x, q.y, q.z, q.w};
                            float *f = v + k * kE;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if constexpr (sizeof(TO) == 4) {
                                    f[j] += __uint_as_float(u[j]);
                                } else {
                                    const float2 g = unpack2<TO>(u[j]);
                                    f[2 * j] += g.x;
                                    f[2 * j + 1] += g.y;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int k = 0; k < 32 / kE; ++k) {
                        const float *f = v + k * kE;
                        if constexpr (sizeof(TO) == 4)
                            *cell[k] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                                                  __float_as_uint(f[3]));
                        else
                            *cell[k] = make_uint4(pack2<TO>(f[0], f[1]), pack2<TO>(f[2], f[3]), pack2<TO>(f[4], f[5]),
                                                  pack2<TO>(f[6], f[7]));
                    }
                }
                if (s + 1 == kTileHalf / kSlab) {
                    // the accumulator is read: the products of the tile after the next may overwrite it
                    tc_fence_before();
                    if (rank == 0)
                        mbar_arrive(bar(T_ACCE + b));
                    else
                        mbar_arrive_remote_relaxed(cluster_map(bar(T_ACCE + b), 0));
                }
                if (a.vec) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (m0 < a.M && n < a.N) tma_store_2d(&tmY, slab_s + buf * Tile::kSlabBytes, n, m0);
                        bulk_commit_group();
                    }
                } else {
                    __syncwarp();
                    for (int r = 0; r < 32; ++r)
                        for (int c = lane; c < kSlab; c += 32)
                            if (m0 + r < a.M && n + c < a.N)
                                y[(m0 + r) * a.ldy + n + c] = slab[(r * 8 + ((c / kE) ^ (r & 7))) * kE + c % kE];
                    __syncwarp();
                }
            }
        }
        // no copy of this warp's may still be under way when the CTA exits
        if (lane == 0) bulk_wait_group_all();
        for (; js < asked; ++js) wait_drain(bar(T_RES + 2 * hw + (js & 1u)), (js >> 1) & 1u, a.err);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its partner may still signal it
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 2 * kTileN);
    }
}

// ---- operands TMA cannot read -----------------------------------------------------

// Rows of K 16-bit values at any pitch -> rows at `ldd`, a multiple of 8 values: eight a thread, their loads
// in flight together, one store. Past K zeros. The kernel behind it may start beside it (it waits before it
// reads).
__global__ void __launch_bounds__(256) pack_rows_kernel(const uint16_t *__restrict__ src, long long lds, long long rows,
                                                        int K, uint16_t *__restrict__ dst, long long ldd)
{
    launch_dependents();
    const long long per = ldd / 8, n = rows * per;
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += 256LL * gridDim.x) {
        const long long r = i / per;
        const int k = static_cast<int>(i - r * per) * 8;
        const uint16_t *p = src + r * lds + k;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = k + e < K ? p[e] : 0u;
        *reinterpret_cast<uint4 *>(dst + r * ldd + k) =
            make_uint4(v[0] | v[1] << 16, v[2] | v[3] << 16, v[4] | v[5] << 16, v[6] | v[7] << 16);
    }
}

long long round_up8(long long v) { return (v + 7) / 8 * 8; }

bool tma_ready(const void *p, long long ld, long long rows)
{
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || ld % 8 == 0);
}

template <typename T, typename TO>
s2_status launch_vec(LinearArgs a, int sms, const s2_linear_act_desc &d, cudaStream_t st)
{
    const T *x = static_cast<const T *>(d.x), *w = static_cast<const T *>(d.w);
    const bool wide = (reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.w) | (d.N > 1 ? d.ldw * 2 : 0)) % 16 == 0;
    // Warps that share a row's K: as many as fill the GPU (32 warps an SM) and have a piece each. Then two pieces
    // in flight are enough, else four: 2560 x 2560 (four warps a row) takes 5.3 us with two and 6.4 with four,
    // 15360 x 2560 (one) 16.6 and 16.2.
    const int pieces = std::max(1, a.K / (wide ? 256 : 32)), pairs = (a.N + 1) / 2;
    a.ks = 1;
    while (a.ks < kVecWarps && a.ks * 2 <= pieces && 1LL * pairs * a.ks < 32LL * sms) a.ks *= 2;
    const unsigned grid = static_cast<unsigned>((1LL * pairs * a.ks + kVecWarps - 1) / kVecWarps);
    if (!wide)
        linear_vec_kernel<T, TO, 1, 8><<<grid, kVecThreads, 0, st>>>(x, w, d.ldw, a);
    else if (a.ks > 1)
        linear_vec_kernel<T, TO, 8, 2><<<grid, kVecThreads, 0, st>>>(x, w, d.ldw, a);
    else
        linear_vec_kernel<T, TO, 8, 4><<<grid, kVecThreads, 0, st>>>(x, w, d.ldw, a);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: launch failed: %s", cudaGetErrorString(e));
}

template <int MB, typename TO>
s2_status launch_rows(LinearArgs a, int ks, const void *x, long long ldx, const void *w, long long ldw, cudaStream_t st)
{
    using R = Rows<MB>;
    CUtensorMap mw, mx;
    if (!s2::make_map_2d(&mw, w, a.K, a.N, ldw * 2, kBK, kRowsN) || !s2::make_map_2d(&mx, x, a.K, a.M, ldx * 2, kBK, MB))
        return s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: cuTensorMapEncodeTiled failed");
    static std::atomic<uint64_t> configured{0};
    const s2_status cs = s2::once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(linear_rows_kernel<MB, TO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   R::kSmemBytes);
        return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: %s", cudaGetErrorString(e));
    });
    if (cs != S2_OK) return cs;
    a.ks = ks;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(ks);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>((a.N + kRowsN - 1) / kRowsN * ks), static_cast<unsigned>((a.M + MB - 1) / MB));
    cfg.blockDim = dim3(kRowsThreads);
    cfg.dynamicSmemBytes = R::kSmemBytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = a.packed ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_rows_kernel<MB, TO>, mw, mx, a);
    return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: launch failed: %s", cudaGetErrorString(e));
}

template <typename TO>
s2_status launch_tile(const LinearArgs &a, int sms, const void *x, long long ldx, const void *w, long long ldw,
                      cudaStream_t st)
{
    CUtensorMap mx, mw;
    if (!s2::make_map_2d(&mx, x, a.K, a.M, ldx * 2, kBK, kTileHalf) ||
        !s2::make_map_2d(&mw, w, a.K, a.N, ldw * 2, kBK, kTileHalf))
        return s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: cuTensorMapEncodeTiled failed");
    // slabs of y and of the residual: 32 rows x 128 bytes, swizzled (16-bit maps move any 16-bit type)
    auto slab_map = [&](CUtensorMap *map, const void *ptr, long long ld) {
        return sizeof(TO) == 4 ? s2::make_map_2d_plain_f32(map, ptr, a.N, a.M, ld * 4, 32, 32)
                               : s2::make_map_2d(map, ptr, a.N, a.M, ld * 2, 64, 32);
    };
    CUtensorMap my = mx, mr = mx;  // unused ones repeat a valid map
    if (a.vec && (!slab_map(&my, a.y, a.ldy) || (a.residual && !slab_map(&mr, a.residual, a.ldr))))
        return s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: cuTensorMapEncodeTiled failed");
    static std::atomic<uint64_t> configured{0};
    const s2_status cs = s2::once_per_device(configured, [] {
        const cudaError_t e = cudaFuncSetAttribute(linear_tile_kernel<TO>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   Tile::kSmemBytes);
        return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: %s", cudaGetErrorString(e));
    });
    if (cs != S2_OK) return cs;
    const long long tiles = (a.M + 255) / 256 * ((a.N + kTileN - 1) / kTileN);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(2 * std::min<long long>(tiles, sms / 2)));
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = Tile::kSmemBytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = a.packed ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, linear_tile_kernel<TO>, mx, mw, mr, my, a);
    return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: launch failed: %s", cudaGetErrorString(e));
}

template <typename TO>
s2_status launch_linear(const LinearArgs &a, int sms, const void *x, long long ldx, const void *w, long long ldw,
                        cudaStream_t st)
{
    const int mb = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 64 ? 64 : 128;
    const long long ctas = (a.N + kRowsN - 1LL) / kRowsN * ((a.M + mb - 1) / mb);
    const int n_k = (a.K + kBK - 1) / kBK;
    // CTAs that share a tile's K: as many as two an SM have room for, two slices each at least
    int ks = 8;
    while (ks > 1 && (ctas * ks > 2LL * sms || n_k < 2 * ks)) ks /= 2;
    // More than 128 rows of x go to the 256 x 256 tiles, unless K is long and these tiles leave so much of the
    // GPU idle that its split pays: 200 x 2560 x 5120 17.6 us in rows against 30.4 in tiles, 800 26.5 / 31.1,
    // 800 x 777 x 1000 13.6 / 21.8, but without a split 1237 x 2560 x 5120 41.0 / 31.7, and with a short K
    // 1237 x 512 x 512 10.8 / 8.6. (Near the border either may win by a tenth: 1000 x 512 x 896 9.7 / 10.8, 1000 x 512 x
    // 1024 12.9 / 11.5.)
    if (a.M > 128 && (ks == 1 || n_k < 16)) {
        if ((a.M + 255) / 256 * ((a.N + kTileN - 1) / kTileN) > (1LL << 30))
            return s2::set_error(S2_UNSUPPORTED, "s2_linear_act: too many tiles");
        return launch_tile<TO>(a, sms, x, ldx, w, ldw, st);
    }
    switch (mb) {
    case 16: return launch_rows<16, TO>(a, ks, x, ldx, w, ldw, st);
    case 32: return launch_rows<32, TO>(a, ks, x, ldx, w, ldw, st);
    case 64: return launch_rows<64, TO>(a, ks, x, ldx, w, ldw, st);
    default: return launch_rows<128, TO>(a, ks, x, ldx, w, ldw, st);
    }
}

s2_status check(const s2_linear_act_desc *d)
{
    if (!d) return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: NULL description");
    if (d->M < 0 || d->N <= 0 || d->K <= 0)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: bad shape (M %lld, N %d, K %d)", d->M, d->N, d->K);
    if (d->M > (1LL << 30) || d->N > (1 << 21) || d->K > (1 << 21))
        return s2::set_error(S2_UNSUPPORTED, "s2_linear_act: at most 2^30 rows, 2^21 columns and 2^21 products a sum");
    if ((d->dtype != S2_F16 && d->dtype != S2_BF16) || (d->out_dtype != d->dtype && d->out_dtype != S2_F32))
        return s2::set_error(S2_UNSUPPORTED, "s2_linear_act: dtypes %d -> %d (fp16 or bf16 to the same or fp32)",
                             d->dtype, d->out_dtype);
    if (d->activation < S2_ACT_NONE || d->activation > S2_ACT_GELU_TANH)
        return s2::set_error(S2_UNSUPPORTED, "s2_linear_act: unknown activation %d", d->activation);
    return S2_OK;
}

size_t workspace_of(const s2_linear_act_desc &d)
{
    if (d.M <= 1) return 0;
    size_t need = 0;
    if (!tma_ready(d.x, d.ldx, d.M)) need += static_cast<size_t>(d.M) * round_up8(d.K) * 2;
    if (!tma_ready(d.w, d.ldw, d.N)) need += static_cast<size_t>(d.N) * round_up8(d.K) * 2;
    return need;
}

s2_status check_operands(const s2_linear_act_desc &d, size_t workspace)
{
    const uintptr_t oe = d.out_dtype == S2_F32 ? 4 : 2;
    if (!d.x || !d.w || !d.y) return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: NULL x, w or y");
    if ((reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.w)) % 2 ||
        (reinterpret_cast<uintptr_t>(d.y) | reinterpret_cast<uintptr_t>(d.residual)) % oe ||
        reinterpret_cast<uintptr_t>(d.bias) % 4)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: a pointer is not aligned to its elements");
    const long long top = 1LL << 40;
    if (d.ldx < d.K || d.ldw < d.K || d.ldy < d.N || (d.residual && d.ldr < d.N))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: a pitch is smaller than its row");
    if (d.ldx > top || d.ldw > top || d.ldy > top || (d.residual && d.ldr > top))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: a pitch beyond any memory");
    const s2::PitchedSpan y{d.y, d.M, static_cast<long long>(d.N * oe), static_cast<long long>(d.ldy * oe)};
    const s2::PitchedSpan r{d.residual, d.M, static_cast<long long>(d.N * oe), static_cast<long long>(d.ldr * oe)};
    const s2::PitchedSpan x{d.x, d.M, 2LL * d.K, 2 * d.ldx}, w{d.w, d.N, 2LL * d.K, 2 * d.ldw}, b = s2::bytes_at(d.bias, 4LL * d.N);
    const bool in_place = d.residual == d.y && d.ldr == d.ldy;
    if (s2::may_overlap(y, x) || s2::may_overlap(y, w) || s2::may_overlap(y, b) || (!in_place && s2::may_overlap(y, r)))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: y overlaps an input");
    if (workspace == 0) return S2_OK;
    if (!d.workspace || d.workspace_bytes < workspace || reinterpret_cast<uintptr_t>(d.workspace) % 16)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: workspace of %zu bytes, 16-byte aligned, needed", workspace);
    const s2::PitchedSpan work = s2::bytes_at(d.workspace, static_cast<long long>(workspace));
    if (s2::may_overlap(work, x) || s2::may_overlap(work, w) || s2::may_overlap(work, b) || s2::may_overlap(work, r) ||
        s2::may_overlap(work, y))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: the workspace overlaps an operand");
    return S2_OK;
}

}  // namespace

extern "C" size_t s2_linear_act_workspace_bytes(const s2_linear_act_desc *d)
{
    s2::clear_error();
    return check(d) == S2_OK ? workspace_of(*d) : 0;
}

extern "C" s2_status s2_linear_act(void *stream, const s2_linear_act_desc *d, int *launches)
{
    s2::clear_error();
    if (launches) *launches = 0;
    s2_status s = check(d);
    if (s != S2_OK) return s;
    if (d->M == 0) return S2_OK;
    if ((s = check_operands(*d, workspace_of(*d))) != S2_OK) return s;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    LinearArgs a;
    a.bias = d->bias;
    a.residual = d->residual;
    a.y = d->y;
    a.M = d->M;
    a.ldr = d->ldr;
    a.ldy = d->ldy;
    a.N = d->N;
    a.K = d->K;
    a.act = d->activation;
    a.fmt = d->dtype == S2_BF16 ? 1u : 0u;
    const uintptr_t oe = d->out_dtype == S2_F32 ? 4 : 2;
    a.vec = (reinterpret_cast<uintptr_t>(d->y) | d->ldy * oe | reinterpret_cast<uintptr_t>(d->residual) |
             (d->residual ? d->ldr * oe : 0)) % 16 == 0;
    a.ks = 1;
    a.packed = 0;
    a.err = d->err ? d->err : s2::operator_error_word();
    int dev = 0, sms = 148;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    int count = 0;
    if (d->M <= 1) {
        const bool f32 = d->out_dtype == S2_F32;
        if (d->dtype == S2_F16)
            s = f32 ? launch_vec<__half, float>(a, sms, *d, st) : launch_vec<__half, __half>(a, sms, *d, st);
        else
            s = f32 ? launch_vec<__nv_bfloat16, float>(a, sms, *d, st)
                    : launch_vec<__nv_bfloat16, __nv_bfloat16>(a, sms, *d, st);
    } else {
        uint16_t *ws = static_cast<uint16_t *>(d->workspace);
        // an operand as TMA reads it: in place, or packed
        auto operand = [&](const void *p, long long ld, long long rows, const void **out, long long *ldo) {
            *out = p;
            *ldo = rows == 1 ? round_up8(d->K) : ld;
            if (tma_ready(p, ld, rows)) return;
            *ldo = round_up8(d->K);
            pack_rows_kernel<<<static_cast<unsigned>(std::min<long long>((rows * *ldo / 8 + 255) / 256, 1 << 20)), 256, 0, st>>>(
                static_cast<const uint16_t *>(p), ld, rows, d->K, ws, *ldo);
            *out = ws;
            ws += rows * *ldo;
            ++count;
        };
        const void *x, *w;
        long long ldx, ldw;
        operand(d->x, d->ldx, d->M, &x, &ldx);
        operand(d->w, d->ldw, d->N, &w, &ldw);
        a.packed = count > 0;
        s = d->out_dtype == S2_F32   ? launch_linear<float>(a, sms, x, ldx, w, ldw, st)
            : d->out_dtype == S2_F16 ? launch_linear<__half>(a, sms, x, ldx, w, ldw, st)
                                     : launch_linear<__nv_bfloat16>(a, sms, x, ldx, w, ldw, st);
    }
    if (s != S2_OK) return s;
    if (launches) *launches = count + 1;
    return S2_OK;
}
