// Group norm with an activation over channels-last activations (s2_group_norm_act).
//
// x [S][P][C], G groups of C / G consecutive channels. Per sample s and group g, over the
// n = P C / G values of the group:
//   m = sum x / n,  v = sum (x - m)^2 / n,  y = act((x - m) / sqrt(v + eps) * w[c] + b[c]).
//
// Statistics: a thread keeps one vector of channels and walks down the rows. It sums d = x - p
// and d^2 about a pivot p of its own (the first value of each run of 8 rows) in fp32 and turns
// every run into (count, mean, M2 = sum of squares about the mean); runs, threads and blocks are
// joined by
//   m = ma + (mb - ma) nb / n,   M2 = M2a + M2b + (mb - ma)^2 na nb / n,
// which loses nothing when the mean is far larger than the spread, and an outlier only reaches
// the run that holds it. What is joined with what depends on the shape alone, never on timing.
//
// A unit (a slice of the groups of one sample) is shared by a team of blocks. The least to read and write is x
// and y once (6.5 TB/s); the statistics stand between the two, so what counts is to hold what was read, and to
// read the next while the last is joined and written. Three kernels:
//  * group_norm_slab_kernel, aligned rows: teams of blocks hold narrow slices in shared memory, several at a
//    time, and load, sum, join and write different ones at once. One read, 4 to 4.9 TB/s.
//  * group_norm_held_kernel: the blocks read their rows into shared memory while they sum them, and write the
//    output from there, one step after the other. For units too small to be worth the above: the blocks of a
//    cluster hold one and exchange their moments through distributed shared memory, without a workspace. And
//    for rows that do not start on 16 bytes, also on a cooperative grid, where rows not held are read twice.
//  * group_norm_ring_kernel, aligned rows of samples too large for the first (four slices of 64 bytes a row do not fit
//    the GPU's shared memory: beyond about 125000 positions, 8 MB a slice): a loading warp streams the rows through a
//    ring of slots with bulk copies, so that the memory never waits for the threads that sum and write; all but what
//    the ring holds at the end of the statistics is read twice.
#include <cuda_runtime.h>

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

constexpr int kThreads = 256;
constexpr int kMaxGroups = 1024;
constexpr int kSliceGroups = 64;  // groups of one unit
constexpr int kMaxCluster = 8;
constexpr int kAhead = 8;         // vectors a thread has in flight while it sums, and the rows of a run
constexpr int kBatch = 4;         // ... while it writes

// How the parts of a unit exchange their moments.
enum Join : int {
    kAlone = 0,    // one block
    kCluster = 1,  // the blocks of a cluster, through distributed shared memory
    kGrid = 2,     // blocks of a cooperative grid, through the workspace
};

// `parts` blocks share a unit, `part_rows` rows each (the last ones fewer); `teams` of them take the units
// in turn.
struct GnArgs {
    const void *x;
    void *y;
    const float *weight, *bias;
    int32_t *err;
    long long P, part_rows, x_row, x_sample, y_row, y_sample;
    int C, G, cpg, slices, slice_groups, units, parts, teams, join, hold, act;
    int group_lanes;  // threads that join one group's moments: a power of two up to 32
    // group_norm_slab_kernel: units that a block holds, boxes of rows of one; `direct`: every block joins the
    // parts for itself, join_lanes lanes a group
    int buffers, boxes, box_rows, direct, join_lanes;
    float eps;
    // a grid's: (mean, M2) per [unit][part][group], (mean, 1 / sigma) per [unit][group]; counters, zero
    // before: parts whose moments are written, units whose norm is. group_norm_slab_kernel has no counters: its
    // moments, [unit][group][part], and norms have all bits set until they are written
    float2 *part, *norm;
    uint32_t *arrived, *ready;
    unsigned long long join_ns;  // how long a wait for the other parts may take
};

struct Moments {
    float n, mean, m2;
};

// Both may be empty; the moments of one alone come through unchanged. The reciprocal is the hardware's
// (1 ulp): it weighs a difference of means, which is 0 for equal ones.
__device__ __forceinline__ Moments join(const Moments &a, const Moments &b)
{
    Moments r;
    r.n = a.n + b.n;
    const float w = __fdividef(b.n, r.n), d = b.mean - a.mean;
    const bool both = a.n > 0.f && b.n > 0.f;
    r.mean = both ? fmaf(d, w, a.mean) : (b.n > 0.f ? b.mean : a.mean);
    r.m2 = both ? fmaf(d * d, a.n * w, a.m2 + b.m2) : a.m2 + b.m2;
    return r;
}

// The sum over `lanes` neighbouring threads, in all of them.
__device__ __forceinline__ float sum_lanes(float v, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// `lanes` neighbouring threads' moments in the first of them.
__device__ __forceinline__ Moments join_lanes(Moments m, int lanes)
{
    for (int o = lanes >> 1; o > 0; o >>= 1) {
        Moments t;
        t.n = __shfl_down_sync(0xffffffffu, m.n, o);
        t.mean = __shfl_down_sync(0xffffffffu, m.mean, o);
        t.m2 = __shfl_down_sync(0xffffffffu, m.m2, o);
        m = join(m, t);
    }
    return m;
}

// Moments of group `sub` of a slice over `parts` parts of `rows` rows each (`total` in all), by group_lanes
// threads a group (sub_lane of them): in the first of these. Eight are asked for at a time, in four chains.
template <bool kGlobal>
__device__ __noinline__ Moments join_parts(const float2 *part, int pitch, int parts, long long rows, long long total,
                                           int cpg, int group_lanes, int sub, int sub_lane, int gs)
{
    Moments chain[4] = {};
    if (sub < gs)
        for (int t0 = sub_lane; t0 < parts; t0 += 8 * group_lanes) {
            float2 q[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int t = t0 + k * group_lanes;
                if (t < parts) q[k] = kGlobal ? __ldcg(part + t * pitch + sub) : part[t * pitch + sub];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int t = t0 + k * group_lanes;
                if (t < parts) {
                    Moments o;
                    o.n = static_cast<float>(max(0LL, min(rows, total - t * rows)) * cpg);
                    o.mean = q[k].x;
                    o.m2 = q[k].y;
                    chain[k & 3] = join(chain[k & 3], o);
                }
            }
        }
    return join_lanes(join(join(chain[0], chain[1]), join(chain[2], chain[3])), group_lanes);
}

// mean and 1 / sigma of a group; 1 / sigma is NaN, and with it the group's output, where the squares have
// overflowed (1 / sqrt(inf) = 0 would make it act(bias))
__device__ __forceinline__ float2 norm_of(const Moments &m, float eps)
{
    const float v = __fdiv_rn(m.m2, m.n);
    return make_float2(m.mean, v <= 3.402823466e38f ? __frsqrt_rn(v + eps) : __int_as_float(0x7fffffff));
}

// VEC elements of T as they are loaded: 16 bytes or one element
template <typename T, int VEC>
struct Raw {
    using type = uint4;
    static __device__ __forceinline__ uint4 load(const T *p, uint64_t policy)
    {
        uint4 v;
        asm volatile("ld.global.L1::no_allocate.L2::cache_hint.v4.u32 {%0, %1, %2, %3}, [%4], %5;"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(p), "l"(policy)
                     : "memory");
        return v;
    }
    static __device__ __forceinline__ void floats(const uint4 &v, float (&f)[VEC])
    {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
        if constexpr (sizeof(T) == 4) {
            static_assert(VEC == 4, "");
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(u[i]);
        } else {
            static_assert(VEC == 8, "");
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 t = unpack2<T>(u[i]);
                f[2 * i] = t.x;
                f[2 * i + 1] = t.y;
            }
        }
    }
};
template <typename T>
struct Raw<T, 1> {
    using type = T;
    static __device__ __forceinline__ T load(const T *p, uint64_t) { return *p; }
    static __device__ __forceinline__ void floats(T v, float (&f)[1]) { f[0] = to_float<T>(v); }
};

// y is not read again here: its lines leave L2 first
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&f)[VEC])
{
    if constexpr (VEC == 1) {
        *p = from_float<T>(f[0]);
    } else if constexpr (sizeof(T) == 4) {
        __stcs(reinterpret_cast<float4 *>(p), make_float4(f[0], f[1], f[2], f[3]));
    } else if constexpr (VEC == 8) {
        __stcs(reinterpret_cast<uint4 *>(p),
               make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7])));
    } else {
        __stcs(reinterpret_cast<uint2 *>(p), make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3])));
    }
}

// A run of vectors of one column, summed about its first: N moments a vector, of VEC / N channels each that
// belong to one group.
template <typename TI, int VEC, int N>
struct Run {
    using R = Raw<TI, VEC>;
    static constexpr int kPer = VEC / N, kPairs = VEC / 2, kSums = N == 1 ? (VEC > 2 ? 2 : 1) : kPairs;
    float p[N];
    uint64_t minus[N == 1 ? 1 : kPairs], s2[kSums], q2[kSums];
    __device__ __forceinline__ Run(const typename R::type &first)
    {
        float f[VEC];
        R::floats(first, f);
#pragma unroll
        for (int e = 0; e < N; ++e) p[e] = f[e * kPer];
#pragma unroll
        for (int k = 0; k < (N == 1 ? 1 : kPairs); ++k)
            minus[k] = pair(-p[N == 1 ? 0 : 2 * k / kPer], -p[N == 1 ? 0 : (2 * k + 1) / kPer]);
#pragma unroll
        for (int k = 0; k < kSums; ++k) s2[k] = q2[k] = 0;
    }
    __device__ __forceinline__ void add(const typename R::type &v)
    {
        float f[VEC];
        R::floats(v, f);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            const uint64_t d = add2(pair(f[2 * k], f[2 * k + 1]), minus[N == 1 ? 0 : k]);
            s2[k % kSums] = add2(s2[k % kSums], d);
            q2[k % kSums] = fma2(d, d, q2[k % kSums]);
        }
    }
    // joins the run's `n` vectors to mo
    __device__ __forceinline__ void end(int n, Moments (&mo)[N]) const
    {
        float sum[N], sq[N];
#pragma unroll
        for (int e = 0; e < N; ++e) sum[e] = sq[e] = 0.f;
#pragma unroll
        for (int k = 0; k < kSums; ++k) {
            const float2 b = floats_of(s2[k]), c = floats_of(q2[k]);
            const int e0 = N == 1 ? 0 : 2 * k / kPer, e1 = N == 1 ? 0 : (2 * k + 1) / kPer;
            sum[e0] += b.x;
            sum[e1] += b.y;
            sq[e0] += c.x;
            sq[e1] += c.y;
        }
        const float cnt = static_cast<float>(n * kPer), inv = __fdividef(1.f, cnt);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            Moments run;
            run.n = cnt;
            run.mean = fmaf(sum[e], inv, p[e]);
            // not below 0 by rounding; 0 * sq keeps the NaN of a value that is not finite (squares that overflow
            // leave inf)
            run.m2 = fmaxf(fmaf(-sum[e] * inv, sum[e], sq[e]), 0.f * sq[e]);
            mo[e] = join(mo[e], run);
        }
    }
};
template <typename TI>
struct Run<TI, 1, 1> {
    float p, sum = 0.f, sq = 0.f;
    __device__ __forceinline__ Run(const TI &first) { p = to_float<TI>(first); }
    __device__ __forceinline__ void add(const TI &v)
    {
        const float d = to_float<TI>(v) - p;
        sum += d;
        sq = fmaf(d, d, sq);
    }
    __device__ __forceinline__ void end(int n, Moments (&mo)[1]) const
    {
        const float cnt = static_cast<float>(n), inv = __fdividef(1.f, cnt);
        mo[0] = join(mo[0], Moments{cnt, fmaf(sum, inv, p), fmaxf(fmaf(-sum * inv, sum, sq), 0.f * sq)});
    }
};

// The moments of a thread's `count` vectors, `step` elements apart; the first `hold` stay in shared memory.
template <typename TI, int VEC, int N>
__device__ __forceinline__ void read_rows(const TI *px, long long step, int count, uint64_t policy, int hold,
                                          typename Raw<TI, VEC>::type *held, Moments (&mo)[N])
{
    using R = Raw<TI, VEC>;
    typename R::type v[kAhead];
    int i = 0;
#pragma unroll 1
    for (; i + kAhead <= count; i += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u, px += step) v[u] = R::load(px, policy);
        if (i + kAhead <= hold) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u) held[(i + u) * kThreads] = v[u];
        } else if (i < hold) {
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (i + u < hold) held[(i + u) * kThreads] = v[u];
        }
        Run<TI, VEC, N> run(v[0]);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) run.add(v[u]);
        run.end(kAhead, mo);
    }
    if (i < count) {
        const int n = count - i;
#pragma unroll
        for (int u = 0; u < kAhead; ++u, px += step)
            if (u < n) v[u] = R::load(px, policy);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u < n && i + u < hold) held[(i + u) * kThreads] = v[u];
        Run<TI, VEC, N> run(v[0]);
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u < n) run.add(v[u]);
        run.end(n, mo);
    }
}

// Columns of vectors of a unit that a block works on at a time (all, unless a single group is wider than
// the block), and a thread's place: one column, every lanes-th row.
struct Place {
    int nb, lanes, col, rl, count;
};
__device__ __forceinline__ Place place_of(int cb, int ncols, long long rows)
{
    Place p;
    p.nb = min(kThreads, ncols - cb);
    p.lanes = kThreads / p.nb;
    p.rl = static_cast<int>(threadIdx.x) / p.nb;
    p.col = cb + static_cast<int>(threadIdx.x) - p.rl * p.nb;
    p.count = p.rl < p.lanes && p.rl < rows ? static_cast<int>((rows - p.rl + p.lanes - 1) / p.lanes) : 0;
    return p;
}

// The block's moments of a unit's groups, from its threads'.
template <int N>
struct BlockMoments {
    float2 entry[N][kThreads];  // (mean, M2) a thread and moment, and of how many values
    float n[kThreads];
    Moments group[kSliceGroups];
};

// The moments of group `sub` over the block's threads at the columns from cb, in the thread of sub_lane 0. Ends
// without a barrier. `sync` is the barrier of the kThreads threads.
template <int VEC, int N, typename Sync>
__device__ __forceinline__ Moments block_moments(BlockMoments<N> &s, Moments (&mo)[N], const Place &p, int cb, int cpg,
                                                 int gs, int group_lanes, int sub, int sub_lane, Sync sync)
{
    sync();
#pragma unroll
    for (int e = 0; e < N; ++e) s.entry[e][threadIdx.x] = make_float2(mo[e].mean, mo[e].m2);
    s.n[threadIdx.x] = mo[0].n;
    sync();
    // down the rows: halves of the row lanes joined until one is left
    for (int left = p.lanes; left > 1;) {
        const int half = (left + 1) / 2;
        if (p.rl + half < left) {
            const int other = threadIdx.x + half * p.nb;
            const float n = s.n[other];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float2 q = s.entry[e][other];
                Moments t;
                t.n = n;
                t.mean = q.x;
                t.m2 = q.y;
                mo[e] = join(mo[e], t);
                s.entry[e][threadIdx.x] = make_float2(mo[e].mean, mo[e].m2);
            }
            s.n[threadIdx.x] = mo[0].n;
        }
        left = half;
        sync();
    }
    // across each group's moments along a row
    constexpr int kPer = VEC / N;
    Moments m = {0.f, 0.f, 0.f};
    if (sub < gs) {
        const int lo = max(sub * cpg / kPer, cb * N), end = min((sub + 1) * cpg / kPer, (cb + p.nb) * N);
        for (int k = lo + sub_lane; k < end; k += group_lanes) {
            const float2 q = s.entry[k % N][k / N - cb];
            Moments t;
            t.n = s.n[0];
            t.mean = q.x;
            t.m2 = q.y;
            m = join(m, t);
        }
    }
    return join_lanes(m, group_lanes);
}

// Joins them to s.group[].
template <int VEC, int N, typename Sync>
__device__ __forceinline__ void join_block(BlockMoments<N> &s, Moments (&mo)[N], const Place &p, int cb, int cpg, int gs,
                                           int group_lanes, int sub, int sub_lane, Sync sync)
{
    const Moments m = block_moments<VEC, N>(s, mo, p, cb, cpg, gs, group_lanes, sub, sub_lane, sync);
    if (sub_lane == 0 && sub < gs) s.group[sub] = join(s.group[sub], m);
}

// y = act((x - mean) scale + shift) of one vector; `minus` is -mean, one for VEC / N channels each. The
// subtraction comes first, as in the formula: values that all equal the mean give the shift itself.
template <typename TI, typename TO, int VEC, int N, int kAct>
__device__ __forceinline__ void finish(const typename Raw<TI, VEC>::type &v, TO *py, const float (&minus)[N],
                                       const float (&scale)[VEC], const float (&shift)[VEC])
{
    float f[VEC];
    Raw<TI, VEC>::floats(v, f);
    if constexpr (VEC == 1) {
        f[0] = activate<kAct>(fmaf(f[0] + minus[0], scale[0], shift[0]));
    } else {
#pragma unroll
        for (int k = 0; k < VEC / 2; ++k) {
            const uint64_t d = add2(pair(f[2 * k], f[2 * k + 1]), pair(minus[2 * k / (VEC / N)], minus[(2 * k + 1) / (VEC / N)]));
            const float2 r = floats_of(activate2<kAct>(
                fma2(d, pair(scale[2 * k], scale[2 * k + 1]), pair(shift[2 * k], shift[2 * k + 1]))));
            f[2 * k] = r.x;
            f[2 * k + 1] = r.y;
        }
    }
    store_vec<TO, VEC>(py, f);
}

// y of a thread's `count` vectors, the first `hold` of them from shared memory.
template <typename TI, typename TO, int VEC, int N, int kAct>
__device__ __forceinline__ void write_rows(const TI *px, long long x_step, TO *py, long long y_step, int count,
                                           uint64_t policy, int hold, const typename Raw<TI, VEC>::type *held,
                                           const float (&minus)[N], const float (&scale)[VEC], const float (&shift)[VEC])
{
    using R = Raw<TI, VEC>;
    const int kept = min(count, hold);
#pragma unroll 2
    for (int k = 0; k < kept; ++k, py += y_step) finish<TI, TO, VEC, N, kAct>(held[k * kThreads], py, minus, scale, shift);
    px += kept * x_step;
    int i = kept;
#pragma unroll 1
    for (; i + kBatch <= count; i += kBatch) {
        typename R::type v[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; ++u, px += x_step) v[u] = R::load(px, policy);
#pragma unroll
        for (int u = 0; u < kBatch; ++u, py += y_step) finish<TI, TO, VEC, N, kAct>(v[u], py, minus, scale, shift);
    }
#pragma unroll 1
    for (; i < count; ++i, px += x_step, py += y_step)
        finish<TI, TO, VEC, N, kAct>(R::load(px, policy), py, minus, scale, shift);
}

// What the output does to the channels of a unit's column `col`; the unit's channels begin at c0, norm[g]:
// mean and 1 / sigma.
template <int VEC, int N>
__device__ __forceinline__ void affine_of(const GnArgs &a, int col, int c0, const float2 *norm, float (&minus)[N],
                                          float (&scale)[VEC], float (&shift)[VEC])
{
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float2 mr = norm[(col * VEC + e * (VEC / N)) / a.cpg];
        minus[e] = -mr.x;
#pragma unroll
        for (int k = 0; k < VEC / N; ++k) {
            const int i = e * (VEC / N) + k, c = c0 + col * VEC + i;
            scale[i] = a.weight ? mr.y * __ldg(a.weight + c) : mr.y;
            shift[i] = a.bias ? __ldg(a.bias + c) : 0.f;
        }
    }
}

// Output of a thread's column of a unit.
template <typename TI, typename TO, int VEC, int N>
__device__ __forceinline__ void write_column(const GnArgs &a, const Place &p, int c0, const float2 *norm, const TI *px,
                                             TO *py, uint64_t policy, int hold, const typename Raw<TI, VEC>::type *held)
{
    float minus[N], scale[VEC], shift[VEC];
    affine_of<VEC, N>(a, p.col, c0, norm, minus, scale, shift);
    const long long xs = p.lanes * a.x_row, ys = p.lanes * a.y_row;
    switch (a.act) {
    case S2_ACT_RELU:
        write_rows<TI, TO, VEC, N, S2_ACT_RELU>(px, xs, py, ys, p.count, policy, hold, held, minus, scale, shift);
        break;
    case S2_ACT_SILU:
        write_rows<TI, TO, VEC, N, S2_ACT_SILU>(px, xs, py, ys, p.count, policy, hold, held, minus, scale, shift);
        break;
    case S2_ACT_GELU:
        write_rows<TI, TO, VEC, N, S2_ACT_GELU>(px, xs, py, ys, p.count, policy, hold, held, minus, scale, shift);
        break;
    case S2_ACT_GELU_TANH:
        write_rows<TI, TO, VEC, N, S2_ACT_GELU_TANH>(px, xs, py, ys, p.count, policy, hold, held, minus, scale, shift);
        break;
    default: write_rows<TI, TO, VEC, N, S2_ACT_NONE>(px, xs, py, ys, p.count, policy, hold, held, minus, scale, shift);
    }
}

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t *p)
{
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// device error codes: the wait for the other parts of a unit, for the ring's loads
enum : int { E_JOIN = 96, E_RING = 97 };

// Waits until *p is `value`; for `most` ns, and *stop ends it.
__device__ __forceinline__ bool wait_value(const uint32_t *p, uint32_t value, volatile int *stop, int32_t *err, uint64_t most)
{
    if (ld_acquire(p) == value) return true;
    const uint64_t t0 = global_timer_ns();
    while (ld_acquire(p) != value)
        if (*stop || global_timer_ns() - t0 > most) {
            if (err) atomicCAS(err, 0, E_JOIN);
            *stop = 1;
            return false;
        }
    return true;
}

// The parts of a unit on a grid join their moments (group[], gs of them): each writes its own, the last to
// arrive joins all of them and publishes the unit's mean and 1 / sigma, the others wait for these. `sync` is
// the barrier of the threads that call this; *stop ends the wait, which is bounded. On return norm[] holds
// the unit's.
template <typename Sync>
__device__ __forceinline__ void join_grid(const GnArgs &a, int unit, int member, const Moments *group, int gs, int sub,
                                          int sub_lane, float2 *norm, volatile int *last, volatile int *stop, Sync sync)
{
    const long long at = static_cast<long long>(unit) * a.parts;
    if (threadIdx.x < gs)
        __stcg(a.part + (at + member) * a.slice_groups + threadIdx.x, make_float2(group[threadIdx.x].mean, group[threadIdx.x].m2));
    sync();
    if (threadIdx.x == 0) {
        __threadfence();
        *last = atomicAdd(a.arrived + unit, 1u) == static_cast<uint32_t>(a.parts) - 1;
        __threadfence();
    }
    sync();
    float2 *joined = a.norm + static_cast<long long>(unit) * a.slice_groups;
    if (*last) {
        const Moments m = join_parts<true>(a.part + at * a.slice_groups, a.slice_groups, a.parts, a.part_rows, a.P, a.cpg,
                                           a.group_lanes, sub, sub_lane, gs);
        if (sub_lane == 0 && sub < gs) {
            norm[sub] = norm_of(m, a.eps);
            __stcg(joined + sub, norm[sub]);
        }
        sync();
        if (threadIdx.x == 0) {
            __threadfence();
            atomicExch(a.ready + unit, 1u);
        }
    } else {
        if (threadIdx.x == 0) wait_value(a.ready + unit, 1, stop, a.err, a.join_ns);
        sync();
        if (threadIdx.x < gs) norm[threadIdx.x] = __ldcg(joined + threadIdx.x);
        sync();
    }
}

// ---- rows held by the blocks ---------------------------------------------------------

// Bound by its steps, one after the other (start, read, exchange, write): 3 x 7973 x 96 fp32 with rows of 101 values,
// one at a time, 15.6 us from memory (13.3 when L2 has x); 2 x 1920 x 512 fp16 on clusters 9.3 us.
template <typename TI, typename TO, int VEC, int N>
__global__ void __launch_bounds__(kThreads, 2) group_norm_held_kernel(const GnArgs a)
{
    extern __shared__ uint4 held_raw[];
    __shared__ BlockMoments<N> s;
    __shared__ float2 received[kMaxCluster][kSliceGroups], norm[kSliceGroups];
    __shared__ int last, stop;
    auto *held = reinterpret_cast<typename Raw<TI, VEC>::type *>(held_raw) + threadIdx.x;
    const int team = static_cast<int>(blockIdx.x) / a.parts, member = static_cast<int>(blockIdx.x) - team * a.parts;
    const int sub = static_cast<int>(threadIdx.x) / a.group_lanes, sub_lane = threadIdx.x % a.group_lanes;
    if (threadIdx.x == 0) stop = 0;
    if (a.join == kCluster) cluster_arrive();  // waited for below: no block writes to one that has not begun
    const long long r0 = member * a.part_rows, rows = max(0LL, min(a.part_rows, a.P - r0));
    const uint64_t policy = l2_evict_first();
    for (int unit = team; unit < a.units; unit += a.teams) {  // a cluster has one unit
        const int smp = unit / a.slices, g0 = (unit - smp * a.slices) * a.slice_groups;
        const int gs = min(a.slice_groups, a.G - g0), c0 = g0 * a.cpg, ncols = gs * a.cpg / VEC;
        const TI *x = static_cast<const TI *>(a.x) + smp * a.x_sample + r0 * a.x_row + c0;
        TO *y = static_cast<TO *>(a.y) + smp * a.y_sample + r0 * a.y_row + c0;
        if (threadIdx.x < gs) s.group[threadIdx.x] = Moments{0.f, 0.f, 0.f};
        Place p;
        for (int cb = 0; cb < ncols; cb += kThreads) {
            p = place_of(cb, ncols, rows);
            Moments mo[N] = {};
            read_rows<TI, VEC, N>(x + p.rl * a.x_row + static_cast<long long>(p.col) * VEC, p.lanes * a.x_row, p.count, policy,
                                  a.hold, held, mo);
            join_block<VEC, N>(s, mo, p, cb, a.cpg, gs, a.group_lanes, sub, sub_lane, [] { __syncthreads(); });
        }
        __syncthreads();
        if (a.join == kGrid) {
            join_grid(a, unit, member, s.group, gs, sub, sub_lane, norm, &last, &stop, [] { __syncthreads(); });
            if (stop) return;
        } else if (a.join == kCluster) {
            cluster_wait();
            for (int i = threadIdx.x; i < kSliceGroups * a.parts; i += kThreads) {
                const int to = i / kSliceGroups, g = i % kSliceGroups;
                if (g < gs) {
                    const uint32_t at = cluster_map(smem_u32(&received[member][g]), static_cast<uint32_t>(to));
                    st_cluster_b32(at, __float_as_uint(s.group[g].mean));
                    st_cluster_b32(at + 4, __float_as_uint(s.group[g].m2));
                }
            }
            __syncwarp();
            cluster_sync();
            const Moments m = join_parts<false>(&received[0][0], kSliceGroups, a.parts, a.part_rows, a.P, a.cpg,
                                                a.group_lanes, sub, sub_lane, gs);
            if (sub_lane == 0 && sub < gs) norm[sub] = norm_of(m, a.eps);
        } else if (threadIdx.x < gs) {
            norm[threadIdx.x] = norm_of(s.group[threadIdx.x], a.eps);
        }
        __syncthreads();
        for (int cb = 0; cb < ncols; cb += kThreads) {
            if (ncols > kThreads) p = place_of(cb, ncols, rows);
            if (p.count > 0)
                write_column<TI, TO, VEC, N>(a, p, c0, norm, x + p.rl * a.x_row + static_cast<long long>(p.col) * VEC,
                                             y + p.rl * a.y_row + static_cast<long long>(p.col) * VEC, policy, a.hold, held);
        }
        __syncthreads();  // the next unit reuses the moments
    }
}

// ---- rows through a ring ---------------------------------------------------------------

constexpr int kSlotPasses = 4;  // rows a thread has in a slot
constexpr int kRunSlots = kAhead / kSlotPasses;
constexpr uint32_t kSlotBytes = kSlotPasses * kThreads * 16;
// 16 bytes written by copies that the compiler does not see, so that the load is spelled out
__device__ __forceinline__ uint4 ld_shared(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// Slots beside the moments, of two blocks an SM.
template <int N>
__host__ __device__ constexpr int ring_slots()
{
    return N == 8 ? 5 : 6;
}

// A part's slots over one unit: slot i holds the unit's rows [i * rows, (i + 1) * rows) of the part.
struct Slots {
    int lanes, rows;  // rows of a pass, of a slot
    int total, held;  // held: the last ones stay in the ring from the statistics to the output
};

template <int kSlots>
__device__ __forceinline__ Slots slots_of(long long rows, int ncols)
{
    Slots p;
    p.lanes = kThreads / ncols;
    p.rows = kSlotPasses * p.lanes;
    p.total = static_cast<int>((rows + p.rows - 1) / p.rows);
    p.held = min(p.total, kSlots);
    return p;
}

// One thread's view of the ring: a place in the sequence of loads, and its own vectors of that slot.
template <int kSlots>
struct Cursor {
    uint32_t mine;  // shared address of the thread's vector of slot 0
    uint32_t full0, empty0;
    volatile int *abort;
    int *err;
    uint32_t slot, phase;
    __device__ __forceinline__ void go(uint32_t q)
    {
        slot = q % kSlots;
        phase = q / kSlots & 1u;
    }
    // A wait that runs out raises `abort`, which ends all later ones at once: the block runs on to its end
    // (every thread meets the same barriers) with the error recorded.
    __device__ __forceinline__ void wait() const { mbar_wait(full0 + 8 * slot, phase, abort, err, E_RING); }
    // the thread's vector of pass k of the slot, `stride` bytes a pass
    __device__ __forceinline__ uint4 get(int k, uint32_t stride) const { return ld_shared(mine + slot * kSlotBytes + k * stride); }
    // The slot's values are used: the next copy may overwrite it. The fence orders this thread's reads before
    // the copy, which writes through another path of shared memory; without it, and with the arrival before
    // the values were used, a copy now and then overtook a read of fp32 rows.
    __device__ __forceinline__ void release() const
    {
        fence_proxy_async_smem();
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(empty0 + 8 * slot);
    }
    __device__ __forceinline__ void next()
    {
        if (++slot == kSlots) {
            slot = 0;
            phase ^= 1u;
        }
    }
};

// The unit's rows of one thread, in the order in which the ring holds them: the held slots, then the others
// again, the latest first. `count`: its rows, `stride`: bytes of a pass.
template <typename TI, typename TO, int N, int kAct, int kSlots>
__device__ __forceinline__ void write_slots(Cursor<kSlots> c, const Slots &p, int count, uint32_t stride, TO *y, long long step,
                                            const float (&minus)[N], const float (&scale)[16 / sizeof(TI)],
                                            const float (&shift)[16 / sizeof(TI)])
{
    constexpr int VEC = 16 / sizeof(TI);
    auto slot = [&](int i, TO *py) __attribute__((always_inline)) {
        uint4 v[kSlotPasses];
#pragma unroll
        for (int k = 0; k < kSlotPasses; ++k) v[k] = c.get(k, stride);
        if ((i + 1) * kSlotPasses <= count) {
#pragma unroll
            for (int k = 0; k < kSlotPasses; ++k, py += step) finish<TI, TO, VEC, N, kAct>(v[k], py, minus, scale, shift);
        } else {
#pragma unroll
            for (int k = 0; k < kSlotPasses; ++k, py += step)
                if (i * kSlotPasses + k < count) finish<TI, TO, VEC, N, kAct>(v[k], py, minus, scale, shift);
        }
        c.release();
        c.next();
    };
    const long long slot_step = kSlotPasses * step;
    const int first = p.total - p.held;
    TO *py = y + first * slot_step;
#pragma unroll 1
    for (int i = first; i < p.total; ++i, py += slot_step) slot(i, py);
    py = y + (first - 1) * slot_step;
#pragma unroll 1
    for (int i = first - 1; i >= 0; --i, py -= slot_step) {
        c.wait();
        slot(i, py);
    }
}

// Bound by the memory: two reads and a write of a unit that L2 does not hold. 21 x 921600 x 128 bf16 silu (236 MB a
// sample) 2.37 ms, 96 % of these three passes at the copy rate, 6.3 TB/s; reads that the threads issue for
// themselves took 2.9 ms. N: moments a vector, 16 / sizeof(TI) / N channels each, which always belong to one group.
template <typename TI, typename TO, int N>
__global__ void __launch_bounds__(kThreads + 32, 2) group_norm_ring_kernel(const GnArgs a)
{
    constexpr int VEC = 16 / sizeof(TI), kSlots = ring_slots<N>();
    extern __shared__ uint4 ring[];
    __shared__ BlockMoments<N> s;
    __shared__ float2 norm[kSliceGroups];
    __shared__ uint64_t bars[2 * kSlots];
    __shared__ int abort_flag, last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int team = static_cast<int>(blockIdx.x) / a.parts, member = static_cast<int>(blockIdx.x) - team * a.parts;
    const long long r0 = member * a.part_rows, rows = max(0LL, min(a.part_rows, a.P - r0));
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kSlots;
    volatile int *abort = &abort_flag;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, kThreads / 32);
        }
        abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();

    if (warp == kThreads / 32) {
        // the loads of all units, as far ahead as slots are free
        const uint64_t once = l2_evict_first(), again = l2_evict_last();
        uint32_t slot = 0, phase = 0, issued = 0;
        bool ok = true;
        for (int unit = team; ok && unit < a.units; unit += a.teams) {
            const int smp = unit / a.slices, g0 = (unit - smp * a.slices) * a.slice_groups;
            const int ncols = min(a.slice_groups, a.G - g0) * a.cpg / VEC;
            const Slots p = slots_of<kSlots>(rows, ncols);
            const TI *x = static_cast<const TI *>(a.x) + smp * a.x_sample + r0 * a.x_row + g0 * a.cpg;
            const uint32_t row_bytes = ncols * 16;
            const bool dense = a.x_row * sizeof(TI) == row_bytes;
            const int loads = 2 * p.total - p.held;
            for (int q = 0; q < loads; ++q, ++issued) {
                const int i = q < p.total ? q : p.total - p.held - 1 - (q - p.total);
                const long long first = static_cast<long long>(i) * p.rows;
                const int n = static_cast<int>(min(static_cast<long long>(p.rows), rows - first));
                // nothing after a time-out: those who gave up release slots that are still being filled
                ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * slot, phase ^ 1u, abort, a.err, E_RING) && !*abort);
                if (!ok) break;
                const uint32_t dst = smem_u32(ring) + slot * kSlotBytes, bar = full0 + 8 * slot;
                if (lane == 0) mbar_arrive_expect_tx(bar, n * row_bytes);
                __syncwarp();
                const TI *src = x + first * a.x_row;
                const uint64_t policy = q < p.total - p.held ? again : once;
                if (dense) {
                    if (lane == 0) bulk_load(dst, src, n * row_bytes, bar, policy);
                } else {
                    for (int r = lane; r < n; r += 32) bulk_load(dst + r * row_bytes, src + r * a.x_row, row_bytes, bar, policy);
                }
                if (++slot == kSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
        // No copy may still be landing when the block ends: wait for the slots' last loads. (After a time-out nobody
        // else may have, also when all were issued before.)
        int dummy = 0;
        for (uint32_t k = 0; k < kSlots && k < issued; ++k) {
            const uint32_t q = issued - 1 - k;
            mbar_wait(full0 + 8 * (q % kSlots), (q / kSlots) & 1u, &dummy, a.err, E_RING);
        }
        return;
    }

    const int sub = static_cast<int>(threadIdx.x) / a.group_lanes, sub_lane = threadIdx.x % a.group_lanes;
    auto sync = [] { named_barrier_sync(1, kThreads); };
    Cursor<kSlots> cur{smem_u32(ring) + threadIdx.x * 16, full0, empty0, abort, a.err, 0, 0};
    uint32_t begin = 0;  // the unit's place in the sequence of loads
    for (int unit = team; unit < a.units; unit += a.teams) {
        const int smp = unit / a.slices, g0 = (unit - smp * a.slices) * a.slice_groups;
        const int gs = min(a.slice_groups, a.G - g0), c0 = g0 * a.cpg, ncols = gs * a.cpg / VEC;
        const Slots p = slots_of<kSlots>(rows, ncols);
        const Place at = place_of(0, ncols, rows);
        const uint32_t stride = p.lanes * ncols * 16;
        if (threadIdx.x < gs) s.group[threadIdx.x] = Moments{0.f, 0.f, 0.f};
        Moments mo[N] = {};
        cur.go(begin);
        for (int i = 0; i < p.total; i += kRunSlots) {
            const int n = min(kRunSlots, p.total - i), valid = min(n * kSlotPasses, at.count - i * kSlotPasses);
            cur.wait();
            Run<TI, VEC, N> run(cur.get(0, stride));
#pragma unroll 1
            for (int k = 0; k < n; ++k) {
                if (k > 0) cur.wait();
                uint4 v[kSlotPasses];
#pragma unroll
                for (int w = 0; w < kSlotPasses; ++w) v[w] = cur.get(w, stride);
                if ((k + 1) * kSlotPasses <= valid) {
#pragma unroll
                    for (int w = 0; w < kSlotPasses; ++w) run.add(v[w]);
                } else {
#pragma unroll
                    for (int w = 0; w < kSlotPasses; ++w)
                        if (k * kSlotPasses + w < valid) run.add(v[w]);
                }
                if (i + k < p.total - p.held) cur.release();
                cur.next();
            }
            if (valid > 0) run.end(valid, mo);
        }
        join_block<VEC, N>(s, mo, at, 0, a.cpg, gs, a.group_lanes, sub, sub_lane, sync);
        sync();
        join_grid(a, unit, member, s.group, gs, sub, sub_lane, norm, &last, abort, sync);

        float minus[N], scale[VEC], shift[VEC];
        affine_of<VEC, N>(a, at.col, c0, norm, minus, scale, shift);
        TO *y = static_cast<TO *>(a.y) + smp * a.y_sample + (r0 + at.rl) * a.y_row + c0 + at.col * VEC;
        const long long step = p.lanes * a.y_row;
        cur.go(begin + p.total - p.held);
        switch (a.act) {
        case S2_ACT_RELU: write_slots<TI, TO, N, S2_ACT_RELU>(cur, p, at.count, stride, y, step, minus, scale, shift); break;
        case S2_ACT_SILU: write_slots<TI, TO, N, S2_ACT_SILU>(cur, p, at.count, stride, y, step, minus, scale, shift); break;
        case S2_ACT_GELU: write_slots<TI, TO, N, S2_ACT_GELU>(cur, p, at.count, stride, y, step, minus, scale, shift); break;
        case S2_ACT_GELU_TANH:
            write_slots<TI, TO, N, S2_ACT_GELU_TANH>(cur, p, at.count, stride, y, step, minus, scale, shift);
            break;
        default: write_slots<TI, TO, N, S2_ACT_NONE>(cur, p, at.count, stride, y, step, minus, scale, shift);
        }
        begin += 2 * p.total - p.held;
    }
}

// ---- slices held by the whole grid -----------------------------------------------------

constexpr int kMaxBuffers = 8;
constexpr int kSlabGroups = 16;
constexpr int kSlabThreads = 128;  // that sum, and as many that write
constexpr int kPartsLane = 10;     // parts of a unit that a lane joins
// buffers beside N moments a vector, of two blocks an SM
constexpr int slab_room(int n) { return 112 * 1024 - n * 2560 - 4096; }

// y of a thread's `count` vectors in shared memory, `stride` bytes apart.
template <typename TI, typename TO, int N, int kAct>
__device__ __forceinline__ void write_slab(uint32_t from, int count, uint32_t stride, TO *py, long long step, const float (&minus)[N],
                                           const float (&scale)[16 / sizeof(TI)], const float (&shift)[16 / sizeof(TI)])
{
    constexpr int VEC = 16 / sizeof(TI);
    int i = 0;
#pragma unroll 1
    for (; i + kBatch <= count; i += kBatch) {
        uint4 v[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) v[k] = ld_shared(from + (i + k) * stride);
#pragma unroll
        for (int k = 0; k < kBatch; ++k, py += step) finish<TI, TO, VEC, N, kAct>(v[k], py, minus, scale, shift);
    }
#pragma unroll 1
    for (; i < count; ++i, py += step) finish<TI, TO, VEC, N, kAct>(ld_shared(from + i * stride), py, minus, scale, shift);
}

// Pairs of floats that are their own flag: all bits set until they are written (a NaN is written as another).
__device__ __forceinline__ uint64_t ld_pair(const float2 *p)
{
    uint64_t v;
    asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(v) : "l"(p) : "memory");
    return v;
}
__device__ __forceinline__ void st_pair(float2 *p, float2 f)
{
    const uint64_t v = pair(f.x != f.x ? __uint_as_float(0x7fffffffu) : f.x, f.y);
    asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" ::"l"(p), "l"(v) : "memory");
}
__device__ __forceinline__ void wait_pair(uint64_t &v, const float2 *p, volatile int *stop, int32_t *err, uint64_t most)
{
    if (v != ~0ull) return;
    const uint64_t t0 = global_timer_ns();
    while ((v = ld_pair(p)) == ~0ull)
        if (*stop || global_timer_ns() - t0 > most) {
            if (err) atomicCAS(err, 0, E_JOIN);
            *stop = 1;
            return;
        }
}
// A group's moments of all parts, by `lanes` neighbouring lanes (`sub` of them): part sub + k lanes in q[k], part 0's
// past the last; returns when all are written.
__device__ __forceinline__ void load_parts(uint64_t (&q)[kPartsLane], const float2 *part, int parts, int lanes, int sub,
                                           volatile int *stop, int32_t *err, uint64_t most)
{
    const uint64_t t0 = global_timer_ns();
    for (;;) {
        bool all = true;
#pragma unroll
        for (int k = 0; k < kPartsLane; ++k) {
            const int t = sub + k * lanes;
            q[k] = ld_pair(part + (t < parts ? t : 0));
        }
#pragma unroll
        for (int k = 0; k < kPartsLane; ++k) all = all && q[k] != ~0ull;
        if (__all_sync(0xffffffffu, all)) return;
        if (__any_sync(0xffffffffu, *stop || global_timer_ns() - t0 > most)) {
            if (err) atomicCAS(err, 0, E_JOIN);
            *stop = 1;
            return;
        }
    }
}
// Their mean and 1 / sigma; w[k]: the parts' shares of the rows, inv_n: 1 / the group's values.
__device__ __forceinline__ float2 norm_of_parts(const uint64_t (&q)[kPartsLane], const float (&w)[kPartsLane], int lanes, float inv_n,
                                                float eps)
{
    const float p0 = __shfl_sync(0xffffffffu, floats_of(q[0]).x, 0, lanes);
    float sum = 0.f, var = 0.f;
#pragma unroll
    for (int k = 0; k < kPartsLane; ++k)
        if (w[k] > 0.f) sum = fmaf(floats_of(q[k]).x - p0, w[k], sum);
    const float mean = p0 + sum_lanes(sum, lanes);
#pragma unroll
    for (int k = 0; k < kPartsLane; ++k) {
        const float d = floats_of(q[k]).x - mean;
        if (w[k] > 0.f) var += fmaf(d * d, w[k], floats_of(q[k]).y * inv_n);
    }
    return norm_of(Moments{1.f, mean, sum_lanes(var, lanes)}, eps);
}
// Until this block has posted its moments of `unit`: when to begin to ask for the others'. It orders no memory.
__device__ __forceinline__ bool wait_posted(const volatile int *posted, int unit, volatile int *stop, int32_t *err, uint64_t most)
{
    const uint64_t t0 = global_timer_ns();
    while (*posted <= unit) {
        __nanosleep(100);
        if (*stop) return false;
        if (global_timer_ns() - t0 > most) {
            if (err) atomicCAS(err, 0, E_JOIN);
            *stop = 1;
            return false;
        }
    }
    return true;
}

// Teams of blocks (one of all of them for large samples) take narrow slices of the channels, 64 bytes a row and
// more; a block holds its rows of the last few units in shared memory. The work on these goes on side by side:
// warps 0-3 sum one and post their block's moments, warps 4-7 write an older one, warp 8 loads the next (and has
// the one behind it brought to L2), warp 9 joins all parts' moments of the groups that are its block's turn,
// warp 10 fetches the results; where the parts are few, warp 10 joins them all itself. What bounds it is how long a
// unit stays in shared memory, about 12 us of which 2.5 for the load, 1.5 for the sums, 5 for the exchange and 2.5
// for the output, at 28 MB for the whole GPU. 11 x 57600 x 512 bf16 silu: 270 us, 4.8 TB/s (346 through the ring,
// which reads twice; 264 without an activation, 286 with gelu_tanh, 373 with gelu, which the writing warps do not
// hide); 6 x 14400 x 512: 42 us (48); 40 x 3600 x 512: 73 us (136 held by clusters). With one role after the other
// in each block the first took 560 us, and 370 while a lane asked for one part's moments after the other.
template <typename TI, typename TO, int N>
__global__ void __launch_bounds__(kThreads + 96, 2) group_norm_slab_kernel(const __grid_constant__ CUtensorMap map, const GnArgs a)
{
    constexpr int VEC = 16 / sizeof(TI);
    extern __shared__ uint4 slab_raw[];
    // the summing threads' (mean, M2), [unit & 1][group][row lane][moment of a row]; their shares of a group's values
    __shared__ float2 moments[2][kSlabThreads * N];
    __shared__ float share[kSlabThreads * N];
    __shared__ float2 norm[kMaxBuffers][kSlabGroups];
    __shared__ uint64_t bars[3 * kMaxBuffers];
    __shared__ int abort_flag;
    __shared__ volatile int posted;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int team = static_cast<int>(blockIdx.x) / a.parts, member = static_cast<int>(blockIdx.x) - team * a.parts;
    const int units = (a.units - team + a.teams - 1) / a.teams;  // the team's: team, team + teams, ...
    const int gs = a.slice_groups, ncols = gs * a.cpg / VEC;
    const long long r0 = member * a.part_rows, rows = min(a.part_rows, a.P - r0);
    const uint32_t base = (smem_u32(slab_raw) + 127u) & ~127u, box_bytes = a.box_rows * ncols * 16, buffer_bytes = a.boxes * box_bytes;
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kMaxBuffers, ready0 = empty0 + 8 * kMaxBuffers;
    volatile int *abort = &abort_flag;
    if (threadIdx.x == 0) {
        for (int i = 0; i < a.buffers; ++i) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, 2 * kSlabThreads / 32);  // the warps that sum and those that write
            mbar_init(ready0 + 8 * i, 1);
        }
        abort_flag = 0;
        posted = 0;
        fence_mbar_init();
    }
    __syncthreads();

    if (warp == kThreads / 32) {
        if (lane != 0) return;
        const uint64_t policy = l2_evict_first();
        int b = 0, u = 0;
        uint32_t phase = 0;
        for (; u < units; ++u) {
            const int unit = team + u * a.teams, smp = unit / a.slices, c0 = (unit - smp * a.slices) * gs * a.cpg;
            // nothing after a time-out: those who gave up release buffers that are still being filled
            if (!mbar_wait(empty0 + 8 * b, phase ^ 1u, abort, a.err, E_RING) || *abort) break;
            mbar_arrive_expect_tx(full0 + 8 * b, buffer_bytes);
            for (int i = 0; i < a.boxes; ++i)
                tma_load_3d(base + b * buffer_bytes + i * box_bytes, &map, full0 + 8 * b, c0, static_cast<int>(r0) + i * a.box_rows, smp,
                            policy);
            // the next unit, whose buffer is still in use, to L2: 11 x 57600 x 512 3 % faster
            const int next = unit + a.teams;
            if (next < a.units)
                for (int i = 0; i < a.boxes; ++i)
                    tma_prefetch_3d(&map, next % a.slices * gs * a.cpg, static_cast<int>(r0) + i * a.box_rows, next / a.slices);
            if (++b == a.buffers) {
                b = 0;
                phase ^= 1u;
            }
        }
        // no copy may still be landing when the block ends (see group_norm_ring_kernel): wait for the buffers' last loads
        int dummy = 0;
        for (int k = max(0, u - a.buffers); k < u; ++k)
            mbar_wait(full0 + 8 * (k % a.buffers), k / a.buffers & 1, &dummy, a.err, E_RING);
        return;
    }
    if (warp > kThreads / 32) {
        const bool joins = warp == kThreads / 32 + 1;
        if (joins && a.direct) return;
        // lanes of a group: all, or few for each of a unit's groups at once
        const int lanes = a.direct ? a.join_lanes : 32, sub = lane % lanes, group = lane / lanes;
        const float inv_rows = 1.f / static_cast<float>(a.P), inv_n = inv_rows / a.cpg;
        float w[kPartsLane];
#pragma unroll
        for (int k = 0; k < kPartsLane; ++k) {
            const int t = sub + k * lanes;
            w[k] = t < a.parts ? static_cast<float>(min(a.part_rows, a.P - t * a.part_rows)) * inv_rows : 0.f;
        }
        uint64_t q[kPartsLane];
        if (joins) {
            // the units' groups go round the team's blocks
            for (int turn = member; turn < units * gs; turn += a.parts) {
                const int u = turn / gs, of = (team + u * a.teams) * gs + turn - u * gs;
                if (!wait_posted(&posted, u, abort, a.err, a.join_ns)) return;
                load_parts(q, a.part + static_cast<long long>(of) * a.parts, a.parts, lanes, sub, abort, a.err, a.join_ns);
                const float2 r = norm_of_parts(q, w, lanes, inv_n, a.eps);
                if (lane == 0) st_pair(a.norm + of, r);
            }
            return;
        }
        int b = 0;
        uint32_t phase = 0;
        for (int u = 0; u < units; ++u) {
            const int of = (team + u * a.teams) * gs;
            // norm[b] is read no more (and will be before the unit is loaded): orders those reads before the writes below
            if (!mbar_wait(empty0 + 8 * b, phase ^ 1u, abort, a.err, E_RING)) return;
            if (!wait_posted(&posted, u, abort, a.err, a.join_ns)) return;
            if (a.direct) {
                load_parts(q, a.part + static_cast<long long>(of + min(group, gs - 1)) * a.parts, a.parts, lanes, sub, abort, a.err, a.join_ns);
                const float2 r = norm_of_parts(q, w, lanes, inv_n, a.eps);
                if (sub == 0 && group < gs) norm[b][group] = r;
            } else if (lane < gs) {
                uint64_t v = ld_pair(a.norm + of + lane);
                wait_pair(v, a.norm + of + lane, abort, a.err, a.join_ns);
                norm[b][lane] = floats_of(v);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(ready0 + 8 * b);
            if (++b == a.buffers) {
                b = 0;
                phase ^= 1u;
            }
        }
        return;
    }

    // one column a thread, every lanes-th row, for the sums and for the output alike. Units are whole slices, so
    // this is the same for all of them.
    const int tid = threadIdx.x % kSlabThreads, lanes = kSlabThreads / ncols, rl = tid / ncols, col = tid - rl * ncols;
    const int count = rl < lanes && rl < rows ? static_cast<int>((rows - rl + lanes - 1) / lanes) : 0;
    const uint32_t mine = base + tid * 16, stride = lanes * ncols * 16;
    int b = 0;
    uint32_t phase = 0;
    if (warp < kSlabThreads / 32) {
        const int sub = tid / a.group_lanes, sub_lane = tid % a.group_lanes;
        // a group's moments of a row lane, of the block
        const int group_cols = a.cpg / (VEC / N), entries = lanes * group_cols;
        const float n = static_cast<float>(rows * a.cpg);
        int to[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const int group = (col * N + k) / group_cols, of_row = col * N + k - group * group_cols;
            to[k] = group * entries + rl * group_cols + of_row;
            if (rl < lanes && group == 0) share[to[k]] = static_cast<float>(count * (VEC / N)) / n;
        }
        for (int u = 0; u < units; ++u) {
            mbar_wait(full0 + 8 * b, phase, abort, a.err, E_RING);
            Moments mo[N] = {};
            const uint32_t from = mine + b * buffer_bytes;
            int i = 0;
#pragma unroll 1
            for (; i + kAhead <= count; i += kAhead) {
                uint4 v[kAhead];
#pragma unroll
                for (int k = 0; k < kAhead; ++k) v[k] = ld_shared(from + (i + k) * stride);
                Run<TI, VEC, N> run(v[0]);
#pragma unroll
                for (int k = 0; k < kAhead; ++k) run.add(v[k]);
                run.end(kAhead, mo);
            }
            if (i < count) {
                Run<TI, VEC, N> run(ld_shared(from + i * stride));
#pragma unroll 1
                for (int k = i; k < count; ++k) run.add(ld_shared(from + k * stride));
                run.end(count - i, mo);
            }
            float2 *entry = moments[u & 1];
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (rl < lanes) entry[to[k]] = make_float2(mo[k].mean, mo[k].m2);
            named_barrier_sync(1, kSlabThreads);
            // joined as sums about the first one's mean, then about the mean of all: two short rounds of shuffles
            const float2 *of = entry + (sub < gs ? sub * entries : 0);
            const float p0 = of[0].x;
            float sum = 0.f, m2 = 0.f;
            for (int k = sub_lane; k < entries; k += a.group_lanes) sum = fmaf(of[k].x - p0, share[k], sum);
            __syncwarp();
            const float mean = p0 + sum_lanes(sum, a.group_lanes);
            for (int k = sub_lane; k < entries; k += a.group_lanes) {
                const float d = of[k].x - mean;
                if (share[k] > 0.f) m2 += fmaf(d * d, share[k] * n, of[k].y);  // not 0 * inf for lanes without rows
            }
            __syncwarp();
            m2 = sum_lanes(m2, a.group_lanes);
            if (sub_lane == 0 && sub < gs)
                st_pair(a.part + (static_cast<long long>(team + u * a.teams) * gs + sub) * a.parts + member, make_float2(mean, m2));
            if (threadIdx.x == 0) posted = u + 1;
            // the buffer is read (see Cursor::release); behind the posting, which others wait for
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(empty0 + 8 * b);
            if (++b == a.buffers) {
                b = 0;
                phase ^= 1u;
            }
        }
        return;
    }
    for (int unit = team; unit < a.units; unit += a.teams) {
        const int smp = unit / a.slices, c0 = (unit - smp * a.slices) * gs * a.cpg;
        mbar_wait(full0 + 8 * b, phase, abort, a.err, E_RING);  // orders the copy before the reads
        mbar_wait(ready0 + 8 * b, phase, abort, a.err, E_RING);
        float minus[N], scale[VEC], shift[VEC];
        affine_of<VEC, N>(a, col, c0, norm[b], minus, scale, shift);
        TO *y = static_cast<TO *>(a.y) + smp * a.y_sample + (r0 + rl) * a.y_row + c0 + col * VEC;
        const uint32_t from = mine + b * buffer_bytes;
        const long long step = lanes * a.y_row;
        switch (a.act) {
        case S2_ACT_RELU: write_slab<TI, TO, N, S2_ACT_RELU>(from, count, stride, y, step, minus, scale, shift); break;
        case S2_ACT_SILU: write_slab<TI, TO, N, S2_ACT_SILU>(from, count, stride, y, step, minus, scale, shift); break;
        case S2_ACT_GELU: write_slab<TI, TO, N, S2_ACT_GELU>(from, count, stride, y, step, minus, scale, shift); break;
        case S2_ACT_GELU_TANH: write_slab<TI, TO, N, S2_ACT_GELU_TANH>(from, count, stride, y, step, minus, scale, shift); break;
        default: write_slab<TI, TO, N, S2_ACT_NONE>(from, count, stride, y, step, minus, scale, shift);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(empty0 + 8 * b);
        if (++b == a.buffers) {
            b = 0;
            phase ^= 1u;
        }
    }
}

// ---- host --------------------------------------------------------------------------

constexpr size_t kHold = 22 * kThreads * 16;  // shared memory for rows, two blocks an SM

// The units of a call and the blocks that share them.
struct Plan {
    int slices, slice_groups, units, parts, teams, join;
    bool ring, slab;
    int buffers, boxes, box_rows, direct, join_lanes;
    long long part_rows;
    size_t smem;
};

size_t elem(int dtype) { return dtype == S2_F32 ? 4 : 2; }

// Moments a vector of 16 bytes has: one for all the channels that surely share a group.
int moments_of(int cpg, int vec)
{
    int n = 1;
    while (cpg % (vec / n) != 0) n *= 2;
    return n;
}

// Vectors of 16 bytes of x (their y 8 or 16 bytes) need every row to start on one.
bool is_wide(const s2_group_norm_act_desc &d)
{
    const size_t ie = elem(d.in_dtype), oe = elem(d.out_dtype), vec = 16 / ie;
    const uintptr_t xb = reinterpret_cast<uintptr_t>(d.x) | d.x_row * ie | (d.samples > 1 ? d.x_sample * ie : 0);
    const uintptr_t yb = reinterpret_cast<uintptr_t>(d.y) | d.y_row * oe | (d.samples > 1 ? d.y_sample * oe : 0);
    return d.channels % vec == 0 && xb % 16 == 0 && yb % (vec * oe) == 0;
}

// Slices for group_norm_slab_kernel: the widest of which as many blocks as there are can hold four. With 4 x 115200
// x 512 bf16 these are 64 bytes wide and take 218 us; two of 128 take 242, the ring 256. However little a block's
// share of a slice: 1 x 24000 x 32 fp16 (5.2 KB) takes 8.3 us and 16.4 through the ring, 1 x 22000 x 48 (7.2 KB) 12.1
// and 22.6, 20 x 9000 x 192 44 and 68. Held by clusters 16 x 5000 x 512 bf16 takes 68 us and 47 here, 400 x 256 x 1280
// 226 and 130.
bool plan_slab(const s2_group_norm_act_desc &d, int sms, Plan &p)
{
    const int size = static_cast<int>(elem(d.in_dtype)), vec = 16 / size, cpg = d.channels / d.groups;
    if (d.x_row >= (1LL << 40) / size || d.x_sample >= (1LL << 40) / size) return false;  // a tensor map's strides
    const long long room = slab_room(moments_of(cpg, vec)) / 4, blocks = 2 * sms;
    for (int sg = std::min(d.groups, kSlabGroups); sg > 0; --sg) {
        const int channels = sg * cpg;
        if (d.groups % sg != 0 || channels % vec != 0 || channels > 256) continue;
        const int width = channels * size;
        if (width < 64) break;
        const int whole = std::max(1, 128 / (width & -width));  // a box is a multiple of 128 bytes
        const long long most = room / width / whole * whole;    // rows of a quarter of the room
        const long long units = 1LL * d.samples * (d.groups / sg);
        if (most == 0 || (d.positions + most - 1) / most > blocks) continue;
        const long long teams = std::min(units, blocks / ((d.positions + most - 1) / most));
        const long long part_rows = (d.positions + blocks / teams - 1) / (blocks / teams);
        const long long boxes = (part_rows + 255) / 256, box_rows = ((part_rows + boxes - 1) / boxes + whole - 1) / whole * whole;
        const long long bytes = boxes * box_rows * width, parts = (d.positions + part_rows - 1) / part_rows;
        if (bytes > room || box_rows > 256) continue;
        if (parts > 32 * kPartsLane) break;
        p.slab = true;
        p.join = kGrid;
        p.part_rows = part_rows;
        p.parts = static_cast<int>(parts);
        p.teams = static_cast<int>(teams);
        p.slice_groups = sg;
        p.slices = d.groups / sg;
        p.units = static_cast<int>(units);
        p.boxes = static_cast<int>(boxes);
        p.box_rows = static_cast<int>(box_rows);
        p.buffers = static_cast<int>(std::min<long long>(kMaxBuffers, 4 * room / bytes));
        p.join_lanes = 32;
        while (p.join_lanes * sg > 32) p.join_lanes /= 2;
        p.direct = parts <= p.join_lanes * kPartsLane;
        p.smem = p.buffers * bytes + 128;
        return true;
    }
    return false;
}

Plan plan_of(const s2_group_norm_act_desc &d, int sms)
{
    const bool wide = is_wide(d);
    const long long size = static_cast<long long>(elem(d.in_dtype)), cpg = d.channels / d.groups;
    const int vec = wide ? static_cast<int>(16 / size) : 1;
    // slices are whole vectors
    int step = 1;
    while (step * cpg % vec != 0) ++step;
    auto slices_of = [&](int sg) { return (d.groups + sg - 1) / sg; };
    auto width = [&](int sg) { return sg * cpg * size; };
    auto bytes_of = [&](int sg) { return d.positions * width(sg); };  // of a unit
    auto halve = [&](int sg) { return std::max(step, sg / 2 / step * step); };
    auto fit = [&](int sg, int members) { return bytes_of(sg) / members <= static_cast<long long>(kHold * 15 / 16); };
    Plan p = {};
    // Below 8 MB the slices' GPU time is no less, and their workspace, which is cleared first, and cooperative
    // launch cost the host 5 us: 2 x 1920 x 512 fp16 10.9 us and 17.2 called one by one, 9.5 and 11.3 by clusters.
    if (wide && d.samples * bytes_of(d.groups) >= (8LL << 20) && plan_slab(d, sms, p)) return p;
    p.slice_groups = std::max(step, std::min(d.groups, kSliceGroups / step * step));
    // The blocks hold the rows of slices that their threads cover with a column each: 6 x 14400 x 512 fp16 in rows of 515
    // values takes 117 us in slices of 256 channels, 156 in whole rows, which are read twice. Only where a single group
    // is wider are columns taken in turns, nothing is held, and the sizes below just choose between cluster and grid.
    while (p.slice_groups * cpg / vec > kThreads && halve(p.slice_groups) < p.slice_groups) p.slice_groups = halve(p.slice_groups);
    const bool holds = p.slice_groups * cpg / vec <= kThreads;
    p.join = kGrid;
    // Held by a cluster, if need be in narrower slices. Reading 128 bytes of each row at a time costs little,
    // 32 do once the memory is the limit: 6 x 14400 x 512 takes 87 us in slices of 32 bytes and 47 on a grid, but
    // 3 x 7973 x 96 (9 MB, rows of 101 values) 15.6 us in slices of 48 and 21.5 on a grid.
    const int narrow = d.samples * bytes_of(d.groups) <= (32LL << 20) ? 32 : 128;
    for (int sg = p.slice_groups;; sg = halve(sg)) {
        if (fit(sg, kMaxCluster)) {
            p.slice_groups = sg;
            p.join = kCluster;
            break;
        }
        if (halve(sg) == sg || width(halve(sg)) < narrow) break;
    }
    if (p.join == kGrid && wide && plan_slab(d, sms, p)) return p;
    // A bulk copy takes the loading warp 60 clocks however short it is: 400 us became 16 ms with rows of 128
    // bytes apart from one another. Packed rows are copied a slot at a time, others have to be long.
    const bool rows_fit = d.x_row * size == width(p.slice_groups) || width(p.slice_groups) >= 1024;
    p.ring = p.join == kGrid && wide && rows_fit && p.slice_groups * cpg / vec <= kThreads;
    if (p.join == kCluster) {
        p.parts = 1;
        while (!fit(p.slice_groups, p.parts)) p.parts *= 2;
        auto few = [&] { return 1LL * d.samples * slices_of(p.slice_groups) * p.parts < sms; };
        while (few() && halve(p.slice_groups) < p.slice_groups && width(halve(p.slice_groups)) >= 64)
            p.slice_groups = halve(p.slice_groups);
        while (few() && p.parts < kMaxCluster && d.positions >= 32 * p.parts) p.parts *= 2;
    }
    p.slices = slices_of(p.slice_groups);
    p.units = d.samples * p.slices;
    p.teams = p.units;
    if (p.join == kGrid) {
        // All units at once up to 8 of them, else three or four in flight, whichever leaves fewer blocks idle in
        // the last round: while some read, others write. 21 x 921600 x 128 bf16: 2.43 ms with two, 2.36 / 2.46 with
        // three / four, 2.47 with all; 11 x 57600 x 512 through the ring: 380, 359 / 348 and 350 us. More when a block's
        // share of a unit would be less than it holds.
        const int blocks = 2 * sms;
        auto rounds = [&](int teams) { return static_cast<double>((p.units + teams - 1) / teams) / (blocks / teams); };
        p.teams = p.units <= 8 ? p.units : (rounds(3) < rounds(4) ? 3 : 4);
        const long long enough = std::max<long long>(1, (bytes_of(p.slice_groups) + kHold - 1) / static_cast<long long>(kHold));
        p.teams = static_cast<int>(std::max<long long>(p.teams, std::min<long long>(p.units, blocks / enough)));
        p.parts = static_cast<int>(std::min<long long>(blocks / p.teams, d.positions));
    }
    if (p.join == kCluster && p.parts == 1) p.join = kAlone;
    p.part_rows = (d.positions + p.parts - 1) / p.parts;
    // no more shared memory than the rows need
    const long long lanes = std::max<long long>(1, kThreads * vec / (p.slice_groups * cpg)), pieces = (p.part_rows + lanes - 1) / lanes;
    p.smem = holds ? std::min<size_t>(kHold, static_cast<size_t>(pieces) * kThreads * (wide ? 16 : size)) : 0;
    return p;
}

size_t round_up16(size_t v) { return (v + 15) / 16 * 16; }
size_t counters_of(const Plan &p) { return p.slab ? 0 : static_cast<size_t>(p.units) * 8; }

size_t workspace_of(const Plan &p)
{
    if (p.join != kGrid) return 0;
    return round_up16(counters_of(p)) + static_cast<size_t>(p.units) * (!p.direct + p.parts) * p.slice_groups * sizeof(float2);
}

int sm_count()
{
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        cudaGetLastError();
    return sms > 0 ? sms : 148;
}

template <typename... Args>
s2_status launch(void (*kernel)(Args...), std::atomic<uint64_t> &configured, size_t most, size_t smem, int threads, const Plan &p,
                 cudaStream_t st, const Args &...args)
{
    const s2_status cs = s2::once_per_device(configured, [&] {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(most));
        return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: %s", cudaGetErrorString(e));
    });
    if (cs != S2_OK) return cs;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    if (p.join == kGrid) {
        attr[0].id = cudaLaunchAttributeCooperative;
        attr[0].val.cooperative = 1;
    } else {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(p.parts);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
    }
    cfg.gridDim = dim3(static_cast<unsigned>(p.teams) * p.parts);
    cfg.blockDim = dim3(static_cast<unsigned>(threads));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
    return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: launch failed: %s", cudaGetErrorString(e));
}

template <typename TI, typename TO, int VEC, int N>
s2_status launch_shape(GnArgs &a, const Plan &p, cudaStream_t st)
{
    static std::atomic<uint64_t> held{0};
    if constexpr (VEC > 1) {
        static std::atomic<uint64_t> ring{0};
        constexpr size_t kBytes = ring_slots<N>() * kSlotBytes;
        if (p.ring) return launch(group_norm_ring_kernel<TI, TO, N>, ring, kBytes, kBytes, kThreads + 32, p, st, a);
        static std::atomic<uint64_t> slab{0};
        if (p.slab) {
            CUtensorMap map;
            const size_t ie = sizeof(TI);
            if (!s2::make_map_3d_plain(&map, a.x, ie, a.C, a.P, (a.units / a.slices), a.x_row * ie,
                                       a.x_sample > 0 ? a.x_sample * ie : a.x_row * ie, a.slice_groups * a.cpg, a.box_rows))
                return s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: cuTensorMapEncodeTiled failed");
            return launch(group_norm_slab_kernel<TI, TO, N>, slab, slab_room(N) + 128, p.smem, kThreads + 96, p, st, map, a);
        }
    }
    a.hold = static_cast<int>(p.smem / (kThreads * sizeof(typename Raw<TI, VEC>::type)));
    return launch(group_norm_held_kernel<TI, TO, VEC, N>, held, kHold, p.smem, kThreads, p, st, a);
}

template <typename TI, typename TO>
s2_status launch_types(GnArgs &a, const Plan &p, bool wide, cudaStream_t st)
{
    constexpr int kWide = 16 / sizeof(TI);
    if (!wide) return launch_shape<TI, TO, 1, 1>(a, p, st);
    switch (moments_of(a.cpg, kWide)) {
    case 1: return launch_shape<TI, TO, kWide, 1>(a, p, st);
    case 2: return launch_shape<TI, TO, kWide, 2>(a, p, st);
    case 4: return launch_shape<TI, TO, kWide, 4>(a, p, st);
    default: return launch_shape<TI, TO, kWide, kWide>(a, p, st);
    }
}

s2_status check(const s2_group_norm_act_desc *d)
{
    if (!d) return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: NULL description");
    if (d->samples < 0 || d->positions < 0 || d->channels <= 0 || d->groups <= 0 || d->channels % d->groups != 0)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: bad shape (samples %d, positions %lld, channels %d, groups %d)",
                             d->samples, d->positions, d->channels, d->groups);
    if (d->groups > kMaxGroups || d->samples > 65535 || d->positions > (1LL << 31))
        return s2::set_error(S2_UNSUPPORTED, "s2_group_norm_act: at most %d groups, 65535 samples and 2^31 positions", kMaxGroups);
    if (d->positions > (1LL << 44) / d->channels)
        return s2::set_error(S2_UNSUPPORTED, "s2_group_norm_act: at most 2^44 values a sample");
    const bool types = (d->in_dtype == S2_F32 && (d->out_dtype == S2_F32 || d->out_dtype == S2_F16 || d->out_dtype == S2_BF16)) ||
                       ((d->in_dtype == S2_F16 || d->in_dtype == S2_BF16) && d->out_dtype == d->in_dtype);
    if (!types)
        return s2::set_error(S2_UNSUPPORTED, "s2_group_norm_act: dtypes %d -> %d (the same, or fp32 to fp16 / bf16)", d->in_dtype, d->out_dtype);
    if (d->activation < S2_ACT_NONE || d->activation > S2_ACT_GELU_TANH)
        return s2::set_error(S2_UNSUPPORTED, "s2_group_norm_act: unknown activation %d", d->activation);
    if (!(d->eps >= 0.f) || d->eps > 1e30f)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: eps must be finite and not negative");
    return S2_OK;
}

bool in_place(const s2_group_norm_act_desc &d)
{
    return d.x == d.y && d.in_dtype == d.out_dtype && d.x_row == d.y_row &&
           (d.samples == 1 || d.x_sample == d.y_sample);
}

// All samples as one pitched matrix when they follow one another at whole rows (then column
// ranges of one buffer are told apart), else as one run of bytes.
s2::PitchedSpan span(const void *p, const s2_group_norm_act_desc &d, long long row, long long sample, long long size)
{
    if (d.samples == 1) return {p, d.positions, d.channels * size, row * size};
    if (sample % row == 0) return {p, (d.samples - 1) * (sample / row) + d.positions, d.channels * size, row * size};
    const long long bytes = ((d.samples - 1) * sample + (d.positions - 1) * row + d.channels) * size;
    return {p, 1, bytes, bytes};
}

}  // namespace

extern "C" size_t s2_group_norm_act_workspace_bytes(const s2_group_norm_act_desc *d)
{
    s2::clear_error();
    if (check(d) != S2_OK || d->samples == 0 || d->positions == 0) return 0;
    return workspace_of(plan_of(*d, sm_count()));
}

extern "C" s2_status s2_group_norm_act(void *stream, const s2_group_norm_act_desc *d, int *launches)
{
    s2::clear_error();
    if (launches) *launches = 0;
    const s2_status cs = check(d);
    if (cs != S2_OK) return cs;
    if (d->samples == 0 || d->positions == 0) return S2_OK;
    if (!d->x || !d->y) return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: NULL x or y");
    const size_t ie = elem(d->in_dtype), oe = elem(d->out_dtype);
    if (reinterpret_cast<uintptr_t>(d->x) % ie || reinterpret_cast<uintptr_t>(d->y) % oe ||
        (reinterpret_cast<uintptr_t>(d->weight) | reinterpret_cast<uintptr_t>(d->bias)) % 4)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: a pointer is not aligned to its elements");
    // (n - 1) strides stay within 2^44 elements, so that no offset below overflows
    auto far = [](long long n, long long stride) { return n > 1 && stride > (1LL << 44) / (n - 1); };
    if (d->x_row > (1LL << 40) || d->y_row > (1LL << 40) || far(d->positions, d->x_row) || far(d->positions, d->y_row) ||
        far(d->samples, d->x_sample) || far(d->samples, d->y_sample))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: a pitch or sample stride beyond any memory");
    if (d->x_row < d->channels || d->y_row < d->channels ||
        (d->samples > 1 && (d->x_sample < (d->positions - 1) * d->x_row + d->channels ||
                            d->y_sample < (d->positions - 1) * d->y_row + d->channels)))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: a pitch is smaller than what it spans");
    const s2::PitchedSpan xs = span(d->x, *d, d->x_row, d->x_sample, static_cast<long long>(ie));
    const s2::PitchedSpan ys = span(d->y, *d, d->y_row, d->y_sample, static_cast<long long>(oe));
    const s2::PitchedSpan ws = s2::bytes_at(d->weight, 4LL * d->channels), bs = s2::bytes_at(d->bias, 4LL * d->channels);
    if (!in_place(*d) && s2::may_overlap(xs, ys)) return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: y overlaps x");
    if (s2::may_overlap(ws, ys) || s2::may_overlap(bs, ys))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: y overlaps weight or bias");
    const Plan p = plan_of(*d, sm_count());
    const size_t need = workspace_of(p);
    if (need > 0 && (!d->workspace || d->workspace_bytes < need || reinterpret_cast<uintptr_t>(d->workspace) % 16))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: workspace of %zu bytes, 16-byte aligned, needed", need);
    const s2::PitchedSpan work = s2::bytes_at(need > 0 ? d->workspace : nullptr, static_cast<long long>(need));
    if (s2::may_overlap(work, xs) || s2::may_overlap(work, ys) || s2::may_overlap(work, ws) || s2::may_overlap(work, bs))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: the workspace overlaps an operand");
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    GnArgs a = {};
    a.x = d->x;
    a.y = d->y;
    a.weight = d->weight;
    a.bias = d->bias;
    a.err = d->err ? d->err : s2::operator_error_word();
    a.P = d->positions;
    a.part_rows = p.part_rows;
    a.x_row = d->x_row;
    a.x_sample = d->samples > 1 ? d->x_sample : 0;
    a.y_row = d->y_row;
    a.y_sample = d->samples > 1 ? d->y_sample : 0;
    a.C = d->channels;
    a.G = d->groups;
    a.cpg = d->channels / d->groups;
    a.slices = p.slices;
    a.slice_groups = p.slice_groups;
    a.units = p.units;
    a.parts = p.parts;
    a.teams = p.teams;
    a.join = p.join;
    a.act = d->activation;
    a.buffers = p.buffers;
    a.boxes = p.boxes;
    a.direct = p.direct;
    a.join_lanes = p.join_lanes;
    a.box_rows = p.box_rows;
    a.group_lanes = 32;
    while (a.group_lanes * p.slice_groups > (p.slab ? kSlabThreads : kThreads)) a.group_lanes /= 2;
    a.eps = d->eps;
    a.join_ns = s2::take_norm_wait();
    if (p.join == kGrid) {
        a.arrived = static_cast<uint32_t *>(d->workspace);
        a.ready = a.arrived + p.units;
        a.norm = reinterpret_cast<float2 *>(static_cast<char *>(d->workspace) + round_up16(counters_of(p)));
        a.part = a.norm + (p.direct ? 0 : static_cast<size_t>(p.units) * p.slice_groups);
        const cudaError_t e = p.slab ? cudaMemsetAsync(d->workspace, 0xff, need, st) : cudaMemsetAsync(d->workspace, 0, counters_of(p), st);
        if (e != cudaSuccess) return s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: %s", cudaGetErrorString(e));
    }
    const bool wide = is_wide(*d);
    s2_status s;
    if (d->in_dtype == S2_F16)
        s = launch_types<__half, __half>(a, p, wide, st);
    else if (d->in_dtype == S2_BF16)
        s = launch_types<__nv_bfloat16, __nv_bfloat16>(a, p, wide, st);
    else if (d->out_dtype == S2_F32)
        s = launch_types<float, float>(a, p, wide, st);
    else if (d->out_dtype == S2_F16)
        s = launch_types<float, __half>(a, p, wide, st);
    else
        s = launch_types<float, __nv_bfloat16>(a, p, wide, st);
    if (s == S2_OK && launches) *launches = 1;
    return s;
}
