// Group norm with an activation over channels-last activations (s2_group_norm_act).
//
// x [S][P][C], G groups of C / G consecutive channels. Per sample s and group g, over the
// n = P C / G values of the group:
//   m = sum x / n,  v = sum (x - m)^2 / n,  y = act((x - m) / sqrt(v + eps) * w[c] + b[c]).
//
// Statistics: a thread keeps one vector of channels and walks down the rows. It sums d = x - p
// and d^2 about a pivot p of its own (the first value of each short run of rows) in fp32 and
// turns every run into (count, mean, M2 = sum of squares about the mean); runs, threads and
// blocks are joined by
//   m = ma + (mb - ma) nb / n,   M2 = M2a + M2b + (mb - ma)^2 na nb / n,
// which loses nothing when the mean is far larger than the spread, and an outlier only reaches
// the run that holds it. Blocks are joined in double, in order: the result does not depend on
// timing.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cstdint>
#include <cstdlib>

#include "s2_act.cuh"
#include "s2_internal.h"
#include "s2_launch.h"
#include "s2_overlap.h"
#include "s2_sm100.cuh"

namespace {

using namespace s2dev;

constexpr int kThreads = 256;
constexpr int kMaxGroups = 1024;
constexpr int kSliceGroups = 64;   // groups of one unit
constexpr int kMaxCluster = 8;
constexpr int kAhead = 8;          // vectors a thread has in flight while it reads

// How the members of a unit exchange their groups' moments.
enum Join : int {
    kAlone = 0,    // one block
    kCluster = 1,  // the blocks of a cluster, through distributed shared memory
    kGrid = 2,     // blocks of a cooperative grid, through the workspace
    kRing = 3,     // the same, one block an SM that streams its rows through a ring (group_norm_ring_kernel)
};

// A unit is the slice of `slice_groups` groups of one sample; `members` blocks share its positions:
// the first `more_rows` of them rows + 1 each, the others `rows`.
struct GnArgs {
    const void *x;
    void *y;
    const float *weight, *bias;
    // members of a grid: [unit][member][group of the slice] (mean, M2), [unit][group] (mean, 1 / sigma),
    // and per unit the members whose moments are written and, once set, that the unit's are (zero before)
    float2 *part, *joined;
    uint32_t *arrived, *ready;
    int32_t *err;
    long long rows, x_row, x_sample, y_row, y_sample;
    int more_rows, C, G, cpg, slices, slice_groups, units, members, teams, join, hold, act;
    int group_lanes;    // threads that join one group's moments: a power of two up to 32
    float eps;
};

struct Moments {
    float n = 0.f, mean = 0.f, m2 = 0.f;
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

// VEC elements of T as they are loaded: 16 bytes or one element
template <typename T, int VEC>
struct Raw {
    using type = uint4;
    static __device__ __forceinline__ uint4 load(const T *p)
    {
        uint4 v;
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(p)
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
    static __device__ __forceinline__ T load(const T *p) { return *p; }
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

// A run: up to kAhead vectors of one column, read, held in shared memory when they come before `hold`,
// and their moments joined to mo: N = 1 those of all values together, N = VEC of each of a vector's
// channels. The pivot is the run's first vector.
template <typename TI, int VEC, int N, bool kFull>
__device__ __forceinline__ void read_run(const TI *px, long long step, int n, int i, int hold,
                                         typename Raw<TI, VEC>::type *held, Moments (&mo)[N])
{
    using R = Raw<TI, VEC>;
    constexpr int kPairs = VEC > 1 ? VEC / 2 : 1, kSums = N == 1 ? (VEC > 2 ? 2 : 1) : kPairs, kPer = VEC / N;
    if (kFull) n = kAhead;
    typename R::type v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
        if (kFull || u < n) v[u] = R::load(px);
        px += step;
    }
    if (i + kAhead <= hold) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (kFull || u < n) held[(i + u) * kThreads] = v[u];
    } else if (i < hold) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (u < n && i + u < hold) held[(i + u) * kThreads] = v[u];
    }
    float f[VEC], p[N], sum[N], sq[N];
    R::floats(v[0], f);
#pragma unroll
    for (int e = 0; e < N; ++e) p[e] = f[e * kPer];
    if constexpr (VEC == 1) {
        sum[0] = sq[0] = 0.f;
#pragma unroll
        for (int u = 1; u < kAhead; ++u)
            if (kFull || u < n) {
                R::floats(v[u], f);
                const float d = f[0] - p[0];
                sum[0] += d;
                sq[0] = fmaf(d, d, sq[0]);
            }
    } else {
        uint64_t minus[N == 1 ? 1 : kPairs], s2[kSums], q2[kSums];
#pragma unroll
        for (int k = 0; k < (N == 1 ? 1 : kPairs); ++k)
            minus[k] = N == 1 ? pair(-p[0], -p[0]) : pair(-p[2 * k < N ? 2 * k : 0], -p[2 * k + 1 < N ? 2 * k + 1 : 0]);
#pragma unroll
        for (int k = 0; k < kSums; ++k) s2[k] = q2[k] = 0;
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (kFull || u < n) {
                R::floats(v[u], f);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    const uint64_t d = add2(pair(f[2 * k], f[2 * k + 1]), minus[N == 1 ? 0 : k]);
                    s2[k % kSums] = add2(s2[k % kSums], d);
                    q2[k % kSums] = fma2(d, d, q2[k % kSums]);
                }
            }
        if constexpr (N == 1) {
            const float2 a = floats_of(kSums == 2 ? add2(s2[0], s2[kSums - 1]) : s2[0]);
            const float2 b = floats_of(kSums == 2 ? add2(q2[0], q2[kSums - 1]) : q2[0]);
            sum[0] = a.x + a.y;
            sq[0] = b.x + b.y;
        } else {
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const float2 a = floats_of(s2[k]), b = floats_of(q2[k]);
                sum[2 * k] = a.x;
                sum[2 * k + 1] = a.y;
                sq[2 * k] = b.x;
                sq[2 * k + 1] = b.y;
            }
        }
    }
    const float cnt = static_cast<float>(n * kPer), inv = __fdividef(1.f, cnt);
#pragma unroll
    for (int e = 0; e < N; ++e) {
        Moments run;
        run.n = cnt;
        run.mean = fmaf(sum[e], inv, p[e]);
        // not below 0 by rounding; 0 * sq keeps the NaN of a value that is not finite
        run.m2 = fmaxf(fmaf(-sum[e] * inv, sum[e], sq[e]), 0.f * sq[e]);
        mo[e] = join(mo[e], run);
    }
}

template <typename TI, int VEC, int N>
__device__ __forceinline__ void read_rows(const TI *px, long long step, int count, int hold,
                                          typename Raw<TI, VEC>::type *held, Moments (&mo)[N])
{
    int i = 0;
#pragma unroll 1
    for (; i + kAhead <= count; i += kAhead, px += kAhead * step) read_run<TI, VEC, N, true>(px, step, kAhead, i, hold, held, mo);
    if (i < count) read_run<TI, VEC, N, false>(px, step, count - i, i, hold, held, mo);
}

// silu and gelu_tanh of two values with one reciprocal for both: 1 / a = b / (a b). e^-z is cut off at 2^60
// (a value below -41 gives -41 * 2^-60 and the like instead of 0), so that a b stays finite. Exponentials
// and reciprocals share a unit of 16 a clock on an SM; at two each a value the output of 16-bit vectors took
// 32 clocks a warp's vector there, at three for two 24, where the memory needs 22.
template <int kAct>
__device__ __forceinline__ uint64_t activate_pair(uint64_t v)
{
    if constexpr (kAct == S2_ACT_SILU || kAct == S2_ACT_GELU_TANH) {
        constexpr float kLog2e = 1.4426950408889634f, kTanh = -2.f * 0.7978845608028654f * kLog2e;
        const uint64_t z = kAct == S2_ACT_SILU ? mul2(v, both(-kLog2e))
                                               : mul2(v, fma2(mul2(v, v), both(kTanh * 0.044715f), both(kTanh)));
        const float2 zf = floats_of(z);
        const float2 d = floats_of(add2(ex2_2(pair(fminf(zf.x, 60.f), fminf(zf.y, 60.f))), both(1.f)));
        float r = d.x * d.y;
        asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(r));
        return mul2(v, mul2(both(r), pair(d.y, d.x)));
    }
    return activate2<kAct>(v);
}

// y = act((x - mean) scale + shift) of one vector; `minus` is -mean, one (kOne) or a pair of channels each.
// The subtraction comes first, as in the formula: values that all equal the mean give the shift itself.
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
            const float2 r = floats_of(activate_pair<kAct>(
                fma2(d, pair(scale[2 * k], scale[2 * k + 1]), pair(shift[2 * k], shift[2 * k + 1]))));
            f[2 * k] = r.x;
            f[2 * k + 1] = r.y;
        }
    }
    store_vec<TO, VEC>(py, f);
}

// y of the thread's vectors: those that are not held once more from global memory, the latest read
// first (they are in L2 the longest), then the held ones.
template <typename TI, typename TO, int VEC, int N, int kAct>
__device__ __forceinline__ void write_rows(const TI *px, long long x_step, TO *py, long long y_step, int count, int hold,
                                           const typename Raw<TI, VEC>::type *held, const float (&minus)[N],
                                           const float (&scale)[VEC], const float (&shift)[VEC])
{
    using R = Raw<TI, VEC>;
    constexpr int kRun = 4;
    int i = count;
    if (i > hold) {
        const TI *qx = px + (count - 1) * x_step;
        TO *qy = py + (count - 1) * y_step;
#pragma unroll 1
        for (; i - kRun >= hold; i -= kRun) {
            typename R::type v[kRun];
#pragma unroll
            for (int u = 0; u < kRun; ++u, qx -= x_step) v[u] = R::load(qx);
#pragma unroll
            for (int u = 0; u < kRun; ++u, qy -= y_step) finish<TI, TO, VEC, N, kAct>(v[u], qy, minus, scale, shift);
        }
#pragma unroll 1
        for (; i > hold; --i, qx -= x_step, qy -= y_step) finish<TI, TO, VEC, N, kAct>(R::load(qx), qy, minus, scale, shift);
    }
#pragma unroll 2
    for (int k = 0; k < i; ++k) {
        finish<TI, TO, VEC, N, kAct>(held[k * kThreads], py, minus, scale, shift);
        py += y_step;
    }
}

__device__ __forceinline__ uint32_t ld_acquire(const uint32_t *p)
{
    uint32_t v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// device error codes: the wait for the other members, for the ring's loads
enum : int { E_JOIN = 96, E_RING = 97 };

// The members' moments of group `sub` of the slice, by group_lanes threads a group (sub_lane of them): in the
// first of these. Eight are asked for at a time and joined in four chains; which thread joins what depends on
// the shape alone.
template <bool kGlobal>
__device__ __noinline__ Moments join_members(const GnArgs &a, const float2 *part, int pitch, int sub, int sub_lane, int gs)
{
    Moments chain[4];
    if (sub < gs)
        for (int t0 = sub_lane; t0 < a.members; t0 += 8 * a.group_lanes) {
            float2 q[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int t = t0 + k * a.group_lanes;
                if (t < a.members) q[k] = kGlobal ? __ldcg(part + t * pitch + sub) : part[t * pitch + sub];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int t = t0 + k * a.group_lanes;
                if (t < a.members) {
                    Moments o;
                    o.n = static_cast<float>((a.rows + (t < a.more_rows)) * a.cpg);
                    o.mean = q[k].x;
                    o.m2 = q[k].y;
                    chain[k & 3] = join(chain[k & 3], o);
                }
            }
        }
    return join_lanes(join(join(chain[0], chain[1]), join(chain[2], chain[3])), a.group_lanes);
}

// mean and 1 / sigma of a group
__device__ __forceinline__ float2 norm_of(const Moments &m, float eps)
{
    return make_float2(m.mean, __frsqrt_rn(__fdiv_rn(m.m2, m.n) + eps));
}

// The members of a grid join a unit's moments (group[], gs of them): each writes its own, the last to arrive
// joins all of them and publishes the unit's, the others wait for these. (Every member joining all for itself
// read 296 x 32 moments 296 times from the same lines of L2: 8 us a unit.) `sync` is the barrier of the
// threads that call this; *stop ends the wait, which is bounded. On return norm[] holds the unit's.
template <typename Sync>
__device__ __forceinline__ void join_grid(const GnArgs &a, int unit, int member, const Moments *group, int gs, int sub,
                                          int sub_lane, float2 *norm, volatile int *last, volatile int *stop, Sync sync)
{
    const long long at = static_cast<long long>(unit) * a.members;
    if (threadIdx.x < gs)
        __stcg(a.part + (at + member) * a.slice_groups + threadIdx.x, make_float2(group[threadIdx.x].mean, group[threadIdx.x].m2));
    sync();
    if (threadIdx.x == 0) {
        __threadfence();
        *last = atomicAdd(a.arrived + unit, 1u) == static_cast<uint32_t>(a.members) - 1;
        __threadfence();
    }
    sync();
    float2 *joined = a.joined + static_cast<long long>(unit) * a.slice_groups;
    if (*last) {
        const Moments m = join_members<true>(a, a.part + at * a.slice_groups, a.slice_groups, sub, sub_lane, gs);
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
        if (threadIdx.x == 0 && ld_acquire(a.ready + unit) == 0) {
            const uint64_t t0 = global_timer_ns();
            while (ld_acquire(a.ready + unit) == 0)
                if (*stop || global_timer_ns() - t0 > kWaitTimeoutNs) {
                    if (a.err) atomicCAS(a.err, 0, E_JOIN);
                    *stop = 1;
                    break;
                }
        }
        sync();
        if (threadIdx.x < gs) norm[threadIdx.x] = __ldcg(joined + threadIdx.x);
        sync();
    }
}

// kOne: the VEC channels of a vector always belong to one group.
template <typename TI, typename TO, int VEC, bool kOne>
__global__ void __launch_bounds__(kThreads, 2) group_norm_kernel(const GnArgs a)
{
    using R = Raw<TI, VEC>;
    constexpr int N = kOne ? 1 : VEC;
    extern __shared__ uint4 held_raw[];
    __shared__ float2 entry[N][kThreads];  // (mean, M2) a thread and channel, and of how many values
    __shared__ float entry_n[kThreads];
    __shared__ Moments group[kSliceGroups];
    __shared__ float2 received[kMaxCluster][kSliceGroups];
    __shared__ float2 norm[kSliceGroups];  // mean, 1 / sqrt(v + eps)
    __shared__ int last, stop;
    typename R::type *held = reinterpret_cast<typename R::type *>(held_raw) + threadIdx.x;
    const int member = static_cast<int>(blockIdx.x) % a.members;
    const long long r0 = member * a.rows + min(member, a.more_rows), rows = a.rows + (member < a.more_rows);
    // for the joins of groups: group_lanes threads a group
    const int sub = static_cast<int>(threadIdx.x) / a.group_lanes, sub_lane = threadIdx.x % a.group_lanes;
    if (threadIdx.x == 0) stop = 0;
    if (a.join == kCluster) cluster_arrive();  // waited for below: no block writes to one that has not begun

    for (int unit = static_cast<int>(blockIdx.x) / a.members; unit < a.units; unit += a.teams) {
        const int s = unit / a.slices, g0 = (unit - s * a.slices) * a.slice_groups;
        const int gs = min(a.slice_groups, a.G - g0), c0 = g0 * a.cpg;
        const int ncols = gs * a.cpg / VEC;
        const int hold = ncols <= kThreads ? a.hold : 0;
        const TI *x = static_cast<const TI *>(a.x) + s * a.x_sample + r0 * a.x_row + c0;
        if (sub_lane == 0 && sub < gs) group[sub] = Moments();

        // Columns of vectors, kThreads of them at a time (all, unless a single group is wider than that):
        // a thread keeps one column and takes every lanes-th row.
        int nb = 0, lanes = 0, col = 0, rl = 0, count = 0;
        auto place = [&](int cb) {
            nb = min(kThreads, ncols - cb);
            lanes = kThreads / nb;
            rl = static_cast<int>(threadIdx.x) / nb;
            col = cb + static_cast<int>(threadIdx.x) - rl * nb;
            count = rl < lanes && rl < rows ? static_cast<int>((rows - rl + lanes - 1) / lanes) : 0;
        };
        for (int cb = 0; cb < ncols; cb += kThreads) {
            place(cb);
            Moments mo[N];
            read_rows<TI, VEC, N>(x + rl * a.x_row + static_cast<long long>(col) * VEC, lanes * a.x_row, count, hold, held, mo);
            // down the rows: halves of the row lanes joined until one is left
            if (cb > 0) __syncthreads();
#pragma unroll
            for (int e = 0; e < N; ++e) entry[e][threadIdx.x] = make_float2(mo[e].mean, mo[e].m2);
            entry_n[threadIdx.x] = mo[0].n;
            __syncthreads();
            for (int left = lanes; left > 1;) {
                const int half = (left + 1) / 2;
                if (rl + half < left) {
                    const int other = threadIdx.x + half * nb;
                    const float n = entry_n[other];
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float2 q = entry[e][other];
                        Moments t;
                        t.n = n;
                        t.mean = q.x;
                        t.m2 = q.y;
                        mo[e] = join(mo[e], t);
                        entry[e][threadIdx.x] = make_float2(mo[e].mean, mo[e].m2);
                    }
                    entry_n[threadIdx.x] = mo[0].n;
                }
                left = half;
                __syncthreads();
            }
            // across the columns of each group (N = 1), or its channels
            Moments m;
            if (sub < gs) {
                constexpr int kUnit = N == 1 ? VEC : 1;
                const int lo = max(sub * a.cpg / kUnit, cb * (VEC / kUnit)) - cb * (VEC / kUnit);
                const int end = min((sub + 1) * a.cpg / kUnit, (cb + nb) * (VEC / kUnit)) - cb * (VEC / kUnit);
                for (int k = lo + sub_lane; k < end; k += a.group_lanes) {
                    const float2 q = N == 1 ? entry[0][k] : entry[k % N][k / N];
                    Moments t;
                    t.n = entry_n[0];
                    t.mean = q.x;
                    t.m2 = q.y;
                    m = join(m, t);
                }
            }
            m = join_lanes(m, a.group_lanes);
            if (sub_lane == 0 && sub < gs) group[sub] = join(group[sub], m);
        }
        __syncthreads();

        // hand the moments to the other members and take theirs
        if (a.join == kAlone) {
            if (threadIdx.x < gs) received[0][threadIdx.x] = make_float2(group[threadIdx.x].mean, group[threadIdx.x].m2);
            __syncthreads();
        } else if (a.join == kCluster) {
            cluster_wait();
            for (int i = threadIdx.x; i < kSliceGroups * a.members; i += kThreads) {
                const int to = i / kSliceGroups, g = i % kSliceGroups;
                if (g < gs) {
                    const uint32_t at = cluster_map(smem_u32(&received[member][g]), static_cast<uint32_t>(to));
                    st_cluster_b32(at, __float_as_uint(group[g].mean));
                    st_cluster_b32(at + 4, __float_as_uint(group[g].m2));
                }
            }
            __syncwarp();
            cluster_sync();
        } else {
            join_grid(a, unit, member, group, gs, sub, sub_lane, norm, &last, &stop, [] { __syncthreads(); });
            if (stop) return;
        }
        if (a.join != kGrid) {
            const Moments m = join_members<false>(a, &received[0][0], kSliceGroups, sub, sub_lane, gs);
            if (sub_lane == 0 && sub < gs) norm[sub] = norm_of(m, a.eps);
            __syncthreads();
        }

        TO *y = static_cast<TO *>(a.y) + s * a.y_sample + r0 * a.y_row + c0;
        for (int cb = 0; cb < ncols; cb += kThreads) {
            if (ncols > kThreads) place(cb);
            if (count == 0) continue;
            float minus[N], scale[VEC], shift[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const int c = col * VEC + e;
                const float2 mr = norm[(kOne ? col * VEC : c) / a.cpg];
                minus[e % N] = -mr.x;
                scale[e] = a.weight ? mr.y * __ldg(a.weight + c0 + c) : mr.y;
                shift[e] = a.bias ? __ldg(a.bias + c0 + c) : 0.f;
            }
            const TI *px = x + rl * a.x_row + static_cast<long long>(col) * VEC;
            TO *py = y + rl * a.y_row + static_cast<long long>(col) * VEC;
            const long long xs = lanes * a.x_row, ys = lanes * a.y_row;
            switch (a.act) {
            case S2_ACT_RELU: write_rows<TI, TO, VEC, N, S2_ACT_RELU>(px, xs, py, ys, count, hold, held, minus, scale, shift); break;
            case S2_ACT_SILU: write_rows<TI, TO, VEC, N, S2_ACT_SILU>(px, xs, py, ys, count, hold, held, minus, scale, shift); break;
            case S2_ACT_GELU: write_rows<TI, TO, VEC, N, S2_ACT_GELU>(px, xs, py, ys, count, hold, held, minus, scale, shift); break;
            case S2_ACT_GELU_TANH:
                write_rows<TI, TO, VEC, N, S2_ACT_GELU_TANH>(px, xs, py, ys, count, hold, held, minus, scale, shift);
                break;
            default: write_rows<TI, TO, VEC, N, S2_ACT_NONE>(px, xs, py, ys, count, hold, held, minus, scale, shift);
            }
        }
        __syncthreads();  // the next unit reuses the moments
    }
}

// ---- large units -----------------------------------------------------------------

constexpr int kRingThreads = 256;             // and a warp that only loads; two blocks an SM
constexpr int kSlotPasses = 4;                // passes of a slot
constexpr int kRunSlots = 2;                  // slots summed about one pivot
constexpr uint32_t kSlotBytes = kSlotPasses * kRingThreads * 16;

// Slots of the ring: what is left beside the joins' shared memory.
template <int N>
__host__ __device__ constexpr int ring_slots()
{
    return 6;
}

// A member's slots over one unit: slot i holds kSlotPasses times `lanes` of its rows.
struct Slots {
    int lanes, rows;  // of a pass, of a slot
    int total, held;  // held: the last ones stay in the ring from the statistics to the output
};

template <int N>
__device__ __forceinline__ Slots slots_of(long long rows, int ncols)
{
    Slots p;
    p.lanes = kRingThreads / ncols;
    p.rows = kSlotPasses * p.lanes;
    p.total = static_cast<int>((rows + p.rows - 1) / p.rows);
    p.held = min(p.total, ring_slots<N>());
    return p;
}

// One thread's view of the ring: a place in the sequence of loads, and its own 16 bytes of a slot.
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
    // A wait that ran out raises `abort`, which ends all later ones at once: the block runs on to its end
    // (every thread meets the same barriers) with the error recorded.
    __device__ __forceinline__ void wait() const { mbar_wait(full0 + 8 * slot, phase, abort, err, E_RING); }
    // the thread's vector of pass k of the slot, `stride` bytes a pass (the ring is only written by copies
    // the compiler does not see, so its loads are spelled out)
    __device__ __forceinline__ uint4 get(int k, uint32_t stride) const
    {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(mine + slot * kSlotBytes + k * stride)
                     : "memory");
        return v;
    }
    __device__ __forceinline__ void release() const
    {
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

// The unit's rows of one thread, in the order in which the ring holds them. `count`: its rows, `stride`:
// vectors of a pass.
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
        c.release();
        c.next();
        if ((i + 1) * kSlotPasses <= count) {
#pragma unroll
            for (int k = 0; k < kSlotPasses; ++k, py += step) finish<TI, TO, VEC, N, kAct>(v[k], py, minus, scale, shift);
        } else {
#pragma unroll
            for (int k = 0; k < kSlotPasses; ++k, py += step)
                if (i * kSlotPasses + k < count) finish<TI, TO, VEC, N, kAct>(v[k], py, minus, scale, shift);
        }
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

// Group norm of units that are shared by the blocks of a cooperative grid. A loading warp streams the
// member's rows through a ring of slots with bulk copies, far ahead of the threads that sum and write,
// so that the memory is never waited for; what the ring can hold is read once. Rows beyond it come a
// second time, the latest first (from L2, as far as it holds them). With a.ahead the ring holds two
// units: the next one's statistics come before this one's output, and the members' join is hidden.
// N: moments a vector, 16 / sizeof(TI) / N channels each, which always belong to one group.
template <typename TI, typename TO, int N>
__global__ void __launch_bounds__(kRingThreads + 32, 2) group_norm_ring_kernel(const GnArgs a)
{
    constexpr int VEC = 16 / sizeof(TI), kPer = VEC / N, kPairs = VEC / 2, kSlots = ring_slots<N>();
    constexpr int kRound = N < 4 ? N : 4;  // moments joined at a time
    using R = Raw<TI, VEC>;
    extern __shared__ uint4 ring[];
    __shared__ float2 entry[kRound][kRingThreads];
    __shared__ float entry_n[kRingThreads];
    __shared__ Moments group[kSliceGroups];
    __shared__ float2 norm[kSliceGroups];
    __shared__ uint64_t bars[2 * kSlots];
    __shared__ int abort_flag, last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int member = static_cast<int>(blockIdx.x) % a.members, team = static_cast<int>(blockIdx.x) / a.members;
    const long long r0 = member * a.rows + min(member, a.more_rows), rows = a.rows + (member < a.more_rows);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kSlots;
    volatile int *abort = &abort_flag;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) {
            mbar_init(full0 + 8 * i, 1);
            mbar_init(empty0 + 8 * i, kRingThreads / 32);
        }
        abort_flag = 0;
        fence_mbar_init();
    }
    __syncthreads();

    if (warp == kRingThreads / 32) {
        uint32_t slot = 0, phase = 0, issued = 0;
        bool ok = true;
        const uint64_t once = l2_evict_first(), again = l2_evict_last();
        for (int unit = team; ok && unit < a.units; unit += a.teams) {
            const int s = unit / a.slices, g0 = (unit - s * a.slices) * a.slice_groups;
            const int ncols = min(a.slice_groups, a.G - g0) * a.cpg / VEC;
            const Slots p = slots_of<N>(rows, ncols);
            const TI *x = static_cast<const TI *>(a.x) + s * a.x_sample + r0 * a.x_row + g0 * a.cpg;
            const uint32_t row_bytes = ncols * 16;
            const bool dense = a.x_row * sizeof(TI) == row_bytes;
            const int loads = 2 * p.total - p.held;
            for (int q = 0; q < loads; ++q, ++issued) {
                const int i = q < p.total ? q : p.total - p.held - 1 - (q - p.total);
                const long long first = static_cast<long long>(i) * p.rows;
                const int n = static_cast<int>(min(static_cast<long long>(p.rows), rows - first));
                ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * slot, phase ^ 1u, abort, a.err, E_RING));
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
        if (!ok) {
            // no copy may still be landing when the block ends: wait for the slots' last loads
            int dummy = 0;
            for (uint32_t k = 0; k < kSlots && k < issued; ++k) {
                const uint32_t q = issued - 1 - k;
                mbar_wait(full0 + 8 * (q % kSlots), (q / kSlots) & 1u, &dummy, a.err, E_RING);
            }
        }
        return;
    }

    const int sub = static_cast<int>(threadIdx.x) / a.group_lanes, sub_lane = threadIdx.x % a.group_lanes;
    Cursor<kSlots> cur{smem_u32(ring) + threadIdx.x * 16, full0, empty0, abort, a.err, 0, 0};
    auto sync = [] { named_barrier_sync(1, kRingThreads); };
    // where the next unit's loads begin in the ring's sequence
    uint32_t begin = 0;

    struct Unit {
        int s, g0, gs, ncols, rl, col, count;
        uint32_t begin;
        Slots p;
    };
    auto describe = [&](int unit) {
        Unit u;
        u.s = unit / a.slices;
        u.g0 = (unit - u.s * a.slices) * a.slice_groups;
        u.gs = min(a.slice_groups, a.G - u.g0);
        u.ncols = u.gs * a.cpg / VEC;
        u.p = slots_of<N>(rows, u.ncols);
        u.rl = static_cast<int>(threadIdx.x) / u.ncols;
        u.col = static_cast<int>(threadIdx.x) - u.rl * u.ncols;
        u.count = u.rl < u.p.lanes && u.rl < rows ? static_cast<int>((rows - u.rl + u.p.lanes - 1) / u.p.lanes) : 0;
        u.begin = begin;
        begin += 2 * u.p.total - u.p.held;
        return u;
    };
    // the unit's moments, handed to its members
    auto statistics = [&](int unit, const Unit &u) {
        Moments mo[N];
        cur.go(u.begin);
        const uint32_t stride = u.p.lanes * u.ncols * 16;
        for (int i = 0; i < u.p.total; i += kRunSlots) {
            constexpr int kSums = N == 1 ? 2 : kPairs;
            float p[N];
            uint64_t minus[N == 1 ? 1 : kPairs], s2[kSums], q2[kSums];
#pragma unroll
            for (int k = 0; k < kSums; ++k) s2[k] = q2[k] = 0;
            const int n = min(kRunSlots, u.p.total - i), valid = min(n * kSlotPasses, u.count - i * kSlotPasses);
            auto add = [&](const uint4 &raw) __attribute__((always_inline)) {
                float f[VEC];
                R::floats(raw, f);
#pragma unroll
                for (int k = 0; k < kPairs; ++k) {
                    const uint64_t d = add2(pair(f[2 * k], f[2 * k + 1]), minus[N == 1 ? 0 : k]);
                    s2[k % kSums] = add2(s2[k % kSums], d);
                    q2[k % kSums] = fma2(d, d, q2[k % kSums]);
                }
            };
            cur.wait();
            {
                float f[VEC];
                R::floats(cur.get(0, stride), f);
#pragma unroll
                for (int e = 0; e < N; ++e) p[e] = f[e * kPer];
#pragma unroll
                for (int k = 0; k < (N == 1 ? 1 : kPairs); ++k)
                    minus[k] = pair(-p[N == 1 ? 0 : 2 * k / kPer], -p[N == 1 ? 0 : (2 * k + 1) / kPer]);
            }
#pragma unroll 1
            for (int v = 0; v < n; ++v) {
                if (v > 0) cur.wait();
                uint4 raw[kSlotPasses];
#pragma unroll
                for (int w = 0; w < kSlotPasses; ++w) raw[w] = cur.get(w, stride);
                if (i + v < u.p.total - u.p.held) cur.release();
                cur.next();
                if ((v + 1) * kSlotPasses <= valid) {
#pragma unroll
                    for (int w = 0; w < kSlotPasses; ++w) add(raw[w]);
                } else {
#pragma unroll
                    for (int w = 0; w < kSlotPasses; ++w)
                        if (v * kSlotPasses + w < valid) add(raw[w]);
                }
            }
            if (valid > 0) {
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
                const float cnt = static_cast<float>(valid * kPer), inv = __fdividef(1.f, cnt);
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    Moments run;
                    run.n = cnt;
                    run.mean = fmaf(sum[e], inv, p[e]);
                    run.m2 = fmaxf(fmaf(-sum[e] * inv, sum[e], sq[e]), 0.f * sq[e]);
                    mo[e] = join(mo[e], run);
                }
            }
        }
        if (sub_lane == 0 && sub < u.gs) group[sub] = Moments();
#pragma unroll
        for (int first = 0; first < N; first += kRound) {
            sync();
#pragma unroll
            for (int e = 0; e < kRound; ++e) entry[e][threadIdx.x] = make_float2(mo[first + e].mean, mo[first + e].m2);
            float n = mo[0].n;
            entry_n[threadIdx.x] = n;
            sync();
            for (int left = u.p.lanes; left > 1;) {
                const int half = (left + 1) / 2;
                if (u.rl + half < left) {
                    const int other = threadIdx.x + half * u.ncols;
                    const float on = entry_n[other];
#pragma unroll
                    for (int e = 0; e < kRound; ++e) {
                        const float2 o = entry[e][other], m = entry[e][threadIdx.x];
                        Moments b, c;
                        b.n = n;
                        b.mean = m.x;
                        b.m2 = m.y;
                        c.n = on;
                        c.mean = o.x;
                        c.m2 = o.y;
                        b = join(b, c);
                        entry[e][threadIdx.x] = make_float2(b.mean, b.m2);
                    }
                    n += on;
                    entry_n[threadIdx.x] = n;
                }
                left = half;
                sync();
            }
            // group `sub`: the moments [sub cpg / kPer, (sub + 1) cpg / kPer) along a row of vectors, those
            // of this round
            Moments m;
            if (sub < u.gs)
                for (int k = sub * a.cpg / kPer + sub_lane; k < (sub + 1) * a.cpg / kPer; k += a.group_lanes) {
                    const int e = k % N - first;
                    if (e >= 0 && e < kRound) {
                        const float2 o = entry[e][k / N];
                        Moments c;
                        c.n = entry_n[0];
                        c.mean = o.x;
                        c.m2 = o.y;
                        m = join(m, c);
                    }
                }
            m = join_lanes(m, a.group_lanes);
            if (sub_lane == 0 && sub < u.gs) group[sub] = join(group[sub], m);
        }
        sync();
        join_grid(a, unit, member, group, u.gs, sub, sub_lane, norm, &last, abort, sync);
    };

    auto output = [&](const Unit &u) {
        float minus[N], scale[VEC], shift[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int c = u.col * VEC + e;
            const float2 mr = norm[min((u.col * VEC + e / kPer * kPer) / a.cpg, u.gs - 1)];
            const int ch = min(u.g0 * a.cpg + c, a.C - 1);
            minus[e / kPer] = -mr.x;
            scale[e] = a.weight ? mr.y * __ldg(a.weight + ch) : mr.y;
            shift[e] = a.bias ? __ldg(a.bias + ch) : 0.f;
        }
        TO *y = static_cast<TO *>(a.y) + u.s * a.y_sample + (r0 + u.rl) * a.y_row + u.g0 * a.cpg + u.col * VEC;
        const long long y_step = u.p.lanes * a.y_row;
        const uint32_t stride = u.p.lanes * u.ncols * 16;
        cur.go(u.begin + u.p.total - u.p.held);
        switch (a.act) {
        case S2_ACT_RELU: write_slots<TI, TO, N, S2_ACT_RELU>(cur, u.p, u.count, stride, y, y_step, minus, scale, shift); break;
        case S2_ACT_SILU: write_slots<TI, TO, N, S2_ACT_SILU>(cur, u.p, u.count, stride, y, y_step, minus, scale, shift); break;
        case S2_ACT_GELU: write_slots<TI, TO, N, S2_ACT_GELU>(cur, u.p, u.count, stride, y, y_step, minus, scale, shift); break;
        case S2_ACT_GELU_TANH:
            write_slots<TI, TO, N, S2_ACT_GELU_TANH>(cur, u.p, u.count, stride, y, y_step, minus, scale, shift);
            break;
        default: write_slots<TI, TO, N, S2_ACT_NONE>(cur, u.p, u.count, stride, y, y_step, minus, scale, shift);
        }
    };

    for (int unit = team; unit < a.units; unit += a.teams) {
        const Unit u = describe(unit);
        statistics(unit, u);
        output(u);
    }
}

// The units, members and shared memory of a call.
struct Plan {
    int slices, slice_groups, units, members, teams, join, hold;
    size_t smem;
};

size_t elem(int dtype) { return dtype == S2_F32 ? 4 : 2; }

// Vectors of 16 bytes of x (their y 8 or 16 bytes) need every row to start on one.
bool is_wide(const s2_group_norm_act_desc &d)
{
    const size_t ie = elem(d.in_dtype), oe = elem(d.out_dtype), vec = 16 / ie;
    const uintptr_t xb = reinterpret_cast<uintptr_t>(d.x) | d.x_row * ie | (d.samples > 1 ? d.x_sample * ie : 0);
    const uintptr_t yb = reinterpret_cast<uintptr_t>(d.y) | d.y_row * oe | (d.samples > 1 ? d.y_sample * oe : 0);
    // slices begin at whole groups, so these have to fall on whole vectors too
    return d.channels % vec == 0 && xb % 16 == 0 && yb % (vec * oe) == 0;
}

constexpr size_t kPiece = kThreads * 16;    // shared memory of one vector a thread
constexpr size_t kHoldTwo = 22 * kPiece;    // held by each of two blocks an SM
constexpr size_t kMaxHold = 50 * kPiece;    // by a block alone

Plan plan_of(const s2_group_norm_act_desc &d, int sms)
{
    const bool wide = is_wide(d);
    const long long size = static_cast<long long>(elem(d.in_dtype)), cpg = d.channels / d.groups;
    const int vec = wide ? static_cast<int>(16 / size) : 1;
    // slices are whole vectors
    int step = 1;
    while (step * cpg % vec != 0) ++step;
    auto slices_of = [&](int sg) { return (d.groups + sg - 1) / sg; };
    auto bytes_of = [&](int sg) { return d.positions * sg * cpg * size; };  // of a unit
    auto fit = [&](int sg, int members, size_t hold) { return (bytes_of(sg) + members - 1) / members <= static_cast<long long>(hold * 15 / 16); };
    Plan p;
    p.slice_groups = std::max(step, std::min(d.groups, kSliceGroups / step * step));
    auto halve = [&](int sg) { return std::max(step, sg / 2 / step * step); };
    auto width = [&](int sg) { return sg * cpg * size; };
    p.smem = kHoldTwo;
    p.join = kGrid;
    for (int sg = p.slice_groups;; sg = halve(sg)) {
        if (fit(sg, kMaxCluster, kHoldTwo)) {
            p.slice_groups = sg;
            p.join = kCluster;
            break;
        }
        if (halve(sg) == sg || width(halve(sg)) < 128) break;
    }
    if (p.join == kCluster) {
        p.members = 1;
        while (!fit(p.slice_groups, p.members, kHoldTwo)) p.members *= 2;
        auto few = [&] { return 1LL * d.samples * slices_of(p.slice_groups) * p.members < sms; };
        while (few() && p.members < kMaxCluster && d.positions >= 32 * p.members) p.members *= 2;
        while (few() && halve(p.slice_groups) < p.slice_groups && width(halve(p.slice_groups)) >= 128) p.slice_groups = halve(p.slice_groups);
    } else {
        while (!fit(p.slice_groups, sms, kHoldTwo) && halve(p.slice_groups) < p.slice_groups && width(halve(p.slice_groups)) >= 64)
            p.slice_groups = halve(p.slice_groups);
        const long long want = (bytes_of(p.slice_groups) + kHoldTwo - 1) / kHoldTwo;
        p.members = static_cast<int>(std::min<long long>(sms, want));
    }
    if (const char *e = getenv("GN_SG")) p.slice_groups = atoi(e);
    if (const char *e = getenv("GN_JOIN")) p.join = atoi(e);
    if (const char *e = getenv("GN_T")) p.members = atoi(e);
    if (const char *e = getenv("GN_HOLD")) p.smem = atoi(e) * kPiece;
    p.slices = slices_of(p.slice_groups);
    p.units = d.samples * p.slices;
    p.teams = p.units;
    if (p.join == kGrid)
        p.teams = std::max(1, std::min(p.units, (p.smem <= kHoldTwo ? 2 : 1) * sms / p.members));
    if (p.join == kRing) p.teams = std::max(1, std::min(p.units, 2 * sms / p.members));
    if (const char *e = getenv("GN_TEAMS")) p.teams = atoi(e);
    if (p.join == kCluster && p.members == 1) p.join = kAlone;
    // no more shared memory than the rows need
    const long long rows = (d.positions + p.members - 1) / p.members, ncols = p.slice_groups * cpg / vec;
    const long long lanes = std::max<long long>(1, kThreads / ncols), pieces = (rows + lanes - 1) / lanes;
    p.smem = std::min<size_t>(p.smem, static_cast<size_t>(pieces) * kThreads * (wide ? 16 : size));
    return p;
}

size_t round_up16(size_t v) { return (v + 15) / 16 * 16; }

size_t workspace_of(const Plan &p)
{
    if (p.join != kGrid && p.join != kRing) return 0;
    return round_up16(static_cast<size_t>(p.units) * 8) +
           static_cast<size_t>(p.units) * (p.members + 1) * p.slice_groups * sizeof(float2);
}

int sm_count()
{
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
        cudaGetLastError();
    return sms > 0 ? sms : 148;
}

template <typename TI, typename TO, int VEC, bool kOne>
s2_status launch(GnArgs &a, const Plan &p, cudaStream_t st)
{
    auto kernel = group_norm_kernel<TI, TO, VEC, kOne>;
    static std::atomic<uint64_t> configured{0};
    const s2_status cs = s2::once_per_device(configured, [&] {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxHold);
        return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: %s", cudaGetErrorString(e));
    });
    if (cs != S2_OK) return cs;
    a.hold = static_cast<int>(p.smem / (kThreads * sizeof(typename Raw<TI, VEC>::type)));
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    if (p.join == kGrid) {
        attr[0].id = cudaLaunchAttributeCooperative;
        attr[0].val.cooperative = 1;
    } else {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = static_cast<unsigned>(p.members);
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
    }
    cfg.gridDim = dim3(static_cast<unsigned>(p.teams) * p.members);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: launch failed: %s", cudaGetErrorString(e));
}

template <typename TI, typename TO, int N>
s2_status launch_ring(const GnArgs &a, const Plan &p, cudaStream_t st)
{
    auto kernel = group_norm_ring_kernel<TI, TO, N>;
    constexpr int kBytes = static_cast<int>(ring_slots<N>() * kSlotBytes);
    static std::atomic<uint64_t> configured{0};
    const s2_status cs = s2::once_per_device(configured, [&] {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: %s", cudaGetErrorString(e));
    });
    if (cs != S2_OK) return cs;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.gridDim = dim3(static_cast<unsigned>(p.teams) * p.members);
    cfg.blockDim = dim3(kRingThreads + 32);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    return e == cudaSuccess ? S2_OK : s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: launch failed: %s", cudaGetErrorString(e));
}

template <typename TI, typename TO>
s2_status launch_types(GnArgs &a, const Plan &p, bool wide, cudaStream_t st)
{
    constexpr int kWide = 16 / sizeof(TI);
    if (p.join == kRing) {
        if (a.cpg % kWide == 0) return launch_ring<TI, TO, 1>(a, p, st);
        if (a.cpg % (kWide / 2) == 0) return launch_ring<TI, TO, 2>(a, p, st);
        if constexpr (kWide == 8)
            if (a.cpg % 2 == 0) return launch_ring<TI, TO, 4>(a, p, st);
        return launch_ring<TI, TO, kWide>(a, p, st);
    }
    if (!wide) return launch<TI, TO, 1, true>(a, p, st);
    return a.cpg % kWide == 0 ? launch<TI, TO, kWide, true>(a, p, st) : launch<TI, TO, kWide, false>(a, p, st);
}

s2_status check(const s2_group_norm_act_desc *d)
{
    if (!d) return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: NULL description");
    if (d->samples < 0 || d->positions < 0 || d->channels <= 0 || d->groups <= 0 || d->channels % d->groups != 0)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: bad shape (samples %d, positions %lld, channels %d, groups %d)",
                             d->samples, d->positions, d->channels, d->groups);
    if (d->groups > kMaxGroups || d->samples > 65535 || d->positions > (1LL << 31))
        return s2::set_error(S2_UNSUPPORTED, "s2_group_norm_act: at most %d groups, 65535 samples and 2^31 positions", kMaxGroups);
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
    if (d->x_row < d->channels || d->y_row < d->channels || d->x_row > (1LL << 40) || d->y_row > (1LL << 40) ||
        (d->samples > 1 && (d->x_sample < (d->positions - 1) * d->x_row + d->channels ||
                            d->y_sample < (d->positions - 1) * d->y_row + d->channels)))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: a pitch is smaller than what it spans");
    if (!in_place(*d) && s2::may_overlap(span(d->x, *d, d->x_row, d->x_sample, static_cast<long long>(ie)),
                                         span(d->y, *d, d->y_row, d->y_sample, static_cast<long long>(oe))))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: y overlaps x");
    const Plan p = plan_of(*d, sm_count());
    const size_t need = workspace_of(p);
    if (need > 0 && (!d->workspace || d->workspace_bytes < need || reinterpret_cast<uintptr_t>(d->workspace) % 16))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: workspace of %zu bytes, 16-byte aligned, needed", need);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    GnArgs a;
    a.x = d->x;
    a.y = d->y;
    a.weight = d->weight;
    a.bias = d->bias;
    a.part = a.joined = nullptr;
    a.arrived = a.ready = nullptr;
    if (p.join == kGrid || p.join == kRing) {
        a.arrived = static_cast<uint32_t *>(d->workspace);
        a.ready = a.arrived + p.units;
        a.joined = reinterpret_cast<float2 *>(static_cast<char *>(d->workspace) + round_up16(static_cast<size_t>(p.units) * 8));
        a.part = a.joined + static_cast<size_t>(p.units) * p.slice_groups;
        const cudaError_t e = cudaMemsetAsync(a.arrived, 0, static_cast<size_t>(p.units) * 8, st);
        if (e != cudaSuccess) return s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: %s", cudaGetErrorString(e));
    }
    a.err = d->err;
    a.rows = d->positions / p.members;
    a.more_rows = static_cast<int>(d->positions % p.members);
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
    a.members = p.members;
    a.teams = p.teams;
    a.join = p.join;
    a.group_lanes = 32;
    while (a.group_lanes * p.slice_groups > (p.join == kRing ? kRingThreads : kThreads)) a.group_lanes /= 2;
    a.act = d->activation;
    a.eps = d->eps;
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
