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
#include <cstdint>

#include "s2_act.cuh"
#include "s2_internal.h"
#include "s2_overlap.h"

namespace {

using namespace s2dev;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxGroups = 1024;
constexpr int kUnroll = 8;  // rows a thread has in flight

struct GnArgs {
    const void *x;
    void *y;
    const float *weight, *bias;
    float2 *part;  // [sample][member][group] (mean, M2)
    long long P, x_row, x_sample, y_row, y_sample;
    int C, G, cpg, members, act;
    float eps;
};

struct Moments {
    float n = 0.f, mean = 0.f, m2 = 0.f;
};

__device__ __forceinline__ Moments join(const Moments &a, const Moments &b)
{
    if (b.n == 0.f) return a;
    Moments r;
    r.n = a.n + b.n;
    const float d = b.mean - a.mean, w = __fdiv_rn(b.n, r.n);
    r.mean = fmaf(d, w, a.mean);
    r.m2 = a.m2 + b.m2 + d * d * a.n * w;
    return r;
}

// VEC elements of T, 16 bytes or one element
template <typename T, int VEC>
struct Vec;
template <typename T>
struct Vec<T, 1> {
    T v;
    __device__ __forceinline__ void load(const T *p) { v = *p; }
    __device__ __forceinline__ void floats(float (&f)[1]) const { f[0] = to_float<T>(v); }
};
template <typename T>
struct Vec<T, 8> {
    uint4 v;
    __device__ __forceinline__ void load(const T *p) { v = *reinterpret_cast<const uint4 *>(p); }
    __device__ __forceinline__ void floats(float (&f)[8]) const
    {
        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = unpack2<T>(u[i]);
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        }
    }
};
template <>
struct Vec<float, 4> {
    float4 v;
    __device__ __forceinline__ void load(const float *p) { v = *reinterpret_cast<const float4 *>(p); }
    __device__ __forceinline__ void floats(float (&f)[4]) const
    {
        f[0] = v.x;
        f[1] = v.y;
        f[2] = v.z;
        f[3] = v.w;
    }
};

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T *p, const float (&f)[VEC])
{
    if constexpr (VEC == 1) {
        *p = from_float<T>(f[0]);
    } else if constexpr (sizeof(T) == 4) {
        static_assert(VEC == 4, "");
        *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
    } else if constexpr (VEC == 8) {
        *reinterpret_cast<uint4 *>(p) =
            make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
    } else {
        *reinterpret_cast<uint2 *>(p) = make_uint2(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]));
    }
}

// Part one: (mean, M2) of every group over the rows of one member of the sample.
template <typename TI, int VEC>
__global__ void __launch_bounds__(kThreads) gn_stats_kernel(const GnArgs a)
{
    __shared__ Moments entry[VEC][kThreads];
    __shared__ Moments group[kMaxGroups];
    const int s = blockIdx.y, member = blockIdx.x;
    const long long r0 = a.P * member / a.members, r1 = a.P * (member + 1) / a.members;
    const TI *x = static_cast<const TI *>(a.x) + s * a.x_sample;
    for (int g = threadIdx.x; g < a.G; g += kThreads) group[g] = Moments();
    const int ncols = a.C / VEC;
    for (int cb = 0; cb < ncols; cb += kThreads) {
        // columns [cb, cb + nb) of vectors, `lanes` rows at a time
        const int nb = min(kThreads, ncols - cb), lanes = kThreads / nb;
        const int col = threadIdx.x % nb, rl = threadIdx.x / nb;
        Moments mo[VEC];
        if (rl < lanes) {
            const TI *px = x + static_cast<long long>(cb + col) * VEC;
            for (long long r = r0 + rl; r < r1; r += 1LL * kUnroll * lanes) {
                Vec<TI, VEC> v[kUnroll];
                const int n = static_cast<int>(min(1LL * kUnroll, (r1 - r + lanes - 1) / lanes));
#pragma unroll
                for (int u = 0; u < kUnroll; ++u)
                    if (u < n) v[u].load(px + (r + 1LL * u * lanes) * a.x_row);
                float p[VEC], sum[VEC], sq[VEC];
                v[0].floats(p);
#pragma unroll
                for (int e = 0; e < VEC; ++e) sum[e] = sq[e] = 0.f;
#pragma unroll
                for (int u = 1; u < kUnroll; ++u)
                    if (u < n) {
                        float f[VEC];
                        v[u].floats(f);
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float d = f[e] - p[e];
                            sum[e] += d;
                            sq[e] = fmaf(d, d, sq[e]);
                        }
                    }
                const float inv = __fdiv_rn(1.f, static_cast<float>(n));
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    Moments run;
                    run.n = static_cast<float>(n);
                    run.mean = fmaf(sum[e], inv, p[e]);
                    // not below 0 by rounding; 0 * sq keeps the NaN of a value that is not finite
                    run.m2 = fmaxf(sq[e] - sum[e] * sum[e] * inv, 0.f * sq[e]);
                    mo[e] = join(mo[e], run);
                }
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) entry[e][threadIdx.x] = mo[e];
        __syncthreads();
        // a warp per group that has channels in [cb, cb + nb) * VEC
        const int c0 = cb * VEC, c1 = (cb + nb) * VEC;
        for (int g = c0 / a.cpg + (threadIdx.x >> 5); g * a.cpg < c1; g += kWarps) {
            const int lo = max(c0, g * a.cpg), w = min(c1, (g + 1) * a.cpg) - lo;
            Moments m;
            for (int i = threadIdx.x & 31; i < lanes * w; i += 32) {
                const int c = lo - c0 + i % w;
                m = join(m, entry[c % VEC][(i / w) * nb + c / VEC]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                Moments t;
                t.n = __shfl_down_sync(0xffffffffu, m.n, o);
                t.mean = __shfl_down_sync(0xffffffffu, m.mean, o);
                t.m2 = __shfl_down_sync(0xffffffffu, m.m2, o);
                m = join(m, t);
            }
            if ((threadIdx.x & 31) == 0) group[g] = join(group[g], m);
        }
    }
    __syncthreads();
    for (int g = threadIdx.x; g < a.G; g += kThreads)
        a.part[(static_cast<long long>(s) * a.members + member) * a.G + g] = make_float2(group[g].mean, group[g].m2);
}

template <int VEC>
__device__ __forceinline__ void activate_vec(float (&f)[VEC], int act)
{
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        if (act == S2_ACT_RELU) f[e] = activate<S2_ACT_RELU>(f[e]);
        if (act == S2_ACT_SILU) f[e] = activate<S2_ACT_SILU>(f[e]);
        if (act == S2_ACT_GELU) f[e] = activate<S2_ACT_GELU>(f[e]);
        if (act == S2_ACT_GELU_TANH) f[e] = activate<S2_ACT_GELU_TANH>(f[e]);
    }
}

// Part two: the members' moments joined, then the rows of one member.
template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(kThreads) gn_apply_kernel(const GnArgs a)
{
    // mean = hi + lo, 1 / sqrt(v + eps)
    __shared__ float hi[kMaxGroups], lo[kMaxGroups], rstd[kMaxGroups];
    const int s = blockIdx.y, member = blockIdx.x;
    const long long r0 = a.P * member / a.members, r1 = a.P * (member + 1) / a.members;
    for (int g = threadIdx.x; g < a.G; g += kThreads) {
        double n = 0.0, mean = 0.0, m2 = 0.0;
        for (int t = 0; t < a.members; ++t) {
            const double nb = static_cast<double>(a.P * (t + 1) / a.members - a.P * t / a.members) * a.cpg;
            if (nb == 0.0) continue;
            const float2 q = a.part[(static_cast<long long>(s) * a.members + t) * a.G + g];
            const double d = q.x - mean, w = nb / (n + nb);
            mean += d * w;
            m2 += q.y + d * d * n * w;
            n += nb;
        }
        hi[g] = static_cast<float>(mean);
        lo[g] = static_cast<float>(mean - hi[g]);
        rstd[g] = static_cast<float>(1.0 / sqrt(m2 / n + a.eps));
    }
    __syncthreads();
    const TI *x = static_cast<const TI *>(a.x) + s * a.x_sample;
    TO *y = static_cast<TO *>(a.y) + s * a.y_sample;
    const int ncols = a.C / VEC;
    for (int cb = 0; cb < ncols; cb += kThreads) {
        const int nb = min(kThreads, ncols - cb), lanes = kThreads / nb;
        const int col = cb + threadIdx.x % nb, rl = threadIdx.x / nb;
        if (rl >= lanes) continue;
        // y = (x - hi) scale + shift: the subtraction first, as the formula has it
        float mean[VEC], scale[VEC], shift[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int c = col * VEC + e, g = c / a.cpg;
            mean[e] = hi[g];
            scale[e] = rstd[g] * (a.weight ? __ldg(a.weight + c) : 1.f);
            shift[e] = (a.bias ? __ldg(a.bias + c) : 0.f) - lo[g] * scale[e];
        }
        for (long long r = r0 + rl; r < r1; r += lanes) {
            Vec<TI, VEC> v;
            v.load(x + r * a.x_row + static_cast<long long>(col) * VEC);
            float f[VEC];
            v.floats(f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = fmaf(f[e] - mean[e], scale[e], shift[e]);
            activate_vec<VEC>(f, a.act);
            store_vec<TO, VEC>(y + r * a.y_row + static_cast<long long>(col) * VEC, f);
        }
    }
}

int members_of(const s2_group_norm_act_desc &d)
{
    const long long want = std::max<long long>(1, 1184 / std::max(1, d.samples));
    return static_cast<int>(std::max<long long>(1, std::min<long long>(want, d.positions / 16)));
}

template <typename TI, typename TO, int VEC>
void launch(const GnArgs &a, int samples, cudaStream_t st)
{
    const dim3 grid(static_cast<unsigned>(a.members), static_cast<unsigned>(samples));
    gn_stats_kernel<TI, VEC><<<grid, kThreads, 0, st>>>(a);
    gn_apply_kernel<TI, TO, VEC><<<grid, kThreads, 0, st>>>(a);
}

template <typename TI, typename TO>
void launch_types(const GnArgs &a, int samples, cudaStream_t st)
{
    constexpr int kWide = 16 / sizeof(TI);
    const uintptr_t out_bytes = kWide * sizeof(TO);
    const bool wide = a.C % kWide == 0 && (reinterpret_cast<uintptr_t>(a.x) | a.x_row * sizeof(TI) |
                                           a.x_sample * sizeof(TI)) % 16 == 0 &&
                      (reinterpret_cast<uintptr_t>(a.y) | a.y_row * sizeof(TO) | a.y_sample * sizeof(TO)) % out_bytes == 0;
    if (wide)
        launch<TI, TO, kWide>(a, samples, st);
    else
        launch<TI, TO, 1>(a, samples, st);
}

size_t elem(int dtype) { return dtype == S2_F32 ? 4 : 2; }

s2_status check(const s2_group_norm_act_desc *d)
{
    if (!d) return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: NULL description");
    if (d->samples < 0 || d->positions < 0 || d->channels <= 0 || d->groups <= 0 || d->channels % d->groups != 0)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: bad shape (samples %d, positions %lld, channels %d, groups %d)",
                             d->samples, d->positions, d->channels, d->groups);
    if (d->groups > kMaxGroups || d->samples > 65535 || d->positions > (1LL << 40))
        return s2::set_error(S2_UNSUPPORTED, "s2_group_norm_act: at most %d groups, 65535 samples and 2^40 positions", kMaxGroups);
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
    return static_cast<size_t>(d->samples) * members_of(*d) * d->groups * sizeof(float2);
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
    const size_t need = s2_group_norm_act_workspace_bytes(d);
    if (need > 0 && (!d->workspace || d->workspace_bytes < need || reinterpret_cast<uintptr_t>(d->workspace) % 16))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_group_norm_act: workspace of %zu bytes, 16-byte aligned, needed", need);
    GnArgs a;
    a.x = d->x;
    a.y = d->y;
    a.weight = d->weight;
    a.bias = d->bias;
    a.part = static_cast<float2 *>(d->workspace);
    a.P = d->positions;
    a.x_row = d->x_row;
    a.x_sample = d->samples > 1 ? d->x_sample : 0;
    a.y_row = d->y_row;
    a.y_sample = d->samples > 1 ? d->y_sample : 0;
    a.C = d->channels;
    a.G = d->groups;
    a.cpg = d->channels / d->groups;
    a.members = members_of(*d);
    a.act = d->activation;
    a.eps = d->eps;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (d->in_dtype == S2_F16)
        launch_types<__half, __half>(a, d->samples, st);
    else if (d->in_dtype == S2_BF16)
        launch_types<__nv_bfloat16, __nv_bfloat16>(a, d->samples, st);
    else if (d->out_dtype == S2_F32)
        launch_types<float, float>(a, d->samples, st);
    else if (d->out_dtype == S2_F16)
        launch_types<float, __half>(a, d->samples, st);
    else
        launch_types<float, __nv_bfloat16>(a, d->samples, st);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return s2::set_error(S2_INFERENCE_FAILED, "s2_group_norm_act: launch failed: %s", cudaGetErrorString(e));
    if (launches) *launches = 2;
    return S2_OK;
}
