// Matrix product with bias, activation and residual (s2_linear_act):
//   y[m][n] = act(sum_k x[m][k] w[n][k] + bias[n]) + residual[m][n],
// x, w fp16 or bf16, the sum and everything after it in fp32, one rounding at the end.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "s2_act.cuh"
#include "s2_internal.h"
#include "s2_overlap.h"

namespace {

using namespace s2dev;

struct LinearArgs {
    const void *x, *w;
    const float *bias;
    const void *residual;
    void *y;
    long long M, ldx, ldw, ldr, ldy;
    int N, K, act;
};

__device__ __forceinline__ float activate_any(float v, int act)
{
    switch (act) {
    case S2_ACT_RELU: return activate<S2_ACT_RELU>(v);
    case S2_ACT_SILU: return activate<S2_ACT_SILU>(v);
    case S2_ACT_GELU: return activate<S2_ACT_GELU>(v);
    case S2_ACT_GELU_TANH: return activate<S2_ACT_GELU_TANH>(v);
    default: return v;
    }
}

constexpr int kTile = 64, kSlice = 16;

template <typename T, typename TO>
__global__ void __launch_bounds__(256) linear_kernel(const LinearArgs a)
{
    __shared__ float xs[kSlice][kTile + 4], ws[kSlice][kTile + 4];
    const long long m0 = 1LL * blockIdx.x * kTile;
    const int n0 = blockIdx.y * kTile;
    const int tm = threadIdx.x / 16 * 4, tn = threadIdx.x % 16 * 4;
    const T *x = static_cast<const T *>(a.x), *w = static_cast<const T *>(a.w);
    float acc[4][4] = {};
    for (int k0 = 0; k0 < a.K; k0 += kSlice) {
        for (int i = threadIdx.x; i < kTile * kSlice; i += 256) {
            const int r = i / kSlice, k = i % kSlice;
            xs[k][r] = m0 + r < a.M && k0 + k < a.K ? to_float<T>(x[(m0 + r) * a.ldx + k0 + k]) : 0.f;
            ws[k][r] = n0 + r < a.N && k0 + k < a.K ? to_float<T>(w[(n0 + r) * a.ldw + k0 + k]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kSlice; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[k][tm + i], ws[k][tn + j], acc[i][j]);
        __syncthreads();
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const long long m = m0 + tm + i;
            const int n = n0 + tn + j;
            if (m >= a.M || n >= a.N) continue;
            float v = activate_any(acc[i][j] + (a.bias ? a.bias[n] : 0.f), a.act);
            if (a.residual) v += to_float<TO>(static_cast<const TO *>(a.residual)[m * a.ldr + n]);
            static_cast<TO *>(a.y)[m * a.ldy + n] = from_float<TO>(v);
        }
}

template <typename T>
void launch(const LinearArgs &a, bool f32_out, cudaStream_t st)
{
    const dim3 grid(static_cast<unsigned>((a.M + kTile - 1) / kTile), static_cast<unsigned>((a.N + kTile - 1) / kTile));
    if (f32_out)
        linear_kernel<T, float><<<grid, 256, 0, st>>>(a);
    else
        linear_kernel<T, T><<<grid, 256, 0, st>>>(a);
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

s2_status check_operands(const s2_linear_act_desc &d)
{
    const uintptr_t oe = d.out_dtype == S2_F32 ? 4 : 2;
    if (!d.x || !d.w || !d.y) return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: NULL x, w or y");
    if ((reinterpret_cast<uintptr_t>(d.x) | reinterpret_cast<uintptr_t>(d.w)) % 2 ||
        (reinterpret_cast<uintptr_t>(d.y) | reinterpret_cast<uintptr_t>(d.residual)) % oe ||
        reinterpret_cast<uintptr_t>(d.bias) % 4)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: a pointer is not aligned to its elements");
    const long long top = 1LL << 40;
    if (d.ldx < d.K || d.ldw < d.K || d.ldy < d.N || (d.residual && d.ldr < d.N) || d.ldx > top || d.ldw > top ||
        d.ldy > top || d.ldr > top)
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: a pitch is smaller than its row");
    const s2::PitchedSpan y{d.y, d.M, static_cast<long long>(d.N * oe), static_cast<long long>(d.ldy * oe)};
    const bool in_place = d.residual == d.y && d.ldr == d.ldy;
    if (s2::may_overlap(y, {d.x, d.M, 2LL * d.K, 2 * d.ldx}) || s2::may_overlap(y, {d.w, d.N, 2LL * d.K, 2 * d.ldw}) ||
        s2::may_overlap(y, {d.bias, 1, 4LL * d.N, 4LL * d.N}) ||
        (!in_place && s2::may_overlap(y, {d.residual, d.M, static_cast<long long>(d.N * oe),
                                          static_cast<long long>(d.ldr * oe)})))
        return s2::set_error(S2_INVALID_ARGUMENT, "s2_linear_act: y overlaps an input");
    return S2_OK;
}

}  // namespace

extern "C" size_t s2_linear_act_workspace_bytes(const s2_linear_act_desc *d)
{
    s2::clear_error();
    check(d);
    return 0;
}

extern "C" s2_status s2_linear_act(void *stream, const s2_linear_act_desc *d, int *launches)
{
    s2::clear_error();
    if (launches) *launches = 0;
    s2_status s = check(d);
    if (s != S2_OK) return s;
    if (d->M == 0) return S2_OK;
    if ((s = check_operands(*d)) != S2_OK) return s;
    LinearArgs a;
    a.x = d->x;
    a.w = d->w;
    a.bias = d->bias;
    a.residual = d->residual;
    a.y = d->y;
    a.M = d->M;
    a.ldx = d->ldx;
    a.ldw = d->ldw;
    a.ldr = d->ldr;
    a.ldy = d->ldy;
    a.N = d->N;
    a.K = d->K;
    a.act = d->activation;
    if (d->dtype == S2_F16)
        launch<__half>(a, d->out_dtype == S2_F32, static_cast<cudaStream_t>(stream));
    else
        launch<__nv_bfloat16>(a, d->out_dtype == S2_F32, static_cast<cudaStream_t>(stream));
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return s2::set_error(S2_INFERENCE_FAILED, "s2_linear_act: launch failed: %s", cudaGetErrorString(e));
    if (launches) *launches = 1;
    return S2_OK;
}
