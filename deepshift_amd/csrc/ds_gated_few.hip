// The gated block for a few tokens, one above all: a token that is served.
//
// Reading the weights is what counts then.  A wave has both halves' rows of one or two results, its lanes share the features, and
// every weight is loaded once, as it lies, and multiplied in vector registers in 32 bits; the tokens come from the caches.  One token
// of 4096 features, 8192 results: bfloat16 26 us, 5.2 TB/s, float32 48 us, 5.6 TB/s (a copy of 2 GiB runs at 4.9).  Which numbers of
// tokens come here, and what they take otherwise, is measured at most_few (ds_gated.hip).
#include "ds_gated.h"

namespace ds {
namespace gated {

// R results of a wave, A pieces of 64 vectors on their way at a time.
template <typename E, int TT, int R, int A>
__global__ __launch_bounds__(256) void few_kernel(Few f)
{
    constexpr int N = 16 / sizeof(E), kPiece = 64 * N, kAll = TT * R * 2;
    __shared__ float sums[4][kAll];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t c0 = ((int64_t)blockIdx.x * 4 + wave) * R;
    const E *w[R][2], *x[TT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[r][h] = (const E *)f.weight + ((c0 + r < f.F ? c0 + r : f.F - 1) + h * f.F) * f.ldw;
#pragma unroll
    for (int t = 0; t < TT; ++t) x[t] = (const E *)f.x + (t < f.T ? t : f.T - 1) * f.ldx;
    float acc[kAll];
#pragma unroll
    for (int k = 0; k < kAll; ++k) acc[k] = 0.f;
    auto multiply = [&](const Vec<E, N> (&v)[R][2], int at, int left) {
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const Vec<E, N> of = load_any<E, N>(x[t] + at, left);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int e = 0; e < N; ++e)
                        acc[(t * R + r) * 2 + h] = fmaf(to_float(v[r][h].v[e]), to_float(of.v[e]), acc[(t * R + r) * 2 + h]);
        }
    };
    int at = lane * N;
    for (int from = 0; from + kPiece * A <= f.D; from += kPiece * A) {
        Vec<E, N> v[A][R][2];
#pragma unroll
        for (int a = 0; a < A; ++a)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int h = 0; h < 2; ++h) __builtin_memcpy(&v[a][r][h], w[r][h] + at + a * kPiece, 16);
#pragma unroll
        for (int a = 0; a < A; ++a) multiply(v[a], at + a * kPiece, N);
        at += kPiece * A;
    }
    for (; at < f.D; at += kPiece) {
        Vec<E, N> v[R][2];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int h = 0; h < 2; ++h) v[r][h] = load_any<E, N>(w[r][h] + at, f.D - at);
        multiply(v, at, f.D - at);
    }
#pragma unroll
    for (int k = 0; k < kAll; ++k)
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) acc[k] += __shfl_xor(acc[k], o);
    if (lane == 0)
#pragma unroll
        for (int k = 0; k < kAll; ++k) sums[wave][k] = acc[k];
    __syncthreads();
    const int t = lane / R;
    const int64_t c = c0 + lane % R;
    if (t >= f.T || c >= f.F) return;
    const float gate = sums[wave][lane * 2] + (f.bias ? to_float(((const E *)f.bias)[c]) : 0.f);
    const float up = sums[wave][lane * 2 + 1] + (f.bias ? to_float(((const E *)f.bias)[f.F + c]) : 0.f);
    ((E *)f.out)[t * f.F + c] = from_float<E>(activation_of(f.activation, gate) * up);
    if (f.halves) f.halves[t * 2 * f.ldz + c] = gate, f.halves[(t * 2 + 1) * f.ldz + c] = up;
}

template <typename E>
int launch_few(const Few &f, hipStream_t st)
{
    auto blocks = [&](int R) { return dim3((unsigned)((f.F + 4 * R - 1) / (4 * R))); };
    if (f.T == 1) hipLaunchKernelGGL((few_kernel<E, 1, 1, 4>), blocks(1), dim3(256), 0, st, f);
    else if (f.T == 2) hipLaunchKernelGGL((few_kernel<E, 2, 1, 4>), blocks(1), dim3(256), 0, st, f);
    else if (f.T <= 4) hipLaunchKernelGGL((few_kernel<E, 4, 2, 2>), blocks(2), dim3(256), 0, st, f);
    else if constexpr (sizeof(E) == 4) {
        if (f.T <= 8) hipLaunchKernelGGL((few_kernel<E, 8, 2, 2>), blocks(2), dim3(256), 0, st, f);
        else hipLaunchKernelGGL((few_kernel<E, 16, 2, 1>), blocks(2), dim3(256), 0, st, f);
    } else {
        return DS_EINVAL;
    }
    return launch_status();
}
template int launch_few<float>(const Few &, hipStream_t);
template int launch_few<bf16_t>(const Few &, hipStream_t);
template int launch_few<f16_t>(const Few &, hipStream_t);

}  // namespace gated
}  // namespace ds
