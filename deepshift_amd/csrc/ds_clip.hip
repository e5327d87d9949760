// The global norm of many tensors, and their clipping by it.
//
//   n = sqrt(sum over all tensors of x^2)        f = min(1, max_norm / (n + 1e-6))        out = f * x
//
// Bound by memory: one pass reads everything, a second one reads and writes it.  Tensors travel in the kernel arguments,
// some two hundred to a launch, so nothing is copied to the device and a call can be captured.
#include "ds_train.h"

namespace ds {

constexpr int kSpans = 128;        // per launch: 4 KB of arguments
constexpr int kClipChunk = 16384;  // elements that a workgroup takes at a time
constexpr int kClipBlocks = 2048;  // partial sums of one launch at most

struct SpanTable {
    const void *src[kSpans];
    void *dst[kSpans];
    int64_t n[kSpans];
    int32_t first[kSpans];  // chunks before this tensor
    uint8_t src_type[kSpans], dst_type[kSpans];
    int count, chunks;
};

// Which tensor holds chunk c: the last one that begins at or before it.  Every lane looks at two.
__device__ __forceinline__ int span_of(const SpanTable &t, int c)
{
    const int lane = threadIdx.x & 63;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kSpans; j += 64) {
        const int i = j + lane;
        n += __popcll(__ballot(i < t.count && t.first[i] <= c));
    }
    return __builtin_amdgcn_readfirstlane(n - 1);
}

// Squares are added up in 64 bits: values of float32 up to its largest have a norm, and the order of the additions, which
// is fixed all the same, would not show.
template <typename E>
__device__ __forceinline__ double square_sum(const E *__restrict__ x, int n)
{
    double s0 = 0, s1 = 0;
    constexpr int N = 16 / sizeof(E);
    int i = 0;
    if (((uintptr_t)x & 15) == 0) {
        const Vec<E, N> *v = (const Vec<E, N> *)x;
        const int units = n / N;
        constexpr int kAhead = 4;
        for (int u = threadIdx.x; u < units; u += 256 * kAhead) {
            Vec<E, N> got[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (u + j * 256 < units) got[j] = v[u + j * 256];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (u + j * 256 >= units) break;
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    const double a = (double)to_float(got[j].v[e]), b = (double)to_float(got[j].v[e + 1]);
                    s0 = fma(a, a, s0);
                    s1 = fma(b, b, s1);
                }
            }
        }
        i = units * N;
    }
    for (i += threadIdx.x; i < n; i += 256) {
        const double a = (double)to_float(x[i]);
        s0 = fma(a, a, s0);
    }
    return s0 + s1;
}

__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// The sum of 256 threads' values, in every thread.
__device__ __forceinline__ double block_sum(double v, double *lds)
{
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__global__ __launch_bounds__(256) void clip_norm_kernel(SpanTable t, double *__restrict__ part)
{
    __shared__ double lds[4];
    double s = 0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = span_of(t, c);
        const int64_t at = (int64_t)(c - t.first[i]) * kClipChunk;
        const int n = (int)min((int64_t)kClipChunk, t.n[i] - at);
        if (t.src_type[i] == DS_F32) s += square_sum((const float *)t.src[i] + at, n);
        else if (t.src_type[i] == DS_BF16) s += square_sum((const bf16_t *)t.src[i] + at, n);
        else s += square_sum((const f16_t *)t.src[i] + at, n);
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// The norm from the partial sums, in the same order in every workgroup.
__device__ __forceinline__ double norm_of(const double *__restrict__ part, int parts, double *lds)
{
    double s = 0;
    for (int i = threadIdx.x; i < parts; i += 256) s += part[i];
    return sqrt(block_sum(s, lds));
}

__global__ __launch_bounds__(256) void clip_join_kernel(const double *__restrict__ part, int parts, float *__restrict__ norm)
{
    __shared__ double lds[4];
    const double n = norm_of(part, parts, lds);
    if (threadIdx.x == 0) *norm = (float)n;
}

template <typename E, typename O>
__device__ __forceinline__ void scale_span(const E *x, O *y, int n, float pre, float f)
{
    constexpr int N = sizeof(E) == 4 && sizeof(O) == 4 ? 4 : 8;
    int i = 0;
    if (((uintptr_t)x % (sizeof(E) * N < 16 ? sizeof(E) * N : 16)) == 0 && ((uintptr_t)y % (sizeof(O) * N < 16 ? sizeof(O) * N : 16)) == 0) {
        const int units = n / N;
        constexpr int kAhead = 4;
        for (int u = threadIdx.x; u < units; u += 256 * kAhead) {
            Vec<E, N> got[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                if (u + j * 256 < units) got[j] = ((const Vec<E, N> *)x)[u + j * 256];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (u + j * 256 >= units) break;
                Vec<O, N> o;
#pragma unroll
                for (int e = 0; e < N; ++e) o.v[e] = from_float<O>(to_float(got[j].v[e]) * pre * f);
                ((Vec<O, N> *)y)[u + j * 256] = o;
            }
        }
        i = units * N;
    }
    for (i += threadIdx.x; i < n; i += 256) y[i] = from_float<O>(to_float(x[i]) * pre * f);
}

template <typename E>
__device__ __forceinline__ void scale_any(const SpanTable &t, int i, int64_t at, int n, float pre, float f)
{
    const E *x = (const E *)t.src[i] + at;
    if (t.dst_type[i] == DS_F32) scale_span(x, (float *)t.dst[i] + at, n, pre, f);
    else if (t.dst_type[i] == DS_BF16) scale_span(x, (bf16_t *)t.dst[i] + at, n, pre, f);
    else scale_span(x, (f16_t *)t.dst[i] + at, n, pre, f);
}

__global__ __launch_bounds__(256) void clip_scale_kernel(SpanTable t, const double *__restrict__ part, int parts,
                                                         float max_norm, float *__restrict__ norm)
{
    __shared__ double lds[4];
    const double n = norm_of(part, parts, lds);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double ratio = (double)max_norm / (n + 1e-6);
    // a factor that float32 would hold with fewer bits is applied in two steps; a norm that is no number stays one
    const float pre = ratio < 0x1p-64 ? 0x1p-64f : 1.f;
    const float f = ratio >= 1.0 ? 1.f : (float)(ratio / pre);
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = span_of(t, c);
        // a factor of one leaves a tensor in place as it is
        if (f == 1.f && t.src[i] == t.dst[i] && t.src_type[i] == t.dst_type[i]) continue;
        const int64_t at = (int64_t)(c - t.first[i]) * kClipChunk;
        const int m = (int)min((int64_t)kClipChunk, t.n[i] - at);
        if (t.src_type[i] == DS_F32) scale_any<float>(t, i, at, m, pre, f);
        else if (t.src_type[i] == DS_BF16) scale_any<bf16_t>(t, i, at, m, pre, f);
        else scale_any<f16_t>(t, i, at, m, pre, f);
    }
}

// The tensors from `from` on that one launch takes; returns the first one that it does not.
int fill_table(const ds_tensor *tensors, int count, int from, SpanTable &t, int64_t *too_many)
{
    t.count = 0;
    int64_t chunks = 0;
    int i = from;
    for (; i < count && t.count < kSpans; ++i) {
        const ds_tensor &x = tensors[i];
        if (x.n == 0) continue;
        const int64_t more = (x.n + kClipChunk - 1) / kClipChunk;
        if (chunks + more > 0x7fffffff - kClipBlocks) {
            if (t.count == 0) *too_many = 1;
            break;
        }
        t.src[t.count] = x.src;
        t.dst[t.count] = x.dst;
        t.n[t.count] = x.n;
        t.src_type[t.count] = (uint8_t)x.src_type;
        t.dst_type[t.count] = (uint8_t)x.dst_type;
        t.first[t.count++] = (int32_t)chunks;
        chunks += more;
    }
    t.chunks = (int)chunks;
    return i;
}

inline size_t clip_bytes(int count) { return (size_t)(count / kSpans + 1) * kClipBlocks * sizeof(double); }

}  // namespace ds

using namespace ds;

DS_EXPORT size_t ds_clip_workspace_bytes(int count) { return count < 0 ? 0 : clip_bytes(count); }

DS_EXPORT int ds_clip(const ds_tensor *tensors, int count, float max_norm, int scale, float *norm, void *workspace,
                      size_t workspace_bytes, ds_stream_t stream)
{
    if (count < 0 || (count > 0 && !tensors) || (!norm && !scale) || !(max_norm >= 0.f || !scale)) return DS_EINVAL;
    for (int i = 0; i < count; ++i) {
        const ds_tensor &x = tensors[i];
        if (x.n < 0 || !element_bytes(x.src_type) || (x.n > 0 && !x.src)) return DS_EINVAL;
        if (scale && (!element_bytes(x.dst_type) || (x.n > 0 && !x.dst))) return DS_EINVAL;
        if ((uintptr_t)x.src % element_bytes(x.src_type) || (scale && (uintptr_t)x.dst % element_bytes(x.dst_type))) return DS_EINVAL;
    }
    if (!workspace || workspace_bytes < clip_bytes(count) || (uintptr_t)workspace % 8) return DS_EWORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    double *part = (double *)workspace;
    SpanTable t;
    int64_t too_many = 0;
    int parts = 0, launches = 0;
    for (int i = 0; i < count;) {
        i = fill_table(tensors, count, i, t, &too_many);
        if (too_many || (size_t)(parts + kClipBlocks) * sizeof(double) > clip_bytes(count)) return DS_ETOOLARGE;
        if (t.chunks == 0) continue;
        const int blocks = t.chunks < kClipBlocks ? t.chunks : kClipBlocks;
        hipLaunchKernelGGL(clip_norm_kernel, dim3(blocks), dim3(256), 0, st, t, part + parts);
        parts += blocks;
        ++launches;
    }
    if (!scale || launches == 0) {
        if (!norm) return DS_OK;
        hipLaunchKernelGGL(clip_join_kernel, dim3(1), dim3(256), 0, st, part, parts, norm);
        return launch_status();
    }
    for (int i = 0, done = 0; i < count; ) {
        i = fill_table(tensors, count, i, t, &too_many);
        if (t.chunks == 0) continue;
        const int blocks = t.chunks < kClipBlocks ? t.chunks : kClipBlocks;
        hipLaunchKernelGGL(clip_scale_kernel, dim3(blocks), dim3(256), 0, st, t, part, parts, max_norm, done++ == 0 ? norm : nullptr);
    }
    return launch_status();
}
