// The global norm of many tensors, and their clipping by it.
//
//   n = sqrt(sum over all tensors of x^2)        f = min(1, max_norm / (n + 1e-6))        out = f * x
//
// Bound by memory: one pass reads everything, a second one reads and writes it, unless the factor is 1 and the tensors stay where
// they are.  Tensors travel in the kernel arguments, some two hundred to a launch, so nothing is copied to the device and a call
// can be captured.  144 bfloat16 tensors of 0.8 G elements take 255 us for the norm (1.6 GB, 6.3 TB/s) and 910 for their float32
// results (4.8 GB, 5.3 TB/s; 1020 us with stores that stay in the caches); the 161 gradients of a ResNet-50 19 us for the norm
// and 4 where nothing is to clip, 54 both passes where something is; six tensors of 0.7 M elements 4 and 5 us.
#include "ds_train.h"

namespace ds {

constexpr int kClipBlocks = 2048;  // partial sums of one launch at most

// The tensors of a launch: 3.9 KB of kernel arguments, 192 tensors where nothing is written elsewhere, else 136.
template <bool ELSEWHERE>
struct SpanTable {
    static constexpr int kSpans = ELSEWHERE ? 136 : 192;
    const void *src[kSpans];
    int64_t n[kSpans];      // elements | type of src << 56 | type of dst << 60
    int32_t first[kSpans];  // chunks before this tensor
    int count, chunks, chunk;
    void *dst[ELSEWHERE ? kSpans : 1];

    __device__ int64_t elements(int i) const { return n[i] & 0xffffffffffffffll; }
    __device__ int src_type(int i) const { return (int)(n[i] >> 56) & 15; }
    __device__ int dst_type(int i) const { return (int)(n[i] >> 60) & 7; }
    __device__ void *to(int i) const { return ELSEWHERE ? dst[i] : const_cast<void *>(src[i]); }

    // Which tensor holds chunk c: the last one that begins at or before it.  Every lane looks at some.
    __device__ int span_of(int c) const
    {
        const int lane = threadIdx.x & 63;
        int found = 0;
#pragma unroll
        for (int j = 0; j < kSpans; j += 64) {
            const int i = j + lane;
            found += __popcll(__ballot(i < count && i < kSpans && first[i < kSpans ? i : 0] <= c));
        }
        return __builtin_amdgcn_readfirstlane(found - 1);
    }
};

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

__global__ __launch_bounds__(256) void clip_norm_kernel(SpanTable<false> t, double *__restrict__ part)
{
    __shared__ double lds[4];
    double s = 0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const int i = t.span_of(c);
        const int64_t at = (int64_t)(c - t.first[i]) * t.chunk;
        const int n = (int)min((int64_t)t.chunk, t.elements(i) - at);
        if (t.src_type(i) == DS_F32) s += square_sum((const float *)t.src[i] + at, n);
        else if (t.src_type(i) == DS_BF16) s += square_sum((const bf16_t *)t.src[i] + at, n);
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

template <bool STREAM, typename E, typename O>
__device__ __forceinline__ void scale_span(const E *x, O *y, int n, float pre, float f)
{
    constexpr int N = sizeof(O) == 4 ? 4 : 8;
    int i = 0;
    constexpr size_t kFrom = sizeof(E) * N < 16 ? sizeof(E) * N : 16, kTo = sizeof(O) * N < 16 ? sizeof(O) * N : 16;
    if ((uintptr_t)x % kFrom == 0 && (uintptr_t)y % kTo == 0) {
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
                if constexpr (STREAM && sizeof(O) * N == 16) store_streaming((Vec<O, N> *)y + u + j * 256, o);
                else ((Vec<O, N> *)y)[u + j * 256] = o;
            }
        }
        i = units * N;
    }
    for (i += threadIdx.x; i < n; i += 256) y[i] = from_float<O>(to_float(x[i]) * pre * f);
}

template <bool STREAM, typename E, typename TABLE>
__device__ __forceinline__ void scale_any(const TABLE &t, int i, int64_t at, int n, float pre, float f)
{
    const E *x = (const E *)t.src[i] + at;
    if (t.dst_type(i) == DS_F32) scale_span<STREAM>(x, (float *)t.to(i) + at, n, pre, f);
    else if (t.dst_type(i) == DS_BF16) scale_span<STREAM>(x, (bf16_t *)t.to(i) + at, n, pre, f);
    else scale_span<STREAM>(x, (f16_t *)t.to(i) + at, n, pre, f);
}

// Chunks are taken from the last one down: what the norm read last is the likeliest to be in cache still.
template <bool ELSEWHERE>
__global__ __launch_bounds__(256) void clip_scale_kernel(SpanTable<ELSEWHERE> t, const double *__restrict__ part, int parts,
                                                         float max_norm, float *__restrict__ norm)
{
    __shared__ double lds[4];
    const double n = norm_of(part, parts, lds);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
    const double ratio = (double)max_norm / (n + 1e-6);
    // a factor that float32 would hold with fewer bits is applied in two steps; a norm that is no number stays one
    const float pre = ratio < 0x1p-64 ? 0x1p-64f : 1.f;
    const float f = ratio >= 1.0 ? 1.f : (float)(ratio / pre);
    // a factor of one leaves tensors in place as they are
    if (!ELSEWHERE && f == 1.f && pre == 1.f) return;
    for (int c = t.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        const int i = t.span_of(c);
        const int64_t at = (int64_t)(c - t.first[i]) * t.chunk;
        const int m = (int)min((int64_t)t.chunk, t.elements(i) - at);
        if (t.src_type(i) == DS_F32) scale_any<ELSEWHERE, float>(t, i, at, m, pre, f);
        else if (t.src_type(i) == DS_BF16) scale_any<ELSEWHERE, bf16_t>(t, i, at, m, pre, f);
        else scale_any<ELSEWHERE, f16_t>(t, i, at, m, pre, f);
    }
}

// The tensors from `from` on that one launch takes; returns the first one that it does not.
template <bool ELSEWHERE>
int fill_table(const ds_tensor *tensors, int count, int from, int chunk, SpanTable<ELSEWHERE> &t)
{
    t.count = 0;
    t.chunk = chunk;
    int64_t chunks = 0;
    int i = from;
    for (; i < count && t.count < t.kSpans; ++i) {
        const ds_tensor &x = tensors[i];
        if (x.n == 0) continue;
        t.src[t.count] = x.src;
        t.n[t.count] = x.n | (int64_t)x.src_type << 56 | (int64_t)x.dst_type << 60;
        if (ELSEWHERE) t.dst[t.count] = x.dst;
        t.first[t.count++] = (int32_t)chunks;
        chunks += (x.n + chunk - 1) / chunk;
    }
    t.chunks = (int)chunks;
    return i;
}

template <bool ELSEWHERE>
int scale_tensors(const ds_tensor *tensors, int count, int chunk, const double *part, int parts, float max_norm, float *norm,
                  hipStream_t st)
{
    SpanTable<ELSEWHERE> t;
    for (int i = 0; i < count;) {
        i = fill_table(tensors, count, i, chunk, t);
        if (t.chunks == 0) continue;
        const int blocks = t.chunks < kClipBlocks ? t.chunks : kClipBlocks;
        hipLaunchKernelGGL((clip_scale_kernel<ELSEWHERE>), dim3(blocks), dim3(256), 0, st, t, part, parts, max_norm, norm);
        norm = nullptr;
    }
    return launch_status();
}

inline size_t clip_bytes(int count) { return (size_t)(count / SpanTable<false>::kSpans + 1) * kClipBlocks * sizeof(double); }

}  // namespace ds

using namespace ds;

DS_EXPORT size_t ds_clip_workspace_bytes(int count) { return count < 0 ? 0 : clip_bytes(count); }

DS_EXPORT int ds_clip(const ds_tensor *tensors, int count, float max_norm, int scale, float *norm, void *workspace,
                      size_t workspace_bytes, ds_stream_t stream)
{
    if (count < 0 || (count > 0 && !tensors) || (!norm && !scale) || !(max_norm >= 0.f || !scale)) return DS_EINVAL;
    int64_t total = 0;
    bool elsewhere = false;
    for (int i = 0; i < count; ++i) {
        const ds_tensor &x = tensors[i];
        const int from = element_bytes(x.src_type), to = scale ? element_bytes(x.dst_type) : from;
        if (x.n < 0 || !from || !to || (x.n > 0 && (!x.src || (scale && !x.dst)))) return DS_EINVAL;
        if ((uintptr_t)x.src % from || (scale && (uintptr_t)x.dst % to)) return DS_EINVAL;
        if (x.n >= (int64_t)1 << 40 || (total += x.n) >= (int64_t)1 << 40) return DS_ETOOLARGE;
        if (scale && x.n > 0 && (x.src != x.dst || x.src_type != x.dst_type)) elsewhere = true;
    }
    if (!workspace || workspace_bytes < clip_bytes(count) || (uintptr_t)workspace % 8) return DS_EWORKSPACE;
    // Chunks of 64 KB and more keep a workgroup's loads together; few elements are cut smaller, to reach every CU.
    int chunk = 16384;
    while (chunk > 2048 && total / chunk < 2 * device_cus()) chunk >>= 1;
    hipStream_t st = (hipStream_t)stream;
    double *part = (double *)workspace;
    SpanTable<false> t;
    int parts = 0;
    for (int i = 0; i < count;) {
        i = fill_table(tensors, count, i, chunk, t);
        if (t.chunks == 0) continue;
        const int blocks = t.chunks < kClipBlocks ? t.chunks : kClipBlocks;
        hipLaunchKernelGGL(clip_norm_kernel, dim3(blocks), dim3(256), 0, st, t, part + parts);
        parts += blocks;
    }
    if (!scale || parts == 0) {
        if (norm) hipLaunchKernelGGL(clip_join_kernel, dim3(1), dim3(256), 0, st, part, parts, norm);
        return launch_status();
    }
    if (elsewhere) return scale_tensors<true>(tensors, count, chunk, part, parts, max_norm, norm, st);
    return scale_tensors<false>(tensors, count, chunk, part, parts, max_norm, norm, st);
}
