// Gated block of a feed-forward layer, and its gradients.
//
//   g = x Wg^T + bg      u = x Wu^T + bu      y = act(g) u                W = [Wg; Wu], 2 F rows
//   dz = [dy u act'(g), dy act(g)]            dx = dz W      dW = dz^T x      db = sum_t dz[t]
//
// One product with both halves forms y in its epilogue; for gradients it leaves g and u too, in 32 bits (rounded to bfloat16 they
// moved dx and dW by as much again as the rounding of dz, which its products need, and of the results).  Going back, one pass
// makes dz of them, in the layout that the products of the vocabulary's cross entropy take, whose two gradient products do the
// rest: 4 T D F operations forward and 8 T D F back, as the formulas have them.
#include "ds_gated.h"

namespace ds {
namespace gated {

// Gradients of a gate and its activation, of one element.
__device__ __forceinline__ void slope_of(int kind, float g, float &act, float &slope)
{
    if (kind == DS_RELU) {
        act = g < 0.f ? 0.f : g, slope = g > 0.f ? 1.f : 0.f;
    } else if (kind == DS_GELU) {
        const float half = 0.5f * erfcf(g * -0.7071067811865476f);
        act = g * half, slope = half + g * exp2f(g * g * (-0.5f * kLog2e)) * 0.3989422804014327f;
    } else {
        const float s = logistic(g), rest = logistic(-g);
        act = kind == DS_SILU ? g * s : s;
        slope = kind == DS_SILU ? fmaf(g * s, rest, s) : s * rest;
    }
}

struct Back {
    const float *halves;  // [T][2][ldz]
    const void *grad;     // [T] rows of ldg
    int64_t ldz, ldg, T;
    int F, activation;
    int rows;             // of a workgroup, a multiple of 8
    void *dz;             // [T] rows of ldp, of `words` elements, zeros behind 2 F
    int64_t ldp;
    int words;
    float *bias_part;     // [workgroups along T][2 F], or NULL
    // float16: dz is held times a power of two that brings the largest to the upper end of its range (loss gradients are small:
    // those below 2^-14 would lose bits, those below 2^-24 everything).  One for all rows: a row whose largest is r times that of all
    // is off by up to 2^-39 / r of its own, which is more than its rounding, 2^-11, below r = 2^-28; dx itself, from the same
    // weights, has 30 powers of two from float16's largest to the least with all bits.
    float *tops;          // the largest finite |dz| of each workgroup of top_kernel, `top_groups` of them
    int top_groups;
    float *factor;        // what the results are multiplied with, but for kProbScale
};

// Eight columns of a row: both halves' gradients, 0 behind F.
template <typename E>
__device__ __forceinline__ void gradients_of(const Back &f, int64_t t, int c, float (&dg)[8], float (&du)[8])
{
    constexpr int N = 16 / sizeof(E);
    const Vec<float, 8> g = *(const Vec<float, 8> *)(f.halves + t * 2 * f.ldz + c);
    const Vec<float, 8> u = *(const Vec<float, 8> *)(f.halves + (t * 2 + 1) * f.ldz + c);
    float dy[8];
#pragma unroll
    for (int k = 0; k < 8; k += N) {
        const Vec<E, N> v = load_any<E, N>((const E *)f.grad + t * f.ldg + c + k, f.F - c - k);
#pragma unroll
        for (int e = 0; e < N; ++e) dy[k + e] = to_float(v.v[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        float act, slope;
        slope_of(f.activation, g.v[e], act, slope);
        dg[e] = c + e < f.F ? dy[e] * (u.v[e] * slope) : 0.f;
        du[e] = c + e < f.F ? dy[e] * act : 0.f;
    }
}

__device__ __forceinline__ int power_above(float top)
{
    int e = 0;
    frexpf(top, &e);
    return top == 0.f ? 0 : e < -100 ? -100 : e > 120 ? 120 : e;
}

// The largest of a workgroup of 256 threads.
__device__ __forceinline__ float largest(float top)
{
    __shared__ float of_wave[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) of_wave[threadIdx.x >> 6] = top;
    __syncthreads();
    return fmaxf(fmaxf(of_wave[0], of_wave[1]), fmaxf(of_wave[2], of_wave[3]));
}

// Eight values to their place in a row of dz; `left` of them exist.
template <typename P>
__device__ __forceinline__ void put_row(uint16_t *row, int col, int left, const float (&v)[8])
{
    if constexpr (P::planes == 1) {
        Vec<uint16_t, 8> o;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const s16x4 four = round4<P>(f32x4{v[h * 4], v[h * 4 + 1], v[h * 4 + 2], v[h * 4 + 3]});
#pragma unroll
            for (int e = 0; e < 4; ++e) o.v[h * 4 + e] = (uint16_t)four[e];
        }
        store_any<uint16_t, 8>(row + col, o, left);
    } else {
        Vec<uint16_t, 8> o[3];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            bf16_t planes[3];
            split_planes(v[e], planes);
#pragma unroll
            for (int q = 0; q < 3; ++q) o[q].v[e] = planes[q].bits;
        }
        if (left >= 8 && col % 8 == 0) {
#pragma unroll
            for (int q = 0; q < 3; ++q) *(Vec<uint16_t, 8> *)(row + (col >> 5) * 96 + q * 32 + (col & 31)) = o[q];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left)
#pragma unroll
                    for (int q = 0; q < 3; ++q) row[((col + e) >> 5) * 96 + q * 32 + ((col + e) & 31)] = o[q].v[e];
        }
    }
}

// A workgroup has 256 columns of both halves of some rows, a thread eight of every eighth row.  Bound by memory.
template <typename P>
__global__ __launch_bounds__(256) void back_kernel(Back f)
{
    typedef typename ElementOf<P>::type E;
    __shared__ float sums[2][8][256];
    const int lane = threadIdx.x % 32, part = threadIdx.x / 32, c = blockIdx.x * 256 + lane * 8;
    float scale = 1.f;
    if constexpr (P::half) {
        float top = 0.f;
        for (int i = threadIdx.x; i < f.top_groups; i += 256) top = fmaxf(top, f.tops[i]);
        const int e = power_above(largest(top));
        scale = ldexpf(kProbScale, -e);
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *f.factor = ldexpf(1.f, e);
    }
    float over_t[2][8];
#pragma unroll
    for (int e = 0; e < 8; ++e) over_t[0][e] = over_t[1][e] = 0.f;
    for (int i = 0; i < f.rows; i += 8) {
        const int64_t t = (int64_t)blockIdx.y * f.rows + i + part;
        if (t >= f.T) break;
        uint16_t *const row = (uint16_t *)f.dz + t * f.ldp;
        if (blockIdx.x == 0 && lane < f.words - 2 * f.F) {
            const int col = 2 * f.F + lane;
#pragma unroll
            for (int q = 0; q < P::planes; ++q) row[P::planes == 1 ? col : (col >> 5) * 96 + q * 32 + (col & 31)] = 0;
        }
        if (c >= f.F) continue;
        float dg[8], du[8];
        gradients_of<E>(f, t, c, dg, du);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            over_t[0][e] += dg[e], over_t[1][e] += du[e];
            if (P::half) dg[e] *= scale, du[e] *= scale;
        }
        put_row<P>(row, c, f.F - c, dg);
        put_row<P>(row, f.F + c, f.F - c, du);
    }
    if (!f.bias_part) return;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 8; ++e) sums[h][part][lane * 8 + e] = over_t[h][e];
    __syncthreads();
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= f.F) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += sums[h][w][threadIdx.x];
        f.bias_part[(int64_t)blockIdx.y * 2 * f.F + h * f.F + v] = s;
    }
}

// The largest finite |dz|, of every workgroup's eighths of rows (one atomic maximum for all waves took 100 us where 1543 rows of
// 2731 columns take 12).
constexpr int kTopGroups = 1024;
__global__ __launch_bounds__(256) void top_kernel(Back f)
{
    const int lane = threadIdx.x % 32, part = threadIdx.x / 32, across = (f.F + 255) / 256;
    const int64_t units = (f.T + 7) / 8 * across;
    float top = 0.f;
    for (int64_t i = blockIdx.x; i < units; i += gridDim.x) {
        const int64_t t = i / across * 8 + part;
        const int c = (int)(i % across) * 256 + lane * 8;
        if (t >= f.T || c >= f.F) continue;
        float dg[8], du[8];
        gradients_of<f16_t>(f, t, c, dg, du);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (fabsf(dg[e]) < INFINITY) top = fmaxf(top, fabsf(dg[e]));
            if (fabsf(du[e]) < INFINITY) top = fmaxf(top, fabsf(du[e]));
        }
    }
    top = largest(top);
    if (threadIdx.x == 0) f.tops[blockIdx.x] = top;
}

struct Call {
    const void *x, *weight;
    int64_t ldx, ldw, T, D, F;
    int type;
    char *ws;
    size_t ws_bytes;
    hipStream_t st;
};

enum { kForward = 1, kBackward = 2 };

struct Plan {
    int Dp, tile, rows, words;
    int64_t ldd, ldp;
    bool pack_x, pack_w, raw, few;
    Choice hidden, weight;
    size_t x, w, dz, bias, slices, tops, factor, bytes;
};

// Up to how many tokens a wave multiplies its weights as they lie, in vector registers: of float32 as long as that is bound by memory
// (then weights are split for the matrix instructions), of 16-bit types as long as the tiles, which are too few to read as fast, take
// longer, the more so where they need operands repacked.  As they lie and by tiles, in us, 8192 results, weights from memory:
//                                  1 token       2         3         4         5         8 tokens
//   4096 features, bfloat16       26   35    31   35   38   35   40   36   58   35   70   36
//   4096, float16                 26   35    27   35   31   36   32   35   37   36   38   36
//   4095, bfloat16                36   74    53   74   44   74   45   75   75   74   78   74
//   4096, float32                 48  215    52  215   53  215   54  215   62  216   64  217   16: 85  132 (split by the tiles)
//   1024, 2731 results, float32    9   34     8   33   10   33   10   33   14   33   14   34    16: 20   36
//   4096, 512 results, float32                                                      27   85    16: 24   85
template <typename P>
int64_t most_few(const void *x, int64_t ldx, const void *weight, int64_t ldw, int64_t D)
{
    return P::planes > 1 ? 16 : in_place(x, ldx, D) && in_place(weight, ldw, D) ? 2 : 4;
}

template <typename P>
Plan plan_of(const void *x, int64_t ldx, const void *weight, int64_t ldw, int64_t T, int64_t D, int64_t F, int what)
{
    constexpr bool kSplit = P::planes > 1;
    Plan p{};
    p.Dp = (int)(kSplit ? (D + 31) / 32 * 32 : (D + 7) / 8 * 8);
    p.ldd = row_elements<P>(D);
    p.few = what == kForward && T <= most_few<P>(x, ldx, weight, ldw, D) && g_tune.vocab_tile == kTuneUnset;
    // not many tokens of float32: weights that are split where they are needed, as the cross entropy's
    p.raw = !p.few && kSplit && what == kForward && (uintptr_t)weight % 16 == 0 && ldw % 4 == 0 && D % 4 == 0 &&
            T <= raw_tokens(2 * F * D, 4, kLoss) && g_tune.vocab_tile == kTuneUnset;
    p.pack_x = !p.few && (kSplit || !in_place(x, ldx, D));
    p.pack_w = !p.few && !p.raw && (kSplit || !in_place(weight, ldw, D));
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t was = at;
        at = align_up(at + n, 256);
        return was;
    };
    if (p.pack_x) p.x = take((size_t)T * p.ldd * 2);
    if (p.pack_w) p.w = take((size_t)2 * F * p.ldd * 2);
    if (what == kForward) {
        p.tile = choose<P>(2 * F, T, D, kShapes, 1, true).tile;
    } else {
        p.words = (int)(kSplit ? (2 * F + 31) / 32 * 32 : (2 * F + 7) / 8 * 8);
        p.ldp = (int64_t)p.words * P::planes;
        // as many as leave every CU two workgroups: a bias's gradient is a sum over the workgroups along T
        p.rows = 64;
        while (p.rows > 8 && (T + p.rows - 1) / p.rows * ((F + 255) / 256) < 2 * device_cus()) p.rows /= 2;
        p.rows = std::max(p.rows, (int)((T + 65534) / 65535 + 7) / 8 * 8);  // the grid's second axis has 65535 workgroups
        p.dz = take((size_t)T * p.ldp * 2);
        p.bias = take((size_t)((T + p.rows - 1) / p.rows) * 2 * F * 4);
        p.hidden = choose<P>(D, T, 2 * F, kGradShapes<P>, 64, false);
        p.weight = choose<P>(D, 2 * F, T, kGradShapes<P>, 64, false);
        size_t slices = 0;
        if (p.hidden.splits > 1) slices = (size_t)p.hidden.splits * T * D * 4;
        if (p.weight.splits > 1) slices = std::max(slices, (size_t)p.weight.splits * 2 * F * D * 4);
        p.slices = take(slices);
        if (P::half) p.tops = take(kTopGroups * 4), p.factor = take(4);
    }
    p.bytes = at ? at : 256;
    return p;
}

int check(const Call &c)
{
    if (c.T < 0 || c.D < 0 || c.F < 0 || !element_bytes(c.type)) return DS_EINVAL;
    if (c.D > 0 && ((c.T > 0 && (!c.x || c.ldx < c.D)) || (c.F > 0 && (!c.weight || c.ldw < c.D)))) return DS_EINVAL;
    const int64_t most = 0x7fffffff - 512;
    if (c.T > most || c.F > most / 2 || c.D > 1000000 || c.ldx > 2000000 || c.ldw > 2000000) return DS_ETOOLARGE;
    return DS_OK;
}

// Operands in place, or repacked.
template <typename P>
int operands(const Call &c, const Plan &p, Operand &x, Operand &w)
{
    typedef typename ElementOf<P>::type E;
    Pack px{}, pw{};
    x = p.pack_x ? Operand{c.ws + p.x, p.ldd} : Operand{c.x, c.ldx};
    w = p.pack_w ? Operand{c.ws + p.w, p.ldd} : Operand{c.weight, c.ldw};
    if (c.D == 0) return DS_OK;
    if (p.pack_x) px = Pack{c.x, c.ldx, c.T, (int)c.D, p.Dp, (uint16_t *)(c.ws + p.x), p.ldd, nullptr, 0, 0, 0};
    if (p.pack_w) pw = Pack{c.weight, c.ldw, 2 * c.F, (int)c.D, p.Dp, (uint16_t *)(c.ws + p.w), p.ldd, nullptr, 0, 0, 0};
    return launch_pack<E>(px, pw, c.st);
}

template <typename P>
int forward(const Call &c, const void *bias, int activation, void *out, float *halves)
{
    const Plan p = plan_of<P>(c.x, c.ldx, c.weight, c.ldw, c.T, c.D, c.F, kForward);
    if (!c.ws || c.ws_bytes < p.bytes || (uintptr_t)c.ws % 256) return DS_EWORKSPACE;
    if (c.T == 0 || c.F == 0) return DS_OK;
    const int64_t ldz = (c.F + 7) / 8 * 8;
    if (p.few)
        return launch_few<typename ElementOf<P>::type>(
            Few{c.x, c.weight, bias, c.ldx, c.ldw, c.F, (int)c.T, (int)c.D, activation, out, halves, ldz}, c.st);
    Args g{};
    DS_TRY(operands<P>(c, p, g.b, g.a));
    g.M = (int)c.F, g.N = (int)c.T, g.K = p.raw ? (int)c.D : p.Dp;
    g.splits = 1, g.k_split = (p.Dp + P::step - 1) / P::step * P::step;
    g.half_bytes = c.F * g.a.ld * (p.raw ? 4 : 2);
    g.bias = bias, g.bias_type = c.type, g.activation = activation;
    g.out = out, g.ldo = c.F;
    g.halves = halves, g.ldz = ldz;
    if constexpr (P::planes > 1)
        if (p.raw) return launch_gate_raw(g, c.st);
    return launch_gate<P>(p.tile, g, c.st);
}

struct Results {
    void *dx, *dweight, *dbias;
};

template <typename P>
int backward(const Call &c, const float *halves, const void *grad, int64_t ldg, int activation, const Results &r)
{
    typedef typename ElementOf<P>::type E;
    const Plan p = plan_of<P>(c.x, c.ldx, c.weight, c.ldw, c.T, c.D, c.F, kBackward);
    if (!c.ws || c.ws_bytes < p.bytes || (uintptr_t)c.ws % 256) return DS_EWORKSPACE;
    const int n = (int)(2 * c.F), T = (int)c.T, D = (int)c.D;
    Operand x, w;
    DS_TRY(operands<P>(c, p, x, w));
    float *const factor = P::half ? (float *)(c.ws + p.factor) : nullptr;
    const int tiles = ceil_div(T, p.rows);
    Back f{halves, grad, (c.F + 7) / 8 * 8, ldg, c.T, (int)c.F, activation, p.rows, c.ws + p.dz, p.ldp, p.words,
           r.dbias ? (float *)(c.ws + p.bias) : nullptr, (float *)(c.ws + p.tops), 0, factor};
    const dim3 grid(ceil_div((int)c.F, 256), tiles);
    if (T > 0 && n > 0) {
        if (P::half) {
            f.top_groups = (int)std::min<int64_t>(kTopGroups, (int64_t)ceil_div(T, 8) * grid.x);
            hipLaunchKernelGGL(top_kernel, dim3(f.top_groups), dim3(256), 0, c.st, f);
        }
        hipLaunchKernelGGL((back_kernel<P>), grid, dim3(256), 0, c.st, f);
    }
    const bool made = T > 0 && n > 0;  // dz, and with it the factor
    if (r.dbias && n > 0) DS_TRY(launch_bias_join<E>(BiasJoin{f.bias_part, n, tiles, n, r.dbias}, nullptr, nullptr, c.st));
    if (D == 0) return launch_status();
    float *const slices = (float *)(c.ws + p.slices);
    Args g[2] = {};
    bool wanted[2], joined[2];
    for (int which = 0; which < 2; ++which) {
        Args &a = g[which];
        wanted[which] = which ? r.dweight && n > 0 : r.dx && T > 0;
        a.a = which ? x : w;
        a.b = Operand{c.ws + p.dz, p.ldp};
        a.M = D;
        a.N = which ? (n + 7) / 8 * 8 : T;
        a.n_store = which ? n : T;
        a.K = which ? T : n;
        a.factor[0] = made ? factor : nullptr;
        a.out = which ? r.dweight : r.dx;
        a.ldo = D;
        a.splits = which ? p.weight.splits : p.hidden.splits;
        a.k_split = ((a.K + a.splits - 1) / a.splits + P::step - 1) / P::step * P::step;
        joined[which] = a.splits > 1;
        a.slice = joined[which] ? slices : nullptr;
    }
    // few workgroups each, and no slices to share: both in one launch
    const int tm = Shapes<P>::m[p.weight.tile], tn = Shapes<P>::n[p.weight.tile];
    const int64_t blocks = ceil_div(D, tm) * ((int64_t)ceil_div(T, tn) * p.hidden.splits + ceil_div(n, tn));
    const bool both = wanted[0] && wanted[1] && !joined[1] && p.hidden.tile == p.weight.tile && blocks <= 2 * device_cus();
    if (both) DS_TRY(launch_product<P>(kHidden, p.weight.tile, g[0], &g[1], c.st));
    for (int which = 0; which < 2; ++which) {
        Args &a = g[which];
        if (!wanted[which]) continue;
        if (!both) DS_TRY(launch_product<P>(which ? kWeight : kHidden, which ? p.weight.tile : p.hidden.tile, a, nullptr, c.st));
        if (joined[which]) DS_TRY(launch_join<P>(slices, a.splits, (int64_t)a.n_store * D, D, a.factor[0], nullptr, a.out, c.st));
    }
    return launch_status();
}

}  // namespace gated
}  // namespace ds

using namespace ds;
using namespace ds::gated;

DS_EXPORT size_t ds_gated_workspace_bytes(const void *x, int64_t ldx, const void *weight, int64_t ldw, int64_t T, int64_t D, int64_t F,
                                          int type, int what)
{
    if (T < 0 || D < 0 || F < 0 || !element_bytes(type) || (what != kForward && what != kBackward)) return 0;
    if (type == DS_F32) return gated::plan_of<Split>(x, ldx, weight, ldw, T, D, F, what).bytes;
    if (type == DS_BF16) return gated::plan_of<Bf16>(x, ldx, weight, ldw, T, D, F, what).bytes;
    return gated::plan_of<F16>(x, ldx, weight, ldw, T, D, F, what).bytes;
}

DS_EXPORT int ds_gated_forward(const void *x, int64_t ldx, const void *weight, int64_t ldw, const void *bias, int activation,
                               int64_t T, int64_t D, int64_t F, int type, void *out, float *halves, void *workspace,
                               size_t workspace_bytes, ds_stream_t stream)
{
    const gated::Call c{x, weight, ldx, ldw, T, D, F, type, (char *)workspace, workspace_bytes, (hipStream_t)stream};
    if (activation < DS_SILU || activation > DS_SIGMOID) return DS_EINVAL;
    DS_TRY(gated::check(c));
    if (T > 0 && F > 0 && !out) return DS_EINVAL;
    if (type == DS_F32) return forward<Split>(c, bias, activation, out, halves);
    if (type == DS_BF16) return forward<Bf16>(c, bias, activation, out, halves);
    return forward<F16>(c, bias, activation, out, halves);
}

DS_EXPORT int ds_gated_backward(const void *x, int64_t ldx, const void *weight, int64_t ldw, const float *halves, const void *grad,
                                int64_t ldg, int activation, int64_t T, int64_t D, int64_t F, int type, void *dx, void *dweight,
                                void *dbias, void *workspace, size_t workspace_bytes, ds_stream_t stream)
{
    const gated::Call c{x, weight, ldx, ldw, T, D, F, type, (char *)workspace, workspace_bytes, (hipStream_t)stream};
    if (activation < DS_SILU || activation > DS_SIGMOID) return DS_EINVAL;
    DS_TRY(gated::check(c));
    if (T > 0 && F > 0 && (!halves || !grad || ldg < F || (uintptr_t)halves % 16)) return DS_EINVAL;
    const Results r{dx, dweight, dbias};
    if (type == DS_F32) return backward<Split>(c, halves, grad, ldg, activation, r);
    if (type == DS_BF16) return backward<Bf16>(c, halves, grad, ldg, activation, r);
    return backward<F16>(c, halves, grad, ldg, activation, r);
}
