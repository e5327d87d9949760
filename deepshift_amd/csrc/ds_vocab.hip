// Softmax cross entropy of a linear head over a large vocabulary, in pieces of the vocabulary, and its gradients.
//
//   s[t][v] = h[t] . W[v] + b[v]      lse[t] = log sum_v exp s[t][v]      loss[t] = lse[t] - s[t][y_t]
//   P[t][v] = g_t (exp(s[t][v] - lse[t]) - [v = y_t])      dh = P W      dW = P^T h      db = sum_t P[t]
//
// The logits are never stored: the forward pass keeps a maximum and a sum of exponentials per tile (T x V / 128 pairs), the
// backward pass computes the logits of a piece of the vocabulary again, leaves that piece's P in a workspace, and forms both
// gradients from it.  Four products of 2 T D V operations for a step, of which three are the formula's own.
#include "ds_vocab.h"

namespace ds {
namespace vocab {

// ---- operands as the products take them --------------------------------------------------------------------------

// Rows of D elements to rows of Dp (a multiple of 8, zeros behind D): 16-bit elements as they are, float32 as three planes.
// Rows whose target is `ignore` (where targets are given) become zeros: tokens that do
// not count leave nothing in the weights' gradient, not even a value that is no number.
template <typename E, int N>
__global__ __launch_bounds__(256) void pack_kernel(const E *__restrict__ x, int64_t ld, int64_t rows, int D, int Dp,
                                                   uint16_t *__restrict__ out, int64_t plane, const void *__restrict__ target,
                                                   int wide, int64_t ignore)
{
    const int units = Dp / N;
    const int64_t total = rows * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / units;
        const int c = (int)(i - r * units) * N;
        Vec<E, N> v{};
        if (target && (wide ? ((const int64_t *)target)[r] : (int64_t)((const int32_t *)target)[r]) == ignore) {
        } else if (c + N <= D) v = *(const Vec<E, N> *)(x + r * ld + c);
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c + e < D) v.v[e] = x[r * ld + c + e];
        uint16_t *to = out + r * Dp + c;
        if constexpr (sizeof(E) == 2) {
            *(Vec<E, N> *)to = v;
        } else {
            Vec<bf16_t, N> p[3];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                bf16_t planes[3];
                split_planes(to_float(v.v[e]), planes);
#pragma unroll
                for (int q = 0; q < 3; ++q) p[q].v[e] = planes[q];
            }
#pragma unroll
            for (int q = 0; q < 3; ++q) *(Vec<bf16_t, N> *)(to + q * plane) = p[q];
        }
    }
}

template <typename E>
int launch_pack(const void *x, int64_t ld, int64_t rows, int D, int Dp, void *out, int64_t plane, const void *target, int wide,
                int64_t ignore, hipStream_t st)
{
    if (rows == 0 || Dp == 0) return DS_OK;
    const int n = vector_elements(sizeof(E), {ld, 8}, {x});
    const int64_t blocks = (rows * (Dp / n) + 255) / 256;
    const dim3 grid((unsigned)(blocks < 8192 ? blocks : 8192));
#define DS_LAUNCH(N)                                                                                                   \
    hipLaunchKernelGGL((pack_kernel<E, N>), grid, dim3(256), 0, st, (const E *)x, ld, rows, D, Dp, (uint16_t *)out, plane, target,  \
                       wide, ignore)
    if (n == 8) { if constexpr (sizeof(E) == 2) DS_LAUNCH(8); }
    else if (n == 4) DS_LAUNCH(4);
    else if (n == 2) DS_LAUNCH(2);
    else DS_LAUNCH(1);
#undef DS_LAUNCH
    return launch_status();
}

// ---- rows ------------------------------------------------------------------------------------------------------

constexpr float kLn2 = 0.6931471805599453f;

// Joins the tiles' maxima and sums: a workgroup has 64 rows, each wave a quarter of the tiles.
__global__ __launch_bounds__(256) void row_kernel(const float2 *__restrict__ stats, const float *__restrict__ picked, int tiles,
                                                  int T, const void *__restrict__ target, int wide, int64_t V, int64_t ignore,
                                                  float *__restrict__ lse, float *__restrict__ loss)
{
    __shared__ float tops[4][64], sums[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, t = blockIdx.x * 64 + lane;
    float top = -INFINITY, sum = 0.f;
    if (t < T) {
#pragma unroll 4
        for (int i = wave; i < tiles; i += 4) {
            const float2 s = stats[(int64_t)i * T + t];
            const float both = fmaxf(top, s.x);
            sum = both == -INFINITY ? sum + s.y : sum * exp2f(top - both) + s.y * exp2f(s.x - both);
            top = both;
        }
    }
    tops[wave][lane] = top, sums[wave][lane] = sum;
    __syncthreads();
    if (wave != 0 || t >= T) return;
#pragma unroll
    for (int w = 1; w < 4; ++w) {
        const float both = fmaxf(top, tops[w][lane]);
        sum = both == -INFINITY ? sum + sums[w][lane] : sum * exp2f(top - both) + sums[w][lane] * exp2f(tops[w][lane] - both);
        top = both;
    }
    const float total = sum == 0.f ? -INFINITY : top + log2f(sum);
    lse[t] = total;
    const int64_t y = wide ? ((const int64_t *)target)[t] : (int64_t)((const int32_t *)target)[t];
    loss[t] = y == ignore ? 0.f : y < 0 || y >= V ? NAN : (total - picked[t]) * kLn2;
}

// Sum of a workgroup's values in a fixed order, in every thread.
template <typename S>
__device__ __forceinline__ S sum_of_block(S v, S *lds)
{
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    S s = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) s += lds[w];
    return s;
}

// total[0]: the sum or the mean of the counted rows' losses, total[1]: one row's share in it.  Without a counted row both the
// loss and the gradients are 0.
__global__ __launch_bounds__(1024) void total_kernel(const float *__restrict__ loss, const void *__restrict__ target, int wide,
                                                     int T, int64_t ignore, int mean, float *__restrict__ total)
{
    __shared__ double lds[16];
    double sum = 0, n = 0;
    for (int t = threadIdx.x; t < T; t += 1024) {
        const int64_t y = wide ? ((const int64_t *)target)[t] : (int64_t)((const int32_t *)target)[t];
        sum += loss[t];
        n += y != ignore;
    }
    sum = sum_of_block(sum, lds);
    n = sum_of_block(n, lds);
    if (threadIdx.x == 0) {
        const double share = mean && n > 0 ? 1.0 / n : 1.0;
        total[0] = (float)(sum * share);
        total[1] = (float)share;
    }
}

// Gradients of single losses: the largest of them in `factor`, each one's share of that in `scale`, so that what the products
// take lies in [-1, 1] whatever the gradients' size.
__global__ __launch_bounds__(1024) void row_scale_kernel(const float *__restrict__ grad, const void *__restrict__ target,
                                                         int wide, int T, int64_t ignore, float *__restrict__ scale,
                                                         float *__restrict__ factor)
{
    __shared__ float lds[16];
    float top = 0.f;
    for (int t = threadIdx.x; t < T; t += 1024) {
        const int64_t y = wide ? ((const int64_t *)target)[t] : (int64_t)((const int32_t *)target)[t];
        const float g = y == ignore ? 0.f : fabsf(grad[t]);
        top = g > top || g != g ? g : top;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float other = __shfl_xor(top, o);
        top = other > top || other != other ? other : top;
    }
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = 0.f;
    for (int w = 0; w < 16; ++w) top = lds[w] > top || lds[w] != lds[w] ? lds[w] : top;
    for (int t = threadIdx.x; t < T; t += 1024) scale[t] = top == 0.f ? 0.f : grad[t] / top;
    if (threadIdx.x == 0) *factor = top;
}

// ---- joins -------------------------------------------------------------------------------------------------------

// The slices of a product in order, behind what earlier pieces of the vocabulary left in `acc`; the last piece's result is
// multiplied and rounded.
template <typename P, typename E>
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ slices, int splits, int64_t n, int M, float *acc,
                                                   int first, int last, const float *f0, const float *f1, E *__restrict__ out,
                                                   int64_t ldo)
{
    const float *const f[2] = {f0, f1};
    const float factor = last ? out_factor<P>(f) : 1.f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float s = first ? 0.f : acc[i];
        for (int k = 0; k < splits; ++k) s += slices[k * n + i];
        if (last) out[i / M * ldo + i % M] = from_float<E>(s * factor);
        else acc[i] = s;
    }
}

template <typename E>
__global__ __launch_bounds__(256) void bias_join_kernel(const float *__restrict__ part, int ld, int tiles, int n, const float *f0,
                                                        const float *f1, E *__restrict__ out)
{
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= n) return;
    float s = 0.f;
#pragma unroll 4
    for (int i = 0; i < tiles; ++i) s += part[(int64_t)i * ld + v];
    out[v] = from_float<E>(s * (f0 ? *f0 : 1.f) * (f1 ? *f1 : 1.f));
}

// ---- plan --------------------------------------------------------------------------------------------------------

constexpr size_t kPieceBytes = (size_t)1 << 30;  // of P, and of repacked weights

template <typename P>
int pick_tile(int64_t m, int64_t n)
{
    const int64_t cus = device_cus();
    const int forced = g_tune.vocab_tile;
    if (forced >= 0 && forced < 3) return forced;
    for (int i = 0; i < 2; ++i)
        if (n > Shapes<P>::n[i] / 2 && m > Shapes<P>::m[i] / 2 &&
            ((m + Shapes<P>::m[i] - 1) / Shapes<P>::m[i]) * ((n + Shapes<P>::n[i] - 1) / Shapes<P>::n[i]) >= cus) return i;
    return n > 64 ? 1 : 2;
}

template <typename P>
int pick_splits(int tile, int64_t m, int64_t n, int64_t k)
{
    const int64_t tiles = ((m + Shapes<P>::m[tile] - 1) / Shapes<P>::m[tile]) * ((n + Shapes<P>::n[tile] - 1) / Shapes<P>::n[tile]);
    if (tiles < 1) return 1;
    const int64_t want = g_tune.vocab_split != kTuneUnset ? (int64_t)g_tune.vocab_split : device_cus() / tiles;
    const int64_t most = (k + kStep - 1) / kStep / 8;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

struct Plan {
    int Dp;               // row length of repacked operands
    int64_t piece, pieces;
    bool pack_h, pack_w;
    int tile_logits, tile_hidden, tile_weight, split_hidden, split_weight;
    int64_t ldp;
    size_t h, w, stats, picked, prob, bias, slices, acc, scale, factor, bytes;
};

inline bool in_place(const void *p, int64_t ld, int64_t D) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && D % 8 == 0; }

template <typename P>
Plan plan_of(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int64_t T, int64_t D, int64_t V, bool grad)
{
    constexpr size_t NP = P::planes;
    Plan p{};
    p.Dp = (int)((D + 7) / 8 * 8);
    p.pack_h = NP > 1 || grad || !in_place(hidden, ldh, D);  // grad: without the rows that do not count
    p.pack_w = NP > 1 || !in_place(weight, ldw, D);
    const int kb = g_tune.vocab_piece_kb;
    const size_t piece_bytes = kb == kTuneUnset ? kPieceBytes : (size_t)kb << 10;
    int64_t most = V;
    auto at_most = [&](size_t per_word) {
        const int64_t n = (int64_t)(piece_bytes / (per_word ? per_word : 1)) / 256 * 256;
        most = n < 256 ? (most < 256 ? most : 256) : n < most ? n : most;
    };
    if (p.pack_w) at_most(NP * (size_t)p.Dp * 2);
    if (grad) at_most(NP * (size_t)T * 2);
    // equal pieces, of whole tiles
    p.pieces = (V + most - 1) / most;
    p.piece = ((V + p.pieces - 1) / p.pieces + 255) / 256 * 256;
    if (p.piece > V) p.piece = V;
    p.pieces = (V + p.piece - 1) / p.piece;
    p.tile_logits = pick_tile<P>(p.piece, T);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t was = at;
        at = align_up(at + n, 256);
        return was;
    };
    if (p.pack_h) p.h = take(NP * (size_t)T * p.Dp * 2);
    if (p.pack_w) p.w = take(NP * (size_t)p.piece * p.Dp * 2);
    if (!grad) {
        const int64_t tiles = (p.piece + Shapes<P>::m[p.tile_logits] - 1) / Shapes<P>::m[p.tile_logits];
        p.stats = take((size_t)(tiles * p.pieces) * T * 8);
        p.picked = take((size_t)T * 4);
    } else {
        p.ldp = (p.piece + 31) / 32 * 32;
        p.tile_hidden = pick_tile<P>(D, T);
        p.tile_weight = pick_tile<P>(D, p.piece);
        p.split_hidden = pick_splits<P>(p.tile_hidden, D, T, p.piece);
        p.split_weight = pick_splits<P>(p.tile_weight, D, p.piece, T);
        p.prob = take(NP * (size_t)T * p.ldp * 2);
        p.bias = take((size_t)((T + Shapes<P>::n[p.tile_logits] - 1) / Shapes<P>::n[p.tile_logits]) * p.ldp * 4);
        size_t slices = 0;
        if (p.split_hidden > 1 || p.pieces > 1) slices = (size_t)p.split_hidden * T * D * 4;
        if (p.split_weight > 1) {
            const size_t n = (size_t)p.split_weight * p.piece * D * 4;
            slices = n > slices ? n : slices;
        }
        p.slices = take(slices);
        if (p.pieces > 1) p.acc = take((size_t)T * D * 4);
        p.scale = take((size_t)T * 4);
        p.factor = take(4);
    }
    p.bytes = at ? at : 256;
    return p;
}

struct Call {
    const void *hidden, *weight, *bias, *target;
    int64_t ldh, ldw, T, D, V, ignore;
    int wide, type;
    char *ws;
    hipStream_t st;
};

inline int check(const Call &c)
{
    if (c.T < 0 || c.D < 0 || c.V < 1 || !element_bytes(c.type)) return DS_EINVAL;
    if (c.T > 0 && (!c.target || (c.D > 0 && (!c.hidden || !c.weight || c.ldh < c.D || c.ldw < c.D)))) return DS_EINVAL;
    const int64_t most = 0x7fffffff - 512;
    if (c.T > most || c.V > most || c.D > 4000000 || c.ldh > 4000000 || c.ldw > 4000000) return DS_ETOOLARGE;
    return DS_OK;
}

template <typename P> struct ElementOf { typedef bf16_t type; };
template <> struct ElementOf<F16> { typedef f16_t type; };
template <> struct ElementOf<Split> { typedef float type; };

template <typename P>
int hidden_operand(const Call &c, const Plan &p, bool counted_only, Operand *o)
{
    if (!p.pack_h) {
        *o = Operand{c.hidden, c.ldh, 0};
        return DS_OK;
    }
    *o = Operand{c.ws + p.h, p.Dp, c.T * p.Dp};
    return launch_pack<typename ElementOf<P>::type>(c.hidden, c.ldh, c.T, (int)c.D, p.Dp, c.ws + p.h, c.T * p.Dp,
                                                    counted_only ? c.target : nullptr, c.wide, c.ignore, c.st);
}

template <typename P>
int weight_operand(const Call &c, const Plan &p, int64_t v0, int64_t n, Operand *o)
{
    typedef typename ElementOf<P>::type E;
    const E *from = (const E *)c.weight + v0 * c.ldw;
    if (!p.pack_w) {
        *o = Operand{from, c.ldw, 0};
        return DS_OK;
    }
    *o = Operand{c.ws + p.w, p.Dp, p.piece * p.Dp};
    return launch_pack<E>(from, c.ldw, n, (int)c.D, p.Dp, c.ws + p.w, p.piece * p.Dp, nullptr, 0, 0, c.st);
}

template <typename P>
Args logit_args(const Call &c, const Plan &p, int64_t v0, int64_t n, const Operand &h, const Operand &w)
{
    Args g{};
    g.a = w, g.b = h;
    g.M = (int)n, g.N = (int)c.T, g.K = p.Dp;
    g.splits = 1, g.k_split = (p.Dp + kStep - 1) / kStep * kStep;
    g.bias = c.bias, g.bias_type = c.type;
    g.target = c.target, g.target_wide = c.wide;
    g.V = c.V, g.ignore = c.ignore, g.v0 = (int)v0;
    return g;
}

#define DS_TRY(what)                    \
    do {                                \
        const int s_ = (what);          \
        if (s_ != DS_OK) return s_;     \
    } while (0)

template <typename P>
int loss(const Call &c, int reduction, float *rows, float *lse, float *total, size_t ws_bytes)
{
    const Plan p = plan_of<P>(c.hidden, c.ldh, c.weight, c.ldw, c.T, c.D, c.V, false);
    if (!c.ws || ws_bytes < p.bytes || (uintptr_t)c.ws % 256) return DS_EWORKSPACE;
    Operand h, w;
    if (c.T > 0) {
        DS_TRY(hidden_operand<P>(c, p, false, &h));
        int tiles = 0;
        for (int64_t v0 = 0; v0 < c.V; v0 += p.piece) {
            const int64_t n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
            DS_TRY(weight_operand<P>(c, p, v0, n, &w));
            Args g = logit_args<P>(c, p, v0, n, h, w);
            g.stats = (float *)(c.ws + p.stats) + (int64_t)tiles * c.T * 2;
            g.picked = (float *)(c.ws + p.picked);
            DS_TRY(launch_product<P>(kLogitStats, p.tile_logits, g, c.st));
            tiles += g.tiles_m;
        }
        hipLaunchKernelGGL(row_kernel, dim3((unsigned)((c.T + 63) / 64)), dim3(256), 0, c.st, (const float2 *)(c.ws + p.stats),
                           (const float *)(c.ws + p.picked), tiles, (int)c.T, c.target, c.wide, c.V, c.ignore, lse, rows);
    }
    if (reduction)
        hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, c.st, rows, c.target, c.wide, (int)c.T, c.ignore,
                           reduction == DS_MEAN, total);
    return launch_status();
}

template <typename P>
int loss_grad(const Call &c, const float *lse, const float *row_grad, const float *grad, const float *share, void *dhidden,
              void *dweight, void *dbias, size_t ws_bytes)
{
    typedef typename ElementOf<P>::type E;
    const Plan p = plan_of<P>(c.hidden, c.ldh, c.weight, c.ldw, c.T, c.D, c.V, true);
    if (!c.ws || ws_bytes < p.bytes || (uintptr_t)c.ws % 256) return DS_EWORKSPACE;
    if (c.T > 0 && row_grad) {
        hipLaunchKernelGGL(row_scale_kernel, dim3(1), dim3(1024), 0, c.st, row_grad, c.target, c.wide, (int)c.T, c.ignore,
                           (float *)(c.ws + p.scale), (float *)(c.ws + p.factor));
        grad = (const float *)(c.ws + p.factor);
    }
    Operand h{}, w{};
    if (c.T > 0) DS_TRY(hidden_operand<P>(c, p, true, &h));
    float *const slices = (float *)(c.ws + p.slices);
    for (int64_t v0 = 0; v0 < c.V; v0 += p.piece) {
        const int64_t n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
        const bool first = v0 == 0, last = v0 + n == c.V;
        int bias_tiles = 0;
        const Operand prob{c.ws + p.prob, p.ldp, c.T * p.ldp};
        if (c.T > 0) {
            DS_TRY(weight_operand<P>(c, p, v0, n, &w));
            Args g = logit_args<P>(c, p, v0, n, h, w);
            g.lse = lse;
            g.row_scale = row_grad ? (const float *)(c.ws + p.scale) : nullptr;
            g.prob = c.ws + p.prob, g.ldp = p.ldp, g.prob_plane = prob.plane;
            g.bias_part = dbias ? (float *)(c.ws + p.bias) : nullptr;
            g.ld_bias_part = (int)p.ldp;
            DS_TRY(launch_product<P>(kLogitProb, p.tile_logits, g, c.st));
            bias_tiles = g.tiles_n;
        }
        if (dbias)
            hipLaunchKernelGGL((bias_join_kernel<E>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, c.st,
                               (const float *)(c.ws + p.bias), (int)p.ldp, bias_tiles, (int)n, grad, share, (E *)dbias + v0);
        if (c.D == 0) continue;
        for (int which = 0; which < 2; ++which) {
            void *out = which ? dweight : dhidden;
            if (!out || (!which && c.T == 0)) continue;
            Args g{};
            g.a = which ? h : w;
            g.b = prob;
            g.M = (int)c.D;
            g.N = which ? (int)((n + 7) / 8 * 8) : (int)c.T;
            g.n_store = which ? (int)n : (int)c.T;
            g.K = which ? (int)c.T : (int)n;
            g.factor[0] = grad, g.factor[1] = share;
            g.out = which ? (void *)((E *)dweight + v0 * c.D) : dhidden;
            g.ldo = c.D, g.out_type = c.type;
            g.splits = which ? p.split_weight : p.split_hidden;
            g.k_split = ((g.K + g.splits - 1) / g.splits + kStep - 1) / kStep * kStep;
            const bool joined = g.splits > 1 || (!which && p.pieces > 1);
            g.slice = joined ? slices : nullptr;
            DS_TRY(launch_product<P>(which ? kWeight : kHidden, which ? p.tile_weight : p.tile_hidden, g, c.st));
            if (!joined) continue;
            const int64_t count = (int64_t)g.n_store * c.D;
            const int64_t blocks = (count + 255) / 256;
            hipLaunchKernelGGL((join_kernel<P, E>), dim3((unsigned)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, c.st, slices,
                               g.splits, count, (int)c.D, which ? nullptr : (float *)(c.ws + p.acc), which || first, which || last,
                               grad, share, (E *)g.out, c.D);
        }
    }
    return launch_status();
}

}  // namespace vocab
}  // namespace ds

using namespace ds;
using namespace ds::vocab;

DS_EXPORT size_t ds_vocab_workspace_bytes(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int64_t T, int64_t D,
                                          int64_t V, int type, int grad)
{
    if (T < 0 || D < 0 || V < 1 || !element_bytes(type)) return 0;
    if (type == DS_F32) return plan_of<Split>(hidden, ldh, weight, ldw, T, D, V, grad).bytes;
    if (type == DS_BF16) return plan_of<Bf16>(hidden, ldh, weight, ldw, T, D, V, grad).bytes;
    return plan_of<F16>(hidden, ldh, weight, ldw, T, D, V, grad).bytes;
}

DS_EXPORT int ds_vocab_loss(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias,
                            const void *target, int target_bytes, int64_t ignore, int64_t T, int64_t D, int64_t V, int type,
                            int reduction, float *rows, float *lse, float *total, void *workspace, size_t workspace_bytes,
                            ds_stream_t stream)
{
    if ((target_bytes != 4 && target_bytes != 8) || reduction < 0 || reduction > DS_MEAN) return DS_EINVAL;
    if ((T > 0 && (!rows || !lse)) || (reduction && !total)) return DS_EINVAL;
    const Call c{hidden, weight, bias, target, ldh, ldw, T, D, V, ignore, target_bytes == 8, type, (char *)workspace,
                 (hipStream_t)stream};
    DS_TRY(check(c));
    if (type == DS_F32) return loss<Split>(c, reduction, rows, lse, total, workspace_bytes);
    if (type == DS_BF16) return loss<Bf16>(c, reduction, rows, lse, total, workspace_bytes);
    return loss<F16>(c, reduction, rows, lse, total, workspace_bytes);
}

DS_EXPORT int ds_vocab_loss_grad(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias,
                                 const void *target, int target_bytes, int64_t ignore, int64_t T, int64_t D, int64_t V, int type,
                                 const float *lse, const float *row_grad, const float *grad, const float *share, void *dhidden,
                                 void *dweight, void *dbias, void *workspace, size_t workspace_bytes, ds_stream_t stream)
{
    if ((target_bytes != 4 && target_bytes != 8) || (row_grad && (grad || share)) || (T > 0 && !lse)) return DS_EINVAL;
    const Call c{hidden, weight, bias, target, ldh, ldw, T, D, V, ignore, target_bytes == 8, type, (char *)workspace,
                 (hipStream_t)stream};
    DS_TRY(check(c));
    if (type == DS_F32) return loss_grad<Split>(c, lse, row_grad, grad, share, dhidden, dweight, dbias, workspace_bytes);
    if (type == DS_BF16) return loss_grad<Bf16>(c, lse, row_grad, grad, share, dhidden, dweight, dbias, workspace_bytes);
    return loss_grad<F16>(c, lse, row_grad, grad, share, dhidden, dweight, dbias, workspace_bytes);
}
