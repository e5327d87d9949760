// Softmax cross entropy of a linear head over a large vocabulary, in pieces of the vocabulary, and its gradients.
//
//   s[t][v] = h[t] . W[v] + b[v]      lse[t] = log sum_v exp s[t][v]      loss[t] = lse[t] - s[t][y_t]
//   P[t][v] = g_t (exp(s[t][v] - lse[t]) - [v = y_t])      dh = P W      dW = P^T h      db = sum_t P[t]
//
// The logits are never stored: the forward pass keeps a maximum and a sum of exponentials per tile (a pair for every 32 to 256
// of them), the backward pass computes the logits of a piece of the vocabulary again, leaves that piece's P in a workspace of
// a bounded size, and forms both gradients from it: four products of 2 T D V operations for a step, of which three are the
// formula's own.  Where loss and gradients are asked for in one call, the forward pass leaves the last piece's exponentials,
// relative to their tiles' maxima, in a workspace, in 32 bits, and a pass over them makes them P: three products for that piece,
// which may be the whole vocabulary.
#include "ds_vocab.h"
#include <algorithm>

namespace ds {
namespace vocab {

// ---- operands as the products take them --------------------------------------------------------------------------

// Rows of D elements to rows of Dp (a multiple of 8 or 32, zeros behind D): 16-bit elements as they are, float32 as three planes.
// Bound by memory: (2048 + 32768) x 1024 float32 in 64 us, 5.5 TB/s.  Loads are 16 bytes wherever a row begins: 50021 x 2049
// bfloat16 take 75 us, element by element 176.
// Rows whose target is `ignore` (where targets are given) become zeros: tokens that do
// not count leave nothing in the weights' gradient, not even a value that is no number.
struct Pack {
    const void *x;
    int64_t ld, rows;
    int D, Dp;
    uint16_t *out;
    int64_t ldo;
    const void *target;
    int wide;
    int64_t ignore;
};

// One operand, or two in one launch, the first by `first` workgroups.
template <typename E>
__global__ __launch_bounds__(256) void pack_kernel(Pack one, Pack two, int first)
{
    constexpr int N = 16 / sizeof(E);
    const bool is_one = (int)blockIdx.x < first;
    const Pack &p = is_one ? one : two;
    const int block = is_one ? blockIdx.x : blockIdx.x - first, blocks = is_one ? first : gridDim.x - first;
    const int units = p.Dp / N;
    const int64_t total = p.rows * units;
    for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < total; i += (int64_t)blocks * 256) {
        const int64_t r = i / units;
        const int c = (int)(i - r * units) * N;
        const E *x = (const E *)p.x + r * p.ld;
        Vec<E, N> v{};
        if (p.target && (p.wide ? ((const int64_t *)p.target)[r] : (int64_t)((const int32_t *)p.target)[r]) == p.ignore) {
        } else if (c + N <= p.D) __builtin_memcpy(&v, x + c, sizeof(v));  // wherever it lies
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c + e < p.D) v.v[e] = x[c + e];
        uint16_t *row = p.out + r * p.ldo;
        if constexpr (sizeof(E) == 2) {
            *(Vec<E, N> *)(row + c) = v;
        } else {
            Vec<bf16_t, N> q[3];
#pragma unroll
            for (int e = 0; e < N; ++e) {
                bf16_t planes[3];
                split_planes(to_float(v.v[e]), planes);
#pragma unroll
                for (int k = 0; k < 3; ++k) q[k].v[e] = planes[k];
            }
#pragma unroll
            for (int k = 0; k < 3; ++k) *(Vec<bf16_t, N> *)(row + (c >> 5) * 96 + k * 32 + (c & 31)) = q[k];
        }
    }
}

template <typename E>
int launch_pack(const Pack &one, const Pack &two, hipStream_t st)
{
    auto blocks = [](const Pack &p) {
        const int64_t b = (p.rows * (p.Dp / (16 / (int)sizeof(E))) + 255) / 256;
        return (int)(b < 8192 ? b : 8192);
    };
    const int first = blocks(one), all = first + blocks(two);
    if (all == 0) return DS_OK;
    hipLaunchKernelGGL((pack_kernel<E>), dim3(all), dim3(256), 0, st, one, two, first);
    return launch_status();
}

// ---- rows ------------------------------------------------------------------------------------------------------

constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ int64_t target_of(const void *target, int wide, int64_t t)
{
    return wide ? ((const int64_t *)target)[t] : (int64_t)((const int32_t *)target)[t];
}

// The sums of every workgroup's rows, and how many of them count.
struct Share { double loss, rows; };

// total[0]: the sum or the mean of the counted rows' losses, total[1]: one row's share in it.  Without a counted row both the
// loss and the gradients are 0.
__device__ __forceinline__ void write_total(double loss, double rows, int mean, float *total)
{
    const double share = mean && rows > 0 ? 1.0 / rows : 1.0;
    total[0] = (float)(loss * share);
    total[1] = (float)share;
}

// A maximum and a sum of exponentials relative to it, joined with another such pair.
__device__ __forceinline__ void join_pair(float &top, float &sum, float top2, float sum2)
{
    const float both = fmaxf(top, top2);
    sum = both == -INFINITY ? sum + sum2 : sum * exp2_of(top - both) + sum2 * exp2_of(top2 - both);
    top = both;
}

// Where the losses of rows go, and what they come from.
struct Rows {
    const float2 *stats;   // [tiles][T]
    const float *picked;
    int tiles, T;
    const void *target;
    int wide;
    int64_t V, ignore;
    float *lse, *loss;
    int reduction;
    Share *shares;
    uint32_t *arrived;
    float *total;
};

__device__ __forceinline__ float log_of_sum(float top, float sum) { return sum == 0.f ? -INFINITY : top + log2f(sum); }

__device__ __forceinline__ float loss_of(const Rows &r, int t, int64_t y, float lse)
{
    return y == r.ignore ? 0.f : y < 0 || y >= r.V ? NAN : (lse - r.picked[t]) * kLn2;
}

// A workgroup's part in the total: its wave's sums of losses and of counted rows, `group` of `groups`.  The one that ends last
// adds up all of them, in order.
__device__ __forceinline__ void add_to_total(const Rows &r, double loss, double counted, int group, int groups)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) loss += __shfl_xor(loss, o), counted += __shfl_xor(counted, o);
    if (groups == 1) {
        if (lane == 0) write_total(loss, counted, r.reduction == DS_MEAN, r.total);
        return;
    }
    uint32_t before = 0;
    if (lane == 0) {
        r.shares[group] = Share{loss, counted};
        before = __hip_atomic_fetch_add(r.arrived, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    if ((int)__builtin_amdgcn_readfirstlane(before) != groups - 1) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    loss = counted = 0;
    for (int i = lane; i < groups; i += 64) loss += r.shares[i].loss, counted += r.shares[i].rows;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) loss += __shfl_xor(loss, o), counted += __shfl_xor(counted, o);
    if (lane == 0) write_total(loss, counted, r.reduction == DS_MEAN, r.total);
}

// Joins the tiles' maxima and sums: a workgroup has kRowsJoined rows, each of its waves a sixteenth of the tiles and each
// quarter of a wave a quarter of those.  Bound by latency: 37 rows of 391 tiles in 4.4 us (18 with 64 rows a workgroup and a
// wave's tiles one after the other), 8192 rows of 512 tiles, 34 MB, in 20.
constexpr int kRowsJoined = 16;

__global__ __launch_bounds__(1024) void row_kernel(Rows r)
{
    __shared__ float tops[64][kRowsJoined], sums[64][kRowsJoined];
    const int row = threadIdx.x % kRowsJoined, part = threadIdx.x / kRowsJoined, t = blockIdx.x * kRowsJoined + row;
    float top = -INFINITY, sum = 0.f;
    if (t < r.T) {
        constexpr int kAhead = 4;
        for (int i = part; i < r.tiles; i += 64 * kAhead) {
            float2 s[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
                s[j] = i + j * 64 < r.tiles ? r.stats[(int64_t)(i + j * 64) * r.T + t] : float2{-INFINITY, 0.f};
#pragma unroll
            for (int j = 0; j < kAhead; ++j) join_pair(top, sum, s[j].x, s[j].y);
        }
    }
    tops[part][row] = top, sums[part][row] = sum;
    __syncthreads();
    if (threadIdx.x >= 64) return;
    // the quarters of a wave join 16 parts each, then each other
    for (int i = part + 4; i < 64; i += 4) join_pair(top, sum, tops[i][row], sums[i][row]);
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) join_pair(top, sum, __shfl_xor(top, o), __shfl_xor(sum, o));
    double mine = 0, counts = 0;
    if (t < r.T && part == 0) {
        const float lse = log_of_sum(top, sum);
        const int64_t y = target_of(r.target, r.wide, t);
        r.lse[t] = lse;
        const float l = loss_of(r, t, y, lse);
        r.loss[t] = l;
        mine = l, counts = y != r.ignore;
    }
    if (r.reduction) add_to_total(r, mine, counts, blockIdx.x, gridDim.x);
}

__global__ void no_rows_kernel(int mean, float *total) { write_total(0, 0, mean, total); }

// Gradients of single losses: the largest finite one in `factor`, each one's share of that in `scale`, so that what the products
// take lies in [-1, 1] whatever the gradients' size, or is no number where its own gradient is none.  With `power` the shares are
// cut into a part from a half to 1, which stays in `scale`, and a power of two.
__global__ __launch_bounds__(1024) void row_scale_kernel(const float *__restrict__ grad, const void *__restrict__ target,
                                                         int wide, int T, int64_t ignore, float *__restrict__ scale,
                                                         float *__restrict__ factor, float *__restrict__ power)
{
    __shared__ float lds[16];
    float top = 0.f;
    for (int t = threadIdx.x; t < T; t += 1024) {
        const float g = fabsf(grad[t]);
        if (target_of(target, wide, t) != ignore && g < INFINITY) top = fmaxf(top, g);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = top;
    __syncthreads();
    top = 0.f;
    for (int w = 0; w < 16; ++w) top = fmaxf(top, lds[w]);
    if (top == 0.f) top = 1.f;
    for (int t = threadIdx.x; t < T; t += 1024) {
        float share = grad[t] / top;
        if (power) {
            int e = 0;
            if (fabsf(share) < INFINITY) share = frexpf(share, &e);
            power[t] = target_of(target, wide, t) == ignore ? 1.f : ldexpf(1.f, e);
        }
        scale[t] = share;
    }
    if (threadIdx.x == 0) *factor = top;
}

// Rows of float16 probabilities times their powers of two, in place.  A row whose gradient is 2^-20 of the largest keeps all bits of
// its probabilities until its own hidden gradient is formed; then every row goes to the common scale, on which the weights'
// gradient sums them and on which float16 holds what is above 2^-39 of the largest.  Bound by memory: 2048 x 32768 in
// 24 us of 540 (bfloat16, which needs none of it, 450).
__global__ __launch_bounds__(256) void power_kernel(f16_t *__restrict__ prob, int64_t ldp, int words, int64_t T,
                                                    const float *__restrict__ power)
{
    const int units = words / 8;
    const int64_t total = T * units;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t t = i / units;
        const float by = power[t];
        if (by == 1.f) continue;
        Vec<f16_t, 8> *const at = (Vec<f16_t, 8> *)(prob + t * ldp) + (i - t * units);
        Vec<f16_t, 8> v = *at;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = from_float<f16_t>(to_float(v.v[e]) * by);
        *at = v;
    }
}

// ---- exponentials to probabilities -----------------------------------------------------------------------------------

// P[t][v] = e[t][v] 2^(top[tile of v][t] - lse[t]) - [v = y_t]; the target's own from its logit.  All in 32 bits until P is rounded to
// the operands' type, once, as where the logits are formed again.  A workgroup has 256 words of some rows, a thread 8 words of
// every eighth of them; its rows' sums are the bias's gradient.  float32's exponentials lie where their planes go, those of 16-bit
// types in a place of their own.
// Bound by memory: 2048 x 32768 float32 exponentials to three planes in 155 us, 0.67 GB at 4.3 TB/s, where forming the logits
// again takes 830; 8192 x 65536 bfloat16 probabilities from 32 bits in 590, 3.2 GB at 5.4 TB/s, where forming the logits again
// takes 3500.  (Kept in 16 bits, and so rounded twice, their pass took 400 and the product before it 3530 instead of 3675, of
// 23500 a step.)
struct Finish {
    void *prob;
    int64_t ldp;
    const float *kept;     // exponentials, rows of ld_kept; of float32 32 of every 48
    int64_t ld_kept;
    int words, tile;       // words of a row, a multiple of 32; words a tile of the logits had
    int rows;              // of a workgroup, a multiple of 8
    int64_t v0, n;         // the piece: its first word, and how many there are
    int tile0;             // and its first tile
    int ld_bias_part;
    Rows of;
    float *bias_part;      // [workgroups along T][ld_bias_part], or NULL
    void *bias_out;        // one workgroup has all rows: the gradient itself, of V words, or NULL
    const float *factor[2];
};
// 64 rows, or 8 where that would leave CUs without work.
inline int finish_rows(int64_t T, int64_t words) { return (T + 63) / 64 * ((words + 255) / 256) >= 2 * device_cus() ? 64 : 8; }

// A row's sum, joined by half a wave, a lane every 32nd tile.
__device__ __forceinline__ float lse_of_row(const Rows &r, int t, int lane)
{
    float top = -INFINITY, sum = 0.f;
    for (int k = lane; k < r.tiles; k += 32) {
        const float2 s = r.stats[(int64_t)k * r.T + t];
        join_pair(top, sum, s.x, s.y);
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) join_pair(top, sum, __shfl_xor(top, o), __shfl_xor(sum, o));
    return log_of_sum(top, sum);
}

// JOIN: every workgroup joins its rows' sums for itself, and one more (the last along the rows) all of them, for the losses;
// else they are in of.lse.
template <typename P, bool JOIN>
__global__ __launch_bounds__(256) void finish_kernel(Finish f)
{
    typedef typename ElementOf<P>::type E;
    constexpr int NP = P::planes;
    __shared__ float sums[8][256];
    const Rows &r = f.of;
    const int lane = threadIdx.x % 32, part = threadIdx.x / 32, word = blockIdx.x * 256 + lane * 8;
    if (JOIN && blockIdx.y == gridDim.y - 1) {
        if (blockIdx.x > 0) return;
        // a wave has 64 rows at a time, a quarter of the tiles
        double loss = 0, counted = 0;
        const int wave = threadIdx.x / 64, row = threadIdx.x % 64;
        float2 *const parts = (float2 *)sums;  // [4][64]
        for (int t0 = 0; t0 < r.T; t0 += 64) {
            const int t = t0 + row;
            float top = -INFINITY, sum = 0.f;
            constexpr int kAhead = 8;
            for (int k = wave; k < r.tiles; k += 4 * kAhead) {
                float2 s[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; ++j)
                    s[j] = t < r.T && k + j * 4 < r.tiles ? r.stats[(int64_t)(k + j * 4) * r.T + t] : float2{-INFINITY, 0.f};
#pragma unroll
                for (int j = 0; j < kAhead; ++j) join_pair(top, sum, s[j].x, s[j].y);
            }
            parts[wave * 64 + row] = float2{top, sum};
            __syncthreads();
            if (wave == 0 && t < r.T) {
#pragma unroll
                for (int w = 1; w < 4; ++w) join_pair(top, sum, parts[w * 64 + row].x, parts[w * 64 + row].y);
                const float lse = log_of_sum(top, sum);
                const int64_t y = target_of(r.target, r.wide, t);
                const float l = loss_of(r, t, y, lse);
                r.lse[t] = lse, r.loss[t] = l;
                loss += l, counted += y != r.ignore;
            }
            __syncthreads();
        }
        if (wave == 0 && r.reduction) add_to_total(r, loss, counted, 0, 1);
        return;
    }
    float over_t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) over_t[e] = 0.f;
    const float2 *tops = r.stats + (int64_t)(f.tile0 + (word < f.words ? word / f.tile : 0)) * r.T;
    uint16_t *const column = (uint16_t *)f.prob + (NP == 1 ? word : (word >> 5) * 96 + (word & 31));
    const float *const kept = f.kept + (NP == 1 ? word : (word >> 5) * 48 + (word & 31));
#pragma unroll JOIN ? 1 : 4
    for (int i = 0; i < f.rows; i += 8) {
        const int t = blockIdx.y * f.rows + i + part;
        if (t >= r.T) break;
        const int64_t y = target_of(r.target, r.wide, t);
        const float lse = JOIN ? lse_of_row(r, t, lane) : r.lse[t];
        if (word >= f.words) continue;
        Vec<uint16_t, 8> *const at = (Vec<uint16_t, 8> *)(column + t * f.ldp);
        Vec<uint16_t, 8> v[NP];
        // four neighbouring lanes' planes take the place of all their exponentials: each lane needs both of its loads for
        // any store, and a wave's loads are one instruction
        const f32x4 e32[2] = {*(const f32x4 *)(kept + t * f.ld_kept), *(const f32x4 *)(kept + t * f.ld_kept + 4)};
        // rows that do not count leave nothing; a target that is no word leaves no number
        const float factor = y == r.ignore ? 0.f : y < 0 || y >= r.V ? NAN : exp2f(tops[t].x - lse);
        float p[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p[e] = y == r.ignore ? 0.f : e32[e / 4][e % 4] * factor;
        const int64_t here = y - f.v0 - word;
        if (here >= 0 && here < 8 && word + here < f.n && y != r.ignore) {
            const float hot = exp2f(r.picked[t] - lse) - 1.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = here == e ? hot : p[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) over_t[e] += p[e];
        if constexpr (NP == 3) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                bf16_t planes[3];
                split_planes<true>(p[e], planes);
#pragma unroll
                for (int q = 0; q < 3; ++q) v[q].v[e] = planes[q].bits;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 four = f32x4{p[h * 4], p[h * 4 + 1], p[h * 4 + 2], p[h * 4 + 3]} * (P::half ? kProbScale : 1.f);
                const s16x4 rounded = round4<P>(four);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[0].v[h * 4 + e] = (uint16_t)rounded[e];
            }
        }
#pragma unroll
        for (int q = 0; q < NP; ++q) at[q * 4] = v[q];
    }
    if (!f.bias_part && !f.bias_out) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[part][lane * 8 + e] = over_t[e];
    __syncthreads();
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v >= f.n) return;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][threadIdx.x];
    if (f.bias_out) ((E *)f.bias_out)[v] = from_float<E>(s * factor_of(f.factor));
    else f.bias_part[(int64_t)blockIdx.y * f.ld_bias_part + v] = s;
}

// ---- joins -------------------------------------------------------------------------------------------------------

// The sums of a bias's tiles, to the gradient of 256 words.
struct BiasJoin {
    const float *part;
    int ld, tiles, n;
    void *out;
};
template <typename E>
__device__ __forceinline__ void join_bias(const BiasJoin &b, int block, float factor)
{
    const int v = block * 256 + threadIdx.x;
    if (v >= b.n) return;
    float s = 0.f;
#pragma unroll 4
    for (int i = 0; i < b.tiles; ++i) s += b.part[(int64_t)i * b.ld + v];
    ((E *)b.out)[v] = from_float<E>(s * factor);
}
template <typename E>
__global__ __launch_bounds__(256) void bias_join_kernel(BiasJoin b, const float *f0, const float *f1)
{
    const float *const f[2] = {f0, f1};
    join_bias<E>(b, blockIdx.x, factor_of(f));
}

// The slices of a product in order, behind what earlier pieces of the vocabulary left in `acc`; the last piece's result is
// multiplied and rounded.  Workgroups from `blocks` on join a bias.
template <typename P, typename E>
__global__ __launch_bounds__(256) void join_kernel(const float *__restrict__ slices, int splits, int64_t n, int M, float *acc,
                                                   int first, int last, const float *f0, const float *f1,
                                                   const float *row_power, E *__restrict__ out, int64_t ldo, int blocks, BiasJoin bias)
{
    const float *const f[2] = {f0, f1};
    if ((int)blockIdx.x >= blocks) {
        join_bias<E>(bias, blockIdx.x - blocks, factor_of(f));
        return;
    }
    const float factor = last ? out_factor<P>(f) : 1.f;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)blocks * 256) {
        float s = first ? 0.f : acc[i];
        constexpr int kAhead = 8;
        for (int k = 0; k < splits; k += kAhead) {
            float got[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) got[j] = k + j < splits ? slices[(k + j) * n + i] : 0.f;
#pragma unroll
            for (int j = 0; j < kAhead; ++j) s += got[j];
        }
        if (last) out[i / M * ldo + i % M] = from_float<E>(s * (P::half && row_power ? factor * row_power[i / M] : factor));
        else acc[i] = s;
    }
}

// ---- plan --------------------------------------------------------------------------------------------------------

// Workspace of a piece's P, and of its repacked weights.  Larger pieces mean fewer slices of the hidden gradient to join (95 us
// a piece for 8192 tokens of 4096 features), smaller ones less memory; the products do not feel it.  The exponentials that a call
// for loss and gradients keeps of 16-bit types take twice as much besides.
constexpr size_t kPieceBytes = (size_t)1 << 30;

// The tile shape of a product, and how many stretches its reduction of k is cut into (1 of `most_splits`): the pair with the
// shortest estimate, rounds of workgroups times their steps and ends; slices are written and read once more by a launch of
// their own.  What decides it, measured: hidden gradients of 1543 x 1000 from 20011 words, float16, 157 us on 128 x 128 tiles
// in two stretches, 76 us on 256 x 256 in eight; 2048 x 1024 from 32768 words, float32, 1113 us (128 x 128, two) and 707 us
// (256 x 128, four); 64 x 512 from 1000 words, float32, 25 us in one stretch, 13 in four; scores of 512 tokens of 1024 features
// over 8000 words, bfloat16, 25, 16, 16 and 19 us from the largest tiles to the smallest.
struct Choice { int tile, splits; };
template <typename P>
Choice choose(int64_t m, int64_t n, int64_t k, int shapes, int most_splits, bool prob)
{
    typedef Shapes<P> S;
    const int cus = device_cus(), tile_knob = g_tune.vocab_tile, split_knob = g_tune.vocab_split;
    const int64_t steps = (k + P::step - 1) / P::step;
    Choice best{0, 1};
    if (m < 1 || n < 1) return best;
    double shortest = 1e300;
    for (int i = 0; i < shapes; ++i) {
        if (tile_knob >= 0 && tile_knob < shapes && i != tile_knob) continue;
        const int64_t tiles = ((m + S::m[i] - 1) / S::m[i]) * ((n + S::n[i] - 1) / S::n[i]);
        const int64_t fill = (int64_t)cus * S::resident[i];
        // stretches of 256 at least, and no more workgroups than two rounds of them
        int most = most_splits;
        if (most > steps * P::step / 256) most = (int)(steps * P::step / 256);
        if (split_knob >= 1) most = most < split_knob ? most : split_knob;
        else if (most > 2 * fill / tiles) most = (int)(2 * fill / tiles);
        if (most < 1) most = 1;
        for (int s = split_knob >= 1 ? most : 1; s <= most; s += 1 + s / 4) {
            const int64_t blocks = tiles * s;
            const double step = blocks <= cus ? S::alone_us[i] : S::step_us[i];
            const double round = (double)((steps + s - 1) / s) * step + S::ends_us[i] + (prob ? S::prob_us[i] : 0);
            const double us = (double)((blocks + fill - 1) / fill) * round + (s > 1 ? 4 + (double)s * m * n * 4 / 3e6 : 0);
            if (us < shortest) shortest = us, best = Choice{i, s};
        }
    }
    return best;
}

struct Plan {
    int Dp;               // features of repacked operands,
    int64_t ldd;          // and what their rows take
    int64_t piece, pieces;
    bool pack_h, pack_w;
    bool keep;            // the last piece's exponentials become its probabilities
    bool few;             // ds_vocab_few.hip's kernels
    int raw;              // float32 weights as they are for the matrix cores, so many at a time, or 0
    int tile_logits, tile_words, tile_tokens;
    Choice hidden, weight;
    int words;            // of a piece's probabilities, a multiple of 32,
    int64_t ldp;          // and what a row of them takes
    size_t h, w, stats, picked, shares, arrived, prob, kept, bias, slices, acc, scale, power, factor, bytes;
};

inline bool in_place(const void *p, int64_t ld, int64_t D) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && D % 8 == 0; }

// Up to how many tokens of float32 read the weights as they are.  Small heads give each workgroup too little to read: 16 tokens of
// 512 features, 1000 words, 44 us a step where planes take 33 (8 tokens: 31 and 34), 16 of 1024, 8000 words, 74 and 78.
constexpr int64_t kManyWeights = 1 << 23;
inline int64_t few_tokens(int64_t weights) { return weights < kManyWeights ? kFewTokens / 2 : kFewTokens; }

// What a call does: the loss, the gradients, or both.
enum { kLoss = 1, kGrad = 2 };

// Up to how many tokens of float32 the matrix instructions take weights as they are, `width` floats at a time, split into planes by
// every tile of 64 tokens; for more, planes for all of them to share are worth what writing and reading them takes, the sooner the
// fewer weights there are, for gradients (whose hidden states are in planes either way) and for weights that come one by one.
// Measured as they are and by planes, in us:
//                                  loss of 24       128         512     a step of 24         128           256           512 tokens
//   1024 features,  8200 words      46   44     47   62     93   94      93   88    117  121     166  152       260  225
//   1024,          16400            45   69     61   72    140  153     108  137    163  169     252  265       412  412
//   1024,          33000            60  126     93  154    243  271     158  242    267  330     424  482       735  753
//   1023 (one by one), 8300         53   42     55   60    106   94     105   88    131  123     180  155       285  228
//   1023,          16400            54   70     67   73    158  153     120  138    176  171     276  267       451  415
//   1023,          33000            66  132    106  159    268  274     174  251    294  338     464  490       805  760
//   2049,          50021           143  389    242  410    767  796     437  706    737  898    1266 1332      2424 2206
constexpr int64_t kManyOddWeights = 7 << 21;
inline int64_t raw_tokens(int64_t weights, int width, int what)
{
    const bool odd = width == 1, grad = what & kGrad;
    if (weights < (odd ? kManyOddWeights : kManyWeights)) return 0;
    return std::min<int64_t>(odd && grad ? 256 : 512, weights >> (15 + odd + grad));
}

template <typename P>
Plan plan_of(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int64_t T, int64_t D, int64_t V, int what)
{
    constexpr size_t NP = P::planes;
    Plan p{};
    p.Dp = (int)(NP > 1 ? (D + 31) / 32 * 32 : (D + 7) / 8 * 8);
    p.ldd = row_elements<P>(D);
    p.few = NP > 1 && T > 0 && T <= few_tokens(V * D) && g_tune.vocab_tile == kTuneUnset;
    p.pack_h = !p.few && (NP > 1 || what & kGrad || !in_place(hidden, ldh, D));  // for gradients: without the rows that do not count
    if (NP > 1 && !p.few && T > 0 && g_tune.vocab_tile == kTuneUnset) {
        const int width = (uintptr_t)weight % 16 == 0 && ldw % 4 == 0 && D % 4 == 0 ? 4 : 1;
        if (T <= raw_tokens(V * D, width, what)) p.raw = width;
    }
    p.pack_w = !p.few && !p.raw && (NP > 1 || !in_place(weight, ldw, D));
    const int kb = g_tune.vocab_piece_kb;
    const size_t piece_bytes = kb == kTuneUnset ? kPieceBytes : (size_t)kb << 10;
    int64_t most = V;
    auto at_most = [&](size_t per_word) {
        const int64_t n = (int64_t)(piece_bytes / (per_word ? per_word : 1)) / 256 * 256;
        most = n < 256 ? (most < 256 ? most : 256) : n < most ? n : most;
    };
    if (p.pack_w) at_most((size_t)p.ldd * 2);
    if (what & kGrad) at_most(NP * (size_t)T * 2);
    // equal pieces, of whole tiles
    p.pieces = (V + most - 1) / most;
    p.piece = ((V + p.pieces - 1) / p.pieces + 255) / 256 * 256;
    if (p.piece > V) p.piece = V;
    p.pieces = (V + p.piece - 1) / p.piece;
    p.keep = what == (kLoss | kGrad) && T <= 65535 * 8;
    p.tile_logits = p.few || p.raw ? 0 : choose<P>(p.piece, T, D, kShapes, 1, what & kGrad).tile;
    p.tile_words = p.few ? kFewWords : p.raw ? kRawWords : Shapes<P>::m[p.tile_logits];
    p.tile_tokens = p.few ? kFewTokens : p.raw ? kRawTokens : Shapes<P>::n[p.tile_logits];
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t was = at;
        at = align_up(at + n, 256);
        return was;
    };
    if (p.pack_h) p.h = take((size_t)T * p.ldd * 2);
    if (p.pack_w) p.w = take((size_t)p.piece * p.ldd * 2);
    if (what & kLoss) {
        const int64_t tiles = (p.piece + p.tile_words - 1) / p.tile_words;
        p.stats = take((size_t)(tiles * p.pieces) * T * 8);
        p.picked = take((size_t)T * 4);
        p.shares = take((size_t)((T + kRowsJoined - 1) / kRowsJoined) * sizeof(Share));
        p.arrived = take(4);
    }
    if (what & kGrad) {
        p.words = (int)((p.piece + 31) / 32 * 32);
        p.ldp = p.words * (int64_t)NP;
        if (p.few) {
            // four workgroups a CU, with 16 words at least
            const int64_t across = D > 0 ? (D + 255) / 256 : 1;
            p.hidden.splits = (int)std::min({(int64_t)64, (4 * device_cus() + across - 1) / across, (p.piece + 15) / 16});
            p.weight.splits = 1;
        } else {
            p.hidden = choose<P>(D, T, p.piece, kGradShapes<P>, 64, false);
            if (p.raw) {
                // two workgroups a CU, with 256 words at least
                const int64_t tiles = std::max<int64_t>(1, (D + kRawWords - 1) / kRawWords * ((T + kRawTokens - 1) / kRawTokens));
                p.hidden.splits = (int)std::max<int64_t>(1, std::min({(int64_t)64, 2 * device_cus() / tiles, p.piece / 256}));
            }
            p.weight = choose<P>(D, p.piece, T, kGradShapes<P>, 64, false);
        }
        p.prob = take((size_t)T * p.ldp * 2);
        // what a workgroup of either pass leaves of its rows
        const int kept_rows = finish_rows(T, p.words), rows = p.keep && kept_rows < p.tile_tokens ? kept_rows : p.tile_tokens;
        p.bias = take((size_t)((T + rows - 1) / rows) * p.words * 4);
        size_t slices = 0;
        if (p.few || p.hidden.splits > 1 || p.pieces > 1) slices = (size_t)p.hidden.splits * T * D * 4;
        if (p.weight.splits > 1) {
            const size_t n = (size_t)p.weight.splits * p.piece * D * 4;
            slices = n > slices ? n : slices;
        }
        // exponentials are probabilities before there is anything in the slices
        const size_t kept = p.keep && NP == 1 ? (size_t)T * p.words * 4 : 0;
        p.kept = p.slices = take(slices > kept ? slices : kept);
        if (p.pieces > 1) p.acc = take((size_t)T * D * 4);
        p.scale = take((size_t)T * 4);
        if (P::half) p.power = take((size_t)T * 4);
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
    size_t ws_bytes;
    hipStream_t st;
};

inline int check(const Call &c)
{
    if (c.T < 0 || c.D < 0 || c.V < 1 || !element_bytes(c.type)) return DS_EINVAL;
    if (c.T > 0 && (!c.target || (c.D > 0 && (!c.hidden || !c.weight || c.ldh < c.D || c.ldw < c.D)))) return DS_EINVAL;
    const int64_t most = 0x7fffffff - 512;
    if (c.T > most || c.V > most || c.D > 1000000 || c.ldh > 2000000 || c.ldw > 2000000) return DS_ETOOLARGE;
    return DS_OK;
}

#define DS_TRY(what)                    \
    do {                                \
        const int s_ = (what);          \
        if (s_ != DS_OK) return s_;     \
    } while (0)

// The operands as the products take them: hidden states once, weights piece by piece.
template <typename P>
struct Operands {
    Operand h, w;
    int64_t w_at = -1;
    bool h_there = false;

    int prepare(const Call &c, const Plan &p, bool counted_only, int64_t v0, int64_t n)
    {
        typedef typename ElementOf<P>::type E;
        const E *from = (const E *)c.weight + v0 * c.ldw;
        Pack ph{}, pw{};
        if (!h_there) {
            h = p.pack_h ? Operand{c.ws + p.h, p.ldd} : Operand{c.hidden, c.ldh};
            if (p.pack_h)
                ph = Pack{c.hidden, c.ldh, c.T, (int)c.D, p.Dp, (uint16_t *)(c.ws + p.h), p.ldd,
                          counted_only ? c.target : nullptr, c.wide, c.ignore};
            h_there = true;
        }
        if (w_at != v0) {
            w = p.pack_w ? Operand{c.ws + p.w, p.ldd} : Operand{from, c.ldw};
            if (p.pack_w) pw = Pack{from, c.ldw, n, (int)c.D, p.Dp, (uint16_t *)(c.ws + p.w), p.ldd, nullptr, 0, 0};
            w_at = v0;
        }
        return launch_pack<E>(ph, pw, c.st);
    }
};

template <typename P>
Args logit_args(const Call &c, const Plan &p, int64_t v0, int64_t n, const Operands<P> &o)
{
    Args g{};
    g.a = o.w, g.b = o.h;
    g.M = (int)n, g.N = (int)c.T, g.K = p.few || p.raw ? (int)c.D : p.Dp;
    g.splits = 1, g.k_split = (p.Dp + P::step - 1) / P::step * P::step;
    g.bias = c.bias, g.bias_type = c.type;
    g.target = c.target, g.target_wide = c.wide;
    g.V = c.V, g.ignore = c.ignore, g.v0 = (int)v0;
    return g;
}

// Whether finish_kernel joins the rows' sums: each of its workgroups does it for its own rows, and one for all, which pays
// while there are few of both (64 tokens, 1000 words, float32: 3 us of a step).
inline bool joined_later(const Plan &p, int64_t T, int tiles) { return p.keep && p.pieces == 1 && T <= 128 && tiles <= 64; }

// One product, of `kind`, by the kernels of the plan; fills in the tile counts.
template <typename P>
int product(const Plan &p, int kind, int tile, Args &g, int64_t T, hipStream_t st)
{
    if (p.raw && kind != kWeight) return launch_raw(kind, p.raw, g, st);
    return p.few ? launch_few(kind, (int)T, g, st) : launch_product<P>(kind, tile, g, nullptr, st);
}

template <typename P>
int loss(const Call &c, const Plan &p, bool counted_only, Operands<P> &o, int reduction, float *rows, float *lse, float *total,
         Rows *of)
{
    if (c.T == 0) {
        if (reduction) hipLaunchKernelGGL(no_rows_kernel, dim3(1), dim3(1), 0, c.st, reduction == DS_MEAN, total);
        return launch_status();
    }
    int tiles = 0;
    for (int64_t v0 = 0; v0 < c.V; v0 += p.piece) {
        const int64_t n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
        // (float32 tokens that do not count never make a tile look at its NaNs: 2048 x 1024 over 32768 words, a twentieth of them
        // NaN, 705 us for the loss instead of 1580)
        DS_TRY(o.prepare(c, p, counted_only || P::planes > 1, v0, n));
        Args g = logit_args<P>(c, p, v0, n, o);
        g.stats = (float *)(c.ws + p.stats) + (int64_t)tiles * c.T * 2;
        g.picked = (float *)(c.ws + p.picked);
        g.arrived = (uint32_t *)(c.ws + p.arrived);
        g.prob = c.ws + p.prob, g.ldp = p.ldp, g.prob_words = p.words;
        g.kept = (float *)(c.ws + p.kept), g.ld_kept = p.words;
        DS_TRY(product<P>(p, p.keep && v0 + n == c.V ? kLogitKeep : kLogitStats, p.tile_logits, g, c.T, c.st));
        tiles += g.tiles_m;
    }
    *of = Rows{(const float2 *)(c.ws + p.stats), (const float *)(c.ws + p.picked), tiles, (int)c.T, c.target, c.wide, c.V, c.ignore,
               lse, rows, reduction, (Share *)(c.ws + p.shares), (uint32_t *)(c.ws + p.arrived), total};
    if (!joined_later(p, c.T, tiles))
        hipLaunchKernelGGL(row_kernel, dim3((unsigned)((c.T + kRowsJoined - 1) / kRowsJoined)), dim3(1024), 0, c.st, *of);
    return launch_status();
}

// What the gradients are asked for with, and where they go.
struct Grads {
    const float *lse, *row_grad, *grad, *share;
    void *dhidden, *dweight, *dbias;
};

template <typename P>
int loss_grad(const Call &c, const Plan &p, Operands<P> &o, const Rows &of, Grads r)
{
    typedef typename ElementOf<P>::type E;
    // rows of float16 whose gradients are of different sizes keep scales of their own until their hidden gradients are formed
    float *const power = P::half && r.row_grad && r.dhidden ? (float *)(c.ws + p.power) : nullptr;
    if (c.T > 0 && r.row_grad) {
        hipLaunchKernelGGL(row_scale_kernel, dim3(1), dim3(1024), 0, c.st, r.row_grad, c.target, c.wide, (int)c.T, c.ignore,
                           (float *)(c.ws + p.scale), (float *)(c.ws + p.factor), power);
        r.grad = (const float *)(c.ws + p.factor);
    }
    float *const slices = (float *)(c.ws + p.slices);
    // the last piece first: its exponentials may be there, and its weights are
    for (int64_t i = 0; i < p.pieces; ++i) {
        const int64_t v0 = (i == 0 ? p.pieces - 1 : i - 1) * p.piece;
        const int64_t n = c.V - v0 < p.piece ? c.V - v0 : p.piece;
        const bool first = i == 0, last = i == p.pieces - 1, kept = p.keep && i == 0;
        int bias_tiles = 0;
        bool bias_left = r.dbias != nullptr;
        const Operand prob{c.ws + p.prob, p.ldp};
        if (c.T > 0) {
            const int rows = kept ? finish_rows(c.T, p.words) : p.tile_tokens;
            bias_tiles = (int)((c.T + rows - 1) / rows);
            // the sums of one workgroup are the gradient, but for the share that a launch which joins the rows only finds
            bias_left = r.dbias && (bias_tiles > 1 || joined_later(p, c.T, of.tiles));
            float *const bias_part = bias_left ? (float *)(c.ws + p.bias) : nullptr;
            void *const bias_out = r.dbias && !bias_left ? (E *)r.dbias + v0 : nullptr;
            if (kept) {
                const int words = ceil_div((int)n, 32) * 32;
                const bool beside = P::planes == 1;
                const Finish f{c.ws + p.prob, p.ldp, (const float *)(c.ws + (beside ? p.kept : p.prob)), beside ? p.words : p.ldp / 2, words, p.tile_words, rows, v0, n, of.tiles - ceil_div((int)n, p.tile_words),
                               p.words, of, bias_part, bias_out, {r.grad, r.share}};
                const unsigned along = ceil_div(words, 256), down = ceil_div((int)c.T, rows);
                if (joined_later(p, c.T, of.tiles))
                    hipLaunchKernelGGL((finish_kernel<P, true>), dim3(along, down + 1), dim3(256), 0, c.st, f);
                else
                    hipLaunchKernelGGL((finish_kernel<P, false>), dim3(along, down), dim3(256), 0, c.st, f);
            } else {
                DS_TRY(o.prepare(c, p, true, v0, n));
                Args g = logit_args<P>(c, p, v0, n, o);
                g.lse = r.lse;
                g.row_scale = r.row_grad ? (const float *)(c.ws + p.scale) : nullptr;
                g.row_power = power;
                g.prob = c.ws + p.prob, g.ldp = p.ldp, g.prob_words = p.words;
                g.factor[0] = r.grad, g.factor[1] = r.share;
                g.bias_out = bias_out, g.bias_part = bias_part;
                g.ld_bias_part = p.words;
                DS_TRY(product<P>(p, kLogitProb, p.tile_logits, g, c.T, c.st));
            }
        }
        BiasJoin bias{(const float *)(c.ws + p.bias), p.words, bias_tiles, (int)n, r.dbias ? (E *)r.dbias + v0 : nullptr};
        // by itself, or along with the join of a product
        auto join_bias_alone = [&] {
            if (bias_left)
                hipLaunchKernelGGL((bias_join_kernel<E>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, c.st, bias, r.grad,
                                   r.share);
            bias_left = false;
        };
        if (c.D == 0) join_bias_alone();
        if (c.D == 0) continue;
        Args g[2] = {};
        bool wanted[2], joined[2];
        for (int which = 0; which < 2; ++which) {
            Args &x = g[which];
            wanted[which] = which ? r.dweight != nullptr : r.dhidden && c.T > 0;
            x.a = which ? o.h : o.w;
            x.b = prob;
            x.M = (int)c.D;
            x.N = which ? (int)((n + 7) / 8 * 8) : (int)c.T;
            x.n_store = which ? (int)n : (int)c.T;
            x.K = which ? (int)c.T : (int)n;
            x.factor[0] = r.grad, x.factor[1] = r.share;
            x.out = which ? (void *)((E *)r.dweight + v0 * c.D) : r.dhidden;
            x.ldo = c.D;
            x.splits = which ? p.weight.splits : p.hidden.splits;
            x.k_split = ((x.K + x.splits - 1) / x.splits + P::step - 1) / P::step * P::step;
            if (p.few) x.k_split = ceil_div(x.K, x.splits);
            x.target = c.target, x.target_wide = c.wide, x.ignore = c.ignore;
            joined[which] = x.splits > 1 || (!which && (p.pieces > 1 || p.few));
            x.slice = joined[which] ? slices : nullptr;
            x.row_power = which ? nullptr : power;
        }
        // few workgroups each, and no slices to share: both in one launch
        const int tm = Shapes<P>::m[p.weight.tile], tn = Shapes<P>::n[p.weight.tile];
        const int64_t across = (int64_t)ceil_div((int)c.T, tn) * p.hidden.splits + ceil_div((int)n, tn);
        const int64_t blocks = ceil_div((int)c.D, tm) * across;
        const bool both = !p.few && !p.raw && !power && wanted[0] && wanted[1] && !joined[1] && p.hidden.tile == p.weight.tile && blocks <= 2 * device_cus();
        if (both) DS_TRY(launch_product<P>(kHidden, p.weight.tile, g[0], &g[1], c.st));
        for (int which = 0; which < 2; ++which) {
            Args &x = g[which];
            if (!wanted[which]) continue;
            const int tile = which ? p.weight.tile : p.hidden.tile;
            if (which && power && c.T > 0) {
                const int words = ceil_div((int)n, 32) * 32;
                const int64_t all = (c.T * (words / 8) + 255) / 256;
                hipLaunchKernelGGL(power_kernel, dim3((unsigned)(all < 16384 ? all : 16384)), dim3(256), 0, c.st,
                                   (f16_t *)(c.ws + p.prob), p.ldp, words, c.T, power);
            }
            if (!both) DS_TRY(product<P>(p, which ? kWeight : kHidden, tile, x, c.T, c.st));
            if (!joined[which]) continue;
            const int64_t count = (int64_t)x.n_store * c.D;
            const int64_t all = (count + 255) / 256;
            const int join = (int)(all < 16384 ? all : 16384), more = bias_left ? ceil_div((int)n, 256) : 0;
            hipLaunchKernelGGL((join_kernel<P, E>), dim3(join + more), dim3(256), 0, c.st, slices, x.splits, count, (int)c.D,
                               which ? nullptr : (float *)(c.ws + p.acc), which || first, which || last, r.grad, r.share,
                               x.row_power, (E *)x.out, c.D, join, bias);
            bias_left = false;
        }
        join_bias_alone();
    }
    return launch_status();
}

struct Outputs {
    int reduction;
    float *rows, *lse, *total;
    Grads grads;
};

template <typename P>
int run(const Call &c, int what, const Outputs &out)
{
    const Plan p = plan_of<P>(c.hidden, c.ldh, c.weight, c.ldw, c.T, c.D, c.V, what);
    if (!c.ws || c.ws_bytes < p.bytes || (uintptr_t)c.ws % 256) return DS_EWORKSPACE;
    Operands<P> o;
    Rows of{};
    if (what & kLoss) DS_TRY(loss<P>(c, p, what & kGrad, o, out.reduction, out.rows, out.lse, out.total, &of));
    if (what & kGrad) DS_TRY(loss_grad<P>(c, p, o, of, out.grads));
    return DS_OK;
}

int run(const Call &c, int what, const Outputs &out)
{
    DS_TRY(check(c));
    if (c.type == DS_F32) return run<Split>(c, what, out);
    if (c.type == DS_BF16) return run<Bf16>(c, what, out);
    return run<F16>(c, what, out);
}

}  // namespace vocab
}  // namespace ds

using namespace ds;
using namespace ds::vocab;

DS_EXPORT size_t ds_vocab_workspace_bytes(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int64_t T, int64_t D,
                                          int64_t V, int type, int what)
{
    if (T < 0 || D < 0 || V < 1 || !element_bytes(type) || what < kLoss || what > (kLoss | kGrad)) return 0;
    if (type == DS_F32) return plan_of<Split>(hidden, ldh, weight, ldw, T, D, V, what).bytes;
    if (type == DS_BF16) return plan_of<Bf16>(hidden, ldh, weight, ldw, T, D, V, what).bytes;
    return plan_of<F16>(hidden, ldh, weight, ldw, T, D, V, what).bytes;
}

DS_EXPORT int ds_vocab_loss(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias,
                            const void *target, int target_bytes, int64_t ignore, int64_t T, int64_t D, int64_t V, int type,
                            int reduction, float *rows, float *lse, float *total, void *workspace, size_t workspace_bytes,
                            ds_stream_t stream)
{
    if ((target_bytes != 4 && target_bytes != 8) || reduction < 0 || reduction > DS_MEAN) return DS_EINVAL;
    if ((T > 0 && (!rows || !lse)) || (reduction && !total)) return DS_EINVAL;
    return run(Call{hidden, weight, bias, target, ldh, ldw, T, D, V, ignore, target_bytes == 8, type, (char *)workspace,
                    workspace_bytes, (hipStream_t)stream},
               kLoss, Outputs{reduction, rows, lse, total, Grads{}});
}

DS_EXPORT int ds_vocab_loss_grad(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias,
                                 const void *target, int target_bytes, int64_t ignore, int64_t T, int64_t D, int64_t V, int type,
                                 const float *lse, const float *row_grad, const float *grad, const float *share, void *dhidden,
                                 void *dweight, void *dbias, void *workspace, size_t workspace_bytes, ds_stream_t stream)
{
    if ((target_bytes != 4 && target_bytes != 8) || (row_grad && (grad || share)) || (T > 0 && !lse)) return DS_EINVAL;
    return run(Call{hidden, weight, bias, target, ldh, ldw, T, D, V, ignore, target_bytes == 8, type, (char *)workspace,
                    workspace_bytes, (hipStream_t)stream},
               kGrad, Outputs{0, nullptr, nullptr, nullptr, Grads{lse, row_grad, grad, share, dhidden, dweight, dbias}});
}

DS_EXPORT int ds_vocab_loss_step(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias,
                                 const void *target, int target_bytes, int64_t ignore, int64_t T, int64_t D, int64_t V, int type,
                                 int reduction, float *rows, float *lse, float *total, void *dhidden, void *dweight, void *dbias,
                                 void *workspace, size_t workspace_bytes, ds_stream_t stream)
{
    if ((target_bytes != 4 && target_bytes != 8) || reduction < 0 || reduction > DS_MEAN) return DS_EINVAL;
    if ((T > 0 && (!rows || !lse)) || (reduction && !total)) return DS_EINVAL;
    return run(Call{hidden, weight, bias, target, ldh, ldw, T, D, V, ignore, target_bytes == 8, type, (char *)workspace,
                    workspace_bytes, (hipStream_t)stream},
               kLoss | kGrad, Outputs{reduction, rows, lse, total,
                                      Grads{lse, nullptr, nullptr, reduction ? total + 1 : nullptr, dhidden, dweight, dbias}});
}
