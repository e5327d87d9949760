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
//
// Distillation from a teacher's best K words is the same with many targets a token, q the softmax of their logits by the
// temperature c:  p = softmax(s / c)      loss[t] = c^2 sum_k q_k (log q_k - log p_k)      P = c g_t (p - q).
// One launch makes q of the teacher's logits and puts the words in ascending order; the tiles find the words that lie in them by
// a search while their operands arrive.
#include "ds_vocab_host.h"

namespace ds {
namespace vocab {

// ---- operands as the products take them --------------------------------------------------------------------------

// Rows of D elements to rows of Dp (a multiple of 8 or 32, zeros behind D): 16-bit elements as they are, float32 as three planes.
// Bound by memory: (2048 + 32768) x 1024 float32 in 64 us, 5.5 TB/s.  Loads are 16 bytes wherever a row begins: 50021 x 2049
// bfloat16 take 75 us, element by element 176.
// Rows whose target is `ignore` (where targets are given) become zeros: tokens that do
// not count leave nothing in the weights' gradient, not even a value that is no number.  The first operand by `first` workgroups.
template <typename E, typename COUNTS>
__device__ __forceinline__ void pack_rows(const Pack &p, int block, int blocks, const COUNTS &counts)
{
    constexpr int N = 16 / sizeof(E);
    const int units = p.Dp / N;
    const int64_t total = p.rows * units;
    for (int64_t i = (int64_t)block * 256 + threadIdx.x; i < total; i += (int64_t)blocks * 256) {
        const int64_t r = i / units;
        const int c = (int)(i - r * units) * N;
        const E *x = (const E *)p.x + r * p.ld;
        Vec<E, N> v{};
        if (!counts(r)) {
        } else if (c + N <= p.D) __builtin_memcpy(&v, x + c, sizeof(v));  // wherever it lies
        else
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (c + e < p.D) v.v[e] = x[c + e];
        uint16_t *row = p.out + r * p.ldo;
        if constexpr (sizeof(E) == 2) {
            *(Vec<E, N> *)(row + c) = v;
            if (p.again) *(Vec<E, N> *)(row + p.again * p.ldo + c) = v;
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
__global__ __launch_bounds__(256) void pack_kernel(Pack one, Pack two, int first)
{
    const bool is_one = (int)blockIdx.x < first;
    const Pack &p = is_one ? one : two;
    const void *const target = p.target;
    const int wide = p.wide;
    const int64_t ignore = p.ignore;
    pack_rows<E>(p, is_one ? blockIdx.x : blockIdx.x - first, is_one ? first : gridDim.x - first, [=](int64_t r) {
        return !target || (wide ? ((const int64_t *)target)[r] : (int64_t)((const int32_t *)target)[r]) != ignore;
    });
}

template <typename E> int pack_blocks(const Pack &p)
{
    const int64_t b = (p.rows * (p.Dp / (16 / (int)sizeof(E))) + 255) / 256;
    return (int)(b < 8192 ? b : 8192);
}
template <typename E>
int launch_pack(const Pack &one, const Pack &two, hipStream_t st)
{
    const int first = pack_blocks<E>(one), all = first + pack_blocks<E>(two);
    if (all == 0) return DS_OK;
    hipLaunchKernelGGL((pack_kernel<E>), dim3(all), dim3(256), 0, st, one, two, first);
    return launch_status();
}

template int launch_pack<float>(const Pack &, const Pack &, hipStream_t);
template int launch_pack<bf16_t>(const Pack &, const Pack &, hipStream_t);
template int launch_pack<f16_t>(const Pack &, const Pack &, hipStream_t);

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
__device__ __forceinline__ void write_total(double loss, double rows, int mean, float *total, float temperature = 1.f)
{
    const double share = mean && rows > 0 ? 1.0 / rows : 1.0;
    total[0] = (float)(loss * share);
    total[1] = (float)(share * temperature);  // (the gradient of a teacher's words is the temperature times P)
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
    // of a teacher: its probabilities of the picked words, so many of each, and its temperature; else NULL, 0 and 1
    const float *taught;
    int words;
    float temperature;
};

__device__ __forceinline__ float log_of_sum(float top, float sum) { return sum == 0.f ? -INFINITY : top + log2f(sum); }

__device__ __forceinline__ float loss_of(const Rows &r, int t, int64_t y, float lse)
{
    return y == r.ignore ? 0.f : y < 0 || y >= r.V ? NAN : (lse - r.picked[t]) * kLn2;
}

// A share of a row's distance from its teacher: every `step`-th of its words from `from` on.
__device__ __forceinline__ float taught_loss(const Rows &r, int t, float lse, int from, int step)
{
    float sum = 0.f;
    const float *const q = r.taught + (int64_t)t * r.words, *const s = r.picked + (int64_t)t * r.words;
#pragma unroll 4
    for (int k = from; k < r.words; k += step) {
        const float p = q[k];
        if (p > 0.f) sum += p * (log2f(p) - (s[k] - lse));  // (places behind the last word hold 0, and their logits nothing)
    }
    return sum;
}

// A workgroup's part in the total: its wave's sums of losses and of counted rows, `group` of `groups`.  The one that ends last
// adds up all of them, in order.
__device__ __forceinline__ void add_to_total(const Rows &r, double loss, double counted, int group, int groups)
{
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) loss += __shfl_xor(loss, o), counted += __shfl_xor(counted, o);
    if (groups == 1) {
        if (lane == 0) write_total(loss, counted, r.reduction == DS_MEAN, r.total, r.temperature);
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
    if (lane == 0) write_total(loss, counted, r.reduction == DS_MEAN, r.total, r.temperature);
}

// ---- a teacher's heavy words ----------------------------------------------------------------------------------------
//
// P is rounded to the operands' type for the gradients' products.  Its own column's size is what a row of the weights' gradient is
// off by then, and words that most tokens teach have columns hundreds of times larger than others.  Of bfloat16 single values were
// off by half of the whole gradient's root mean square, beyond their own rounding (8192 tokens, 64 of 65536 words, as often as text
// has them; of 65 to 8192 tokens over 1000 words by 0.16, over 2000 by 0.21, over 4096 by 0.32).  So P keeps its rounding's remainder
// for groups of 256 words that hold such a word, and the weights' gradient takes both: 0.03 to 0.1 of it then over 65536 words,
// whose step of 8192 x 4096 takes 11.2 ms instead of 10.9; the workspace holds P and the hidden states twice.  A single word's P is
// near -1, which rounds to itself.  Words that only the student finds likely, token for token, are rounded as the cross entropy's are.
//
// Up to kTwiceAll tokens, which costs nothing beside the weights, and up to kTwiceWords words all groups have it: less than 0.001 of
// the root mean square there.  A step in us without it, with groups that are looked for, and with all:
//      tokens, features, words           none  marked   all         tokens, features, words           none  marked   all
//         65      512     1000             30      38    30            512     1024     4096            68      88    74
//        128      512     1000             31      41    31           2048     1024     4096           136     174   158
//       1024      512     1000             50      63    54           4096     1024     2000           151     184   182
//       8192      512     1000            130     155   145           8192     4096     4096           804    1000  1031
constexpr int64_t kTwiceAll = 64, kTwiceWords = 4096;

struct Marks {
    const int *sorted;
    const float *taught;
    const int *target;   // [T] 0: the token counts,
    const float *grad;   // [T] unless this is 0; or NULL
    int64_t T, V;
    int K;
    uint8_t *twice;      // [groups of 256 words]
};

// By one workgroup, while others join the rows (8192 tokens of 64 words: 55 us instead of 22, by itself 30): of up to 512 tokens and
// 16384 words, one token of every stretch, the words' sums of squared probabilities, whole numbers of 2^-20, in two tables by a hash
// of the word each.  A word whose sums are a hundred-and-twenty-eighth of all in both of them marks its group: all that have as much
// themselves, and one of some 10000 others that share their places with such words in both.  A stretch's token is its first that
// counts and has a gradient, looked for from a place that moves by the golden ratio from stretch to stretch: at the same place of
// each, tokens of equal sequences would all stand at one place of theirs.
__device__ __forceinline__ void mark_heavy(const Marks &m)
{
    constexpr int kBuckets = 4096, kSample = 512;
    __shared__ uint32_t sums[2][kBuckets];
    __shared__ int sample[kSample];  // tokens, -1 where none of a stretch counts
    __shared__ unsigned long long all;
    for (int i = threadIdx.x; i < kBuckets; i += blockDim.x) sums[0][i] = 0, sums[1][i] = 0;
    if (threadIdx.x == 0) all = 0;
    const int64_t groups = (m.V + 255) / 256;
    for (int64_t i = threadIdx.x; i < groups; i += blockDim.x) m.twice[i] = 0;
    __threadfence();
    const int most = min(kSample, 16384 / m.K), step = (int)((m.T + most - 1) / most), stretches = (int)((m.T + step - 1) / step);
    const int places = stretches * m.K;
    for (int i = threadIdx.x; i < stretches; i += blockDim.x) {
        const int first = i * step, count = (int)min((int64_t)step, m.T - first);
        const int from = (int)((uint64_t)(uint32_t)(i * 2654435769u) * count >> 32);
        int found = -1;
        constexpr int kAhead = 8;
        for (int j = 0; j < count && found < 0; j += kAhead) {
            int at[kAhead], target[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                at[k] = from + min(j + k, count - 1);
                at[k] = first + (at[k] < count ? at[k] : at[k] - count);
                target[k] = m.grad && m.grad[at[k]] == 0.f ? -1 : m.target[at[k]];
            }
#pragma unroll
            for (int k = kAhead - 1; k >= 0; --k) found = target[k] == 0 ? at[k] : found;
        }
        sample[i] = found;
    }
    __syncthreads();
    auto over_sample = [&](auto found) {
#pragma unroll 4
        for (int i = threadIdx.x; i < places; i += blockDim.x) {
            const int t = sample[i / m.K];
            if (t < 0) continue;
            const int64_t at = (int64_t)t * m.K + i % m.K;
            const float q = m.taught[at];
            const uint32_t id = (uint32_t)m.sorted[at], sum = (uint32_t)(q * q * 0x1p20f);
            if (sum > 0) found(id, sums[0][id * 2654435769u >> 20], sums[1][id * 3242174889u >> 20], sum);
        }
    };
    unsigned long long mine = 0;
    over_sample([&](uint32_t, uint32_t &one, uint32_t &two, uint32_t sum) {
        atomicAdd(&one, sum);
        atomicAdd(&two, sum);
        mine += sum;
    });
    atomicAdd(&all, mine);
    __syncthreads();
    over_sample([&](uint32_t id, uint32_t &one, uint32_t &two, uint32_t) {
        if (min(one, two) * 128ull >= all) m.twice[id / 256] = 1;
    });
}
__global__ __launch_bounds__(1024) void mark_kernel(Marks m) { mark_heavy(m); }

// Joins the tiles' maxima and sums: a workgroup has kRowsJoined rows, each of its waves a sixteenth of the tiles and each
// quarter of a wave a quarter of those.  Bound by latency: 37 rows of 391 tiles in 4.4 us (18 with 64 rows a workgroup and a
// wave's tiles one after the other), 8192 rows of 512 tiles, 34 MB, in 20.
constexpr int kRowsJoined = 16;

// MARK: the last workgroup marks a teacher's heavy words meanwhile.
template <bool MARK>
__global__ __launch_bounds__(1024) void row_kernel(Rows r, Marks m)
{
    const int groups = MARK ? gridDim.x - 1 : gridDim.x;
    if constexpr (MARK)
        if ((int)blockIdx.x == groups) {
            mark_heavy(m);
            return;
        }
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
    float away = 0.f;
    if (r.taught) {
        if (t < r.T) away = taught_loss(r, t, log_of_sum(top, sum), part, 4);
#pragma unroll
        for (int o = 16; o < 64; o <<= 1) away += __shfl_xor(away, o);
        away *= kLn2 * r.temperature * r.temperature;
    }
    if (t < r.T && part == 0) {
        const float lse = log_of_sum(top, sum);
        const int64_t y = target_of(r.target, r.wide, t);
        r.lse[t] = lse;
        const float l = !r.taught ? loss_of(r, t, y, lse) : y == r.ignore ? 0.f : y >= r.V ? NAN : away;
        r.loss[t] = l;
        mine = l, counts = y != r.ignore;
    }
    if (r.reduction) add_to_total(r, mine, counts, blockIdx.x, groups);
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
    const int *taught_ids; // TAUGHT: [T][words of a teacher], as Args has them
    const uint8_t *twice;  // and these two
    int64_t again;
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
// TAUGHT: of the words that a teacher has for the row, those among the workgroup's 256 are found by the half wave that has the
// row, 32 at a time, and each is handed to the lane that has its word.
template <typename P, bool JOIN, bool TAUGHT = false>
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
            float lse = 0.f, away = 0.f;
            if (t < r.T && (TAUGHT || wave == 0)) {
                top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) join_pair(top, sum, parts[w * 64 + row].x, parts[w * 64 + row].y);
                lse = log_of_sum(top, sum);
            }
            if constexpr (TAUGHT) {
                float *const shares = sums[2];  // [4][64], behind the parts
                if (t < r.T) shares[wave * 64 + row] = taught_loss(r, t, lse, wave, 4);
                __syncthreads();
                away = (shares[row] + shares[64 + row] + shares[128 + row] + shares[192 + row]) * (kLn2 * r.temperature * r.temperature);
            }
            if (wave == 0 && t < r.T) {
                const int64_t y = target_of(r.target, r.wide, t);
                const float l = !TAUGHT ? loss_of(r, t, y, lse) : y == r.ignore ? 0.f : y >= r.V ? NAN : away;
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
    const bool both = f.again && (!f.twice || f.twice[f.v0 / 256 + blockIdx.x]);
#pragma unroll JOIN || TAUGHT ? 1 : 4
    for (int i = 0; i < f.rows; i += 8) {
        const int t = blockIdx.y * f.rows + i + part;
        if (t >= r.T) break;
        const int64_t y = target_of(r.target, r.wide, t);
        const float lse = JOIN ? lse_of_row(r, t, lane) : r.lse[t];
        float taught[8];
        if constexpr (TAUGHT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) taught[e] = 0.f;
            const int64_t row = (int64_t)t * r.words;
            const int from = (int)f.v0 + blockIdx.x * 256, to = (int)f.v0 + min((int)f.n, (int)blockIdx.x * 256 + 256), half = threadIdx.x & 32;
            for (int k = 0; k < r.words; k += 32) {
                const int id = k + lane < r.words ? f.taught_ids[row + k + lane] : 0x7fffffff;
                const bool inside = id >= from && id < to;
                const float q = inside ? r.taught[row + k + lane] : 0.f;
                uint32_t left = (uint32_t)(__ballot(inside) >> half);
                while (__any(left != 0)) {
                    const int of = half + (left ? __ffs(left) - 1 : 0);
                    const int here = __shfl(id, of) - from - lane * 8;
                    const float probability = __shfl(q, of);
#pragma unroll
                    for (int e = 0; e < 8; ++e) taught[e] += left && here == e ? probability : 0.f;
                    left &= left - 1;
                }
                if (__all(id >= to)) break;  // they are in ascending order
            }
        }
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
        if constexpr (TAUGHT) {
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = y == r.ignore ? 0.f : p[e] - taught[e];
        } else if (here >= 0 && here < 8 && word + here < f.n && y != r.ignore) {
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
        if constexpr (TAUGHT && NP == 1 && !P::half)
            if (both) {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[0].v[e] = from_float<bf16_t>(rounding_of(p[e])).bits;
                *(Vec<uint16_t, 8> *)(column + (t + f.again) * f.ldp) = v[0];
            }
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

// ---- a teacher's words -------------------------------------------------------------------------------------------------

// What a teacher says of every token: its best words' numbers and logits, K of each.
struct Teacher {
    const void *ids;
    int wide;
    const void *logits;
    int type, K;
    int64_t T, V;
    float temperature;
    int *sorted;       // [T][K] numbers in ascending order, 0x7fffffff behind the last
    float *taught;     // [T][K] their probabilities
    int *target;       // [T] 0, -1 where there is no word, V where the probabilities are no numbers or a word is none
    float *factor;     // the temperature
};
constexpr int kMostTaught = 1024;

// What stands at a place: a word's number, below 0 where there is none, and its logit.
__device__ __forceinline__ int64_t word_at(const Teacher &f, int64_t at, float &logit)
{
    const int64_t word = f.wide ? ((const int64_t *)f.ids)[at] : (int64_t)((const int32_t *)f.ids)[at];
    logit = f.type == DS_F32 ? ((const float *)f.logits)[at]
            : f.type == DS_BF16 ? to_float(((const bf16_t *)f.logits)[at]) : to_float(((const f16_t *)f.logits)[at]);
    return logit == -INFINITY ? -1 : word;
}

// Probabilities of a token's words, in the order of their numbers: a workgroup has a token, a thread a word, whose place is how
// many come before it (the comparisons of 64 words take less time than their loads: 8192 tokens in 12 us).
template <int MOST>
__device__ __forceinline__ void teach(const Teacher &f, int64_t t)
{
    __shared__ int ids[MOST];
    __shared__ float tops[MOST / 64], sums[MOST / 64];
    __shared__ int found[MOST / 64];
    const int k = threadIdx.x, wave = k >> 6, lane = k & 63, waves = blockDim.x >> 6;
    int id = 0x7fffffff, seen = 0;  // 1: a word, 2: something that is none, or no number
    float logit = -INFINITY;
    if (k < f.K) {
        const int64_t word = word_at(f, t * f.K + k, logit);
        if (word < 0) logit = -INFINITY;
        else if (word >= f.V || !(logit < INFINITY)) logit = -INFINITY, seen = 3;
        else id = (int)word, seen = 1;
    }
    float top = logit;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o)), seen |= __shfl_xor(seen, o);
    ids[k] = id;
    if (lane == 0) tops[wave] = top, found[wave] = seen;
    __syncthreads();
    for (int w = 0; w < waves; ++w) top = fmaxf(top, tops[w]), seen |= found[w];
    const float warmth = kLog2e / f.temperature;
    float e = id == 0x7fffffff ? 0.f : exp2f((logit - top) * warmth), sum = e;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if (lane == 0) sums[wave] = sum;
    int place = 0;
    for (int i = 0; i < f.K; ++i) place += ids[i] < id || (ids[i] == id && i < k);
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < waves; ++w) sum += sums[w];
    if (k < f.K) f.sorted[t * f.K + place] = id, f.taught[t * f.K + place] = id == 0x7fffffff ? 0.f : e / sum;
    if (k == 0) f.target[t] = seen == 0 ? -1 : seen & 2 ? (int)f.V : 0;
    if (k == 0 && t == 0) *f.factor = f.temperature;
}
__global__ __launch_bounds__(kMostTaught) void teacher_kernel(Teacher f) { teach<kMostTaught>(f, blockIdx.x); }

// Operands too, in one launch, up to kTaughtBeside tokens of 256 words (one of five to eight that a small call takes; of many tokens
// waves without words would cost more): hidden states look for themselves whether a token has any.
constexpr int kTaughtBeside = 1024;
template <typename E>
__global__ __launch_bounds__(256) void teacher_pack_kernel(Teacher f, Pack one, Pack two, int first)
{
    const int block = blockIdx.x - (int)f.T;
    if (block < 0) {
        teach<256>(f, blockIdx.x);
    } else if (block < first) {
        pack_rows<E>(one, block, first, [&](int64_t r) {
            bool any = !one.target;
            float logit;
            for (int k = 0; k < f.K && !any; ++k) any = word_at(f, r * f.K + k, logit) >= 0;
            return any;
        });
    } else {
        pack_rows<E>(two, block - first, gridDim.x - (int)f.T - first, [](int64_t) { return true; });
    }
}

// ---- joins -------------------------------------------------------------------------------------------------------

// The sums of a bias's tiles, to the gradient of 256 words.
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

template <typename E> int launch_bias_join(const BiasJoin &b, const float *f0, const float *f1, hipStream_t st)
{
    hipLaunchKernelGGL((bias_join_kernel<E>), dim3(ceil_div(b.n, 256)), dim3(256), 0, st, b, f0, f1);
    return launch_status();
}
template int launch_bias_join<float>(const BiasJoin &, const float *, const float *, hipStream_t);
template int launch_bias_join<bf16_t>(const BiasJoin &, const float *, const float *, hipStream_t);
template int launch_bias_join<f16_t>(const BiasJoin &, const float *, const float *, hipStream_t);

template <typename P> int launch_join(const float *slices, int splits, int64_t count, int M, const float *f0, const float *f1, void *out,
                                      hipStream_t st)
{
    typedef typename ElementOf<P>::type E;
    const int64_t all = (count + 255) / 256;
    const int blocks = (int)(all < 16384 ? all : 16384);
    if (blocks == 0) return DS_OK;
    hipLaunchKernelGGL((join_kernel<P, E>), dim3(blocks), dim3(256), 0, st, slices, splits, count, M, (float *)nullptr, 1, 1, f0, f1,
                       (const float *)nullptr, (E *)out, (int64_t)M, blocks, BiasJoin{});
    return launch_status();
}
template int launch_join<Split>(const float *, int, int64_t, int, const float *, const float *, void *, hipStream_t);
template int launch_join<Bf16>(const float *, int, int64_t, int, const float *, const float *, void *, hipStream_t);
template int launch_join<F16>(const float *, int, int64_t, int, const float *, const float *, void *, hipStream_t);

// ---- plan --------------------------------------------------------------------------------------------------------

// Workspace of a piece's P, and of its repacked weights.  Larger pieces mean fewer slices of the hidden gradient to join (95 us
// a piece for 8192 tokens of 4096 features), smaller ones less memory; the products do not feel it.  The exponentials that a call
// for loss and gradients keeps of 16-bit types take twice as much besides.
constexpr size_t kPieceBytes = (size_t)1 << 30;

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
    size_t sorted, taught, target, temperature, twice;  // a teacher's words
    int again;            // the remainders of P are there: 1 for marked groups, 2 for all
};

template <typename P>
Plan plan_of(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int64_t T, int64_t D, int64_t V, int what, int words = 0)
{
    constexpr size_t NP = P::planes;
    Plan p{};
    p.Dp = (int)(NP > 1 ? (D + 31) / 32 * 32 : (D + 7) / 8 * 8);
    p.ldd = row_elements<P>(D);
    p.few = NP > 1 && !words && T > 0 && T <= few_tokens(V * D) && g_tune.vocab_tile == kTuneUnset;
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
    if (words) {
        p.sorted = take((size_t)T * words * 4), p.taught = take((size_t)T * words * 4);
        p.target = take((size_t)T * 4), p.temperature = take(4);
        if (NP == 1 && !P::half && what & kGrad && words > 1) p.again = T <= kTwiceAll || V <= kTwiceWords ? 2 : 1;
        if (p.again == 1) p.twice = take((size_t)((V + 255) / 256));
    }
    const size_t copies = p.again ? 2 : 1;
    if (p.pack_h) p.h = take(copies * T * p.ldd * 2);
    if (p.pack_w) p.w = take((size_t)p.piece * p.ldd * 2);
    if (what & kLoss) {
        const int64_t tiles = (p.piece + p.tile_words - 1) / p.tile_words;
        p.stats = take((size_t)(tiles * p.pieces) * T * 8);
        p.picked = take((size_t)T * (words ? words : 1) * 4);
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
        p.prob = take(copies * T * p.ldp * 2);
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
    Teacher teacher;   // K 0: none, target has the words
};

inline int check(const Call &c)
{
    if (c.T < 0 || c.D < 0 || c.V < 1 || !element_bytes(c.type)) return DS_EINVAL;
    if (c.T > 0 && (!c.target || (c.D > 0 && (!c.hidden || !c.weight || c.ldh < c.D || c.ldw < c.D)))) return DS_EINVAL;
    const int64_t most = 0x7fffffff - 512;
    if (c.T > most || c.V > most || c.D > 1000000 || c.ldh > 2000000 || c.ldw > 2000000) return DS_ETOOLARGE;
    return DS_OK;
}

inline void launch_teacher(const Teacher &t, hipStream_t st)
{
    hipLaunchKernelGGL(teacher_kernel, dim3((unsigned)t.T), dim3(ceil_div(t.K, 64) * 64), 0, st, t);
}

// The operands as the products take them: hidden states once, weights piece by piece.
template <typename P>
struct Operands {
    Operand h, w;
    int64_t w_at = -1;
    bool h_there = false;
    bool untaught = false;   // the teacher's words are still to be put in order

    int prepare(const Call &c, const Plan &p, bool counted_only, int64_t v0, int64_t n)
    {
        typedef typename ElementOf<P>::type E;
        const E *from = (const E *)c.weight + v0 * c.ldw;
        Pack ph{}, pw{};
        if (!h_there) {
            h = p.pack_h ? Operand{c.ws + p.h, p.ldd} : Operand{c.hidden, c.ldh};
            if (p.pack_h)
                ph = Pack{c.hidden, c.ldh, c.T, (int)c.D, p.Dp, (uint16_t *)(c.ws + p.h), p.ldd,
                          counted_only ? c.target : nullptr, c.wide, c.ignore, p.again ? c.T : 0};
            h_there = true;
        }
        if (w_at != v0) {
            w = p.pack_w ? Operand{c.ws + p.w, p.ldd} : Operand{from, c.ldw};
            if (p.pack_w) pw = Pack{from, c.ldw, n, (int)c.D, p.Dp, (uint16_t *)(c.ws + p.w), p.ldd, nullptr, 0, 0, 0};
            w_at = v0;
        }
        if (untaught) {
            untaught = false;
            const Teacher &t = c.teacher;
            const int first = pack_blocks<E>(ph), all = first + pack_blocks<E>(pw);
            if (all > 0 && t.K <= 256 && t.T <= kTaughtBeside) {
                hipLaunchKernelGGL((teacher_pack_kernel<E>), dim3((unsigned)t.T + all), dim3(256), 0, c.st, t, ph, pw, first);
                return launch_status();
            }
            launch_teacher(t, c.st);
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
    g.taught_ids = c.teacher.sorted, g.taught = c.teacher.taught, g.taught_words = c.teacher.K;
    g.warmth = c.teacher.K ? 1.f / c.teacher.temperature : 1.f;
    return g;
}

// Whether finish_kernel joins the rows' sums: each of its workgroups does it for its own rows, and one for all, which pays
// while there are few of both (64 tokens, 1000 words, float32: 3 us of a step) and of a teacher's words.
inline bool joined_later(const Call &c, const Plan &p, int tiles)
{
    return p.keep && p.pieces == 1 && c.T <= 128 && tiles <= 64 && c.teacher.K <= 64 && p.again != 1;
}

inline Marks marks_of(const Call &c, const Plan &p, const float *row_grad)
{
    return Marks{c.teacher.sorted, c.teacher.taught, c.teacher.target, row_grad, c.T, c.V, c.teacher.K, (uint8_t *)(c.ws + p.twice)};
}

// One product, of `kind`, by the kernels of the plan; fills in the tile counts.
template <typename P>
int product(const Plan &p, int kind, int tile, Args &g, int64_t T, hipStream_t st)
{
    if (g.taught_words && kind <= kLogitProb) {
        if constexpr (P::planes > 1)
            if (p.raw) return launch_taught_raw(kind, p.raw, g, st);
        return launch_taught<P>(kind, tile, g, st);
    }
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
               lse, rows, reduction, (Share *)(c.ws + p.shares), (uint32_t *)(c.ws + p.arrived), total, c.teacher.taught, c.teacher.K,
               c.teacher.K ? c.teacher.temperature : 1.f};
    const unsigned groups = (unsigned)((c.T + kRowsJoined - 1) / kRowsJoined);
    if (p.again == 1) hipLaunchKernelGGL(row_kernel<true>, dim3(groups + 1), dim3(1024), 0, c.st, *of, marks_of(c, p, nullptr));
    else if (!joined_later(c, p, tiles)) hipLaunchKernelGGL(row_kernel<false>, dim3(groups), dim3(1024), 0, c.st, *of, Marks{});
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
    // the temperature, where no row's share has it
    if (c.teacher.K && c.T > 0 && !r.share) r.share = c.teacher.factor;
    float *const slices = (float *)(c.ws + p.slices);
    const uint8_t *const twice = p.again == 1 ? (const uint8_t *)(c.ws + p.twice) : nullptr;
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
            bias_left = r.dbias && (bias_tiles > 1 || joined_later(c, p, of.tiles));
            float *const bias_part = bias_left ? (float *)(c.ws + p.bias) : nullptr;
            void *const bias_out = r.dbias && !bias_left ? (E *)r.dbias + v0 : nullptr;
            if (kept) {
                const int words = ceil_div((int)n, 32) * 32;
                const bool beside = P::planes == 1;
                const Finish f{c.ws + p.prob, p.ldp, (const float *)(c.ws + (beside ? p.kept : p.prob)), beside ? p.words : p.ldp / 2, words, p.tile_words, rows, v0, n, of.tiles - ceil_div((int)n, p.tile_words),
                               p.words, of, bias_part, bias_out, {r.grad, r.share}, c.teacher.sorted, twice, p.again ? c.T : 0};
                const unsigned along = ceil_div(words, 256), down = ceil_div((int)c.T, rows);
                if (joined_later(c, p, of.tiles) && c.teacher.K)
                    hipLaunchKernelGGL((finish_kernel<P, true, true>), dim3(along, down + 1), dim3(256), 0, c.st, f);
                else if (joined_later(c, p, of.tiles))
                    hipLaunchKernelGGL((finish_kernel<P, true>), dim3(along, down + 1), dim3(256), 0, c.st, f);
                else if (c.teacher.K)
                    hipLaunchKernelGGL((finish_kernel<P, false, true>), dim3(along, down), dim3(256), 0, c.st, f);
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
                g.twice = twice, g.again = p.again ? c.T : 0;
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
            x.K = which ? (int)c.T * (p.again == 2 ? 2 : 1) : (int)n;
            if (which) x.twice = twice, x.v0 = (int)v0;
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
int run(Call c, int what, const Outputs &out)
{
    const Plan p = plan_of<P>(c.hidden, c.ldh, c.weight, c.ldw, c.T, c.D, c.V, what, c.teacher.K);
    if (!c.ws || c.ws_bytes < p.bytes || (uintptr_t)c.ws % 256) return DS_EWORKSPACE;
    if (c.teacher.K) {
        Teacher &t = c.teacher;
        t.sorted = (int *)(c.ws + p.sorted), t.taught = (float *)(c.ws + p.taught);
        t.target = (int *)(c.ws + p.target), t.factor = (float *)(c.ws + p.temperature);
        // from here on tokens without a word are those that do not count
        c.target = t.target, c.wide = 0, c.ignore = -1;
    }
    Operands<P> o;
    if (c.teacher.K && c.T > 0) {
        if (what & kLoss) o.untaught = true;
        else launch_teacher(c.teacher, c.st);
        if (!(what & kLoss) && p.again == 1) hipLaunchKernelGGL(mark_kernel, dim3(1), dim3(1024), 0, c.st, marks_of(c, p, out.grads.row_grad));
    }
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

DS_EXPORT size_t ds_distill_workspace_bytes(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, int64_t T, int64_t D,
                                            int64_t V, int type, int words, int what)
{
    if (T < 0 || D < 0 || V < 1 || !element_bytes(type) || words < 1 || words > kMostTaught || what < kLoss || what > (kLoss | kGrad))
        return 0;
    if (type == DS_F32) return plan_of<Split>(hidden, ldh, weight, ldw, T, D, V, what, words).bytes;
    if (type == DS_BF16) return plan_of<Bf16>(hidden, ldh, weight, ldw, T, D, V, what, words).bytes;
    return plan_of<F16>(hidden, ldh, weight, ldw, T, D, V, what, words).bytes;
}

// `what` and where its results go, of a teacher's words.
static int run_taught(const Teacher &teacher, int id_bytes, Call c, int what, const Outputs &out)
{
    if (id_bytes != 4 && id_bytes != 8) return DS_EINVAL;
    if (teacher.K < 1 || teacher.K > kMostTaught || !element_bytes(teacher.type)) return DS_EINVAL;
    if (!(teacher.temperature >= 0x1p-20f && teacher.temperature <= 0x1p20f)) return DS_EINVAL;
    if (c.T > 0 && (!teacher.ids || !teacher.logits)) return DS_EINVAL;
    if (c.T > 0xffffffff / (ceil_div(teacher.K, 64) * 64)) return DS_ETOOLARGE;  // threads of teacher_kernel
    c.teacher = teacher;
    c.target = teacher.ids;
    return run(c, what, out);
}

DS_EXPORT int ds_distill_loss(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias, const void *ids,
                              int id_bytes, const void *logits, int logits_type, int words, float temperature, int64_t T, int64_t D,
                              int64_t V, int type, int reduction, float *rows, float *lse, float *total, void *workspace,
                              size_t workspace_bytes, ds_stream_t stream)
{
    if (reduction < 0 || reduction > DS_MEAN || (T > 0 && (!rows || !lse)) || (reduction && !total)) return DS_EINVAL;
    const Teacher teacher{ids, id_bytes == 8, logits, logits_type, words, T, V, temperature, nullptr, nullptr, nullptr, nullptr};
    return run_taught(teacher, id_bytes, Call{hidden, weight, bias, nullptr, ldh, ldw, T, D, V, -1, 0, type, (char *)workspace,
                                              workspace_bytes, (hipStream_t)stream, Teacher{}},
                      kLoss, Outputs{reduction, rows, lse, total, Grads{}});
}

DS_EXPORT int ds_distill_loss_grad(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias, const void *ids,
                                   int id_bytes, const void *logits, int logits_type, int words, float temperature, int64_t T,
                                   int64_t D, int64_t V, int type, const float *lse, const float *row_grad, const float *grad,
                                   const float *share, void *dhidden, void *dweight, void *dbias, void *workspace,
                                   size_t workspace_bytes, ds_stream_t stream)
{
    if ((row_grad && (grad || share)) || (T > 0 && !lse)) return DS_EINVAL;
    const Teacher teacher{ids, id_bytes == 8, logits, logits_type, words, T, V, temperature, nullptr, nullptr, nullptr, nullptr};
    return run_taught(teacher, id_bytes, Call{hidden, weight, bias, nullptr, ldh, ldw, T, D, V, -1, 0, type, (char *)workspace,
                                              workspace_bytes, (hipStream_t)stream, Teacher{}},
                      kGrad, Outputs{0, nullptr, nullptr, nullptr, Grads{lse, row_grad, grad, share, dhidden, dweight, dbias}});
}

DS_EXPORT int ds_distill_loss_step(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias, const void *ids,
                                   int id_bytes, const void *logits, int logits_type, int words, float temperature, int64_t T,
                                   int64_t D, int64_t V, int type, int reduction, float *rows, float *lse, float *total, void *dhidden,
                                   void *dweight, void *dbias, void *workspace, size_t workspace_bytes, ds_stream_t stream)
{
    if (reduction < 0 || reduction > DS_MEAN || (T > 0 && (!rows || !lse)) || (reduction && !total)) return DS_EINVAL;
    const Teacher teacher{ids, id_bytes == 8, logits, logits_type, words, T, V, temperature, nullptr, nullptr, nullptr, nullptr};
    return run_taught(teacher, id_bytes, Call{hidden, weight, bias, nullptr, ldh, ldw, T, D, V, -1, 0, type, (char *)workspace,
                                              workspace_bytes, (hipStream_t)stream, Teacher{}},
                      kLoss | kGrad, Outputs{reduction, rows, lse, total,
                                             Grads{lse, nullptr, nullptr, reduction ? total + 1 : nullptr, dhidden, dweight, dbias}});
}

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
                    workspace_bytes, (hipStream_t)stream, Teacher{}},
               kLoss, Outputs{reduction, rows, lse, total, Grads{}});
}

DS_EXPORT int ds_vocab_loss_grad(const void *hidden, int64_t ldh, const void *weight, int64_t ldw, const void *bias,
                                 const void *target, int target_bytes, int64_t ignore, int64_t T, int64_t D, int64_t V, int type,
                                 const float *lse, const float *row_grad, const float *grad, const float *share, void *dhidden,
                                 void *dweight, void *dbias, void *workspace, size_t workspace_bytes, ds_stream_t stream)
{
    if ((target_bytes != 4 && target_bytes != 8) || (row_grad && (grad || share)) || (T > 0 && !lse)) return DS_EINVAL;
    return run(Call{hidden, weight, bias, target, ldh, ldw, T, D, V, ignore, target_bytes == 8, type, (char *)workspace,
                    workspace_bytes, (hipStream_t)stream, Teacher{}},
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
                    workspace_bytes, (hipStream_t)stream, Teacher{}},
               kLoss | kGrad, Outputs{reduction, rows, lse, total,
                                      Grads{lse, nullptr, nullptr, reduction ? total + 1 : nullptr, dhidden, dweight, dbias}});
}
