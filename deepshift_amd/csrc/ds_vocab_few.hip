// The vocabulary's cross entropy for a few tokens of float32.
//
// Each weight takes part in a handful of products then, and reading it is what counts: once for the logits, once for the hidden
// states' gradient, and the weights' gradient is written once.  Splitting float32 weights into planes for the matrix
// instructions first moves 10 bytes for every 4 of them, so these kernels multiply them as they are, in vector registers, and
// are bound by memory up to some eight tokens, then by vector instructions.  The loss, and a step, in us:
//   1 token of 2707 features, 62215 words     129 (5.2 TB/s), 490     by planes 703, 1220
//   4 tokens of 2048, 50021 words             100, 282                373, 690
//   16 tokens                                 160, 374                375, 679
#include "ds_vocab.h"

namespace ds {
namespace vocab {

// Four neighbours at any address that a float may have; those from `left` on are zeros.
__device__ __forceinline__ f32x4 load4(const float *p, int left)
{
    f32x4 v{0.f, 0.f, 0.f, 0.f};
    if (left >= 4) {
        __builtin_memcpy(&v, p, 16);
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (e < left) v[e] = p[e];
    }
    return v;
}

// Element `v` of a row of P, from its planes.
__device__ __forceinline__ float prob_at(const uint16_t *row, int v)
{
    const bf16_t *p = (const bf16_t *)row + (v >> 5) * 96 + (v & 31);
    return to_float(p[0]) + (to_float(p[32]) + to_float(p[64]) * (1.f / 256)) * (1.f / 256);
}

// Logits of kFewWords words and up to TT tokens.  A wave has eight of the words, four at a time (eight at a time take more
// registers and no less time), its lanes share the features; every weight is loaded once, the next ones while these are
// multiplied.  The hidden states come from the caches.  What becomes of the logits is what product_tile does with them, in the
// same places.
template <int KIND, int TT>
__global__ __launch_bounds__(256) void few_logits_kernel(Args g)
{
    constexpr int R = 4, kMine = kFewWords / 4;  // words at a time, words of a wave
    __shared__ float logits[TT][kFewWords], sums[8][kFewWords];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, m0 = blockIdx.x * kFewWords;
    const float *const W = (const float *)g.a.at, *const H = (const float *)g.b.at;
    if (KIND != kProb && blockIdx.x == 0 && threadIdx.x == 0) *g.arrived = 0;
    // tokens that do not count may hold anything, and leave nothing in gradients
    bool counts[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) counts[t] = t < g.N && (KIND == kStats || target_at(g, t) != g.ignore);
#pragma unroll 1
    for (int r0 = 0; r0 < kMine; r0 += R) {
        const float *row[R];
#pragma unroll
        for (int r = 0; r < R; ++r) row[r] = W + (int64_t)min(m0 + wave * kMine + r0 + r, g.M - 1) * g.a.ld;
        float acc[R * TT];
#pragma unroll
        for (int i = 0; i < R * TT; ++i) acc[i] = 0.f;
        f32x4 next[R];
#pragma unroll
        for (int r = 0; r < R; ++r) next[r] = load4(row[r] + lane * 4, g.K - lane * 4);
        for (int d = lane * 4; d - lane * 4 < g.K; d += 256) {
            f32x4 w[R], h[TT];
#pragma unroll
            for (int r = 0; r < R; ++r) w[r] = next[r], next[r] = load4(row[r] + d + 256, g.K - d - 256);
#pragma unroll
            for (int t = 0; t < TT; ++t) h[t] = load4(H + (counts[t] ? t : 0) * g.b.ld + d, counts[t] ? g.K - d : 0);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int t = 0; t < TT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[r * TT + t] = fmaf(w[r][e], h[t][e], acc[r * TT + t]);
        }
        const int which = spread_sums<32, R * TT>(acc, lane);
        const int word = wave * kMine + r0 + which / TT, m = m0 + word;
        logits[which % TT][word] = m < g.M ? fmaf(acc[0], kLog2e, bias_at(g, g.v0 + m) * kLog2e) : -INFINITY;
    }
    __syncthreads();
    // half a wave has a token, a lane a word
    const int word = threadIdx.x % 32, m = m0 + word;
    float over_t = 0.f;
    for (int t = threadIdx.x / 32; t < g.N; t += 8) {
        const float x = logits[t][word];
        const int64_t y = target_at(g, t);
        const bool hot = y - g.v0 == m && m < g.M;
        uint16_t *const row = (uint16_t *)g.prob + t * g.ldp + m0 * 3;
        if (KIND == kProb) {
            const float lse = g.lse[t];
            const float scale = y < 0 || y >= g.V ? NAN : g.row_scale ? g.row_scale[t] : prob_factor_of(g.factor);
            const float p = y == g.ignore ? 0.f : (exp2f(x - lse) - (hot ? 1.f : 0.f)) * scale;
            over_t += p;
            bf16_t planes[3];
            split_planes<true>(p, planes);
            if (m < g.prob_words)
#pragma unroll
                for (int q = 0; q < 3; ++q) row[q * 32 + word] = planes[q].bits;
        } else {
            if (hot) g.picked[t] = x;
            float top = x;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
            const float e = exp2f(x - (top == -INFINITY ? 0.f : top));
            if (KIND == kKeep && m < g.prob_words) ((float *)row)[word] = e;
            float sum = e;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) sum += __shfl_xor(sum, o);
            if (word == 0) ((float2 *)g.stats)[(int64_t)blockIdx.x * g.N + t] = float2{top, sum};
        }
    }
    if (KIND != kProb || !g.bias_out) return;
    sums[threadIdx.x / 32][word] = over_t;
    __syncthreads();
    if (threadIdx.x < 32 && m < g.M) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += sums[i][word];
        ((float *)g.bias_out)[m] = s * factor_of(g.factor);
    }
}

// Up to 64 words' probabilities of all tokens, from a wave's lanes (a word each) to where all of them read them, token by token.
template <int TT>
struct Shared {
    float p[64][TT];

    __device__ __forceinline__ void put(const Operand &prob, int tokens, int v, bool real)
    {
        const int lane = threadIdx.x & 63;
        float mine[TT];
#pragma unroll
        for (int t = 0; t < TT; ++t)
            mine[t] = t < tokens && real ? prob_at((const uint16_t *)prob.at + t * prob.ld, v) : 0.f;
#pragma unroll
        for (int t = 0; t < TT; ++t) p[lane][t] = mine[t];
        __builtin_amdgcn_wave_barrier();
    }
};

// dh[t][d] = sum_v P[t][v] W[v][d]: a workgroup has 256 features and a stretch of words, each of its waves a quarter of them; a
// lane has four features of all tokens.  Probabilities come from LDS, one read for all lanes (from a lane's register, 16 tokens
// took 140 us where they take 99; four 75 and 69).  410 MB of weights at 6 TB/s.
template <int TT>
__global__ __launch_bounds__(256) void few_hidden_kernel(Args g)
{
    __shared__ union {
        Shared<TT> prob[4];
        f32x4 parts[4][TT][64];
    } lds;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = blockIdx.x * 256 + lane * 4;
    const int stretch = min(g.K - (int)blockIdx.y * g.k_split, g.k_split), quarter = (stretch + 3) / 4;
    const int from = blockIdx.y * g.k_split + wave * quarter, to = from + min(quarter, stretch - wave * quarter);
    const float *const W = (const float *)g.a.at;
    f32x4 acc[TT];
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int v0 = from; v0 < to; v0 += 64) {
        const int words = min(64, to - v0);
        __builtin_amdgcn_wave_barrier();
        lds.prob[wave].put(g.b, g.N, v0 + lane, lane < words);
        constexpr int kAhead = TT <= 4 ? 16 : 8;
#pragma unroll 1
        for (int j0 = 0; j0 < words; j0 += kAhead) {
            f32x4 w[kAhead];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) w[j] = load4(W + (int64_t)(v0 + j0 + j) * g.a.ld + d, j0 + j < words ? g.M - d : 0);
            // (words past the end are zeros, of weights and of probabilities)
#pragma unroll
            for (int j = 0; j < kAhead; ++j)
#pragma unroll
                for (int t = 0; t < TT; ++t) {
                    const float pj = lds.prob[wave].p[j0 + j][t];
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(pj, w[j][e], acc[t][e]);
                }
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TT; ++t) lds.parts[wave][t][lane] = acc[t];
    __syncthreads();
    const float *const flat = (const float *)lds.parts;
    for (int i = threadIdx.x; i < TT * 256; i += 256) {
        const int t = i / 256, col = blockIdx.x * 256 + i % 256;
        if (t >= g.N || col >= g.M) continue;
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s += flat[(w * TT + t) * 256 + i % 256];
        g.slice[((int64_t)blockIdx.y * g.n_store + t) * g.M + col] = s;
    }
}

// dW[v][d] = sum_t P[t][v] h[t][d]: a wave has up to 64 words (g.k_split) of 256 features, a lane four features of all tokens.
// Bound by memory: 410 MB in 67 us, 6.1 TB/s, for four tokens.
template <int TT>
__global__ __launch_bounds__(256) void few_weight_kernel(Args g)
{
    __shared__ Shared<TT> prob[4];
    const int across = (g.M + 255) / 256, down = blockIdx.x / across;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, d = (blockIdx.x - down * across) * 256 + lane * 4;
    const int v0 = (down * 4 + wave) * g.k_split, words = min(g.k_split, g.n_store - v0);
    if (words <= 0) return;
    f32x4 h[TT];
    const float factor = factor_of(g.factor);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
        const bool counts = t < g.K && target_at(g, t) != g.ignore;
        h[t] = load4((const float *)g.a.at + (counts ? t : 0) * g.a.ld + d, counts ? g.M - d : 0);
    }
    prob[wave].put(g.b, g.K, v0 + lane, lane < words);
    const int left = g.M - d;
    float *out = (float *)g.out + v0 * g.ldo + d;
#pragma unroll 4
    for (int j = 0; j < words; ++j, out += g.ldo) {
        f32x4 o{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TT; ++t) {
            const float pj = prob[wave].p[j][t];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(pj, h[t][e], o[e]);
        }
        o *= factor;
        if (left >= 4) {
            __builtin_memcpy(out, &o, 16);
        } else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
                if (e < left) out[e] = o[e];
        }
    }
}

template <int TT>
int launch_few_tokens(int kind, Args &g, hipStream_t st)
{
    const dim3 threads(256);
    if (kind == kHidden) {
        hipLaunchKernelGGL((few_hidden_kernel<TT>), dim3(ceil_div(g.M, 256), g.splits), threads, 0, st, g);
    } else if (kind == kWeight) {
        // 64 words a wave, down to four where CUs would be without work
        const int64_t across = ceil_div(g.M, 256), all = across * g.n_store / (16 * device_cus());
        g.k_split = (int)(all < 4 ? 4 : all < 64 ? all : 64);
        const int64_t blocks = across * ceil_div(g.n_store, 4 * g.k_split);
        if (blocks > 0x7fffffff) return DS_ETOOLARGE;
        hipLaunchKernelGGL((few_weight_kernel<TT>), dim3((unsigned)blocks), threads, 0, st, g);
    } else {
        g.tiles_m = ceil_div(g.M, kFewWords), g.tiles_n = 1;
        if (kind == kLogitStats)
            hipLaunchKernelGGL((few_logits_kernel<kStats, TT>), dim3(g.tiles_m), threads, 0, st, g);
        else if (kind == kLogitKeep)
            hipLaunchKernelGGL((few_logits_kernel<kKeep, TT>), dim3(g.tiles_m), threads, 0, st, g);
        else
            hipLaunchKernelGGL((few_logits_kernel<kProb, TT>), dim3(g.tiles_m), threads, 0, st, g);
    }
    return launch_status();
}

int launch_few(int kind, int tokens, Args &g, hipStream_t st)
{
    if (tokens == 1) return launch_few_tokens<1>(kind, g, st);
    if (tokens == 2) return launch_few_tokens<2>(kind, g, st);
    if (tokens <= 4) return launch_few_tokens<4>(kind, g, st);
    if (tokens <= 8) return launch_few_tokens<8>(kind, g, st);
    return launch_few_tokens<16>(kind, g, st);
}

}  // namespace vocab
}  // namespace ds
