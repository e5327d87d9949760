// Gated linear recurrence along a sequence, channel by channel, and its gradients.
//
//   a_t = 1 / (1 + exp(-g_t))        h_t = a_t h_{t-1} + (1 - a_t) x_t
//   l_t = dh_t + a_{t+1} l_{t+1}     dx_t = (1 - a_t) l_t     dg_t = l_t (h_{t-1} - x_t) a_t (1 - a_t)     dh_0 = a_1 l_1
//
// A stretch of tokens takes a state h to A h + H, with A the product of its a and H what it leaves of nothing, and two
// stretches in a row join to one.  A workgroup has 64 V channels of one sequence and kSteps tokens a wave: each wave finds
// A and H of its own tokens from registers, the waves' are exchanged through LDS, and each goes over its tokens once more with
// the state that it then knows.  So all is read once and the next tokens are on their way meanwhile; nothing waits for
// another workgroup.  Going back, m_t = a_t l_t is found the same way from the end, m_t = a_t (dh_t + m_{t+1}), along with the
// states, which are formed again from those that the forward pass leaves of every workgroup's first tokens.
// States, products and sums are float32; results are rounded once.
//
// Bound by memory: 8 sequences of 8192 tokens and 4096 channels, bfloat16, forward in 350 to 410 us (cards differ), 3.9 to 4.6 TB/s,
// backward in 570 to 654, 4.1 to 4.7 TB/s, where a copy of 2 GiB runs at 4.9; 2048 channels of float32 in 336 and 530.  Sequences that
// end early take hardly less, since the longest one's workgroups are waited for (half of the tokens: 352 and 568, float32 312 and
// 458, on one card).  What that took: loads that are as many in every turn and stores that leave through a
// descriptor, so that nothing but the loads of a turn is waited for (with conditions around both, and 16 waves a workgroup,
// whose registers spilled, the two took 2.9 ms together).
//
// Few channels and many tokens leave CUs without work: there the sequence is cut into segments, a first launch finds each
// one's A and H (and m), and the second begins where those before it end.
#include "ds_train.h"
#include <algorithm>

namespace ds {
namespace recur {

constexpr int kSteps = 8;  // tokens of a wave at a time

struct Sequence {
    const void *at;
    int64_t batch, token;  // elements from one to the next
};

struct Args {
    Sequence x, gate, grad;
    const float *state, *grad_last;  // [B][D] or NULL
    const void *lengths;             // [B] or NULL
    int wide;
    void *out, *dx, *dgate;          // [B][T][D]
    float *last, *dstate;            // [B][D]
    float *kept;                     // [B][blocks][D]: states before every block of tokens
    float2 *ends;                    // [segments][B][D]: what a segment makes of a state, and of nothing
    int64_t T, blocks;
    int B, D, groups, segments;
    int64_t segment;                 // tokens of one, whole blocks
};

// Both sides of a gate, each to a few units in its last place: exp of -|g| with the part of |g| log2 e that its rounding leaves.
__device__ __forceinline__ void sides(float g, float &a, float &away)
{
    constexpr float kHi = 1.44269502162933349609375f, kLo = 1.92596299112661746887e-8f, kLn2 = 0.6931471805599453f;
    const float x = -fabsf(g), y = x * kHi, rest = fmaf(x, kLo, fmaf(x, kHi, -y));
    float e = __builtin_amdgcn_exp2f(y);
    e = y > -126.f ? fmaf(e, rest * kLn2, e) : 0.f;  // (also where y is infinite and the rest no number)
    const float near = __builtin_amdgcn_rcpf(1.f + e), far = e * near;
    a = g >= 0.f ? near : far, away = g >= 0.f ? far : near;
    if (g != g) a = away = g;
}

typedef __amdgpu_buffer_rsrc_t Buffer;

// What lies from `at` on, within 32-bit offsets; an offset of kNowhere stores nothing.
constexpr int kNowhere = (int)0x80000000u;
__device__ __forceinline__ Buffer buffer_of(void *at) { return __builtin_amdgcn_make_buffer_rsrc(at, 0, 0x7fffffff, 0x00020000); }

template <typename E, int V>
__device__ __forceinline__ void put(Buffer to, int offset, const float (&v)[V])
{
    Vec<E, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = from_float<E>(v[e]);
    if constexpr (sizeof(o) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(uint32_t, o), to, offset, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(uint16_t, o), to, offset, 0, 0);
}

// Until every wave's LDS is written; loads and stores of memory stay on their way.
__device__ __forceinline__ void meet()
{
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Which channels of which sequence this workgroup has, and which of its tokens.
struct Place {
    int64_t b, from, to, end;  // the segment's tokens; those from `end` on hold nothing
    int segment, c;
    bool real;                 // lanes past the last channel look at the first, and store nothing

    __device__ Place(const Args &g, int V)
    {
        const int id = blockIdx.x, group = id % g.groups, rest = id / g.groups;
        segment = rest % g.segments, b = rest / g.segments;
        c = (group * 64 + (threadIdx.x & 63)) * V;
        real = c < g.D;
        if (!real) c = 0;
        from = segment * g.segment, to = min(g.T, from + g.segment);
        int64_t length = g.T;
        if (g.lengths) {
            length = g.wide ? ((const int64_t *)g.lengths)[b] : (int64_t)((const int32_t *)g.lengths)[b];
            length = length < 0 ? 0 : min(length, g.T);
        }
        end = max(from, min(length, to));
    }
    // how many of a wave's tokens from t on there are, and hold something
    __device__ __forceinline__ int tokens(int64_t t) const { return (int)max((int64_t)0, min(to - t, (int64_t)kSteps)); }
    __device__ __forceinline__ int full(int64_t t) const { return (int)max((int64_t)0, min(end - t, (int64_t)kSteps)); }
};

// A wave's next tokens; instead of those that hold nothing the last one that does is loaded again, for nobody to look at.  So
// there are always as many loads on their way, and what waits for one block's does not wait for stores behind them.
template <typename E, int V>
__device__ __forceinline__ void load(Vec<E, V> (&v)[kSteps], const Sequence &s, const Place &p, int64_t t)
{
    const E *row = (const E *)s.at + p.b * s.batch + t * s.token;
    const int last = p.full(t) - 1;
    if (last < 0) row = (const E *)s.at + p.b * s.batch + (p.end - 1) * s.token;
#pragma unroll
    for (int r = 0; r < kSteps; ++r) v[r] = *(const Vec<E, V> *)(row + (r <= last ? r : last < 0 ? 0 : last) * s.token + (uint32_t)p.c);
}

template <int V>
__device__ __forceinline__ void state_at(const float *s, int64_t i, float (&h)[V])
{
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = s ? s[i + e] : 0.f;
}

// ENDS: finds only what a segment makes of a state.
template <typename E, int V, int W, bool ENDS>
__global__ __launch_bounds__(W * 64) void forward_kernel(Args g)
{
    constexpr int kBlock = W * kSteps;
    __shared__ float2 ends[2][W][V][64];
    const Place p(g, V);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t state = p.b * g.D + p.c;
    float carry[V], product[V];
#pragma unroll
    for (int e = 0; e < V; ++e) carry[e] = 0.f, product[e] = 1.f;
    if (!ENDS) {
        state_at<V>(g.state, state, carry);
        for (int i = 0; i < p.segment; ++i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 s = g.ends[(int64_t)i * g.B * g.D + state + e];
                carry[e] = fmaf(s.x, carry[e], s.y);
            }
    }
    Vec<E, V> x[kSteps], gate[kSteps];
    auto next = [&](int64_t t0) {
        if (p.end == p.from) return;
        load<E, V>(x, g.x, p, t0 + wave * kSteps);
        load<E, V>(gate, g.gate, p, t0 + wave * kSteps);
    };
    next(p.from);
    int turn = 0;
    for (int64_t t0 = p.from; t0 < p.to; t0 += kBlock, turn ^= 1) {
        const int64_t mine = t0 + wave * kSteps;
        const int full = p.full(mine), tokens = p.tokens(mine);
        float a[kSteps][V], b[kSteps][V], A[V], H[V];
#pragma unroll
        for (int r = 0; r < kSteps; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float away;
                sides(to_float(gate[r].v[e]), a[r][e], away), b[r][e] = away * to_float(x[r].v[e]);
            }
        if (full < kSteps)
#pragma unroll
            for (int r = 0; r < kSteps; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) a[r][e] = r < full ? a[r][e] : 1.f, b[r][e] = r < full ? b[r][e] : 0.f;
        next(t0 + kBlock);
        if (W > 1 || ENDS)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                A[e] = a[0][e], H[e] = b[0][e];
#pragma unroll
                for (int r = 1; r < kSteps; ++r) H[e] = fmaf(a[r][e], H[e], b[r][e]), A[e] *= a[r][e];
            }
        float h[V];
        if (!ENDS && g.kept) {
            const Buffer kept = buffer_of(g.kept + (p.b * g.blocks + t0 / kBlock) * g.D);
#pragma unroll
            for (int e = 0; e < V; ++e) put<float, 1>(kept, wave == 0 && p.real ? (p.c + e) * 4 : kNowhere, {carry[e]});
        }
        if constexpr (W > 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) ends[turn][wave][e][lane] = float2{A[e], H[e]};
            meet();
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float2 s = ends[turn][w][e][lane];
                    h[e] = w == 0 || w == wave ? carry[e] : h[e];
                    carry[e] = fmaf(s.x, carry[e], s.y);
                    if (ENDS) product[e] *= s.x;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = carry[e];
                if (ENDS) carry[e] = fmaf(A[e], carry[e], H[e]), product[e] *= A[e];
            }
        }
        if (ENDS) continue;
        const Buffer out = buffer_of((E *)g.out + (p.b * g.T + mine) * g.D);
#pragma unroll
        for (int r = 0; r < kSteps; ++r) {
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = fmaf(a[r][e], h[e], b[r][e]);
                o[e] = r < full ? h[e] : 0.f;
            }
            put<E, V>(out, r < tokens && p.real ? (int)((r * g.D + p.c) * sizeof(E)) : kNowhere, o);
        }
        if (W == 1)
#pragma unroll
            for (int e = 0; e < V; ++e) carry[e] = h[e];
    }
    if (wave != 0 || !p.real) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (ENDS) g.ends[(int64_t)p.segment * g.B * g.D + state + e] = float2{product[e], carry[e]};
        else if (p.segment == g.segments - 1) g.last[state + e] = carry[e];
    }
}

// ENDS: finds only what a segment makes of a gradient that comes from behind it.
template <typename E, int V, int W, bool ENDS>
__global__ __launch_bounds__(W * 64) void backward_kernel(Args g)
{
    constexpr int kBlock = W * kSteps;
    __shared__ float2 ends[2][W][V][64];
    __shared__ float backs[2][W][V][64];
    const Place p(g, V);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t state = p.b * g.D + p.c;
    float carry[V], product[V];
#pragma unroll
    for (int e = 0; e < V; ++e) carry[e] = 0.f, product[e] = 1.f;
    if (!ENDS) {
        state_at<V>(g.grad_last, state, carry);
        for (int i = g.segments - 1; i > p.segment; --i)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float2 s = g.ends[(int64_t)i * g.B * g.D + state + e];
                carry[e] = fmaf(s.x, carry[e], s.y);
            }
    }
    Vec<E, V> x[kSteps], gate[kSteps], grad[kSteps];
    float entry[V];
    auto next = [&](int64_t t0) {
        if (t0 < p.from) t0 = p.from;
        if (!ENDS) state_at<V>(g.kept, (p.b * g.blocks + t0 / kBlock) * g.D + p.c, entry);
        if (p.end == p.from) return;
        const int64_t t = t0 + wave * kSteps;
        load<E, V>(gate, g.gate, p, t);
        if (g.grad.at) load<E, V>(grad, g.grad, p, t);
        if (!ENDS) load<E, V>(x, g.x, p, t);
    };
    const int64_t first = p.to > p.from ? p.from + (p.to - p.from - 1) / kBlock * kBlock : p.from - kBlock;
    if (p.to > p.from) next(first);
    int turn = 0;
    for (int64_t t0 = first; t0 >= p.from; t0 -= kBlock, turn ^= 1) {
        const int64_t mine = t0 + wave * kSteps;
        const int full = p.full(mine), tokens = p.tokens(mine);
        float a[kSteps][V], away[kSteps][V], v[kSteps][V], dh[kSteps][V], A[V], H[V], M[V], h[V], m[V];
#pragma unroll
        for (int r = 0; r < kSteps; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sides(to_float(gate[r].v[e]), a[r][e], away[r][e]);
                v[r][e] = ENDS ? 0.f : to_float(x[r].v[e]);
                dh[r][e] = g.grad.at ? to_float(grad[r].v[e]) : 0.f;
            }
        if (full < kSteps)
#pragma unroll
            for (int r = 0; r < kSteps; ++r)
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    a[r][e] = r < full ? a[r][e] : 1.f, away[r][e] = r < full ? away[r][e] : 0.f;
                    v[r][e] = r < full ? v[r][e] : 0.f, dh[r][e] = r < full ? dh[r][e] : 0.f;
                }
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = ENDS ? 0.f : entry[e];
        next(t0 - kBlock);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            A[e] = 1.f, H[e] = 0.f, M[e] = 0.f;
#pragma unroll
            for (int r = 0; r < kSteps; ++r) {
                A[e] *= a[r][e];
                if (!ENDS) H[e] = fmaf(a[r][e], H[e], away[r][e] * v[r][e]);
            }
#pragma unroll
            for (int r = kSteps - 1; r >= 0; --r) M[e] = a[r][e] * (dh[r][e] + M[e]);
        }
        if constexpr (W > 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) ends[turn][wave][e][lane] = float2{A[e], H[e]}, backs[turn][wave][e][lane] = M[e];
            meet();
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float2 s[W];
#pragma unroll
                for (int w = 0; w < W; ++w) s[w] = ends[turn][w][e][lane];
                if (!ENDS)
#pragma unroll
                    for (int w = 0; w < W - 1; ++w) h[e] = w < wave ? fmaf(s[w].x, h[e], s[w].y) : h[e];
#pragma unroll
                for (int w = W - 1; w >= 0; --w) {
                    m[e] = w == W - 1 || w == wave ? carry[e] : m[e];
                    carry[e] = fmaf(s[w].x, carry[e], backs[turn][w][e][lane]);
                    if (ENDS) product[e] *= s[w].x;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                m[e] = carry[e];
                carry[e] = fmaf(A[e], carry[e], M[e]);
                if (ENDS) product[e] *= A[e];
            }
        }
        if (ENDS) continue;
        float before[kSteps][V];
#pragma unroll
        for (int r = 0; r < kSteps; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                before[r][e] = h[e] - v[r][e];
                h[e] = fmaf(a[r][e], h[e], away[r][e] * v[r][e]);
            }
        const Buffer to_x = buffer_of((E *)g.dx + (p.b * g.T + mine) * g.D), to_gate = buffer_of((E *)g.dgate + (p.b * g.T + mine) * g.D);
#pragma unroll
        for (int r = kSteps - 1; r >= 0; --r) {
            float dx[V], dg[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float l = dh[r][e] + m[e];
                dx[e] = r < full ? away[r][e] * l : 0.f;
                dg[e] = r < full ? dx[e] * a[r][e] * before[r][e] : 0.f;
                m[e] = a[r][e] * l;
            }
            const int to = r < tokens && p.real ? (int)((r * g.D + p.c) * sizeof(E)) : kNowhere;
            put<E, V>(to_x, g.dx ? to : kNowhere, dx);
            put<E, V>(to_gate, g.dgate ? to : kNowhere, dg);
        }
    }
    if (wave != 0 || !p.real) return;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        if (ENDS) g.ends[(int64_t)p.segment * g.B * g.D + state + e] = float2{product[e], carry[e]};
        else if (p.segment == 0 && g.dstate) g.dstate[state + e] = carry[e];
    }
}

// How the work is cut: channels of a lane, waves of a workgroup, segments of a sequence.
struct Plan {
    int V, W, groups, segments;
    int64_t block, blocks, segment;
    size_t bytes;
};

// Waves of a workgroup by the number of tokens alone, so that both passes cut a sequence into the same blocks.
inline int waves(int64_t T) { return T <= kSteps ? 1 : T <= 4 * kSteps ? 4 : 8; }

inline Plan plan_of(int64_t B, int64_t T, int64_t D, int type, bool pairs)
{
    Plan p{};
    const int cus = device_cus();
    p.W = waves(T);
    p.block = p.W * kSteps, p.blocks = (T + p.block - 1) / p.block;
    auto workgroups = [&](int V) { return B * ((D + 64 * V - 1) / (64 * V)); };
    // Two channels a lane where that leaves every CU a workgroup, or enough tokens to cut for two of them; segments where half
    // of the CUs would have none, for two workgroups a CU.  Measured, us forward and backward, bfloat16:
    //                            one channel                two channels
    //   8 x 8192 x 4096          456, 665                   410, 654        (in two segments 561, 810)
    //   4 x 4096 x 4096          130, 199                   161, 271        (two channels in four segments 140, 224)
    //   2 x 4096 x 4096          110, 184  (4: 89, 123)     153, 257        (4: 82, 120, 8: 67, 112, 16: 70, 117)
    //   1 x 65536 x 2048        1856, 2662 (16: 342, 448)  2404, 3925       (16: 329, 439, 32: 294, 429, 64: 292, 462)
    //   1 x 1024 x 1024           30, -    (8: 11)           41, -          (8: 12)
    //   3 x 4096 x 4096          132, 191  (4: 117, 168, 8: 114, 165, 16: 121, 178), where one channel a lane leaves a quarter of
    // the CUs without work, and the rule cuts nothing.
    const bool two = workgroups(2) >= cus || (2 * workgroups(1) <= cus && workgroups(2) * (p.blocks / 2) >= 2 * cus);
    p.V = type != DS_F32 && pairs && two ? 2 : 1;
    p.groups = (int)((D + 64 * p.V - 1) / (64 * p.V));
    const int64_t all = std::max<int64_t>(1, workgroups(p.V));
    int64_t segments = 2 * all <= cus ? std::min<int64_t>(2 * cus / all, p.blocks / 2) : 1;
    if (g_tune.recur_segments != kTuneUnset) segments = std::min<int64_t>(g_tune.recur_segments, p.blocks);
    if (segments < 1) segments = 1;
    const int64_t each = std::max<int64_t>(1, (p.blocks + segments - 1) / segments);
    p.segment = each * p.block;
    p.segments = (int)std::max<int64_t>(1, (p.blocks + each - 1) / each);
    p.bytes = p.segments > 1 ? (size_t)p.segments * B * D * sizeof(float2) : 0;
    return p;
}

template <typename E, int V, int W>
int launch(const Args &g, bool backward, int64_t grid, hipStream_t st)
{
    const dim3 blocks((unsigned)grid), threads(W * 64);
    if (backward) {
        if (g.segments > 1) hipLaunchKernelGGL((backward_kernel<E, V, W, true>), blocks, threads, 0, st, g);
        hipLaunchKernelGGL((backward_kernel<E, V, W, false>), blocks, threads, 0, st, g);
    } else {
        if (g.segments > 1) hipLaunchKernelGGL((forward_kernel<E, V, W, true>), blocks, threads, 0, st, g);
        hipLaunchKernelGGL((forward_kernel<E, V, W, false>), blocks, threads, 0, st, g);
    }
    return launch_status();
}
template <typename E, int V>
int launch(const Args &g, int W, bool backward, int64_t grid, hipStream_t st)
{
    if (W == 1) return launch<E, V, 1>(g, backward, grid, st);
    if (W == 4) return launch<E, V, 4>(g, backward, grid, st);
    return launch<E, V, 8>(g, backward, grid, st);
}

inline bool in_pairs(const Sequence &s) { return (uintptr_t)s.at % 4 == 0 && s.batch % 2 == 0 && s.token % 2 == 0; }

int check(int64_t B, int64_t T, int64_t D, int type)
{
    if (B < 0 || T < 0 || D < 0 || !element_bytes(type)) return DS_EINVAL;
    const int64_t most = 0x7fffffff;
    if (D > (1 << 25) || B > most || (D > 0 && B > most / ((D + 63) / 64))) return DS_ETOOLARGE;
    if (T > ((int64_t)1 << 40) || (D > 0 && B > 0 && T > ((int64_t)1 << 60) / (B * D))) return DS_ETOOLARGE;
    return DS_OK;
}

int run(Args g, int type, bool pairs, bool backward, void *ws, size_t ws_bytes, hipStream_t st)
{
    const Plan p = plan_of(g.B, g.T, g.D, type, pairs && g.D % 2 == 0);
    if (p.segments > 1 && (!ws || ws_bytes < p.bytes || (uintptr_t)ws % 256)) return DS_EWORKSPACE;
    g.ends = (float2 *)ws;
    g.blocks = p.blocks, g.groups = p.groups, g.segments = p.segments, g.segment = p.segment;
    const int64_t grid = (int64_t)g.B * p.groups * p.segments;
    if (grid > 0x7fffffff) return DS_ETOOLARGE;
    if (type == DS_F32) return launch<float, 1>(g, p.W, backward, grid, st);
    if (type == DS_BF16) return p.V == 2 ? launch<bf16_t, 2>(g, p.W, backward, grid, st) : launch<bf16_t, 1>(g, p.W, backward, grid, st);
    return p.V == 2 ? launch<f16_t, 2>(g, p.W, backward, grid, st) : launch<f16_t, 1>(g, p.W, backward, grid, st);
}

}  // namespace recur
}  // namespace ds

using namespace ds;
using namespace ds::recur;

DS_EXPORT int64_t ds_recur_blocks(int64_t T)
{
    const int64_t block = recur::waves(T) * kSteps;
    return T < 1 ? 0 : (T + block - 1) / block;
}

DS_EXPORT size_t ds_recur_workspace_bytes(int64_t B, int64_t T, int64_t D, int type)
{
    if (check(B, T, D, type) != DS_OK) return 0;
    // whatever the operands' alignment lets the lanes have
    return std::max(plan_of(B, T, D, type, false).bytes, plan_of(B, T, D, type, D % 2 == 0).bytes);
}

DS_EXPORT int ds_recur_forward(const void *x, int64_t x_batch, int64_t x_token, const void *gate, int64_t gate_batch,
                               int64_t gate_token, const float *state, const void *lengths, int length_bytes, void *out, float *last,
                               float *kept, int64_t B, int64_t T, int64_t D, int type, void *workspace, size_t workspace_bytes,
                               ds_stream_t stream)
{
    const int s = check(B, T, D, type);
    if (s != DS_OK) return s;
    if (lengths && length_bytes != 4 && length_bytes != 8) return DS_EINVAL;
    if (B == 0 || D == 0) return DS_OK;
    if (!last || (T > 0 && (!x || !gate || !out))) return DS_EINVAL;
    Args g{};
    g.x = Sequence{x, x_batch, x_token}, g.gate = Sequence{gate, gate_batch, gate_token};
    g.state = state, g.lengths = lengths, g.wide = length_bytes == 8;
    g.out = out, g.last = last, g.kept = kept;
    g.B = (int)B, g.T = T, g.D = (int)D;
    return run(g, type, in_pairs(g.x) && in_pairs(g.gate) && (uintptr_t)out % 4 == 0, false, workspace, workspace_bytes,
               (hipStream_t)stream);
}

DS_EXPORT int ds_recur_backward(const void *x, int64_t x_batch, int64_t x_token, const void *gate, int64_t gate_batch,
                                int64_t gate_token, const void *grad, int64_t grad_batch, int64_t grad_token, const float *grad_last,
                                const void *lengths, int length_bytes, const float *kept, void *dx, void *dgate, float *dstate,
                                int64_t B, int64_t T, int64_t D, int type, void *workspace, size_t workspace_bytes,
                                ds_stream_t stream)
{
    const int s = check(B, T, D, type);
    if (s != DS_OK) return s;
    if (lengths && length_bytes != 4 && length_bytes != 8) return DS_EINVAL;
    if (B == 0 || D == 0) return DS_OK;
    if (T > 0 && (!x || !gate || !kept)) return DS_EINVAL;
    Args g{};
    g.x = Sequence{x, x_batch, x_token}, g.gate = Sequence{gate, gate_batch, gate_token};
    g.grad = Sequence{grad, grad_batch, grad_token};
    g.grad_last = grad_last, g.lengths = lengths, g.wide = length_bytes == 8;
    g.kept = const_cast<float *>(kept), g.dx = dx, g.dgate = dgate, g.dstate = dstate;
    g.B = (int)B, g.T = T, g.D = (int)D;
    const bool pairs = in_pairs(g.x) && in_pairs(g.gate) && in_pairs(g.grad) && ((uintptr_t)dx | (uintptr_t)dgate) % 4 == 0;
    return run(g, type, pairs, true, workspace, workspace_bytes, (hipStream_t)stream);
}
