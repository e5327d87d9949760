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

template <typename E, int V>
__device__ __forceinline__ Vec<E, V> at(const Sequence &s, int64_t b, int64_t t, int c)
{
    return *(const Vec<E, V> *)((const E *)s.at + b * s.batch + t * s.token + c);
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
        end = min(length, to);
    }
};

template <typename E, int V>
__device__ __forceinline__ void put(void *base, const Args &g, const Place &p, int64_t t, const float (&v)[V])
{
    Vec<E, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = from_float<E>(v[e]);
    if (p.real) store_streaming((Vec<E, V> *)((E *)base + (p.b * g.T + t) * g.D + p.c), o);
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
    auto load = [&](int64_t t0) {
#pragma unroll
        for (int r = 0; r < kSteps; ++r) {
            const int64_t t = t0 + wave * kSteps + r;
            if (t < p.end) x[r] = at<E, V>(g.x, p.b, t, p.c), gate[r] = at<E, V>(g.gate, p.b, t, p.c);
        }
    };
    load(p.from);
    int turn = 0;
    for (int64_t t0 = p.from; t0 < p.to; t0 += kBlock, turn ^= 1) {
        float a[kSteps][V], b[kSteps][V], A[V], H[V];
#pragma unroll
        for (int e = 0; e < V; ++e) A[e] = 1.f, H[e] = 0.f;
#pragma unroll
        for (int r = 0; r < kSteps; ++r) {
            const bool there = t0 + wave * kSteps + r < p.end;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float away = 0.f;
                a[r][e] = 1.f, b[r][e] = 0.f;
                if (there) sides(to_float(gate[r].v[e]), a[r][e], away), b[r][e] = away * to_float(x[r].v[e]);
                if (W > 1 || ENDS) H[e] = fmaf(a[r][e], H[e], b[r][e]), A[e] *= a[r][e];
            }
        }
        load(t0 + kBlock);
        float h[V];
        if (!ENDS && g.kept && wave == 0 && p.real)
#pragma unroll
            for (int e = 0; e < V; ++e) g.kept[(p.b * g.blocks + t0 / kBlock) * g.D + p.c + e] = carry[e];
        if constexpr (W > 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) ends[turn][wave][e][lane] = float2{A[e], H[e]};
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e) {
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    const float2 s = ends[turn][w][e][lane];
                    if (w == wave) h[e] = carry[e];
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
#pragma unroll
        for (int r = 0; r < kSteps; ++r) {
            const int64_t t = t0 + wave * kSteps + r;
            if (t >= p.to) break;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = fmaf(a[r][e], h[e], b[r][e]);
                o[e] = t < p.end ? h[e] : 0.f;
            }
            put<E, V>(g.out, g, p, t, o);
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
    float entry[V], next_entry[V];
    auto load = [&](int64_t t0) {
        if (t0 < p.from) return;
#pragma unroll
        for (int r = 0; r < kSteps; ++r) {
            const int64_t t = t0 + wave * kSteps + r;
            if (t >= p.end) continue;
            if (!ENDS) x[r] = at<E, V>(g.x, p.b, t, p.c);
            gate[r] = at<E, V>(g.gate, p.b, t, p.c);
            if (g.grad.at) grad[r] = at<E, V>(g.grad, p.b, t, p.c);
        }
        if (!ENDS) state_at<V>(g.kept, (p.b * g.blocks + t0 / kBlock) * g.D + p.c, next_entry);
    };
    const int64_t first = p.to > p.from ? p.from + (p.to - p.from - 1) / kBlock * kBlock : p.from - kBlock;
    load(first);
    int turn = 0;
    for (int64_t t0 = first; t0 >= p.from; t0 -= kBlock, turn ^= 1) {
        float a[kSteps][V], away[kSteps][V], v[kSteps][V], dh[kSteps][V], A[V], H[V], M[V];
#pragma unroll
        for (int e = 0; e < V; ++e) A[e] = 1.f, H[e] = 0.f, M[e] = 0.f, entry[e] = next_entry[e];
#pragma unroll
        for (int r = 0; r < kSteps; ++r) {
            const bool there = t0 + wave * kSteps + r < p.end;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                a[r][e] = 1.f, away[r][e] = 0.f, v[r][e] = 0.f, dh[r][e] = 0.f;
                if (there) {
                    sides(to_float(gate[r].v[e]), a[r][e], away[r][e]);
                    if (!ENDS) v[r][e] = to_float(x[r].v[e]);
                    if (g.grad.at) dh[r][e] = to_float(grad[r].v[e]);
                }
                A[e] *= a[r][e];
                if (!ENDS) H[e] = fmaf(a[r][e], H[e], away[r][e] * v[r][e]);
            }
        }
#pragma unroll
        for (int r = kSteps - 1; r >= 0; --r)
#pragma unroll
            for (int e = 0; e < V; ++e) M[e] = a[r][e] * (dh[r][e] + M[e]);
        load(t0 - kBlock);
        float h[V], m[V];
        if constexpr (W > 1) {
#pragma unroll
            for (int e = 0; e < V; ++e) ends[turn][wave][e][lane] = float2{A[e], H[e]}, backs[turn][wave][e][lane] = M[e];
            __syncthreads();
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if (!ENDS) {
                    h[e] = entry[e];
#pragma unroll
                    for (int w = 0; w < W - 1; ++w) {
                        const float2 s = ends[turn][w][e][lane];
                        if (w < wave) h[e] = fmaf(s.x, h[e], s.y);
                    }
                }
#pragma unroll
                for (int w = W - 1; w >= 0; --w) {
                    const float s = ends[turn][w][e][lane].x;
                    if (w == wave) m[e] = carry[e];
                    carry[e] = fmaf(s, carry[e], backs[turn][w][e][lane]);
                    if (ENDS) product[e] *= s;
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                h[e] = entry[e], m[e] = carry[e];
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
                before[r][e] = h[e];
                h[e] = fmaf(a[r][e], h[e], away[r][e] * v[r][e]);
            }
#pragma unroll
        for (int r = kSteps - 1; r >= 0; --r) {
            const int64_t t = t0 + wave * kSteps + r;
            float dx[V], dg[V];
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float l = dh[r][e] + m[e];
                const bool there = t < p.end;
                dx[e] = there ? away[r][e] * l : 0.f;
                dg[e] = there ? dx[e] * a[r][e] * (before[r][e] - v[r][e]) : 0.f;
                m[e] = a[r][e] * l;
            }
            if (t >= p.to) continue;
            if (g.dx) put<E, V>(g.dx, g, p, t, dx);
            if (g.dgate) put<E, V>(g.dgate, g, p, t, dg);
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
inline int waves(int64_t T) { return T <= kSteps ? 1 : T <= 8 * kSteps ? 4 : 16; }

inline Plan plan_of(int64_t B, int64_t T, int64_t D, int type, bool pairs)
{
    Plan p{};
    const int cus = device_cus();
    p.W = waves(T);
    p.block = p.W * kSteps, p.blocks = (T + p.block - 1) / p.block;
    auto workgroups = [&](int V) { return B * ((D + 64 * V - 1) / (64 * V)); };
    p.V = type != DS_F32 && pairs && (p.W == 16 || workgroups(2) >= cus) ? 2 : 1;
    p.groups = (int)((D + 64 * p.V - 1) / (64 * p.V));
    const int64_t all = std::max<int64_t>(1, workgroups(p.V));
    int64_t segments = std::min<int64_t>(cus / all, p.blocks / 2);
    if (g_tune.recur_segments != kTuneUnset) segments = std::min<int64_t>(g_tune.recur_segments, p.blocks);
    if (segments < 1) segments = 1;
    const int64_t each = std::max<int64_t>(1, (p.blocks + segments - 1) / segments);
    p.segment = each * p.block;
    p.segments = (int)std::max<int64_t>(1, (p.blocks + each - 1) / each);
    p.bytes = p.segments > 1 ? (size_t)p.segments * B * D * sizeof(float2) : 0;
    if (p.bytes == 0) p.bytes = 256;
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
    return launch<E, V, 16>(g, backward, grid, st);
}

inline bool in_pairs(const Sequence &s) { return (uintptr_t)s.at % 4 == 0 && s.batch % 2 == 0 && s.token % 2 == 0; }

int check(int64_t B, int64_t T, int64_t D, int type)
{
    if (B < 0 || T < 0 || D < 0 || !element_bytes(type)) return DS_EINVAL;
    const int64_t most = 0x7fffffff;
    if (D > most - 128 || B > most || (D > 0 && B > most / ((D + 63) / 64))) return DS_ETOOLARGE;
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
