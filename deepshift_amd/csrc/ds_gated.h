// The gated block's product (ds_gated.hip): product_tile of ds_vocab.h with rows of both halves of the weights by turns of a unit
// in every tile, so that a lane has a gate and what it goes with in registers of its own.
#pragma once
#include "ds_vocab_host.h"

namespace ds {
namespace gated {

using namespace vocab;

// Launches it with tiles of shape `tile` (Shapes<P>, whose rows are of both halves); a translation unit per P.
template <typename P> int launch_gate(int tile, Args &g, hipStream_t st);
// float32 weights as they are
int launch_gate_raw(Args &g, hipStream_t st);

// A few tokens, whose operands lie as the caller's do (ds_gated_few.hip).
struct Few {
    const void *x, *weight, *bias;
    int64_t ldx, ldw, F;
    int T, D, activation;
    void *out;            // [T][F]
    float *halves;        // as Args has them
    int64_t ldz;
};
template <typename E> int launch_few(const Few &f, hipStream_t st);

template <typename P, int BM, int BN, int WM, int WN, int STAGES>
int launch_gate_tiled(Args &g, hipStream_t st)
{
    g.tiles_m = ceil_div(g.M, BM / 2), g.tiles_n = ceil_div(g.N, BN);
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n;
    if (blocks > 0x7fffffff) return DS_ETOOLARGE;
    hipLaunchKernelGGL((product_kernel<P, BM, BN, WM, WN, false, false, kGate, STAGES>), dim3((unsigned)blocks), dim3(WM * WN * 64), 0,
                       st, g);
    return launch_status();
}

// 16-bit types: every wave has both halves of its results, two units along m at least.
template <typename P>
int launch_gate_16(int tile, Args &g, hipStream_t st)
{
    if (tile == 0) return launch_gate_tiled<P, 256, 256, 2, 4, 2>(g, st);
    if (tile == 1) return launch_gate_tiled<P, 128, 128, 2, 2, 2>(g, st);
    if (tile == 2) return launch_gate_tiled<P, 128, 64, 2, 2, 3>(g, st);
    return launch_gate_tiled<P, 64, 64, 1, 2, 3>(g, st);
}

}  // namespace gated
}  // namespace ds
