// The gated block's product on float32 operands, as three bfloat16 planes each.
#include "ds_gated.h"

namespace ds {
namespace gated {

template <> int launch_gate<Split>(int tile, Args &g, hipStream_t st)
{
    if (tile == 0) return launch_gate_tiled<Split, 256, 128, 4, 2, 2>(g, st);
    if (tile == 1) return launch_gate_tiled<Split, 128, 128, 2, 4, 3>(g, st);
    if (tile == 2) return launch_gate_tiled<Split, 64, 64, 2, 2, 6>(g, st);
    return launch_gate_tiled<Split, 32, 32, 1, 2, 6>(g, st);
}

int launch_gate_raw(Args &g, hipStream_t st)
{
    g.tiles_m = ceil_div(g.M, kRawWords / 2), g.tiles_n = ceil_div(g.N, kRawTokens);
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n;
    if (blocks > 0x7fffffff) return DS_ETOOLARGE;
    hipLaunchKernelGGL((raw_kernel<kGate, 4>), dim3((unsigned)blocks), dim3(256), 0, st, g);
    return launch_status();
}

}  // namespace gated
}  // namespace ds
