// The logits' products on float32 operands, as three bfloat16 planes each, where every token has words of a teacher's.
#include "ds_vocab.h"

namespace ds {
namespace vocab {

template <> int launch_taught<Split>(int kind, int tile, Args &g, hipStream_t st)
{
    if (tile == 0) return launch_taught_tiled<Split, 256, 128, 4, 2, 2>(kind, g, st);
    if (tile == 1) return launch_taught_tiled<Split, 128, 128, 2, 4, 3>(kind, g, st);
    if (tile == 2) return launch_taught_tiled<Split, 64, 64, 2, 2, 6>(kind, g, st);
    return launch_taught_tiled<Split, 32, 32, 1, 2, 6>(kind, g, st);
}

template <int WIDTH>
int launch_raw_width(int kind, const Args &g, dim3 grid, hipStream_t st)
{
    if (kind == kLogitStats) hipLaunchKernelGGL((taught_raw_kernel<kStats, WIDTH>), grid, dim3(256), 0, st, g);
    else if (kind == kLogitKeep) hipLaunchKernelGGL((taught_raw_kernel<kKeep, WIDTH>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((taught_raw_kernel<kProb, WIDTH>), grid, dim3(256), 0, st, g);
    return launch_status();
}

int launch_taught_raw(int kind, int width, Args &g, hipStream_t st)
{
    g.tiles_m = ceil_div(g.M, kRawWords), g.tiles_n = ceil_div(g.N, kRawTokens);
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n;
    if (blocks > 0x7fffffff) return DS_ETOOLARGE;
    const dim3 grid((unsigned)blocks);
    return width == 4 ? launch_raw_width<4>(kind, g, grid, st) : launch_raw_width<1>(kind, g, grid, st);
}

}  // namespace vocab
}  // namespace ds
