// The products of the vocabulary's cross entropy on float32 operands, as three bfloat16 planes each.
#include "ds_vocab.h"

namespace ds {
namespace vocab {

template <> int launch_product<Split>(int kind, int tile, Args &g, Args *other, hipStream_t st)
{
    if (tile == 0) return launch_tiled<Split, 256, 128, 4, 2, 2>(kind, g, other, st);
    if (tile == 1) return launch_tiled<Split, 128, 128, 2, 4, 3>(kind, g, other, st);
    if (tile == 2) return launch_tiled<Split, 64, 64, 2, 2, 6>(kind, g, other, st);
    return launch_tiled<Split, 32, 32, 1, 2, 6, false>(kind, g, other, st);
}

template <int WIDTH>
int launch_raw_tiles(int kind, const Args &g, dim3 grid, hipStream_t st)
{
    const dim3 threads(256);
    if (kind == kLogitStats) hipLaunchKernelGGL((raw_kernel<kStats, WIDTH>), grid, threads, 0, st, g);
    else if (kind == kLogitKeep) hipLaunchKernelGGL((raw_kernel<kKeep, WIDTH>), grid, threads, 0, st, g);
    else if (kind == kLogitProb) hipLaunchKernelGGL((raw_kernel<kProb, WIDTH>), grid, threads, 0, st, g);
    else hipLaunchKernelGGL((raw_kernel<kOut, WIDTH>), grid, threads, 0, st, g);
    return launch_status();
}

int launch_raw(int kind, int width, Args &g, hipStream_t st)
{
    g.tiles_m = ceil_div(g.M, kRawWords), g.tiles_n = ceil_div(g.N, kRawTokens);
    const int64_t blocks = (int64_t)g.tiles_m * g.tiles_n * g.splits;
    if (blocks > 0x7fffffff) return DS_ETOOLARGE;
    return width == 4 ? launch_raw_tiles<4>(kind, g, dim3((unsigned)blocks), st) : launch_raw_tiles<1>(kind, g, dim3((unsigned)blocks), st);
}

}  // namespace vocab
}  // namespace ds
