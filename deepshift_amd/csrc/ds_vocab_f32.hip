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

}  // namespace vocab
}  // namespace ds
