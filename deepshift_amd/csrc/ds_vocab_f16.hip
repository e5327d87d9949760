// The products of the vocabulary's cross entropy on float16 operands.
#include "ds_vocab.h"

namespace ds {
namespace vocab {

template <> int launch_product<F16>(int kind, int tile, Args &g, Args *other, hipStream_t st)
{
    if (tile == 0) return launch_tiled<F16, 256, 256, 2, 4, 2>(kind, g, other, st);
    if (tile == 1) return launch_tiled<F16, 128, 128, 2, 2, 2>(kind, g, other, st);
    if (tile == 2) return launch_tiled<F16, 128, 64, 4, 1, 3>(kind, g, other, st);
    return launch_tiled<F16, 64, 64, 2, 2, 3>(kind, g, other, st);
}

}  // namespace vocab
}  // namespace ds
