// The logits' products on float16 operands where every token has words of a teacher's.
#include "ds_vocab.h"

namespace ds {
namespace vocab {

template <> int launch_taught<F16>(int kind, int tile, Args &g, hipStream_t st) { return launch_taught_16<F16>(kind, tile, g, st); }

}  // namespace vocab
}  // namespace ds
