// The logits' products on bfloat16 operands where every token has words of a teacher's.
#include "ds_vocab.h"

namespace ds {
namespace vocab {

template <> int launch_taught<Bf16>(int kind, int tile, Args &g, hipStream_t st) { return launch_taught_16<Bf16>(kind, tile, g, st); }

}  // namespace vocab
}  // namespace ds
