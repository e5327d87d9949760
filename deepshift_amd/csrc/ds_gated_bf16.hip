// The gated block's product on bfloat16 operands.
#include "ds_gated.h"

namespace ds {
namespace gated {

template <> int launch_gate<Bf16>(int tile, Args &g, hipStream_t st) { return launch_gate_16<Bf16>(tile, g, st); }

}  // namespace gated
}  // namespace ds
