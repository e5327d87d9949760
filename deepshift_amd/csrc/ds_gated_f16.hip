// The gated block's product on float16 operands.
#include "ds_gated.h"

namespace ds {
namespace gated {

template <> int launch_gate<F16>(int tile, Args &g, hipStream_t st) { return launch_gate_16<F16>(tile, g, st); }

}  // namespace gated
}  // namespace ds
