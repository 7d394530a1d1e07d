// Linear layers on 8-bit operands with scales (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_f8(GemmArgs& g, hipStream_t s) { return gemm_fwd<F8, FWD>(g, s); }
}  // namespace lin
}  // namespace nerf
