// Linear layers on 8-bit operands with scales (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_f8(GemmArgs& g, hipStream_t s) { return g.out_dt == F32 ? gemm_forward<F8W>(g, s) : gemm_forward<F8>(g, s); }
}  // namespace lin
}  // namespace nerf
