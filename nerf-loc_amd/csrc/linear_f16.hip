// Linear layers, float16 operands (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_f16(int layout, GemmArgs& g, hipStream_t s) { return gemm<F16>(layout, g, s); }
}  // namespace lin
}  // namespace nerf
