// Linear layers, bfloat16 operands (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_bf16(int layout, GemmArgs& g, hipStream_t s) { return gemm<BF16>(layout, g, s); }
}  // namespace lin
}  // namespace nerf
