// Linear layers, float32 operands (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_f32(int layout, GemmArgs& g, hipStream_t s) { return gemm<F32>(layout, g, s); }
}  // namespace lin
}  // namespace nerf
