// Linear layers, bfloat16 operands (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_bf16(int layout, GemmArgs& g, hipStream_t s) { return gemm<BF16>(layout, g, s); }
int panel_grad_bf16(GemmArgs& g, const PanelGrad& a, hipStream_t s) { return launch_panel_grad<BF16>(g, a, s); }
}  // namespace lin
}  // namespace nerf
