// Linear layers, float16 operands (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_f16(int layout, GemmArgs& g, hipStream_t s) { return gemm<F16>(layout, g, s); }
int panel_grad_f16(GemmArgs& g, const PanelGrad& a, hipStream_t s) { return launch_panel_grad<F16>(g, a, s); }
}  // namespace lin
}  // namespace nerf
