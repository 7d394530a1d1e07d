// Linear layers on 8-bit operands with scales (linear.h).
#include "linear_dispatch.h"

namespace nerf {
namespace lin {
int gemm_f8(GemmArgs& g, hipStream_t s) {
    switch (g.out_dt) {
        case F32: return gemm_forward<F8W, F32>(g, s);
        case BF16: return gemm_forward<F8, BF16>(g, s);
        default: return gemm_forward<F8, F16>(g, s);
    }
}
}  // namespace lin
}  // namespace nerf
