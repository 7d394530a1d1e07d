// Which tile a product of linear.h runs on.
#pragma once
#include "linear.h"

namespace nerf {
namespace lin {

// LDS-DMA moves 16-byte chunks between 16-byte aligned places: rows of both operands have to start on 16 bytes, and no
// chunk may hold the end of a row's valid part and something else (the zeros behind it are the loader's, chunk by chunk).
template <int DT>
inline bool dma_ok(int layout, const GemmArgs& g) {
    constexpr int E = elem_size(DT), CE = 16 / E;
    for (int s = 0; s < g.nseg; ++s) {
        const Seg& sg = g.seg[s];
        if (((uintptr_t)sg.a | (uintptr_t)sg.b) & 15) return false;
        if ((sg.lda * E) % 16 || (sg.ldb * E) % 16) return false;
        if (sg.lda * E * 256 >= (1ll << 31) || sg.ldb * E * 256 >= (1ll << 31)) return false;      // 32-bit offsets in a tile
        const bool ta = layout == DW, tb = layout != FWD;
        if ((!ta || !tb) && sg.red % CE) return false;
        if (ta && g.P % CE) return false;
        if (tb && g.Q % CE) return false;
    }
    return true;
}

template <int DT, int LAY>
int gemm_fwd(GemmArgs& g, hipStream_t s) {
    const long long big = ((g.P + 127) / 128) * ((g.Q + 127) / 128) * g.splits;
    if (big >= 256) return launch<DT, LAY, 128, 128, 2, 2, false>(g, s);
    return launch<DT, LAY, 64, 64, 2, 2, false>(g, s);
}

template <int DT>
int gemm(int layout, GemmArgs& g, hipStream_t s) {
    switch (layout) {
        case FWD: return gemm_fwd<DT, FWD>(g, s);
        case DX: return gemm_fwd<DT, DX>(g, s);
        default: return gemm_fwd<DT, DW>(g, s);
    }
}

}  // namespace lin
}  // namespace nerf
