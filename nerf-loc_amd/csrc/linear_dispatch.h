// Which tile a product of linear.h runs on.
#pragma once
#include "linear_rows.h"

namespace nerf {
namespace lin {

// LDS-DMA moves 16-byte chunks between 16-byte aligned places: rows of both operands have to start on 16 bytes.  A chunk
// that holds a row's end must hold zeros behind it where the row runs along the reduction (the neighbour's values would
// be added); along C's rows or columns anything may follow, if it belongs to the buffer.
template <int DT>
inline bool dma_ok(int layout, const GemmArgs& g) {
    constexpr int E = elem_size(DT), CE = 16 / E;
    for (int s = 0; s < g.nseg; ++s) {
        const Seg& sg = g.seg[s];
        if (((uintptr_t)sg.a | (uintptr_t)sg.b) & 15) return false;
        if ((sg.lda * E) % 16 || (sg.ldb * E) % 16) return false;
        if (sg.lda * E * 256 >= (1ll << 31) || sg.ldb * E * 256 >= (1ll << 31)) return false;      // 32-bit offsets in a tile
        const long long row_a = layout == DW ? g.P : sg.red, row_b = layout == FWD ? sg.red : g.Q;
        if ((row_a % CE && !sg.a_padded) || (row_b % CE && !sg.b_padded)) return false;
    }
    return true;
}

// The tile.  256 x 256 reads its operands least often and pays once every compute unit has one and sixteen k-tiles to work
// through; 256 x 128 the same with half the outputs; below, and for short reductions, where filling and draining the
// pipeline is the time, 128 x 64 runs three workgroups a unit beside each other, and 64 x 64 spreads what little there is.
// Tiles that would cover over an eighth more than the outputs need are left to the smaller ones, but for 256 x 256 in 16 and
// 8 bits, where reading less outweighs it (32768 x 576 x 4096 bf16 204 us, with 256 x 128 228; 65536 x 320 x 2048 float32 994
// and with 128 x 64 699; its dW 65536 x 128 x 320 151 and 68).
// Measured (us; 256 x 256, 256 x 128, 128 x 128, 128 x 64, 64 x 64):
//   bf16 8192 x 4096 x 4096    258  295  318    -  444      bf16 4096 x 2048 x 2048   61  42  48  53  61
//   bf16 4096 x 1024 x 4096    110   70   61   53   62      fp32 65536 x 256 x 320   111 107 108  98 101
//   fp32 4096 x 4096 x 4096    994 1033 1098 1066 1099      8-bit 32768 x 1024 x 1024  83 75 66  65  74
template <int DT, int ODT, int LAY>
int gemm_tiles(GemmArgs& g, hipStream_t s) {
    auto tiles = [&](int p, int q) { return ((g.P + p - 1) / p) * ((g.Q + q - 1) / q) * g.splits; };
    if (!dma_ok<DT>(LAY, g)) {
        // 128 columns a tile unless the last tile's empty part would be over a tenth of the work (130 columns: half of it)
        const bool full = (g.Q + 127) / 128 * 128 * 10 <= (g.Q + 63) / 64 * 64 * 11;
        if (full && tiles(128, 128) >= 256) return launch<DT, ODT, LAY, 128, 128, 2, 2, REGS>(g, s);
        if (tiles(128, 64) >= 400) return launch<DT, ODT, LAY, 128, 64, 2, 2, REGS>(g, s);
        return launch<DT, ODT, LAY, 64, 64, 2, 2, REGS>(g, s);
    }
    if constexpr (LAY != DW && elem_size(DT) == 2) {
        if (rows_ok(g)) return launch_rows<DT, LAY == DX>(g, s);
    }
    const long long red = g.splits > 1 ? g.red_part : g.seg[0].red + (g.nseg > 1 ? g.seg[1].red : 0);
    const bool deep = red * elem_size(DT) >= 16 * 128;
    if constexpr (LAY == FWD && DT != F8W) {       // the reduction-major layouts and the widened operands do not fit its registers
        // float32 is bound by its matrix instructions: whole rounds of the card count (16384 x 1096 x 1024 511 us, with
        // 256 x 128 407), and columns in vain (65536 x 192 x 1024 264, with 128 x 64 207)
        const bool worth = DT != F32 || (tile_fits(g.P, g.Q, 256, 256) && (tiles(256, 256) + 255) / 256 * 2 <= (tiles(256, 128) + 255) / 256);
        if (deep && worth && tiles(256, 256) >= 256) return launch<DT, ODT, LAY, 256, 256, 2, 4, DMA16>(g, s);
    }
    // dW is cut to fill the card once, its last parts may be empty
    if (deep && tile_fits(g.P, g.Q, 256, 128) && tiles(256, 128) >= (LAY == DW ? 192 : 256)) return launch<DT, ODT, LAY, 256, 128, 4, 2, DMA16>(g, s);
    if (tiles(128, 64) >= 400) return launch<DT, ODT, LAY, 128, 64, 2, 2, DMA16>(g, s);
    return launch<DT, ODT, LAY, 64, 64, 2, 2, DMA16>(g, s);
}

template <int DT, int ODT>
int gemm_forward(GemmArgs& g, hipStream_t s) {
    constexpr int D = DT == F8 ? F8W : DT;       // few rows: widening is hidden behind the weights' loads
    if (g.P <= 16) return launch_few_rows<D, ODT, 1>(g, s);
    if (g.P <= 32) return launch_few_rows<D, ODT, 2>(g, s);
    if (g.P <= FEW_ROWS) return launch_few_rows<D, ODT, 4>(g, s);
    return gemm_tiles<DT, ODT, FWD>(g, s);
}

template <int DT>
int gemm(int layout, GemmArgs& g, hipStream_t s) {
    switch (layout) {
        case FWD: return gemm_forward<DT, DT>(g, s);
        case DX: return gemm_tiles<DT, DT, DX>(g, s);
        default: return gemm_tiles<DT, DT, DW>(g, s);
    }
}

}  // namespace lin
}  // namespace nerf
