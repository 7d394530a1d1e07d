// Many samples through a narrow layer (16-bit types, up to 256 inputs and outputs): the time is the samples' way through
// memory, so nothing may stand between them and the next ones.  A workgroup keeps the whole weight matrix in LDS and its
// eight waves walk the samples on their own, without a barrier: 16 RF rows at a time, straight from memory into MFMA
// fragments.  Each fragment register is asked for again, for the wave's next rows, as soon as its products are issued, so
// every wave always has its next 16 RF rows under way.
//
// C[p, q] = sum_r A(p, r) B(q, r): q sits on the MFMA's A side, so that a lane ends up with four consecutive columns of
// one row per fragment; two fragments are turned into 8 consecutive columns per lane (64 bytes of each row per store) by
// two permlane swaps.
#pragma once
#include "linear.h"

namespace nerf {
namespace lin {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// Two fragments' columns of a row: lane group g holds 4 columns of each, 16 f + 4 g .. + 4.  Afterwards (or before, the
// exchange undoes itself when run backwards) it holds 8 consecutive ones, 8 g .. + 8.  A swap exchanges a bit of the
// lane's group with the item's.
__device__ __forceinline__ void swap32(unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}
__device__ __forceinline__ void swap16(unsigned& a, unsigned& b) {
    const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
    a = r[0];
    b = r[1];
}

template <int DT>
__device__ __forceinline__ unsigned pack2(float a, float b) {
    if constexpr (DT == BF16) {
        const bf16x2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(unsigned, v);
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(unsigned, v);
    }
}
template <int DT>
__device__ __forceinline__ void unpack2(unsigned v, float& a, float& b) {
    if constexpr (DT == BF16) {
        a = __uint_as_float(v << 16);
        b = __uint_as_float(v & 0xffff0000u);
    } else {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        const f16x2 t = __builtin_bit_cast(f16x2, v);
        a = (float)t[0];
        b = (float)t[1];
    }
}

// The packed columns of two fragments (lo: the first two of a lane's four, hi: the others) to or from 8 g .. + 8 of the
// row's 32 at p; n: columns left from there.
__device__ __forceinline__ void store_row(unsigned (&lo)[2], unsigned (&hi)[2], unsigned short* p, long long n) {
    swap32(lo[0], lo[1]);
    swap32(hi[0], hi[1]);
    swap16(lo[0], lo[1]);
    swap16(hi[0], hi[1]);
    const unsigned w[4] = {lo[0], hi[0], lo[1], hi[1]};
    if (n >= 8) __builtin_memcpy(p, w, 16);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) p[j] = (unsigned short)(w[j >> 1] >> (16 * (j & 1)));
    }
}
__device__ __forceinline__ void load_row(unsigned (&lo)[2], unsigned (&hi)[2], const unsigned short* p, long long n) {
    unsigned w[4] = {0, 0, 0, 0};
    if (n >= 8) __builtin_memcpy(w, p, 16);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) w[j >> 1] |= (unsigned)p[j] << (16 * (j & 1));
    }
    lo[0] = w[0]; hi[0] = w[1]; lo[1] = w[2]; hi[1] = w[3];
    swap16(lo[0], lo[1]);
    swap16(hi[0], hi[1]);
    swap32(lo[0], lo[1]);
    swap32(hi[0], hi[1]);
}

// H x NF 16-column fragments of C, KS 32-element steps of the reduction; TB: B lies reduction-major.  With H = 2 two waves
// share the rows and halve the columns: 32 rows x 256 columns of sums, 256 inputs of 32 rows and the weights' fragments
// do not fit one wave's 256 registers (measured with spills: 310 us for 786432 x 256 x 256).
template <int DT, int NF, int KS, int RF, int H, bool TB>
__global__ void __launch_bounds__(512) rows_kernel(const GemmArgs g) {
    static_assert(NF % 2 == 0 && KS >= 2 && elem_size(DT) == 2, "whole pairs of fragments, whole swizzled rows");
    constexpr int ROWB = KS * 64, ROWS = RF * 16;
    __shared__ __align__(1024) unsigned char wlds[H * NF * 16 * ROWB];
    __shared__ __align__(16) float blds[H * NF * 16];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, gr = lane >> 4;
    const int Q = (int)g.Q, K = (int)g.seg[0].red;
    const long long lda = g.seg[0].lda, blocks = (g.P + ROWS - 1) / ROWS, stride = (long long)gridDim.x * (8 / H);
    const int half = wave % H * NF * 16;         // this wave's first column

    u32x4 x[RF][KS];
    unsigned row_off[RF];
#pragma unroll
    for (int r = 0; r < RF; ++r) row_off[r] = (unsigned)((r * 16 + i) * (int)lda + gr * 8) * 2;
    // a wave's rows as a buffer: rows and reduction elements behind the end lie outside it and read as zeros
    const void* at = nullptr;
    unsigned off[RF];
    auto aim = [&](long long blk) {
        const long long p0 = blk * ROWS, left = g.P - p0;
        at = static_cast<const char*>(g.seg[0].a) + p0 * lda * 2;
#pragma unroll
        for (int r = 0; r < RF; ++r) off[r] = r * 16 + i < left ? row_off[r] : OUTSIDE;
    };
    auto fetch = [&](int s) {
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, 0x7fffffff, 0x00020000);
#pragma unroll
        for (int r = 0; r < RF; ++r) {
            unsigned o = off[r];
            if (s * 32 + 32 > K && s * 32 + gr * 8 >= K) o = OUTSIDE;
            x[r][s] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, s * 64, 0));
        }
    };
    long long blk = (long long)blockIdx.x * (8 / H) + wave / H;
    if (blk < blocks) {
        aim(blk);
#pragma unroll
        for (int s = 0; s < KS; ++s) fetch(s);
    }

    // weights: row q of LDS holds B(q, 0 .. 32 KS), chunk c of each eight at c ^ (q & 7); zeros outside the matrix
    if constexpr (!TB) {
        for (int t = tid; t < H * NF * 16 * KS * 4; t += 512) {
            const int q = t / (KS * 4), c = t % (KS * 4);
            uint4 v = make_uint4(0, 0, 0, 0);
            if (q < Q && c * 8 < K) v = *reinterpret_cast<const uint4*>(static_cast<const char*>(g.seg[0].b) + ((long long)q * g.seg[0].ldb + c * 8) * 2);
            *reinterpret_cast<uint4*>(wlds + q * ROWB + ((c & ~7) | ((c ^ q) & 7)) * 16) = v;
        }
    } else {
        // 8 x 8 blocks turned in registers: eight reduction rows of eight columns in, eight chunks of a column's rows out
        for (int t = tid; t < H * NF * 2 * KS * 4; t += 512) {
            const int c = t / (H * NF * 2), q0 = t % (H * NF * 2) * 8;
            unsigned in[8][4];
#pragma unroll
            for (int r = 0; r < 8; ++r) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (c * 8 + r < K && q0 < Q) v = *reinterpret_cast<const uint4*>(static_cast<const char*>(g.seg[0].b) + ((long long)(c * 8 + r) * g.seg[0].ldb + q0) * 2);
                in[r][0] = v.x; in[r][1] = v.y; in[r][2] = v.z; in[r][3] = v.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int q = q0 + j;
                unsigned out[4];
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    out[k] = __builtin_amdgcn_perm(in[2 * k + 1][j >> 1], in[2 * k][j >> 1], j & 1 ? 0x07060302 : 0x05040100);
                *reinterpret_cast<uint4*>(wlds + q * ROWB + ((c & ~7) | ((c ^ q) & 7)) * 16) = make_uint4(out[0], out[1], out[2], out[3]);
            }
        }
    }
    for (int t = tid; t < H * NF * 16; t += 512) blds[t] = g.bias && t < Q ? ld_elem(g.bias, t, DT) : 0.f;
    __syncthreads();

    const unsigned char* wl = wlds + (half + i) * ROWB;
    // a step's weight fragments are read while the step before it is worked on; the first step's are those of every block
    i32x4 w[2][NF];
    auto weights = [&](int s) {
        const int place = ((4 * s & ~7) | (((4 * s + gr) & 7) ^ (i & 7))) * 16;
#pragma unroll
        for (int j = 0; j < NF; ++j) w[s & 1][j] = *reinterpret_cast<const i32x4*>(wl + j * 16 * ROWB + place);
    };
    static_assert(KS % 2 == 0, "the first step's fragments follow the last one's");
    weights(0);
    for (; blk < blocks; blk += stride) {
        const bool more = blk + stride < blocks;
        if (more) aim(blk + stride);
        f32x4 acc[RF][NF];
#pragma unroll
        for (int j = 0; j < NF; ++j) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(blds + half + j * 16 + gr * 4);
#pragma unroll
            for (int r = 0; r < RF; ++r) acc[r][j] = b;
        }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            weights((s + 1) % KS);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NF; ++j)
#pragma unroll
                for (int r = 0; r < RF; ++r) mma<DT>(acc[r][j], w[s & 1][j], __builtin_bit_cast(i32x4, x[r][s]));
            if (more) fetch(s);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < RF; ++r) {
            const long long p = blk * ROWS + r * 16 + i;
            const bool live = p < g.P;
#pragma unroll
            for (int J = 0; J < NF; J += 2) {
                const long long q = half + J * 16 + gr * 8, n = live ? g.Q - q : 0;
                unsigned lo[2], hi[2];
                f32x4 v[2] = {acc[r][J], acc[r][J + 1]};
                auto pack = [&] {
#pragma unroll
                    for (int j = 0; j < 2; ++j) { lo[j] = pack2<DT>(v[j][0], v[j][1]); hi[j] = pack2<DT>(v[j][2], v[j][3]); }
                };
                auto apply = [&](int act) {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[j][k] = act_fn(v[j][k], act);
                };
                if (g.z) {
                    pack();
                    store_row(lo, hi, static_cast<unsigned short*>(g.z) + p * g.ldz + q, n);
                }
                if (g.act == NERF_ACT_RELU) apply(NERF_ACT_RELU);
                else if (g.act == NERF_ACT_GELU) apply(NERF_ACT_GELU);
                else if (g.act == NERF_ACT_SILU) apply(NERF_ACT_SILU);
                if (g.res) {
                    load_row(lo, hi, static_cast<const unsigned short*>(g.res) + p * g.ldr + q, n);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float a, b;
                        unpack2<DT>(lo[j], a, b);
                        v[j][0] += a; v[j][1] += b;
                        unpack2<DT>(hi[j], a, b);
                        v[j][2] += a; v[j][3] += b;
                    }
                }
                pack();
                store_row(lo, hi, static_cast<unsigned short*>(g.y) + p * g.ldy + q, n);
            }
        }
    }
}

template <int DT, bool TB, int NF, int H, int KS>
int launch_rows2(GemmArgs& g, hipStream_t s) {
    const long long rows = 8 / H * 32, groups = (g.P + rows - 1) / rows;
    hipLaunchKernelGGL((rows_kernel<DT, NF, KS, 2, H, TB>), dim3((unsigned)(groups < 256 ? groups : 256)), dim3(512), 0, s, g);
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}
template <int DT, bool TB, int NF, int H>
int launch_rows1(GemmArgs& g, hipStream_t s) {
    const long long k = g.seg[0].red;
    if (k <= 64) return launch_rows2<DT, TB, NF, H, 2>(g, s);
    if (k <= 128) return launch_rows2<DT, TB, NF, H, 4>(g, s);
    return launch_rows2<DT, TB, NF, H, 8>(g, s);
}
template <int DT, bool TB>
int launch_rows(GemmArgs& g, hipStream_t s) {
    if (g.Q <= 64) return launch_rows1<DT, TB, 4, 1>(g, s);
    if (g.Q <= 128) return launch_rows1<DT, TB, 8, 1>(g, s);
    return launch_rows1<DT, TB, 8, 2>(g, s);
}

}  // namespace lin
}  // namespace nerf
