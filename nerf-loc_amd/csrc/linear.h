// Linear layers of any size: C[p, q] = sum_r A(p, r) B(q, r) on the matrix cores with the layer's epilogue, for the
// three products of a layer y = act(x W^T + b) + r:
//
//     forward   C = y   p = sample  q = output   r = input    A = x  [p][r]     B = W [q][r]
//     dx        C = dx  p = sample  q = input    r = output   A = gz [p][r]     B = W [r][q]   (B reduction-major)
//     dW        C = dW  p = output  q = input    r = sample   A = gz [r][p]     B = x [r][q]   (both reduction-major)
//
// Each operand is read as it lies in memory; the transposition of a reduction-major one happens between LDS and the
// registers (ds_read_b64_tr_b16 for 16-bit types, single-word reads for float32).  Sums are float32 throughout.
#pragma once
#include "common.h"

namespace nerf {
namespace lin {

// F8: e4m3 operands on the 8-bit matrix instructions; F8W: the same operands widened to bf16 first (exact), see mma8w
enum { F32 = NERF_DT_F32, BF16 = NERF_DT_BF16, F16 = NERF_DT_F16, F8 = 3, F8W = 4 };
constexpr bool is_f8(int dt) { return dt >= F8; }
constexpr int elem_size(int dt) { return dt == F32 ? 4 : is_f8(dt) ? 1 : 2; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) unsigned char lds_u8;

// One piece of the reduction: the input of a layer may come in two pieces side by side.
struct Seg {
    const void *a, *b;
    long long lda, ldb;          // elements between rows of the operand as it lies in memory
    long long red;               // length of the reduction over this piece
    bool a_padded, b_padded;     // rows go on with zeros to a whole number of 16-byte chunks
};

struct GemmArgs {
    Seg seg[2];
    int nseg;
    long long P, Q;              // rows and columns of C
    int splits;                  // the reduction is cut into this many parts (nseg = 1) ...
    long long red_part;          // ... of this many elements each (a multiple of the tile's)
    float* partial;              // [splits][P][Q] float32 sums instead of the epilogue, or null
    // epilogue: y = act(C s_p s_q + bias) + res; z = the argument of act
    const void *bias, *res;
    void *y, *z;
    long long ldr, ldy, ldz;
    const float *sp, *sq;        // 8-bit operands: scales of the rows of A and of B
    int act;
    int out_dt;                  // type of y, bias, res, z: the operands' own, or named by the call for 8-bit ones
    unsigned tiles_p, tiles_q;
};

// A product of few tiles and a long reduction is cut until about 256 workgroups of 64 x 64 have work, each with four
// k-tiles at least; linear.hip adds the parts up and runs the epilogue on the sums.  (73 x 409 x 3280 float32: 86 us in
// one part.)
inline int splits_for(long long P, long long Q, long long red, int elem) {
    const long long tiles = ((P + 63) / 64) * ((Q + 63) / 64), k_tiles = (red * elem + 127) / 128;
    if (tiles > 128 || k_tiles < 8) return 1;
    const long long s = 256 / tiles < k_tiles / 4 ? 256 / tiles : k_tiles / 4;
    return s < 1 ? 1 : (int)s;
}
// Whether tiles of bp x bq cover [P, Q] with at most an eighth more than those of 128 x 64 would
inline bool tile_fits(long long P, long long Q, int bp, int bq) {
    return (P + bp - 1) / bp * bp * ((Q + bq - 1) / bq * bq) * 8 <= (P + 127) / 128 * 128 * ((Q + 63) / 64 * 64) * 9;
}
constexpr long long FEW_ROWS = 64;       // up to here few_rows_kernel takes the forward product

// what the three products need of the operands' layouts
enum Layout { FWD = 0, DX = 1, DW = 2 };

int gemm_f32(int layout, GemmArgs& g, hipStream_t s);
int gemm_bf16(int layout, GemmArgs& g, hipStream_t s);
int gemm_f16(int layout, GemmArgs& g, hipStream_t s);
int gemm_f8(GemmArgs& g, hipStream_t s);                 // out_dt names the epilogue's type
// dx = (g act'(z)) W in one kernel with what else the backward needs of gz = g act'(z) (linear_rows.h)
struct PanelGrad {
    const void* z;
    void* gz;                    // [P][ldgz], written
    long long ldz, ldgz;
    float* colsum;               // [PANEL_GRAD_GROUPS][red], written, or null
};
constexpr int PANEL_GRAD_GROUPS = 256;
int panel_grad_bf16(GemmArgs& g, const PanelGrad& a, hipStream_t s);
int panel_grad_f16(GemmArgs& g, const PanelGrad& a, hipStream_t s);
// out [rows, cols] (rows ldo apart) = sum over n parts [rows][cols], in a fixed order (linear.hip)
int part_sum(int dtype, const float* parts, int n, long long rows, long long cols, void* out, long long ldo, hipStream_t s);

// ---------------------------------------------------------------------------------------------- scalars and epilogue
__device__ __forceinline__ float ld_elem(const void* p, long long i, int dt) {
    if (dt == F32) return reinterpret_cast<const float*>(p)[i];
    if (dt == BF16) return (float)reinterpret_cast<const __bf16*>(p)[i];
    return (float)reinterpret_cast<const _Float16*>(p)[i];
}
__device__ __forceinline__ void st_elem(void* p, long long i, float v, int dt) {
    if (dt == F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == BF16) reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
    else reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
}
// Eight consecutive elements at any element: 16-byte accesses need no alignment on this hardware's global memory.
template <int DT>
__device__ __forceinline__ void ld8(const void* p, long long i, float (&v)[8]) {
    if constexpr (DT == F32) {
        __builtin_memcpy(v, reinterpret_cast<const float*>(p) + i, 32);
    } else if constexpr (DT == BF16) {
        bf16x8 a;
        __builtin_memcpy(&a, reinterpret_cast<const __bf16*>(p) + i, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
    } else {
        f16x8 a;
        __builtin_memcpy(&a, reinterpret_cast<const _Float16*>(p) + i, 16);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (float)a[j];
    }
}
template <int DT>
__device__ __forceinline__ void st8(void* p, long long i, const float (&v)[8]) {
    if constexpr (DT == F32) {
        __builtin_memcpy(reinterpret_cast<float*>(p) + i, v, 32);
    } else if constexpr (DT == BF16) {
        bf16x8 a;
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = (__bf16)v[j];
        __builtin_memcpy(reinterpret_cast<__bf16*>(p) + i, &a, 16);
    } else {
        f16x8 a;
#pragma unroll
        for (int j = 0; j < 8; ++j) a[j] = (_Float16)v[j];
        __builtin_memcpy(reinterpret_cast<_Float16*>(p) + i, &a, 16);
    }
}

// The normal distribution's integral, Phi(z) = erfc(-z / sqrt 2) / 2, and exp(-z^2 / 2) beside it.  The tail
// erfc(x) exp(x^2) is t P(t) with t = 1 / (1 + 0.4 x): P of degree 8, fitted over the whole half line to a relative
// 1.3e-7 (weighted least squares, reweighted towards equal error).  In float32 z Phi(z) is off by at most 4e-7, and the
// lower tail keeps its leading digits (2.5e-6 down to z = -5).  About 20 instructions, where erfcf() takes 60.
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }     // 1 ulp; tiny results become 0
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float x = fabsf(z) * 0.70710678118654752f;
    const float t = __builtin_amdgcn_rcpf(fmaf(0.4f, x, 1.f));
    float p = 0.050261341f;
    p = fmaf(p, t, -0.18289855f);
    p = fmaf(p, t, 0.16908108f);
    p = fmaf(p, t, -0.0056041828f);
    p = fmaf(p, t, 0.14143002f);
    p = fmaf(p, t, 0.1685423f);
    p = fmaf(p, t, 0.20784266f);
    p = fmaf(p, t, 0.22566959f);
    p = fmaf(p, t, 0.22567587f);
    e = exp2_fast(x * x * -1.4426950408889634f);
    const float tail = 0.5f * t * p * e;
    return z < 0.f ? tail : 1.f - tail;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(z * -1.4426950408889634f)); }

// relu keeps NaN: a comparison that is false for it selects z.
__device__ __forceinline__ float act_fn(float z, int act) {
    float e;
    switch (act) {
        case NERF_ACT_RELU: return z <= 0.f ? 0.f : z;
        case NERF_ACT_GELU: return z * normal_cdf(z, e);
        case NERF_ACT_SILU: return z * sigmoid(z);
        default: return z;
    }
}
// Beyond +-100 the derivatives are 0 and 1 to the last bit; held there so that an infinite z (float16 reaches it) does
// not multiply a vanished factor.
__device__ __forceinline__ float act_grad(float z, int act) {
    z = z > 100.f ? 100.f : z < -100.f ? -100.f : z;
    switch (act) {
        case NERF_ACT_GELU: {
            float e;
            const float c = normal_cdf(z, e);
            return fmaf(z * 0.39894228040143268f, e, c);
        }
        case NERF_ACT_SILU: {
            const float p = sigmoid(z);
            return p * fmaf(z, 1.f - p, 1.f);
        }
        default: return 1.f;
    }
}
// g act'(z).  relu's 0 is chosen, not multiplied: an infinite g behind a closed relu stays out.
__device__ __forceinline__ float through_act(float g, float z, int act) {
    if (act == NERF_ACT_RELU) return z <= 0.f ? 0.f : g;
    return g * act_grad(z, act);
}
// Eight columns of one row.  Both ways out (a whole group by 16-byte accesses, the last columns one by one) share the
// arithmetic in between.
template <int DT>
__device__ __forceinline__ void some8(const void* p, long long i, bool whole, int n, float (&v)[8]) {
    if (whole) ld8<DT>(p, i, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = j < n ? ld_elem(p, i + j, DT) : 0.f;
    }
}
template <int DT>
__device__ __forceinline__ void put_some8(void* p, long long i, bool whole, int n, const float (&v)[8]) {
    if (whole) st8<DT>(p, i, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (j < n) st_elem(p, i + j, v[j], DT);
    }
}
// DT: type of bias, residual, z and y.  SCALED: sums of 8-bit operands, to be scaled by row and column first.
template <int DT, bool SCALED>
__device__ __forceinline__ void epilogue8(const GemmArgs& g, long long p, long long q, float (&v)[8]) {
    const bool whole = q + 8 <= g.Q;
    const int n = whole ? 8 : (int)(g.Q - q);
    float t[8];
    if constexpr (SCALED) {
        const float s = g.sp[p];
        some8<F32>(g.sq, q, whole, n, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] * s * t[j];
    }
    if (g.bias) {
        some8<DT>(g.bias, q, whole, n, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
    if (g.z) put_some8<DT>(g.z, p * g.ldz + q, whole, n, v);
    if (g.act == NERF_ACT_RELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = act_fn(v[j], NERF_ACT_RELU);
    } else if (g.act == NERF_ACT_GELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = act_fn(v[j], NERF_ACT_GELU);
    } else if (g.act == NERF_ACT_SILU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = act_fn(v[j], NERF_ACT_SILU);
    }
    if (g.res) {
        some8<DT>(g.res, p * g.ldr + q, whole, n, t);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += t[j];
    }
    put_some8<DT>(g.y, p * g.ldy + q, whole, n, v);
}

// ---------------------------------------------------------------------------------------------- one operand's tile
// A tile holds 128 bytes of reduction (BK elements) for OUT rows of C (columns for B).  In LDS it lies as in memory,
// [OUT][BK] or, reduction-major, [BK][OUT], in 16-byte chunks.  The chunks of a row are permuted so that the 16 lanes
// that read one fragment column together fall on different banks:
//   [OUT][BK]            chunk c of row o sits at c ^ (o & 7)
//   [BK][OUT] 16-bit     32-byte unit u of row k at u ^ ((k & 3) | (k >> 3 & 1) << 2)
//   [BK][OUT] float32    64-byte unit u of row k at u ^ (k >> 2 & 3)
// Chunk L (row-major) of the tile is fetched by lane L, so the LDS side is linear, as LDS-DMA wants it, and the
// permutation is on the memory side, inside lines that are fetched whole anyway.
template <int DT, int TR, int OUT, int NT>
struct Tile {
    static constexpr int E = elem_size(DT);
    static constexpr int BK = 128 / E;
    static constexpr int BYTES = OUT * 128;
    static constexpr int CH = BYTES / 16 / NT;                  // chunks per thread
    static constexpr int CE = 16 / E;                           // elements per chunk
    static constexpr int ROWC = TR ? OUT * E / 16 : 8;          // chunks per row
    static constexpr int ROWB = ROWC * 16;
    static_assert(BYTES % (16 * NT) == 0, "whole chunks per thread");

    __device__ __forceinline__ static int row_of(int L) { return L / ROWC; }
    // first element of chunk L within its row
    __device__ __forceinline__ static int col_of(int L) {
        const int row = L / ROWC, slot = L % ROWC;
        if constexpr (!TR) return (slot ^ (row & 7)) * CE;
        else if constexpr (E == 2) {
            const int f = ((row & 3) | ((row >> 3 & 1) << 2)) & (OUT / 16 - 1);
            return (((slot >> 1) ^ f) << 4) + (slot & 1) * 8;
        } else {
            const int f = (row >> 2 & 3) & (OUT / 16 - 1);
            return (((slot >> 2) ^ f) << 4) + (slot & 3) * 4;
        }
    }
    // fragment: lane (i = lane % 16, g = lane / 16) holds outer index o0 + i and reduction elements
    // (4 s + g) CE .. + CE of the tile (s = 0, 1)
    __device__ __forceinline__ static i32x4 frag(const unsigned char* tile, int o0, int s, int lane) {
        const int i = lane & 15, g = lane >> 4;
        if constexpr (!TR) {
            return *reinterpret_cast<const i32x4*>(tile + (o0 + i) * 128 + (((4 * s + g) ^ (i & 7)) << 4));
        } else if constexpr (E == 2) {
            const int f = ((i >> 2) | ((g & 1) << 2)) & (OUT / 16 - 1);
            const int k = s * 32 + g * 8 + (i >> 2);
            const unsigned char* a = tile + k * ROWB + (((o0 >> 4) ^ f) << 5) + (i & 3) * 8;
            typedef __attribute__((address_space(3))) s16x4* lds4;
            union { s16x4 h[2]; i32x4 v; } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(a));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(a + 4 * ROWB));
            return u.v;
        } else {
            const int f = g & (OUT / 16 - 1);
            const int k = s * 16 + g * 4;
            const unsigned char* a = tile + k * ROWB + (((o0 >> 4) ^ f) << 6) + i * 4;
            i32x4 v;
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const int*>(a + j * ROWB);
            return v;
        }
    }
};

__device__ __forceinline__ void mma8w(f32x4& c, const i32x4& a, const i32x4& b);
template <int DT>
__device__ __forceinline__ void mma(f32x4& c, const i32x4& a, const i32x4& b) {
    if constexpr (DT == BF16)
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else if constexpr (DT == F16)
        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else if constexpr (DT == F32) {
        const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    } else if constexpr (DT == F8W) mma8w(c, a, b);
}
__device__ __forceinline__ void mma8(f32x4& c, const i32x4 (&a)[2], const i32x4 (&b)[2]) {
    i32x8 x, y;
#pragma unroll
    for (int j = 0; j < 4; ++j) { x[j] = a[0][j]; x[4 + j] = a[1][j]; y[j] = b[0][j]; y[4 + j] = b[1][j]; }
    // scale operands 0: the products enter unscaled
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 0, 0, 0, 0, 0, 0);
}

// The 8-bit instruction adds its products in groups of eight at a resolution of 2^-13 of the group's largest, cutting
// off what lies below (measured: a relative 1.4e-5 on rows of quantised normal numbers).  bf16 and fp16 results, rounded
// to 2^-9 and 2^-12, do not show it; float32 results would, so theirs come from the bf16 instruction on the widened
// numbers, at half the rate.
__device__ __forceinline__ bf16x8 widen(unsigned lo, unsigned hi) {
    unsigned o[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const unsigned v = j ? hi : lo;
        const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8(v, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(v, true);
        const float a0 = a[0], a1 = a[1], b0 = b[0], b1 = b[1];     // scalars: a bit_cast of a vector's element takes its first
        // every e4m3 number is a bf16 number: the upper halves of the floats
        o[2 * j] = __builtin_amdgcn_perm(__float_as_uint(a1), __float_as_uint(a0), 0x07060302);
        o[2 * j + 1] = __builtin_amdgcn_perm(__float_as_uint(b1), __float_as_uint(b0), 0x07060302);
    }
    bf16x8 r;
    __builtin_memcpy(&r, o, 16);
    return r;
}
__device__ __forceinline__ void mma8w(f32x4& c, const i32x4& a, const i32x4& b) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(a[0], a[1]), widen(b[0], b[1]), c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(a[2], a[3]), widen(b[2], b[3]), c, 0, 0, 0);
}

// LDS-DMA of 16 bytes per lane to lds .. lds + 1024: written as asm because hipcc, once it sees such a load, waits for
// all of them before any LDS read.  A lane whose offset is not below the buffer's 2^31 - 1 bytes gets zeros.
constexpr unsigned OUTSIDE = 0x80000000u;
__device__ __forceinline__ i32x4 buffer_of(const void* p) {
    const unsigned long long a = reinterpret_cast<unsigned long long>(p);
    i32x4 r;
    r[0] = __builtin_amdgcn_readfirstlane((int)(unsigned)a);
    r[1] = __builtin_amdgcn_readfirstlane((int)(unsigned)(a >> 32)) & 0xffff;
    r[2] = 0x7fffffff;
    r[3] = 0x00020000;
    return r;
}
__device__ __forceinline__ void dma16(unsigned lds, unsigned voff, const i32x4& rsrc) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory", "m0");
}

// The first `have` (1 .. CE - 1) elements at p, zeros behind them.  Not unrolled: it runs once at a row's end.
template <int E>
__device__ __forceinline__ uint4 part_chunk(const char* p, int have) {
    unsigned long long lo = 0, hi = 0;
#pragma unroll 1
    for (int j = 0; j < have; ++j) {
        const unsigned long long v = E == 4 ? reinterpret_cast<const unsigned*>(p)[j]
                                   : E == 2 ? reinterpret_cast<const unsigned short*>(p)[j] : reinterpret_cast<const unsigned char*>(p)[j];
        const int at = j * E;
        if (at < 8) lo |= v << (8 * at);
        else hi |= v << (8 * (at - 8));
    }
    return make_uint4((unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32));
}

// The 16 bytes at v moved down by n (0 .. 15), zeros from above.
__device__ __forceinline__ uint4 move_down(const uint4& v, int n) {
    unsigned long long lo = (unsigned long long)v.y << 32 | v.x, hi = (unsigned long long)v.w << 32 | v.z;
    const int b = 8 * (n & 7);
    if (n >= 8) { lo = hi; hi = 0; }
    if (b) {
        lo = lo >> b | hi << (64 - b);
        hi >>= b;
    }
    return make_uint4((unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32));
}

// How an operand's tile reaches LDS.
//   DMA16  by LDS-DMA in 16-byte chunks: rows on 16 bytes, whole chunks throughout
//   REGS   through registers, any alignment (16-byte global loads take it).  Word-wise LDS-DMA of unaligned float32 rows
//          was no faster (4096^3 with rows of 4095: 1359 us against 1314): each row's lines are fetched twice either way
enum Way { REGS = 0, DMA16 = 1 };

// One operand's side of the main loop.  A tile's pieces lie at fixed offsets from its first element, worked out once per
// piece of the reduction; only a k-tile that runs over the reduction's end looks at them again.
template <int DT, int TR, int OUT, int NT, int WAY>
struct Loader {
    using T = Tile<DT, TR, OUT, NT>;
    static constexpr int N = T::CH;          // chunks per thread
    uint4 st[WAY == REGS ? T::CH : 1];
    unsigned off[N];             // bytes from the tile's first element
    int down[WAY == REGS && TR ? T::CH : 1];
    bool fast, edge;

    __device__ __forceinline__ static int row_of(int i, int tid) { return T::row_of(i * NT + tid); }
    __device__ __forceinline__ static int col_of(int i, int tid) { return T::col_of(i * NT + tid); }

    // outs: rows of C this operand has from the tile's first on
    __device__ __forceinline__ void start(long long ld, long long outs, int tid) {
        const int no = (int)(outs < OUT ? outs : OUT);
        if constexpr (WAY != REGS) {
            // what lies behind the last row of C reads as zeros
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = row_of(i, tid), col = col_of(i, tid);
                off[i] = (TR ? col : row) < no ? (unsigned)(row * (int)ld + col) * T::E : OUTSIDE;
            }
        } else {
            // what lies behind the last row of C repeats it or is anything: it is never stored.  A chunk that runs over a
            // reduction-major row's end is read from its last 16 bytes instead and moved down.
            fast = ld * T::E * 256 < (1ll << 31) && (!TR || no >= T::CE);
            edge = TR && no < OUT;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                int row = row_of(i, tid), col = col_of(i, tid);
                if (!TR && row >= no) row = no - 1;
                if constexpr (TR) {
                    const int c = col + T::CE <= no ? col : no - T::CE;
                    down[i] = col < no ? (col - c) * T::E : 0;
                    col = c;
                }
                off[i] = fast ? (unsigned)(row * (int)ld + col) * T::E : 0u;
            }
        }
    }
    // base: the tile's first element at this k-tile; done / reds: the reduction in front of it and what is left from there
    __device__ __forceinline__ void fetch(const char* base, long long ld, long long outs, long long done, long long reds, int tid, unsigned lds) {
        if constexpr (WAY != REGS) {
            const i32x4 rsrc = buffer_of(base);
            const unsigned at = lds + __builtin_amdgcn_readfirstlane(tid >> 6) * 1024;
            if (reds >= T::BK) {
#pragma unroll
                for (int i = 0; i < N; ++i) dma16(at + i * NT * 16, off[i], rsrc);
            } else {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    dma16(at + i * NT * 16, (TR ? row_of(i, tid) : col_of(i, tid)) < reds ? off[i] : OUTSIDE, rsrc);
            }
        } else if (fast && reds >= T::BK) {
#pragma unroll
            for (int i = 0; i < N; ++i) __builtin_memcpy(&st[i], base + off[i], 16);
            if constexpr (TR) {
                if (edge) {
#pragma unroll
                    for (int i = 0; i < N; ++i) st[i] = move_down(st[i], down[i]);
                }
            }
        } else if (fast && (TR || done + reds >= T::CE)) {
            // the reduction's last k-tile: zeros behind its end
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int at = TR ? row_of(i, tid) : col_of(i, tid), nr = (int)reds;
                st[i] = make_uint4(0, 0, 0, 0);
                if (at < nr) {
                    const int back = TR || at + T::CE <= nr ? 0 : at + T::CE - nr;        // elements to start earlier
                    __builtin_memcpy(&st[i], base + (long long)off[i] - back * T::E, 16);
                    st[i] = move_down(st[i], TR ? down[i % (TR ? N : 1)] : back * T::E);
                }
            }
        } else {
            const long long rows = TR ? reds : outs, cols = TR ? outs : reds;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int row = row_of(i, tid), col = col_of(i, tid);
                uint4 v = make_uint4(0, 0, 0, 0);
                if (row < rows && col < cols) {
                    const char* p = base + (row * ld + col) * T::E;
                    const long long have = cols - col;
                    if (have >= T::CE) __builtin_memcpy(&v, p, 16);
                    else v = part_chunk<T::E>(p, (int)have);
                }
                st[i] = v;
            }
        }
    }
    __device__ __forceinline__ void put(unsigned char* tile, int tid) {
        if constexpr (WAY == REGS) {
#pragma unroll
            for (int i = 0; i < N; ++i) *reinterpret_cast<uint4*>(tile + (i * NT + tid) * 16) = st[i];
        }
    }
};

template <int WP, int WQ>
__host__ __device__ constexpr int epi_bytes() { return 16 * (WQ + 4) * 4; }

// BP x BQ of C per workgroup of WVP x WVQ waves; ODT: the epilogue's type.
template <int DT, int ODT, int LAY, int BP, int BQ, int WVP, int WVQ, int WAY>
__global__ void __launch_bounds__(WVP* WVQ * 64) gemm_kernel(const GemmArgs g) {
    constexpr int NT = WVP * WVQ * 64;
    constexpr int TA = LAY == DW, TB = LAY != FWD;
    constexpr int WP = BP / WVP, WQ = BQ / WVQ, FP = WP / 16, FQ = WQ / 16;
    using LA = Loader<DT, TA, BP, NT, WAY>;
    using LB = Loader<DT, TB, BQ, NT, WAY>;
    constexpr bool DMA = WAY != REGS;
    using TAt = typename LA::T;
    using TBt = typename LB::T;
    constexpr int BK = TAt::BK, E = TAt::E;
    constexpr int STAGE = TAt::BYTES + TBt::BYTES;
    // three k-tiles in LDS for the smallest tile, whose k-tiles are worked off faster than memory answers (512 x 512 x 4096
    // bf16 18.9 -> 15.7 us, gradients of 1000 x 1000 x 1000 fp16 30.1 -> 27.6), and for dW's largest, whose operands come from memory once (786432 x
    // 256 x 256 bf16 183 -> 159, 65536 x 1024 x 1024 178 -> 157; float32 223 -> 225); the others gain nothing from it
    constexpr int NS = WAY != REGS && !is_f8(DT) && ((BP == 64 && BQ == 64) || (LAY == DW && BP == 256 && E == 2)) ? 3 : 2;
    constexpr int EPI = WVP * WVQ * epi_bytes<WP, WQ>(), LDS = NS * STAGE > EPI ? NS * STAGE : EPI;
    static_assert(LDS <= 160 * 1024, "LDS of one compute unit");
    __shared__ __align__(1024) unsigned char smem[LDS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int wp = (wave / WVQ) * WP, wq = (wave % WVQ) * WQ;

    // workgroup -> part and tile: consecutive workgroups go to the 8 XCDs in turn, so XCD x takes the x-th eighth of them,
    // part by part, and within one walks 8 rows of tiles column by column: its L2 then holds both operands' panels (dW of
    // 196608 x 256 x 256 bf16 53 us, with the tiles of a part on XCDs of their own 61)
    const unsigned n_tiles = g.tiles_p * g.tiles_q, all = n_tiles * gridDim.y;
    unsigned t = blockIdx.y * n_tiles + blockIdx.x;
    {
        const unsigned x = t & 7, i = t >> 3, each = all >> 3, more = all & 7;
        t = x * each + (x < more ? x : more) + i;
    }
    const unsigned part = gridDim.y > 1 ? t / n_tiles : 0;
    t -= part * n_tiles;
    const unsigned per = 8 * g.tiles_q, grp = t / per, first = grp * 8;
    const unsigned rows = g.tiles_p - first < 8 ? g.tiles_p - first : 8, in = t - grp * per;
    const long long p0 = (long long)(first + in % rows) * BP, q0 = (long long)(in / rows) * BQ;

    const long long r_lo = (long long)part * g.red_part;
    long long red[2] = {g.seg[0].red, g.nseg > 1 ? g.seg[1].red : 0};
    if (g.splits > 1) red[0] = red[0] - r_lo < g.red_part ? red[0] - r_lo : g.red_part;
    const int nt0 = (int)((red[0] + BK - 1) / BK), nt = nt0 + (int)((red[1] + BK - 1) / BK);

    LA la;
    LB lb;
    const unsigned lds0 = (unsigned)(unsigned long long)(lds_u8*)smem;
    auto fetch = [&](int kt, int buf) {
        const int s = kt >= nt0;
        const Seg& sg = g.seg[s];
        if (kt == nt0) {         // the second piece has a row stride of its own
            la.start(sg.lda, g.P - p0, tid);
            lb.start(sg.ldb, g.Q - q0, tid);
        }
        const long long r = (long long)(s ? kt - nt0 : kt) * BK, left = red[s] - r, ra = r_lo + r;
        const char* pa = reinterpret_cast<const char*>(sg.a) + (TA ? ra * sg.lda + p0 : p0 * sg.lda + ra) * E;
        const char* pb = reinterpret_cast<const char*>(sg.b) + (TB ? ra * sg.ldb + q0 : q0 * sg.ldb + ra) * E;
        la.fetch(pa, sg.lda, g.P - p0, ra, left, tid, lds0 + buf * STAGE);
        lb.fetch(pb, sg.ldb, g.Q - q0, ra, left, tid, lds0 + buf * STAGE + TAt::BYTES);
    };
    la.start(g.seg[0].lda, g.P - p0, tid);
    lb.start(g.seg[0].ldb, g.Q - q0, tid);
    auto put = [&](int buf) {
        la.put(smem + buf * STAGE, tid);
        lb.put(smem + buf * STAGE + TAt::BYTES, tid);
    };

    f32x4 acc[FP][FQ];
#pragma unroll
    for (int i = 0; i < FP; ++i)
#pragma unroll
        for (int j = 0; j < FQ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Two k-tiles (or NS) are in LDS, and the fragments of the next half tile are on their way to registers while the matrix cores
    // work on this one's: the one barrier of an iteration sits between the halves, where everything the second half needs
    // has been read, so the tile's buffer is free for the k-tile after the next, and the next one's loads have had a whole
    // iteration to land.
    auto landed = [&] {
        if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if constexpr (DT == F8) {
        fetch(0, 0);
        put(0);
        landed();
        for (int kt = 0; kt < nt; ++kt) {
            const int buf = kt & 1;
            if (kt + 1 < nt) fetch(kt + 1, buf ^ 1);
            const unsigned char* ta = smem + buf * STAGE;
            const unsigned char* tb = ta + TAt::BYTES;
            i32x4 b[FQ][2];
#pragma unroll
            for (int j = 0; j < FQ; ++j)
#pragma unroll
                for (int s = 0; s < 2; ++s) b[j][s] = TBt::frag(tb, wq + j * 16, s, lane);
#pragma unroll
            for (int i = 0; i < FP; ++i) {
                i32x4 a[2];
#pragma unroll
                for (int s = 0; s < 2; ++s) a[s] = TAt::frag(ta, wp + i * 16, s, lane);
#pragma unroll
                for (int j = 0; j < FQ; ++j) mma8(acc[i][j], b[j], a);
            }
            if constexpr (DMA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if constexpr (!DMA) { if (kt + 1 < nt) put(buf ^ 1); }
            __syncthreads();
        }
    } else {
        struct Half { i32x4 a[FP], b[FQ]; };
        Half h0, h1;
        auto read = [&](Half& h, int buf, int s) {
            const unsigned char* ta = smem + buf * STAGE;
            const unsigned char* tb = ta + TAt::BYTES;
#pragma unroll
            for (int j = 0; j < FQ; ++j) h.b[j] = TBt::frag(tb, wq + j * 16, s, lane);
#pragma unroll
            for (int i = 0; i < FP; ++i) h.a[i] = TAt::frag(ta, wp + i * 16, s, lane);
        };
        auto work = [&](const Half& h) {
#pragma unroll
            for (int i = 0; i < FP; ++i)
#pragma unroll
                for (int j = 0; j < FQ; ++j) mma<DT>(acc[i][j], h.b[j], h.a[i]);
        };
        fetch(0, 0);
        put(0);
        if (nt > 1) {
            fetch(1, 1);
            put(1);
        }
#pragma unroll
        for (int k = 2; k < NS; ++k)
            if (nt > k) fetch(k, k);
        // all but the stages behind the one that is needed may still be on their way
        auto ready = [&](int kt) {
            if (NS > 2 && kt + NS - 2 < nt) {
                asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * (LA::N + LB::N)) : "memory");
                __syncthreads();
            } else landed();
        };
        ready(0);
        if constexpr (!DMA) { if (nt > 2) fetch(2, 0); }
        read(h0, 0, 0);
        int buf = 0;
        for (int kt = 0; kt < nt; ++kt) {
            const int next = buf + 1 == NS ? 0 : buf + 1;
            read(h1, buf, 1);
            __builtin_amdgcn_sched_barrier(0);
            work(h0);
            __builtin_amdgcn_sched_barrier(0);
            ready(kt + 1);
            if (kt + NS < nt) {
                if constexpr (DMA) fetch(kt + NS, buf);
                else {
                    put(buf);
                    if (kt + 3 < nt) fetch(kt + 3, 0);
                }
            }
            if (kt + 1 < nt) read(h0, next, 0);
            __builtin_amdgcn_sched_barrier(0);
            work(h1);
            __builtin_amdgcn_sched_barrier(0);
            buf = next;
        }
        __syncthreads();
    }

    // The accumulator holds four columns of one row of C per lane and fragment; through 16 x WQ floats of LDS per wave
    // it turns into eight columns per lane, whole lines per row, for the epilogue's reads and stores.
    float* slab = reinterpret_cast<float*>(smem) + wave * (epi_bytes<WP, WQ>() / 4);
    constexpr int LPR = WQ / 8, RPP = 64 / LPR;
#pragma unroll
    for (int i = 0; i < FP; ++i) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int j = 0; j < FQ; ++j)
            *reinterpret_cast<f32x4*>(slab + (lane & 15) * (WQ + 4) + j * 16 + (lane >> 4) * 4) = acc[i][j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 16; r += RPP) {
            const int row = r + lane / LPR, col = (lane % LPR) * 8;
            if (RPP > 16 && row >= 16) continue;
            const long long p = p0 + wp + i * 16 + row, q = q0 + wq + col;
            float v[8];
            const f32x4 lo = *reinterpret_cast<const f32x4*>(slab + row * (WQ + 4) + col);
            const f32x4 hi = *reinterpret_cast<const f32x4*>(slab + row * (WQ + 4) + col + 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) { v[j] = lo[j]; v[4 + j] = hi[j]; }
            if (p < g.P && q < g.Q) {
                if (g.partial) {
                    float* o = g.partial + ((long long)part * g.P + p) * g.Q + q;
                    if (q + 8 <= g.Q) __builtin_memcpy(o, v, 32);
                    else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) if (q + j < g.Q) o[j] = v[j];
                    }
                } else epilogue8<ODT, is_f8(DT)>(g, p, q, v);
            }
        }
    }
}

template <int DT, int ODT, int LAY, int BP, int BQ, int WVP, int WVQ, int WAY>
int launch(GemmArgs& g, hipStream_t s) {
    const long long tp = (g.P + BP - 1) / BP, tq = (g.Q + BQ - 1) / BQ;
    // a launch counts its threads in 32 bits
    NERF_REQUIRE(tp * tq < (1ll << 32) / (WVP * WVQ * 64), "linear: %lld x %lld outputs are too many for one launch", g.P, g.Q);
    g.tiles_p = (unsigned)tp;
    g.tiles_q = (unsigned)tq;
    auto k = gemm_kernel<DT, ODT, LAY, BP, BQ, WVP, WVQ, WAY>;
    hipLaunchKernelGGL(k, dim3((unsigned)(tp * tq), g.splits), dim3(WVP * WVQ * 64), 0, s, g);
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}

// ---------------------------------------------------------------------------------------------- few rows
// One to 64 samples: every weight is read once and used a few times, so the time is the weights' way from memory.  A
// workgroup owns 16 outputs; its NW waves take 64-byte steps of the reduction in turn (together whole lines of 16 weight
// rows), straight from memory into fragments, U steps in flight each, and add their sums in LDS.
template <int DT>
__device__ __forceinline__ i32x4 chunk_at(const char* p, long long have) {
    constexpr int E = elem_size(DT), CE = 16 / E;
    i32x4 v = {0, 0, 0, 0};
    if (have >= CE) __builtin_memcpy(&v, p, 16);
    else if (have > 0) {
        const uint4 t = part_chunk<E>(p, (int)have);
        v = i32x4{(int)t.x, (int)t.y, (int)t.z, (int)t.w};
    }
    return v;
}

template <int DT, int ODT, int MT, int NW>
__global__ void __launch_bounds__(NW * 64) few_rows_kernel(const GemmArgs g) {
    constexpr int E = elem_size(DT), CE = 16 / E, STEP = 4 * CE, U = (MT == 1 ? 8 : MT == 2 ? 4 : 2) / (DT == F8W ? 2 : 1);
    __shared__ __align__(16) float sums[NW][MT][16][20];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, c = (lane >> 4) * CE;
    const long long q0 = (long long)blockIdx.x * 16, q = q0 + i < g.Q ? q0 + i : g.Q - 1;
    f32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    int turn = 0;                // steps go round the waves across both pieces
    for (int sgi = 0; sgi < g.nseg; ++sgi) {
        const Seg& sg = g.seg[sgi];
        const char* w = reinterpret_cast<const char*>(sg.b) + (q * sg.ldb + c) * E;
        const char* x[MT];
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const long long p = m * 16 + i < g.P ? m * 16 + i : g.P - 1;     // rows behind the last repeat it
            x[m] = reinterpret_cast<const char*>(sg.a) + (p * sg.lda + c) * E;
        }
        const int whole = (int)(sg.red / STEP), steps = (int)((sg.red + STEP - 1) / STEP);
        int st = (wave - turn) & (NW - 1);
        for (; st + (U - 1) * NW < whole; st += U * NW) {
            i32x4 a[U], b[U][MT];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long long o = (long long)(st + u * NW) * 64;
                __builtin_memcpy(&a[u], w + o, 16);
#pragma unroll
                for (int m = 0; m < MT; ++m) __builtin_memcpy(&b[u][m], x[m] + o, 16);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
#pragma unroll
                for (int m = 0; m < MT; ++m) mma<DT>(acc[m], a[u], b[u][m]);
                if constexpr (DT == F8W) __builtin_amdgcn_sched_barrier(0);      // widen one step at a time: registers
            }
        }
        for (; st < steps; st += NW) {
            const long long o = (long long)st * 64, have = sg.red - (long long)st * STEP - c;
            const i32x4 a = chunk_at<DT>(w + o, have);
#pragma unroll
            for (int m = 0; m < MT; ++m) mma<DT>(acc[m], a, chunk_at<DT>(x[m] + o, have));
        }
        turn = (turn + steps) & (NW - 1);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<f32x4*>(&sums[wave][m][i][(lane >> 4) * 4]) = acc[m];
    __syncthreads();
    for (int t = threadIdx.x; t < MT * 32; t += NW * 64) {
        const int p = t >> 1, col = (t & 1) * 8;
        float v[8] = {};
        for (int k = 0; k < NW; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += sums[k][p >> 4][p & 15][col + j];
        if (p < g.P && q0 + col < g.Q) epilogue8<ODT, is_f8(DT)>(g, p, q0 + col, v);
    }
}

template <int DT, int ODT, int MT>
int launch_few_rows(GemmArgs& g, hipStream_t s) {
    const dim3 grid((unsigned)((g.Q + 15) / 16));
    // sixteen waves (eight where widening needs the registers) once each has two steps to take, else four
    constexpr int MANY = DT == F8W ? 8 : 16;
    const long long bytes = (g.seg[0].red + (g.nseg > 1 ? g.seg[1].red : 0)) * elem_size(DT);
    if (bytes >= 32 * 64) hipLaunchKernelGGL((few_rows_kernel<DT, ODT, MT, MANY>), grid, dim3(MANY * 64), 0, s, g);
    else hipLaunchKernelGGL((few_rows_kernel<DT, ODT, MT, 4>), grid, dim3(256), 0, s, g);
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}

}  // namespace lin
}  // namespace nerf
