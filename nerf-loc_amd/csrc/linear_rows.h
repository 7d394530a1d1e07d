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
#include <utility>

#include "linear.h"

namespace nerf {
namespace lin {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// f(0), f(1), ... f(N - 1) with constant arguments: arrays indexed by them stay in registers, where a loop that the
// compiler unrolls late can leave them in scratch memory
template <class F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F&& f) { each_of(f, std::make_integer_sequence<int, N>{}); }

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

// The packed columns of two fragments (lo: the first two of a lane's four, hi: the others) and the 16 bytes 8 g .. + 8 of
// the row's 32 columns.
__device__ __forceinline__ u32x4 to_row(unsigned (&lo)[2], unsigned (&hi)[2]) {
    swap32(lo[0], lo[1]);
    swap32(hi[0], hi[1]);
    swap16(lo[0], lo[1]);
    swap16(hi[0], hi[1]);
    return u32x4{lo[0], hi[0], lo[1], hi[1]};
}
__device__ __forceinline__ void from_row(const u32x4& v, unsigned (&lo)[2], unsigned (&hi)[2]) {
    lo[0] = v[0]; hi[0] = v[1]; lo[1] = v[2]; hi[1] = v[3];
    swap16(lo[0], lo[1]);
    swap16(hi[0], hi[1]);
    swap32(lo[0], lo[1]);
    swap32(hi[0], hi[1]);
}

// H x NF 16-column fragments of C, KS 32-element steps of the reduction; TB: B lies reduction-major.  With H = 2 (129 to
// 256 outputs with a residual; without one panel_kernel takes them) two waves share the rows and halve the columns: 32 rows
// x 256 columns of sums, 256 inputs of 32 rows and the weights' fragments do not fit one wave's 256 registers (measured
// with spills: 310 us for 786432 x 256 x 256, against 212).  Z, RES: the epilogue stores its argument, adds a residual.
//
// From a block's first load to its last store there is no branch: loads and stores retire in order, and behind a branch
// that may or may not have issued some the compiler waits as if it had issued none, that is, for the stores of the block
// before.  What lies outside the matrices is masked by offsets outside the buffers instead.
template <int DT, int NF, int KS, int RF, int H, bool TB, bool Z, bool RES>
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
        // behind the last block nothing is inside: no branch may stand between the loads, it would make the compiler wait
        // for all of them
        const long long p0 = blk * ROWS, left = g.P - p0;
        at = left > 0 ? static_cast<const char*>(g.seg[0].a) + p0 * lda * 2 : static_cast<const char*>(g.seg[0].a);
#pragma unroll
        for (int r = 0; r < RF; ++r) off[r] = r * 16 + i < left ? row_off[r] : OUTSIDE;
    };
    const int kleft = K - gr * 8;
    // eight columns of a row of y, z or the residual: its offset from the block's first row
    auto spot = [&](long long p0, long long ld, int r, int J) {
        const int q = half + J * 16 + gr * 8;
        return p0 + r * 16 + i < g.P && q < Q ? (unsigned)((r * 16 + i) * (int)ld + q) * 2 : OUTSIDE;
    };
    auto rows_of = [&](const void* p, long long p0, long long ld) {
        return __builtin_amdgcn_make_buffer_rsrc(static_cast<char*>(const_cast<void*>(p)) + p0 * ld * 2, 0, 0x7fffffff, 0x00020000);
    };
    auto fetch = [&](int r, int s) {
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(at), 0, 0x7fffffff, 0x00020000);
        return __builtin_amdgcn_raw_buffer_load_b128(rs, s * 32 < kleft ? off[r] : OUTSIDE, s * 64, 0);
    };
    long long blk = (long long)blockIdx.x * (8 / H) + wave / H;
    aim(blk);
    each<KS>([&](auto s) { each<RF>([&](auto r) { x[r][s] = fetch(r, s); }); });

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
    // a step's weight fragments are read while the step before it is worked on, the first step's at the last one; with a
    // residual, whose rows take the registers, right before their use
    constexpr int WB = RES ? 1 : 2;
    i32x4 w[WB][NF];
    auto weights = [&](int s) {
        const int place = ((4 * s & ~7) | (((4 * s + gr) & 7) ^ (i & 7))) * 16;
#pragma unroll
        for (int j = 0; j < NF; ++j) w[s % WB][j] = *reinterpret_cast<const i32x4*>(wl + j * 16 * ROWB + place);
    };
    static_assert(KS % 2 == 0, "the first step's fragments follow the last one's");
    if constexpr (!RES) weights(0);
    for (; blk < blocks; blk += stride) {
        const long long p0 = blk * ROWS;
        aim(blk + stride);
        u32x4 res[RES ? RF : 1][RES ? NF / 2 : 1];
        if constexpr (RES) {
            const auto rs = rows_of(g.res, p0, g.ldr);
#pragma unroll
            for (int r = 0; r < RF; ++r)
#pragma unroll
                for (int J = 0; J < NF; J += 2)
                    res[r][J / 2] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, spot(p0, g.ldr, r, J), 0, 0));
        }
        f32x4 acc[RF][NF];
        each<NF>([&](auto j) {
            const f32x4 b = *reinterpret_cast<const f32x4*>(blds + half + j * 16 + gr * 4);
            each<RF>([&](auto r) { acc[r][j] = b; });
        });
        each<KS>([&](auto s) {
            weights(RES ? int(s) : (s + 1) % KS);
            __builtin_amdgcn_sched_barrier(0);
            each<NF>([&](auto j) { each<RF>([&](auto r) { mma<DT>(acc[r][j], w[s % WB][j], __builtin_bit_cast(i32x4, x[r][s])); }); });
            each<RF>([&](auto r) { x[r][s] = fetch(r, s); });
            __builtin_amdgcn_sched_barrier(0);
        });
        auto pack = [](const f32x4& a, const f32x4& b, unsigned (&lo)[2], unsigned (&hi)[2]) {
            lo[0] = pack2<DT>(a[0], a[1]);
            hi[0] = pack2<DT>(a[2], a[3]);
            lo[1] = pack2<DT>(b[0], b[1]);
            hi[1] = pack2<DT>(b[2], b[3]);
        };
        if constexpr (Z) {
            const auto rs = rows_of(g.z, p0, g.ldz);
            each<RF>([&](auto r) {
                each<NF / 2>([&](auto J) {
                    unsigned lo[2], hi[2];
                    pack(acc[r][2 * J], acc[r][2 * J + 1], lo, hi);
                    __builtin_amdgcn_raw_buffer_store_b128(to_row(lo, hi), rs, spot(p0, g.ldz, r, 2 * J), 0, 0);
                });
            });
        }
        const auto rs = rows_of(g.y, p0, g.ldy);
        each<RF>([&](auto r) {
            each<NF / 2>([&](auto J) {
                f32x4 v[2] = {acc[r][2 * J], acc[r][2 * J + 1]};
                unsigned lo[2], hi[2];
                each<2>([&](auto j) {
                    f32x4 t = v[j];
                    if (g.act == NERF_ACT_RELU) t = f32x4{act_fn(t[0], NERF_ACT_RELU), act_fn(t[1], NERF_ACT_RELU), act_fn(t[2], NERF_ACT_RELU), act_fn(t[3], NERF_ACT_RELU)};
                    else if (g.act == NERF_ACT_GELU) t = f32x4{act_fn(t[0], NERF_ACT_GELU), act_fn(t[1], NERF_ACT_GELU), act_fn(t[2], NERF_ACT_GELU), act_fn(t[3], NERF_ACT_GELU)};
                    else if (g.act == NERF_ACT_SILU) t = f32x4{act_fn(t[0], NERF_ACT_SILU), act_fn(t[1], NERF_ACT_SILU), act_fn(t[2], NERF_ACT_SILU), act_fn(t[3], NERF_ACT_SILU)};
                    v[j] = t;
                });
                if constexpr (RES) {
                    from_row(res[r][J], lo, hi);
                    each<2>([&](auto j) {
                        float a, b, c, d;
                        unpack2<DT>(lo[j], a, b);
                        unpack2<DT>(hi[j], c, d);
                        v[j] += f32x4{a, b, c, d};
                    });
                }
                pack(v[0], v[1], lo, hi);
                __builtin_amdgcn_raw_buffer_store_b128(to_row(lo, hi), rs, spot(p0, g.ldy, r, 2 * J), 0, 0);
            });
        });
    }
}

// The weight fragments of 64 columns from q0 of a reduction-major matrix: through LDS, turned in registers 8 x 8 at a time.
template <int KS>
__device__ __forceinline__ void turned_weights(const GemmArgs& g, unsigned char* smem, int q0, i32x4 (&w)[KS][4]) {
    constexpr int ROWC = KS * 4, ROWB = KS * 64;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, gr = lane >> 4, Q = (int)g.Q, K = (int)g.seg[0].red;
    for (int k = tid; k < 32 * ROWC; k += 512) {
        const int c = k / 32, q = k % 32 * 8;
        unsigned in[8][4];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (c * 8 + r < K && q < Q) v = *reinterpret_cast<const uint4*>(static_cast<const char*>(g.seg[0].b) + ((long long)(c * 8 + r) * g.seg[0].ldb + q) * 2);
            in[r][0] = v.x; in[r][1] = v.y; in[r][2] = v.z; in[r][3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned out[4];
#pragma unroll
            for (int m = 0; m < 4; ++m)
                out[m] = __builtin_amdgcn_perm(in[2 * m + 1][j >> 1], in[2 * m][j >> 1], j & 1 ? 0x07060302 : 0x05040100);
            *reinterpret_cast<uint4*>(smem + (q + j) * ROWB + ((c & ~7) | ((c ^ (q + j)) & 7)) * 16) = make_uint4(out[0], out[1], out[2], out[3]);
        }
    }
    __syncthreads();
    each<KS>([&](auto s) {
        each<4>([&](auto j) {
            const int c = 4 * s + gr, q = q0 + j * 16 + i;
            w[s][j] = *reinterpret_cast<const i32x4*>(smem + q * ROWB + ((c & ~7) | ((c ^ q) & 7)) * 16);
        });
    });
    __syncthreads();
}

// ---------------------------------------------------------------------------------------------- 129 to 256 outputs
// The same with the sides exchanged: a wave keeps 64 columns of the weights in registers (32 fragments at 256 inputs) and
// the samples come through LDS, where all four column groups find them, 64 rows a stage and several stages under way:
// the loads in flight are no longer what the registers hold.  (rows_kernel on 786432 x 256 x 256 bf16: 212 us, of which
// the products alone take 84, with the loads 141, with the stores 104.)
//
// Everything a wave asks of memory inside the loop is counted: D loads to LDS and E stores a stage, issued without a
// branch, so stage t has landed once all but the E + (S - 2)(D + E) youngest are done.
template <int DT, int KS, bool TB, bool Z>
__global__ void __launch_bounds__(512) panel_kernel(const GemmArgs g) {
    constexpr int ROWC = KS * 4, ROWB = KS * 64, TILE = 64, STAGE = TILE * ROWB;
    constexpr int S = KS == 8 ? 4 : KS == 4 ? 6 : 8;
    constexpr int D = TILE * ROWC / 512, E = Z ? 8 : 4, YOUNGER = E + (S - 2) * (D + E);
    static_assert(D * 512 == TILE * ROWC && YOUNGER < 64 && 256 * ROWB <= S * STAGE && S * STAGE <= 128 * 1024, "stages");
    __shared__ __align__(1024) unsigned char smem[S * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, gr = lane >> 4;
    const int q0 = (wave & 3) * 64, r0 = (wave >> 2) * 32;       // this wave's columns and rows of a tile
    const int Q = (int)g.Q, K = (int)g.seg[0].red;
    const long long lda = g.seg[0].lda, tiles = (g.P + TILE - 1) / TILE;
    const unsigned lds0 = (unsigned)(unsigned long long)(lds_u8*)smem;

    // chunk c of row p of a tile sits at c ^ (p & 7); lane L of the tile's loads fetches what belongs at its place
    unsigned off[D];
    int row[D];
    each<D>([&](auto d) {
        const int L = d * 512 + tid, slot = L % ROWC;
        row[d] = L / ROWC;
        const int c = (slot & ~7) | ((slot ^ row[d]) & 7);
        off[d] = c * 8 < K ? (unsigned)(row[d] * (int)lda + c * 8) * 2 : OUTSIDE;
    });
    auto fetch = [&](long long t, int stage) {
        const long long p0 = t * TILE, left = g.P - p0;          // behind the last tile: nothing is inside
        const i32x4 rsrc = buffer_of(static_cast<const char*>(g.seg[0].a) + (left > 0 ? p0 * lda * 2 : 0));
        const unsigned at = lds0 + stage * STAGE + wave * 1024;
        each<D>([&](auto d) { dma16(at + d * 8192, row[d] < left ? off[d] : OUTSIDE, rsrc); });
    };

    i32x4 w[KS][4];
    f32x4 bias[4];
    long long t = blockIdx.x;
    if constexpr (!TB) {
        each<S - 1>([&](auto k) { fetch(t + k * (long long)gridDim.x, k); });
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(g.seg[0].b), 0, 0x7fffffff, 0x00020000);
        each<KS>([&](auto s) {
            each<4>([&](auto j) {
                const int q = q0 + j * 16 + i, r = s * 32 + gr * 8;
                const unsigned o = q < Q && r < K ? (unsigned)(q * (int)g.seg[0].ldb + r) * 2 : OUTSIDE;
                w[s][j] = __builtin_bit_cast(i32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0));
            });
        });
    } else {
        turned_weights<KS>(g, smem, q0, w);
        each<S - 1>([&](auto k) { fetch(t + k * (long long)gridDim.x, k); });
    }
    each<4>([&](auto j) {
        const int q = q0 + j * 16 + gr * 4;
        auto b = [&](int k) { return g.bias && q + k < Q ? ld_elem(g.bias, q + k, DT) : 0.f; };
        bias[j] = f32x4{b(0), b(1), b(2), b(3)};
    });
    // the weights and the bias have arrived (and with them, once, the first stages): from here on the count is the loop's
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

    const unsigned char* frag = smem + (r0 + i) * ROWB;
    int stage = 0;
    for (; t < tiles; t += gridDim.x) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(YOUNGER) : "memory");
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        // every wave has read the stage before this one: it takes the tile S - 1 ahead
        fetch(t + (S - 1) * (long long)gridDim.x, stage == 0 ? S - 1 : stage - 1);
        f32x4 acc[2][4];
        each<4>([&](auto j) { each<2>([&](auto r) { acc[r][j] = bias[j]; }); });
        const unsigned char* x = frag + stage * STAGE;
        each<KS>([&](auto s) {
            const int place = ((4 * s & ~7) | (((4 * s + gr) & 7) ^ (i & 7))) * 16;
            i32x4 a[2];
            each<2>([&](auto r) { a[r] = *reinterpret_cast<const i32x4*>(x + r * 16 * ROWB + place); });
            each<4>([&](auto j) { each<2>([&](auto r) { mma<DT>(acc[r][j], w[s][j], a[r]); }); });
        });
        const long long p0 = t * TILE + r0;
        auto out = [&](void* base, long long ld) {
            const auto rs = __builtin_amdgcn_make_buffer_rsrc(static_cast<char*>(base) + p0 * ld * 2, 0, 0x7fffffff, 0x00020000);
            each<2>([&](auto r) {
                each<2>([&](auto J) {
                    const f32x4 &u = acc[r][2 * J], &v = acc[r][2 * J + 1];
                    unsigned lo[2] = {pack2<DT>(u[0], u[1]), pack2<DT>(v[0], v[1])}, hi[2] = {pack2<DT>(u[2], u[3]), pack2<DT>(v[2], v[3])};
                    const int q = q0 + J * 32 + gr * 8;
                    const unsigned o = p0 + r * 16 + i < g.P && q < Q ? (unsigned)((r * 16 + i) * (int)ld + q) * 2 : OUTSIDE;
                    __builtin_amdgcn_raw_buffer_store_b128(to_row(lo, hi), rs, o, 0, 0);
                });
            });
        };
        if constexpr (Z) out(g.z, g.ldz);
        auto apply = [&](auto act) {
            each<2>([&](auto r) {
                each<4>([&](auto j) {
                    const f32x4 v = acc[r][j];
                    acc[r][j] = f32x4{act_fn(v[0], act), act_fn(v[1], act), act_fn(v[2], act), act_fn(v[3], act)};
                });
            });
        };
        if (g.act == NERF_ACT_RELU) apply(std::integral_constant<int, NERF_ACT_RELU>{});
        else if (g.act == NERF_ACT_GELU) apply(std::integral_constant<int, NERF_ACT_GELU>{});
        else if (g.act == NERF_ACT_SILU) apply(std::integral_constant<int, NERF_ACT_SILU>{});
        out(g.y, g.ldy);
        stage = stage + 1 == S ? 0 : stage + 1;
    }
    // the loads behind the last tile write (zeros) to this workgroup's LDS: they end before it does
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The input gradient of a layer of 65 to 256 outputs and up to 256 inputs together with the pass in front of it: dx = gz W
// with gz = g act'(z) formed on the way, written once for the weight gradient, and its column sums.  g and z come to LDS as in
// panel_kernel, 32 rows a stage; each thread takes what its own lane has fetched (so its own wait is enough), puts gz in
// g's place and in memory, and the one barrier of a tile stands behind that: it also says that every wave is done with the
// tile before, whose stage is then filled again.  A thread meets the same 8 columns in every tile: their sums stay in
// registers.  Bound by memory: g, z, gz and dx once each
// (786432 x 256 x 256 bf16, relu: 308 us = 5.2 TB/s; gelu 314).
template <int DT, int KS>
__global__ void __launch_bounds__(512) panel_grad_kernel(const GemmArgs g, const PanelGrad a) {
    constexpr int ROWC = KS * 4, ROWB = KS * 64, ROWS = 32, HALF = ROWS * ROWB, STAGE = 2 * HALF;
    constexpr int S = KS == 8 ? 4 : 8, C = ROWS * ROWC / 512;
    // a tile's memory operations, in order: C stores of gz, 2 C loads to LDS, 2 stores of dx
    constexpr int YOUNGER = 2 + (S - 2) * (3 * C + 2);
    static_assert(C * 512 == ROWS * ROWC && YOUNGER < 64 && 256 * ROWB <= S * STAGE && S * STAGE <= 128 * 1024 && (ROWC == 16 || ROWC == 32), "stages");
    __shared__ __align__(1024) unsigned char smem[S * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = lane & 15, gr = lane >> 4;
    const int q0 = (wave & 3) * 64, r0 = (wave >> 2) * 16;
    const int Q = (int)g.Q, K = (int)g.seg[0].red;
    const long long ldg = g.seg[0].lda, tiles = (g.P + ROWS - 1) / ROWS;
    const unsigned lds0 = (unsigned)(unsigned long long)(lds_u8*)smem;

    // this thread's chunk of a tile's row, the same in each of its rows (they are 8 or 16 or 32 apart)
    const int row0 = tid / ROWC, slot = tid % ROWC, col = ((slot & ~7) | ((slot ^ row0) & 7)) * 8;
    static_assert((512 / ROWC) % 8 == 0, "the permutation repeats");
    auto at_row = [&](int c) { return row0 + c * (512 / ROWC); };
    auto fetch = [&](long long t, int stage) {
        const long long p0 = t * ROWS, left = col < K ? g.P - p0 : 0, from = t < tiles ? p0 : 0;     // behind the last tile: nothing is inside
        const i32x4 rg = buffer_of(static_cast<const char*>(g.seg[0].a) + from * ldg * 2), rz = buffer_of(static_cast<const char*>(a.z) + from * a.ldz * 2);
        const unsigned at = lds0 + stage * STAGE + wave * 1024;
        each<C>([&](auto c) {
            const int r = at_row(c);
            dma16(at + c * 8192, r < left ? (unsigned)(r * (int)ldg + col) * 2 : OUTSIDE, rg);
            dma16(at + HALF + c * 8192, r < left ? (unsigned)(r * (int)a.ldz + col) * 2 : OUTSIDE, rz);
        });
    };

    i32x4 w[KS][4];
    turned_weights<KS>(g, smem, q0, w);
    long long t = blockIdx.x;
    each<S - 1>([&](auto k) { fetch(t + k * (long long)gridDim.x, k); });
    float sum[8] = {};
    const unsigned char* frag = smem + (r0 + i) * ROWB;
    int stage = 0;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    for (; t < tiles; t += gridDim.x) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(YOUNGER) : "memory");
        const long long p0 = t * ROWS;
        unsigned char* mine = smem + stage * STAGE + tid * 16;
        u32x4 gz[C];
        auto gate = [&](auto act) {
            each<C>([&](auto c) {
                const u32x4 gv = *reinterpret_cast<const u32x4*>(mine + c * 8192), zv = *reinterpret_cast<const u32x4*>(mine + HALF + c * 8192);
                u32x4 out;
                each<4>([&](auto j) {
                    const unsigned gj = gv[int(j)], zj = zv[int(j)];
                    float g0, g1, z0, z1;
                    unpack2<DT>(gj, g0, g1);
                    unpack2<DT>(zj, z0, z1);
                    g0 = through_act(g0, z0, act);
                    g1 = through_act(g1, z1, act);
                    sum[2 * j] += g0;
                    sum[2 * j + 1] += g1;
                    out[int(j)] = pack2<DT>(g0, g1);
                });
                *reinterpret_cast<u32x4*>(mine + c * 8192) = out;
                gz[c] = out;
            });
        };
        if (g.act == NERF_ACT_RELU) gate(std::integral_constant<int, NERF_ACT_RELU>{});
        else if (g.act == NERF_ACT_GELU) gate(std::integral_constant<int, NERF_ACT_GELU>{});
        else gate(std::integral_constant<int, NERF_ACT_SILU>{});
        {
            const auto rs = __builtin_amdgcn_make_buffer_rsrc(static_cast<char*>(a.gz) + p0 * a.ldgz * 2, 0, 0x7fffffff, 0x00020000);
            each<C>([&](auto c) {
                const int r = at_row(c);
                __builtin_amdgcn_raw_buffer_store_b128(gz[c], rs, p0 + r < g.P && col < K ? (unsigned)(r * (int)a.ldgz + col) * 2 : OUTSIDE, 0, 0);
            });
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
        fetch(t + (S - 1) * (long long)gridDim.x, stage == 0 ? S - 1 : stage - 1);
        f32x4 acc[4];
        each<4>([&](auto j) { acc[j] = f32x4{0.f, 0.f, 0.f, 0.f}; });
        const unsigned char* x = frag + stage * STAGE;
        each<KS>([&](auto s) {
            const int place = ((4 * s & ~7) | (((4 * s + gr) & 7) ^ (i & 7))) * 16;
            const i32x4 v = *reinterpret_cast<const i32x4*>(x + place);
            each<4>([&](auto j) { mma<DT>(acc[j], w[s][j], v); });
        });
        const auto rs = __builtin_amdgcn_make_buffer_rsrc(static_cast<char*>(g.y) + (p0 + r0) * g.ldy * 2, 0, 0x7fffffff, 0x00020000);
        each<2>([&](auto J) {
            const f32x4 &u = acc[2 * J], &v = acc[2 * J + 1];
            unsigned lo[2] = {pack2<DT>(u[0], u[1]), pack2<DT>(v[0], v[1])}, hi[2] = {pack2<DT>(u[2], u[3]), pack2<DT>(v[2], v[3])};
            const int q = q0 + J * 32 + gr * 8;
            const unsigned o = p0 + r0 + i < g.P && q < Q ? (unsigned)(i * (int)g.ldy + q) * 2 : OUTSIDE;
            __builtin_amdgcn_raw_buffer_store_b128(to_row(lo, hi), rs, o, 0, 0);
        });
        stage = stage + 1 == S ? 0 : stage + 1;
    }
    // the loads behind the last tile write (zeros) to this workgroup's LDS: they end before it is used again
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (!a.colsum) return;
    __syncthreads();
    float* sums = reinterpret_cast<float*>(smem);
    each<8>([&](auto j) { sums[row0 * (ROWC * 8) + col + j] = sum[j]; });
    __syncthreads();
    if (tid < K) {
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 512 / ROWC; ++r) s += sums[r * (ROWC * 8) + tid];
        a.colsum[(long long)blockIdx.x * K + tid] = s;
    }
}

template <int DT, bool TB, int KS>
int launch_panel1(GemmArgs& g, hipStream_t s) {
    const long long tiles = (g.P + 63) / 64;
    const dim3 grid((unsigned)(tiles < 256 ? tiles : 256));
    if constexpr (TB) hipLaunchKernelGGL((panel_kernel<DT, KS, TB, false>), grid, dim3(512), 0, s, g);
    else if (g.z) hipLaunchKernelGGL((panel_kernel<DT, KS, TB, true>), grid, dim3(512), 0, s, g);
    else hipLaunchKernelGGL((panel_kernel<DT, KS, TB, false>), grid, dim3(512), 0, s, g);
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}
template <int DT, bool TB>
int launch_panel(GemmArgs& g, hipStream_t s) {
    const long long k = g.seg[0].red;
    if (k <= 64) return launch_panel1<DT, TB, 2>(g, s);
    if (k <= 128) return launch_panel1<DT, TB, 4>(g, s);
    return launch_panel1<DT, TB, 8>(g, s);
}

template <int DT, bool TB, int NF, int H, int KS>
int launch_rows2(GemmArgs& g, hipStream_t s) {
    const long long rows = 8 / H * 32, groups = (g.P + rows - 1) / rows;
    const dim3 grid((unsigned)(groups < 256 ? groups : 256));
    if constexpr (TB) hipLaunchKernelGGL((rows_kernel<DT, NF, KS, 2, H, TB, false, false>), grid, dim3(512), 0, s, g);
    else if (g.z && g.res) hipLaunchKernelGGL((rows_kernel<DT, NF, KS, 2, H, TB, true, true>), grid, dim3(512), 0, s, g);
    else if (g.z) hipLaunchKernelGGL((rows_kernel<DT, NF, KS, 2, H, TB, true, false>), grid, dim3(512), 0, s, g);
    else if (g.res) hipLaunchKernelGGL((rows_kernel<DT, NF, KS, 2, H, TB, false, true>), grid, dim3(512), 0, s, g);
    else hipLaunchKernelGGL((rows_kernel<DT, NF, KS, 2, H, TB, false, false>), grid, dim3(512), 0, s, g);
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
// Whether the streaming kernel takes a product: enough rows to keep every wave going, both sides within its registers and
// LDS, outputs in whole 16-byte groups.
inline bool rows_ok(const GemmArgs& g) {
    const long long k = g.seg[0].red;
    if (g.nseg != 1 || g.partial || g.Q > 256 || k > 256 || g.Q % 8 || g.P < (g.Q <= 128 || k <= 128 ? 65536 : 131072)) return false;
    auto rows = [](const void* p, long long ld) { return !p || (((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld < (1ll << 24)); };
    return rows(g.y, g.ldy) && rows(g.z, g.ldz) && rows(g.res, g.ldr);
}
template <int DT, bool TB>
int launch_rows(GemmArgs& g, hipStream_t s) {
    if (g.Q <= 64) return launch_rows1<DT, TB, 4, 1>(g, s);
    if (g.Q <= 128) return launch_rows1<DT, TB, 8, 1>(g, s);
    if (!g.res) return launch_panel<DT, TB>(g, s);
    return launch_rows1<DT, TB, 8, 2>(g, s);
}

template <int DT>
int launch_panel_grad(GemmArgs& g, const PanelGrad& a, hipStream_t s) {
    const dim3 grid(PANEL_GRAD_GROUPS);
    if (g.seg[0].red <= 128) hipLaunchKernelGGL((panel_grad_kernel<DT, 4>), grid, dim3(512), 0, s, g, a);
    else hipLaunchKernelGGL((panel_grad_kernel<DT, 8>), grid, dim3(512), 0, s, g, a);
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}

}  // namespace lin
}  // namespace nerf
