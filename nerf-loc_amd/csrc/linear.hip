// C entry points of the linear layers, and the passes around their products: the gradient through the activation with
// the bias gradient's column sums, and the sums over the parts of a split reduction.
#include <algorithm>

#include "linear.h"

namespace nerf {
namespace lin {

// gz = g act'(z) over blocks of `rows` samples, and the block's column sums.  One thread owns 8 columns (a 16-byte load
// of 16-bit types) of every (256 / groups)-th sample of its block; the sums of a column meet in LDS in a fixed order.
// Bound by memory: reads g and z, writes gz, once.
struct ActGradArgs {
    const void *g, *z;
    long long ldg, ldz;
    void* gz;                    // [M][ldgz] or null: N columns and zeros behind them
    long long ldgz;
    float* colsum;               // [blocks][N] or null
    void* db;                    // [N]: the sums themselves, where one block holds all samples; or null
    long long M, N, rows;
    int act;
};
constexpr int AG_COLS = 64;      // columns per workgroup: 8 threads across, 32 samples at a time
template <int DT>
__global__ void __launch_bounds__(256) act_grad_kernel(const ActGradArgs a) {
    __shared__ float part[32][AG_COLS + 4];
    const int tx = threadIdx.x & 7, ty = threadIdx.x >> 3;
    const long long q = (long long)blockIdx.x * AG_COLS + tx * 8;
    const long long lo = (long long)blockIdx.y * a.rows, hi = lo + a.rows < a.M ? lo + a.rows : a.M;
    float sum[8] = {};
    const bool whole = q + 8 <= a.N;
    if (q < a.N) {
        for (long long p = lo + ty; p < hi; p += 32) {
            float g[8], z[8];
            if (whole) {
                ld8<DT>(a.g, p * a.ldg + q, g);
                if (a.act != NERF_ACT_NONE) {
                    ld8<DT>(a.z, p * a.ldz + q, z);
#pragma unroll
                    for (int j = 0; j < 8; ++j) g[j] = through_act(g[j], z[j], a.act);
                }
                if (a.gz) st8<DT>(a.gz, p * a.ldgz + q, g);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    g[j] = 0.f;
                    if (q + j < a.N) {
                        g[j] = ld_elem(a.g, p * a.ldg + q + j, DT);
                        if (a.act != NERF_ACT_NONE) g[j] = through_act(g[j], ld_elem(a.z, p * a.ldz + q + j, DT), a.act);
                    }
                    if (a.gz && q + j < a.ldgz) st_elem(a.gz, p * a.ldgz + q + j, g[j], DT);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += g[j];
        }
    }
    if (!a.colsum && !a.db) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) part[ty][tx * 8 + j] = sum[j];
    __syncthreads();
    if (threadIdx.x < AG_COLS) {
        const long long c = (long long)blockIdx.x * AG_COLS + threadIdx.x;
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) s += part[r][threadIdx.x];
        if (c < a.N) {
            if (a.db) st_elem(a.db, c, s, DT);
            else a.colsum[(long long)blockIdx.y * a.N + c] = s;
        }
    }
}

// out[i] (rows of `cols` elements, ldo apart) = sum over n parts.  A workgroup owns 16 consecutive elements and has 64
// threads read every 64th part of each: few outputs still fill the card, and a thread's loads are independent.  The
// order of the additions is fixed.
template <int DT>
__global__ void __launch_bounds__(1024) part_sum_kernel(const float* parts, int n, long long all, long long cols, void* out, long long ldo) {
    __shared__ float sums[64][17];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const long long i = (long long)blockIdx.x * 16 + tx;
    float s = 0.f;
    if (i < all) {
#pragma unroll 8
        for (int k = ty; k < n; k += 64) s += parts[(long long)k * all + i];
    }
    sums[ty][tx] = s;
    __syncthreads();
    if (threadIdx.x < 256) {         // 16 elements x 16: four of the 64 each, then a tree in the wave
        const int c = threadIdx.x >> 4, r = threadIdx.x & 15;
        s = (sums[r][c] + sums[r + 16][c]) + (sums[r + 32][c] + sums[r + 48][c]);
#pragma unroll
        for (int d = 8; d >= 1; d >>= 1) s += __shfl_xor(s, d, 64);
        const long long o = (long long)blockIdx.x * 16 + c;
        if (r == 0 && o < all) st_elem(out, (o / cols) * ldo + o % cols, s, DT);
    }
}
// The same for many elements and few parts: one thread each, in turns (a launch counts its threads in 32 bits).
constexpr long long WIDE_GROUPS = 1 << 20;
template <int DT>
__global__ void __launch_bounds__(256) part_sum_wide_kernel(const float* parts, int n, long long all, long long cols, void* out, long long ldo) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        float s = 0.f;
#pragma unroll 8
        for (int k = 0; k < n; ++k) s += parts[(long long)k * all + i];
        st_elem(out, (i / cols) * ldo + i % cols, s, DT);
    }
}

template <int DT>
static void part_sum_launch(const float* parts, int n, long long all, long long cols, void* out, long long ldo, hipStream_t s) {
    // 64 threads an element pay where one each would leave the card half empty (128 parts of 65536: 16 us against 12)
    if (all <= 16384) hipLaunchKernelGGL(part_sum_kernel<DT>, dim3((unsigned)((all + 15) / 16)), dim3(1024), 0, s, parts, n, all, cols, out, ldo);
    else hipLaunchKernelGGL(part_sum_wide_kernel<DT>, dim3((unsigned)std::min((all + 255) / 256, WIDE_GROUPS)), dim3(256), 0, s, parts, n, all, cols, out, ldo);
}
int part_sum(int dtype, const float* parts, int n, long long rows, long long cols, void* out, long long ldo, hipStream_t s) {
    switch (dtype) {
        case F32: part_sum_launch<F32>(parts, n, rows * cols, cols, out, ldo, s); break;
        case BF16: part_sum_launch<BF16>(parts, n, rows * cols, cols, out, ldo, s); break;
        default: part_sum_launch<F16>(parts, n, rows * cols, cols, out, ldo, s); break;
    }
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}

// The epilogue on the sums of a split product: one thread adds eight columns' parts, in order.
template <int DT, bool SCALED>
__global__ void __launch_bounds__(256) finish_kernel(const GemmArgs g, int parts) {
    const long long groups = (g.Q + 7) / 8, t = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long p = t / groups, q = t % groups * 8;
    if (p >= g.P) return;
    const bool whole = q + 8 <= g.Q;
    const int n = whole ? 8 : (int)(g.Q - q);
    float v[8] = {};
    for (int k = 0; k < parts; ++k) {
        float t8[8];
        some8<F32>(g.partial, ((long long)k * g.P + p) * g.Q + q, whole, n, t8);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += t8[j];
    }
    epilogue8<DT, SCALED>(g, p, q, v);
}

// Rows copied to places on 16 bytes, zeros behind their ends to a whole chunk: all the operands of a product that need it
// in one launch, one chunk a thread.
struct PackArgs {
    struct Job {
        const char* src;
        uint4* dst;
        long long ld, rows, cols, chunks;        // chunks: of a row
        unsigned first;                          // workgroup
    } job[4];
    int jobs;
};
template <int E>
__global__ void __launch_bounds__(256) pack_kernel(const PackArgs a) {
    constexpr int CE = 16 / E;
    int n = 0;
    while (n + 1 < a.jobs && blockIdx.x >= a.job[n + 1].first) ++n;
    const PackArgs::Job& j = a.job[n];
    const long long t = (long long)(blockIdx.x - j.first) * 256 + threadIdx.x, row = t / j.chunks, c = t % j.chunks * CE;
    if (row >= j.rows) return;
    uint4 v;
    const char* p = j.src + (row * j.ld + c) * E;
    if (c + CE <= j.cols) __builtin_memcpy(&v, p, 16);
    else v = part_chunk<E>(p, (int)(j.cols - c));
    j.dst[t] = v;
}

static int dispatch_gemm(int dtype, int layout, GemmArgs& g, hipStream_t s) {
    if (dtype != F8) g.out_dt = dtype;
    switch (dtype) {
        case F32: return gemm_f32(layout, g, s);
        case BF16: return gemm_bf16(layout, g, s);
        case F16: return gemm_f16(layout, g, s);
        default: return gemm_f8(g, s);
    }
}

static size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

// A matrix as a product reads it, and where its packed copy goes if it needs one.
struct Mat {
    const void* p;
    long long ld, rows, cols;
    bool padded;
};
// Rows on 16 bytes, and whole chunks
static bool dma_rows(const Mat& m, int e) { return ((uintptr_t)m.p & 15) == 0 && (m.ld * e) % 16 == 0 && (m.padded || (m.cols * e) % 16 == 0); }
static long long packed_ld(long long cols, int e) { return (cols * e + 15) / 16 * 16 / e; }
static size_t packed_bytes(const Mat& m, int e) { return align256((size_t)m.rows * packed_ld(m.cols, e) * e); }
static long long packed_groups(const Mat& m, int e) { return (m.rows * (packed_ld(m.cols, e) * e / 16) + 255) / 256; }

// One product with its copies and its split: what it takes of the workspace, and the launches.
struct Product {
    int dtype, layout;
    Mat a[2], b[2];
    int nseg;
    long long P, Q;
    long long red[2];
    bool can_split;

    // Unaligned rows are fetched line by line twice; a copy costs its bytes both ways and a launch.  Forward it pays once
    // there are two tiles a compute unit (fewer wait for latency, not for bytes) and the copy is short against the product;
    // where an operand lies reduction-major, and there is only one to copy, earlier.  Measured (us, as they lie and copied;
    // copy over product by the estimates below):
    //   forward fp16 4096 x 4096 x 4095 308 151   65536 x 256 x 319 66 56 (1.4)   4097 x 515 x 1021 23 29 (1.4, 297 tiles)
    //   forward fp32 65536 x 256 x 319 160 141 (0.5)   30000 x 64 x 1001 48 82 (1.8)   2000 x 1000 x 1001 50 57 (0.3, 256 tiles)
    //   dx fp16 4097 x 515 x 1021 43 29 (0.9)   1000 x 200 x 3001 16 18 (3.2)      dx fp32 8000 x 255 x 255 33 32 (0.6)
    //   dW fp16 4097 x 515 x 1021 70 37 (1.4)   30000 x 64 x 1001 54 57 (5.3)      dW fp32 8000 x 255 x 255 43 41 (1.0)
    bool packs() const {
        const int e = elem_size(dtype);
        double copy_us = 0, products = 0;
        long long groups = 0;
        for (int s = 0; s < nseg; ++s) {
            products += (double)P * Q * red[s];
            for (const Mat& m : {a[s], b[s]}) {
                if (m.rows >= (1ll << 31) || m.cols * e >= (1ll << 22)) return false;
                if (!dma_rows(m, e)) {
                    copy_us += (double)m.rows * m.cols * e * 2 / 5e6;
                    groups += packed_groups(m, e);
                }
            }
        }
        if (groups == 0 || groups >= (1ll << 24) || (layout == FWD && P <= FEW_ROWS)) return false;
        copy_us += 5;
        if (layout == FWD && ((P + 127) / 128) * ((Q + 63) / 64) < 512) return false;
        const double aligned_us = products * 2 / (dtype == F32 ? 130e6 : 700e6);
        return copy_us < aligned_us * (dtype != F32 ? 2 : layout == DW ? 1.1 : 0.6);
    }
    int splits() const {
        if (!can_split || nseg != 1 || (layout == FWD && P <= FEW_ROWS)) return 1;
        return splits_for(P, Q, red[0], elem_size(dtype));
    }
    size_t bytes() const {
        size_t n = 0;
        if (packs())
            for (int s = 0; s < nseg; ++s)
                for (const Mat& m : {a[s], b[s]})
                    if (!dma_rows(m, elem_size(dtype))) n += packed_bytes(m, elem_size(dtype));
        if (splits() > 1) n += align256((size_t)splits() * P * Q * 4);
        return n;
    }
    // given: parts that the caller has set up and will add up itself (g.partial, g.red_part)
    int run(GemmArgs& g, char* ws, hipStream_t st, int given = 1) {
        const int e = elem_size(dtype), sp = splits();
        if (packs()) {
            PackArgs pa = {};
            long long groups = 0;
            for (int s = 0; s < nseg; ++s)
                for (Mat* m : {&a[s], &b[s]})
                    if (!dma_rows(*m, e)) {
                        const long long ldd = packed_ld(m->cols, e);
                        pa.job[pa.jobs++] = {static_cast<const char*>(m->p), reinterpret_cast<uint4*>(ws), m->ld, m->rows, m->cols, ldd * e / 16, (unsigned)groups};
                        groups += packed_groups(*m, e);
                        m->p = ws;
                        ws += packed_bytes(*m, e);
                        m->ld = ldd;
                        m->padded = true;
                    }
            const dim3 grid((unsigned)groups);
            if (e == 4) hipLaunchKernelGGL(pack_kernel<4>, grid, dim3(256), 0, st, pa);
            else if (e == 2) hipLaunchKernelGGL(pack_kernel<2>, grid, dim3(256), 0, st, pa);
            else hipLaunchKernelGGL(pack_kernel<1>, grid, dim3(256), 0, st, pa);
            NERF_LAUNCH_CHECK();
        }
        for (int s = 0; s < nseg; ++s) g.seg[s] = {a[s].p, b[s].p, a[s].ld, b[s].ld, red[s], a[s].padded, b[s].padded};
        g.nseg = nseg;
        g.P = P;
        g.Q = Q;
        g.splits = given;
        if (sp == 1) return dispatch_gemm(dtype, layout, g, st);
        const long long unit = 128;              // whole k-tiles; shorter parts cost more to add up than they save
        g.red_part = ((red[0] + sp - 1) / sp + unit - 1) / unit * unit;
        g.splits = (int)((red[0] + g.red_part - 1) / g.red_part);
        g.partial = reinterpret_cast<float*>(ws);
        int rc = dispatch_gemm(dtype, layout, g, st);
        if (rc != NERF_OK) return rc;
        const dim3 grid((unsigned)((P * ((Q + 7) / 8) + 255) / 256));
        auto finish = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(256), 0, st, g, g.splits); };
        const bool scaled = dtype == F8;
        switch (g.out_dt) {
            case F32: scaled ? finish(finish_kernel<F32, true>) : finish(finish_kernel<F32, false>); break;
            case BF16: scaled ? finish(finish_kernel<BF16, true>) : finish(finish_kernel<BF16, false>); break;
            default: scaled ? finish(finish_kernel<F16, true>) : finish(finish_kernel<F16, false>); break;
        }
        NERF_LAUNCH_CHECK();
        return NERF_OK;
    }
};

static Product forward_product(int dtype, const void* x0, long long ldx0, int k0, const void* x1, long long ldx1, int k1,
                               const void* w, long long ldw, long long M, int N) {
    const int e = elem_size(dtype);
    Product f = {};
    f.dtype = dtype;
    f.layout = FWD;
    f.nseg = k1 > 0 ? 2 : 1;
    f.a[0] = {x0, ldx0, M, k0, false};
    f.a[1] = {x1, ldx1, M, k1, false};
    f.b[0] = {w, ldw, N, k0, false};
    f.b[1] = {static_cast<const char*>(w) + (size_t)k0 * e, ldw, N, k1, false};
    f.P = M;
    f.Q = N;
    f.red[0] = k0;
    f.red[1] = k1;
    f.can_split = true;
    return f;
}

// Column sums: about 512 blocks of samples, at least 64 samples each; up to 256 samples one block that writes db itself,
// a launch less where launches are the time.
static long long colsum_rows(long long M) {
    if (M <= 256) return M;
    const long long r = (M + 511) / 512;
    return r < 64 ? 64 : r;
}
static int colsum_blocks(long long M) { return M ? (int)((M + colsum_rows(M) - 1) / colsum_rows(M)) : 0; }

// dW = gz^T x has a long reduction (the samples) and few outputs: cut into as many parts as fill the card once (one tile
// of 256 x 128 a compute unit, three of 128 x 64), not below 512 samples a part.  (One part too many is a second round:
// 65536 x 256 x 320 float32 in 258 workgroups of 256 x 128 217 us, in 255 117.)
static int dw_splits(long long M, long long N, long long K) {
    const bool wide = tile_fits(N, K, 256, 128);
    const long long tiles = wide ? ((N + 255) / 256) * ((K + 127) / 128) : ((N + 127) / 128) * ((K + 63) / 64);
    long long s = (wide ? 256 : 768) / tiles;
    const long long most = (M + 511) / 512;
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}

// The backward pass: gz where the layer has an activation, the column sums' parts, then scratch of one product at a time
// (its copies, the parts of dW).
struct Backward {
    int dtype, act;
    long long M, N, k[2];
    const void *g, *x[2], *w;
    long long ldg, ldx[2], ldw;

    bool through() const { return act != NERF_ACT_NONE; }
    long long ldgz() const { return packed_ld(N, elem_size(dtype)); }
    size_t colsum_at() const { return through() ? align256((size_t)M * ldgz() * elem_size(dtype)) : 0; }
    size_t scratch_at() const { return colsum_at() + align256((size_t)colsum_blocks(M) * N * 4); }
    Mat gz(char* ws) const {
        if (through()) return {ws, ldgz(), M, N, true};
        return {g, ldg, M, N, false};
    }
    Product dx(int piece, char* ws) const {
        Product f = {};
        f.dtype = dtype;
        f.layout = DX;
        f.nseg = 1;
        f.a[0] = gz(ws);
        f.b[0] = {static_cast<const char*>(w) + (piece ? (size_t)k[0] * elem_size(dtype) : 0), ldw, N, k[piece], false};
        f.P = M;
        f.Q = k[piece];
        f.red[0] = N;
        f.can_split = true;
        return f;
    }
    Product dw(int piece, char* ws) const {
        Product f = {};
        f.dtype = dtype;
        f.layout = DW;
        f.nseg = 1;
        f.a[0] = gz(ws);
        f.b[0] = {x[piece], ldx[piece], M, k[piece], false};
        f.P = N;
        f.Q = k[piece];
        f.red[0] = M;
        return f;
    }
    // the parts of dW stand behind its copies
    size_t dw_parts(int piece) const {
        const int s = dw_splits(M, N, k[piece]);
        return s > 1 ? align256((size_t)s * N * k[piece] * 4) : 0;
    }
    size_t bytes(bool want_x0, bool want_x1, bool want_w) const {
        size_t n = 0;
        char* ws = nullptr;
        for (int piece = 0; piece < 2; ++piece) {
            if (k[piece] == 0) continue;
            if (piece ? want_x1 : want_x0) n = std::max(n, dx(piece, ws).bytes());
            if (want_w) n = std::max(n, dw(piece, ws).bytes() + dw_parts(piece));
        }
        return scratch_at() + n;
    }
};

// Whether panel_grad_kernel takes the gradient with respect to an input piece: from 32768 rows on, and 256 outputs and
// inputs together.  Measured (us, the whole backward apart and with it; relu, gelu in bf16):
//   16384 x 256 x 256    36  36    37  38      196608 x 256 x 256   174 144   179 152     196608 x 256 x 64   128  99   134 116
//   32768 x 256 x 256    53  49    55  54      786432 x 256 x 256   647 513   662 516     196608 x 128 x 128   89  84    98  91
//   65536 x 256 x 256    87  77    89  83       65536 x 256 x 128    64  58    67  66      65536 x 128 x 64    34  35    37  39
static bool panel_grad_ok(const GemmArgs& g, const PanelGrad& a) {
    const Seg& s = g.seg[0];
    auto rows = [](const void* p, long long ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0 && ld < (1ll << 22); };
    return g.act != NERF_ACT_NONE && g.P >= 32768 && s.red > 64 && s.red <= 256 && s.red % 8 == 0 && g.Q <= 256 && g.Q % 8 == 0 && s.red + g.Q >= 256 &&
           rows(s.a, s.lda) && rows(s.b, s.ldb) && rows(g.y, g.ldy) && rows(a.z, a.ldz) && rows(a.gz, a.ldgz);
}

static bool dtype_ok(int d) { return d == F32 || d == BF16 || d == F16; }
static bool act_ok(int a) { return a >= NERF_ACT_NONE && a <= NERF_ACT_SILU; }

constexpr long long MAX_DIM = 1ll << 24;       // inputs and outputs of a layer
constexpr long long MAX_ROWS = 1ll << 31;

#define NERF_LINEAR_WORKSPACE(who, need)                                                                                \
    NERF_REQUIRE(workspace_bytes >= (need) && ((need) == 0 || workspace), who ": workspace of %zu bytes, %zu needed",   \
                 workspace_bytes, (size_t)(need));                                                                      \
    NERF_REQUIRE(((uintptr_t)workspace & 255) == 0, who ": the workspace must start on 256 bytes")
#define NERF_LINEAR_SIZES(who)                                                                                          \
    NERF_REQUIRE(M >= 0 && M < MAX_ROWS && N >= 1 && N <= MAX_DIM, who ": bad sizes M=%lld N=%d", M, N);              \
    NERF_REQUIRE(k0 >= 1 && k0 <= MAX_DIM && k1 >= 0 && k1 <= MAX_DIM, who ": bad input widths %d, %d", k0, k1)

}  // namespace lin
}  // namespace nerf

using namespace nerf;
using namespace nerf::lin;

extern "C" size_t nerf_linear_workspace_bytes(int dtype, const void* x0, long long ldx0, int k0, const void* x1, long long ldx1,
                                              int k1, const void* w, long long ldw, long long M, int N) {
    if (!dtype_ok(dtype) || M < 0 || M >= MAX_ROWS || N < 1 || N > MAX_DIM || k0 < 1 || k0 > MAX_DIM || k1 < 0 || k1 > MAX_DIM) return 0;
    return forward_product(dtype, x0, ldx0, k0, x1, ldx1, k1, w, ldw, M, N).bytes();
}

extern "C" int nerf_linear(int dtype, const void* x0, long long ldx0, int k0, const void* x1, long long ldx1, int k1,
                           const void* w, long long ldw, const void* bias, int activation, const void* residual,
                           long long ldr, void* y, long long ldy, void* z, long long ldz, long long M, int N,
                           void* workspace, size_t workspace_bytes, void* stream) {
    NERF_REQUIRE(dtype_ok(dtype), "nerf_linear: unknown type %d", dtype);
    NERF_REQUIRE(act_ok(activation), "nerf_linear: unknown activation %d", activation);
    NERF_LINEAR_SIZES("nerf_linear");
    if (M == 0) return NERF_OK;      // before the pointers: empty tensors have none
    NERF_REQUIRE(x0 && w && y && (k1 == 0 || x1), "nerf_linear: null pointer");
    NERF_REQUIRE(ldx0 >= k0 && (k1 == 0 || ldx1 >= k1) && ldw >= (long long)k0 + k1 && ldy >= N && (!residual || ldr >= N) && (!z || ldz >= N),
                 "nerf_linear: a row stride is below its row's length");
    Product f = forward_product(dtype, x0, ldx0, k0, x1, ldx1, k1, w, ldw, M, N);
    NERF_LINEAR_WORKSPACE("nerf_linear", f.bytes());
    GemmArgs g = {};
    g.bias = bias;
    g.res = residual;
    g.y = y;
    g.z = z;
    g.ldr = ldr;
    g.ldy = ldy;
    g.ldz = ldz;
    g.act = activation;
    g.out_dt = dtype;
    return f.run(g, static_cast<char*>(workspace), as_stream(stream));
}

extern "C" size_t nerf_linear_q8_workspace_bytes(const void* xq, long long ldx, const void* wq, long long ldw, long long M, int N, int K) {
    if (M < 0 || M >= MAX_ROWS || N < 1 || N > MAX_DIM || K < 1 || K > MAX_DIM) return 0;
    return forward_product(F8, xq, ldx, K, nullptr, 0, 0, wq, ldw, M, N).bytes();
}

extern "C" int nerf_linear_q8(const void* xq, long long ldx, const float* x_scale, const void* wq, long long ldw,
                              const float* w_scale, int out_dtype, const void* bias, int activation, const void* residual,
                              long long ldr, void* y, long long ldy, long long M, int N, int K, void* workspace,
                              size_t workspace_bytes, void* stream) {
    NERF_REQUIRE(dtype_ok(out_dtype), "nerf_linear_q8: unknown type %d", out_dtype);
    NERF_REQUIRE(act_ok(activation), "nerf_linear_q8: unknown activation %d", activation);
    const int k0 = K, k1 = 0;
    NERF_LINEAR_SIZES("nerf_linear_q8");
    if (M == 0) return NERF_OK;
    NERF_REQUIRE(xq && wq && x_scale && w_scale && y, "nerf_linear_q8: null pointer");
    NERF_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), "nerf_linear_q8: a row stride is below its row's length");
    Product f = forward_product(F8, xq, ldx, K, nullptr, 0, 0, wq, ldw, M, N);
    NERF_LINEAR_WORKSPACE("nerf_linear_q8", f.bytes());
    GemmArgs g = {};
    g.bias = bias;
    g.res = residual;
    g.y = y;
    g.ldr = ldr;
    g.ldy = ldy;
    g.sp = x_scale;
    g.sq = w_scale;
    g.act = activation;
    g.out_dt = out_dtype;
    return f.run(g, static_cast<char*>(workspace), as_stream(stream));
}

static Backward backward_of(int dtype, int activation, const void* g, long long ldg, const void* x0, long long ldx0, int k0,
                            const void* x1, long long ldx1, int k1, const void* w, long long ldw, long long M, int N) {
    return {dtype, activation, M, N, {k0, k1}, g, {x0, x1}, w, ldg, {ldx0, ldx1}, ldw};
}

extern "C" size_t nerf_linear_backward_workspace_bytes(int dtype, const void* g, long long ldg, int activation, const void* x0,
                                                       long long ldx0, int k0, const void* x1, long long ldx1, int k1,
                                                       const void* w, long long ldw, int want_dx0, int want_dx1, int want_dw,
                                                       long long M, int N) {
    if (!dtype_ok(dtype) || !act_ok(activation) || M < 0 || M >= MAX_ROWS || N < 1 || N > MAX_DIM || k0 < 1 || k0 > MAX_DIM ||
        k1 < 0 || k1 > MAX_DIM)
        return 0;
    return backward_of(dtype, activation, g, ldg, x0, ldx0, k0, x1, ldx1, k1, w, ldw, M, N).bytes(want_dx0, want_dx1, want_dw);
}

extern "C" int nerf_linear_backward(int dtype, const void* g, long long ldg, const void* z, long long ldz, int activation,
                                    const void* x0, long long ldx0, int k0, const void* x1, long long ldx1, int k1,
                                    const void* w, long long ldw, void* dx0, long long lddx0, void* dx1, long long lddx1,
                                    void* dw, void* db, long long M, int N, void* workspace, size_t workspace_bytes,
                                    void* stream) {
    NERF_REQUIRE(dtype_ok(dtype), "nerf_linear_backward: unknown type %d", dtype);
    NERF_REQUIRE(act_ok(activation), "nerf_linear_backward: unknown activation %d", activation);
    NERF_LINEAR_SIZES("nerf_linear_backward");
    const long long K = (long long)k0 + k1;
    hipStream_t s = as_stream(stream);
    if (M == 0) {       // no samples: the parameters' gradients are sums over nothing (before the pointers: empty tensors have none)
        int rc = NERF_OK;
        if (dw) rc = part_sum(dtype, nullptr, 0, N, K, dw, K, s);
        if (db && rc == NERF_OK) rc = part_sum(dtype, nullptr, 0, 1, N, db, N, s);
        return rc;
    }
    NERF_REQUIRE(g && (activation == NERF_ACT_NONE || z), "nerf_linear_backward: null gradient or pre-activation");
    NERF_REQUIRE(!dw || (x0 && (k1 == 0 || x1)), "nerf_linear_backward: the weight gradient needs the layer's input");
    NERF_REQUIRE((!dx0 && !dx1) || w, "nerf_linear_backward: the input gradient needs the weights");
    NERF_REQUIRE(!dx1 || k1 > 0, "nerf_linear_backward: no second input piece to take a gradient of");
    NERF_REQUIRE(ldg >= N && (activation == NERF_ACT_NONE || ldz >= N) && (!dw || (ldx0 >= k0 && (k1 == 0 || ldx1 >= k1))) &&
                     (!w || ldw >= K) && (!dx0 || lddx0 >= k0) && (!dx1 || lddx1 >= k1),
                 "nerf_linear_backward: a row stride is below its row's length");
    const Backward bw = backward_of(dtype, activation, g, ldg, x0, ldx0, k0, x1, ldx1, k1, w, ldw, M, N);
    NERF_LINEAR_WORKSPACE("nerf_linear_backward", bw.bytes(dx0 != nullptr, dx1 != nullptr, dw != nullptr));
    char* base = static_cast<char*>(workspace);
    const int e = elem_size(dtype);

    const bool through = bw.through() && (dx0 || dx1 || dw);
    float* colsum = reinterpret_cast<float*>(base + bw.colsum_at());
    int fused = -1;              // the piece whose dx comes with gz
    for (int piece = 0; piece < 2 && through && e == 2 && fused < 0; ++piece) {
        void* dx = piece ? dx1 : dx0;
        if (!dx) continue;
        const Product f = bw.dx(piece, base);
        GemmArgs a = {};
        a.seg[0] = {g, f.b[0].p, ldg, ldw, N, false, false};
        a.nseg = 1;
        a.P = M;
        a.Q = f.Q;
        a.splits = 1;
        a.y = dx;
        a.ldy = piece ? lddx1 : lddx0;
        a.act = activation;
        const PanelGrad pg = {z, base, ldz, bw.ldgz(), db ? colsum : nullptr};
        if (!panel_grad_ok(a, pg)) continue;
        fused = piece;
        int rc = dtype == BF16 ? panel_grad_bf16(a, pg, s) : panel_grad_f16(a, pg, s);
        if (rc == NERF_OK && db) rc = part_sum(dtype, colsum, PANEL_GRAD_GROUPS, 1, N, db, N, s);
        if (rc != NERF_OK) return rc;
    }
    if (fused < 0 && (through || db)) {
        ActGradArgs a = {};
        a.g = g;
        a.z = z;
        a.ldg = ldg;
        a.ldz = ldz;
        a.gz = through ? base : nullptr;
        a.ldgz = bw.ldgz();
        const bool one = colsum_blocks(M) == 1;
        a.colsum = db && !one ? colsum : nullptr;
        a.db = one ? db : nullptr;
        a.M = M;
        a.N = N;
        a.rows = colsum_rows(M);
        a.act = activation;
        const dim3 grid((unsigned)((N + AG_COLS - 1) / AG_COLS), (unsigned)colsum_blocks(M));
        switch (dtype) {
            case F32: hipLaunchKernelGGL(act_grad_kernel<F32>, grid, dim3(256), 0, s, a); break;
            case BF16: hipLaunchKernelGGL(act_grad_kernel<BF16>, grid, dim3(256), 0, s, a); break;
            default: hipLaunchKernelGGL(act_grad_kernel<F16>, grid, dim3(256), 0, s, a); break;
        }
        NERF_LAUNCH_CHECK();
        if (a.colsum) {
            const int rc = part_sum(dtype, colsum, colsum_blocks(M), 1, N, db, N, s);
            if (rc != NERF_OK) return rc;
        }
    }

    for (int piece = 0; piece < 2; ++piece) {
        const int k = piece ? k1 : k0;
        if (k == 0) continue;
        void* dx = piece ? dx1 : dx0;
        if (dx && piece != fused) {
            GemmArgs a = {};
            a.y = dx;
            a.ldy = piece ? lddx1 : lddx0;
            const int rc = bw.dx(piece, base).run(a, base + bw.scratch_at(), s);
            if (rc != NERF_OK) return rc;
        }
        if (dw) {
            Product f = bw.dw(piece, base);
            GemmArgs a = {};
            char* out = static_cast<char*>(dw) + (piece ? (size_t)k0 * e : 0);
            int sp = dw_splits(M, N, k);
            if (sp > 1) {
                const long long unit = 128 / e;          // whole k-tiles
                a.red_part = ((M + sp - 1) / sp + unit - 1) / unit * unit;
                sp = (int)((M + a.red_part - 1) / a.red_part);
                a.partial = reinterpret_cast<float*>(base + bw.scratch_at() + f.bytes());
            } else {
                a.y = out;
                a.ldy = K;
            }
            int rc = f.run(a, base + bw.scratch_at(), s, sp);
            if (rc != NERF_OK) return rc;
            if (a.partial) {
                rc = part_sum(dtype, a.partial, sp, N, k, out, K, s);
                if (rc != NERF_OK) return rc;
            }
        }
    }
    return NERF_OK;
}
