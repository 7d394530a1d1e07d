// C entry points of the linear layers, and the passes around their products: the gradient through the activation with
// the bias gradient's column sums, and the sums over the parts of a split reduction.
#include "linear.h"

namespace nerf {
namespace lin {

// gz = g act'(z) over blocks of `rows` samples, and the block's column sums.  One thread owns 8 columns (a 16-byte load
// of 16-bit types) of every (256 / groups)-th sample of its block; the sums of a column meet in LDS in a fixed order.
// Bound by memory: reads g and z, writes gz, once.
struct ActGradArgs {
    const void *g, *z;
    long long ldg, ldz;
    void* gz;                    // [M][N] or null
    float* colsum;               // [blocks][N] or null
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
                    for (int j = 0; j < 8; ++j) g[j] *= act_grad(z[j], a.act);
                }
                if (a.gz) st8<DT>(a.gz, p * a.N + q, g);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    g[j] = 0.f;
                    if (q + j < a.N) {
                        g[j] = ld_elem(a.g, p * a.ldg + q + j, DT);
                        if (a.act != NERF_ACT_NONE) g[j] *= act_grad(ld_elem(a.z, p * a.ldz + q + j, DT), a.act);
                        if (a.gz) st_elem(a.gz, p * a.N + q + j, g[j], DT);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum[j] += g[j];
        }
    }
    if (!a.colsum) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) part[ty][tx * 8 + j] = sum[j];
    __syncthreads();
    if (threadIdx.x < AG_COLS) {
        const long long c = (long long)blockIdx.x * AG_COLS + threadIdx.x;
        float s = 0.f;
#pragma unroll
        for (int r = 0; r < 32; ++r) s += part[r][threadIdx.x];
        if (c < a.N) a.colsum[(long long)blockIdx.y * a.N + c] = s;
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
// The same for many elements and few parts: one thread each.
template <int DT>
__global__ void __launch_bounds__(256) part_sum_wide_kernel(const float* parts, int n, long long all, long long cols, void* out, long long ldo) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= all) return;
    float s = 0.f;
#pragma unroll 8
    for (int k = 0; k < n; ++k) s += parts[(long long)k * all + i];
    st_elem(out, (i / cols) * ldo + i % cols, s, DT);
}

template <int DT>
static void part_sum_launch(const float* parts, int n, long long all, long long cols, void* out, long long ldo, hipStream_t s) {
    // 64 threads an element pay where one each would leave the card half empty (128 parts of 65536: 16 us against 12)
    if (all <= 16384) hipLaunchKernelGGL(part_sum_kernel<DT>, dim3((unsigned)((all + 15) / 16)), dim3(1024), 0, s, parts, n, all, cols, out, ldo);
    else hipLaunchKernelGGL(part_sum_wide_kernel<DT>, dim3((unsigned)((all + 255) / 256)), dim3(256), 0, s, parts, n, all, cols, out, ldo);
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

static int dispatch_gemm(int dtype, int layout, GemmArgs& g, hipStream_t s) {
    g.out_dt = dtype;
    switch (dtype) {
        case F32: return gemm_f32(layout, g, s);
        case BF16: return gemm_bf16(layout, g, s);
        default: return gemm_f16(layout, g, s);
    }
}

// Column sums: about 512 blocks of samples, at least 64 samples each.
static long long colsum_rows(long long M) {
    const long long r = (M + 511) / 512;
    return r < 64 ? 64 : r;
}
static int colsum_blocks(long long M) { return (int)((M + colsum_rows(M) - 1) / colsum_rows(M)); }

// dW = gz^T x has a long reduction (the samples) and few outputs: cut until about 512 workgroups of 128 x 128 have work,
// not below 512 samples a part.
static int dw_splits(long long M, long long N, long long K) {
    const long long tiles = ((N + 127) / 128) * ((K + 127) / 128);
    long long s = (512 + tiles - 1) / tiles;
    const long long most = (M + 511) / 512;
    if (s > most) s = most;
    return s < 1 ? 1 : (int)s;
}

static size_t align256(size_t b) { return (b + 255) & ~(size_t)255; }

struct Workspace {
    size_t gz, colsum, partial, all;
};
static Workspace backward_workspace(int dtype, long long M, long long N, long long k0, long long k1, int act) {
    Workspace w;
    w.gz = 0;
    w.colsum = act == NERF_ACT_NONE ? 0 : align256((size_t)M * N * elem_size(dtype));
    w.partial = w.colsum + align256((size_t)colsum_blocks(M) * N * 4);
    size_t part = 0;
    for (long long k : {k0, k1}) {
        const int sp = k > 0 ? dw_splits(M, N, k) : 1;
        if (sp > 1 && (size_t)sp * N * k * 4 > part) part = (size_t)sp * N * k * 4;
    }
    w.all = w.partial + align256(part);
    return w;
}

static bool dtype_ok(int d) { return d == F32 || d == BF16 || d == F16; }
static bool act_ok(int a) { return a >= NERF_ACT_NONE && a <= NERF_ACT_SILU; }

constexpr long long MAX_DIM = 1ll << 24;       // inputs and outputs of a layer
constexpr long long MAX_ROWS = 1ll << 31;

#define NERF_LINEAR_SIZES(who)                                                                                          \
    NERF_REQUIRE(M >= 0 && M < MAX_ROWS && N >= 1 && N <= MAX_DIM, who ": bad sizes M=%lld N=%d", M, N);              \
    NERF_REQUIRE(k0 >= 1 && k0 <= MAX_DIM && k1 >= 0 && k1 <= MAX_DIM, who ": bad input widths %d, %d", k0, k1)

}  // namespace lin
}  // namespace nerf

using namespace nerf;
using namespace nerf::lin;

extern "C" int nerf_linear(int dtype, const void* x0, long long ldx0, int k0, const void* x1, long long ldx1, int k1,
                           const void* w, long long ldw, const void* bias, int activation, const void* residual,
                           long long ldr, void* y, long long ldy, void* z, long long ldz, long long M, int N, void* stream) {
    NERF_REQUIRE(dtype_ok(dtype), "nerf_linear: unknown type %d", dtype);
    NERF_REQUIRE(act_ok(activation), "nerf_linear: unknown activation %d", activation);
    NERF_LINEAR_SIZES("nerf_linear");
    if (M == 0) return NERF_OK;      // before the pointers: empty tensors have none
    NERF_REQUIRE(x0 && w && y && (k1 == 0 || x1), "nerf_linear: null pointer");
    NERF_REQUIRE(ldx0 >= k0 && (k1 == 0 || ldx1 >= k1) && ldw >= (long long)k0 + k1 && ldy >= N && (!residual || ldr >= N) && (!z || ldz >= N),
                 "nerf_linear: a row stride is below its row's length");
    const int e = elem_size(dtype);
    GemmArgs g = {};
    g.seg[0] = {x0, w, ldx0, ldw, k0};
    g.seg[1] = {x1, static_cast<const char*>(w) + (size_t)k0 * e, ldx1, ldw, k1};
    g.nseg = k1 > 0 ? 2 : 1;
    g.P = M;
    g.Q = N;
    g.splits = 1;
    g.bias = bias;
    g.res = residual;
    g.y = y;
    g.z = z;
    g.ldr = ldr;
    g.ldy = ldy;
    g.ldz = ldz;
    g.act = activation;
    return dispatch_gemm(dtype, FWD, g, as_stream(stream));
}

extern "C" int nerf_linear_q8(const void* xq, long long ldx, const float* x_scale, const void* wq, long long ldw,
                              const float* w_scale, int out_dtype, const void* bias, int activation, const void* residual,
                              long long ldr, void* y, long long ldy, long long M, int N, int K, void* stream) {
    NERF_REQUIRE(dtype_ok(out_dtype), "nerf_linear_q8: unknown type %d", out_dtype);
    NERF_REQUIRE(act_ok(activation), "nerf_linear_q8: unknown activation %d", activation);
    const int k0 = K, k1 = 0;
    NERF_LINEAR_SIZES("nerf_linear_q8");
    if (M == 0) return NERF_OK;
    NERF_REQUIRE(xq && wq && x_scale && w_scale && y, "nerf_linear_q8: null pointer");
    NERF_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!residual || ldr >= N), "nerf_linear_q8: a row stride is below its row's length");
    GemmArgs g = {};
    g.seg[0] = {xq, wq, ldx, ldw, K};
    g.nseg = 1;
    g.P = M;
    g.Q = N;
    g.splits = 1;
    g.bias = bias;
    g.res = residual;
    g.y = y;
    g.ldr = ldr;
    g.ldy = ldy;
    g.sp = x_scale;
    g.sq = w_scale;
    g.act = activation;
    g.out_dt = out_dtype;
    return gemm_f8(g, as_stream(stream));
}

extern "C" size_t nerf_linear_backward_workspace_bytes(int dtype, long long M, int N, int k0, int k1, int activation) {
    if (!dtype_ok(dtype) || !act_ok(activation) || M < 0 || M >= MAX_ROWS || N < 1 || N > MAX_DIM || k0 < 1 || k0 > MAX_DIM ||
        k1 < 0 || k1 > MAX_DIM)
        return 0;
    return backward_workspace(dtype, M, N, k0, k1, activation).all;
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
    const Workspace ws = backward_workspace(dtype, M, N, k0, k1, activation);
    NERF_REQUIRE(workspace_bytes >= ws.all && (ws.all == 0 || workspace), "nerf_linear_backward: workspace of %zu bytes, %zu needed",
                 workspace_bytes, ws.all);
    NERF_REQUIRE(((uintptr_t)workspace & 255) == 0, "nerf_linear_backward: the workspace must start on 256 bytes");
    char* base = static_cast<char*>(workspace);
    const int e = elem_size(dtype);

    const bool through = activation != NERF_ACT_NONE && (dx0 || dx1 || dw);
    float* colsum = reinterpret_cast<float*>(base + ws.colsum);
    if (through || db) {
        ActGradArgs a = {};
        a.g = g;
        a.z = z;
        a.ldg = ldg;
        a.ldz = ldz;
        a.gz = through ? base + ws.gz : nullptr;
        a.colsum = db ? colsum : nullptr;
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
        if (db) {
            const int rc = part_sum(dtype, colsum, colsum_blocks(M), 1, N, db, N, s);
            if (rc != NERF_OK) return rc;
        }
    }
    const void* gz = through ? base + ws.gz : g;
    const long long ldgz = through ? N : ldg;

    for (int piece = 0; piece < 2; ++piece) {
        const int k = piece ? k1 : k0;
        if (k == 0) continue;
        const char* wp = static_cast<const char*>(w) + (piece ? (size_t)k0 * e : 0);
        void* dx = piece ? dx1 : dx0;
        if (dx) {
            GemmArgs a = {};
            a.seg[0] = {gz, wp, ldgz, ldw, N};
            a.nseg = 1;
            a.P = M;
            a.Q = k;
            a.splits = 1;
            a.y = dx;
            a.ldy = piece ? lddx1 : lddx0;
            const int rc = dispatch_gemm(dtype, DX, a, s);
            if (rc != NERF_OK) return rc;
        }
        if (dw) {
            GemmArgs a = {};
            a.seg[0] = {gz, piece ? x1 : x0, ldgz, piece ? ldx1 : ldx0, M};
            a.nseg = 1;
            a.P = N;
            a.Q = k;
            a.splits = dw_splits(M, N, k);
            char* out = static_cast<char*>(dw) + (piece ? (size_t)k0 * e : 0);
            if (a.splits > 1) {
                const long long unit = 128;              // a multiple of every type's k-tile
                a.red_part = ((M + a.splits - 1) / a.splits + unit - 1) / unit * unit;
                a.splits = (int)((M + a.red_part - 1) / a.red_part);
                a.partial = reinterpret_cast<float*>(base + ws.partial);
            } else {
                a.y = out;
                a.ldy = K;
            }
            int rc = dispatch_gemm(dtype, DW, a, s);
            if (rc != NERF_OK) return rc;
            if (a.partial) {
                rc = part_sum(dtype, a.partial, a.splits, N, k, out, K, s);
                if (rc != NERF_OK) return rc;
            }
        }
    }
    return NERF_OK;
}
