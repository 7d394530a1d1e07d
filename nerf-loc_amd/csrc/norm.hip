// Root-mean-square norm behind a residual addition, forward, backward and with an 8-bit output:
//
//     h = x + r                      (float32; stored rounded to the type)
//     y = w h rstd,   rstd = 1 / sqrt(mean(h^2) + eps)
//     8 bits: s = max(max|y| / 448, 2^-126) per row, q = e4m3(y / s) with one rounding of 1 / s
//     dx = dr = gh + rstd (gy w) - h rstd^3 mean(gy w h),   dw = sum over rows of gy h rstd
//
// A row stays in the registers of the ROWT threads that own it from its one read to its one write; its sums meet in the
// wave by shuffles and, above 64 threads, in LDS.  Bound by memory.
#include "linear.h"

namespace nerf {
namespace lin {

constexpr float E4M3_MAX = 448.f;
constexpr float SCALE_MIN = 1.1754943508222875e-38f;        // 2^-126: a row of zeros divides by it

struct NormArgs {
    const void *x, *r, *w;
    void *h, *y;
    unsigned char* q;
    float *scale, *rstd;
    long long ldx, ldr, ldh, ldy, ldq, M;
    int N;
    float eps;
};
struct NormGradArgs {
    const void *gy, *gh, *h, *w;
    const float* rstd;
    void* dx;
    float* dw_part;              // [blocks][N] or null
    void* dw;                    // [N]: the sums themselves, where one workgroup has all rows; or null
    long long ldgy, ldgh, ldh, lddx, M;
    int N;
};

// eight elements from column c, zeros behind column n
template <int DT>
__device__ __forceinline__ void row8(const void* p, long long base, int c, int n, float (&v)[8]) {
    if (c + 8 <= n) ld8<DT>(p, base + c, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < n ? ld_elem(p, base + c + j, DT) : 0.f;
    }
}
template <int DT>
__device__ __forceinline__ void put8(void* p, long long base, int c, int n, const float (&v)[8]) {
    if (c + 8 <= n) st8<DT>(p, base + c, v);
    else {
#pragma unroll
        for (int j = 0; j < 8; ++j) if (c + j < n) st_elem(p, base + c + j, v[j], DT);
    }
}

// Eight elements as they lie in memory.
template <int DT>
struct Raw {
    static constexpr int E = elem_size(DT);
    unsigned v[2 * E];
    __device__ __forceinline__ void get(const void* p, long long base, int c, int n) {
        const char* q = static_cast<const char*>(p) + (base + c) * E;
        if (c + 8 <= n) __builtin_memcpy(v, q, 8 * E);
        else {
#pragma unroll
            for (int j = 0; j < 2 * E; ++j) v[j] = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (c + j < n) {
                    if constexpr (E == 4) v[j] = reinterpret_cast<const unsigned*>(q)[j];
                    else v[j >> 1] |= (unsigned)reinterpret_cast<const unsigned short*>(q)[j] << (16 * (j & 1));
                }
            }
        }
    }
    __device__ __forceinline__ void put(float (&f)[8]) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (DT == F32) f[j] = __uint_as_float(v[j]);
            else if constexpr (DT == BF16) f[j] = __uint_as_float(j & 1 ? v[j >> 1] & 0xffff0000u : v[j >> 1] << 16);
            else {
                const unsigned short u = (unsigned short)(v[j >> 1] >> (16 * (j & 1)));
                f[j] = (float)__builtin_bit_cast(_Float16, u);
            }
        }
    }
};

// Sum (or, of absolute values' bits, the maximum: NaN above infinity above all numbers) over the ROWT threads of a row.
template <int ROWT>
__device__ __forceinline__ float row_sum(float v, float* shared) {
    constexpr int W = ROWT < 64 ? ROWT : 64;
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
    if constexpr (ROWT > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < ROWT / 64; ++i) v += shared[i];
    }
    return v;
}
template <int ROWT>
__device__ __forceinline__ unsigned row_max(unsigned v, float* shared) {
    constexpr int W = ROWT < 64 ? ROWT : 64;
#pragma unroll
    for (int d = W / 2; d >= 1; d >>= 1) {
        const unsigned o = __shfl_xor(v, d, 64);
        v = o > v ? o : v;
    }
    if constexpr (ROWT > 64) {
        __syncthreads();
        if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = __uint_as_float(v);
        __syncthreads();
        v = 0;
#pragma unroll
        for (int i = 0; i < ROWT / 64; ++i) {
            const unsigned o = __float_as_uint(shared[i]);
            v = o > v ? o : v;
        }
    }
    return v;
}

template <int DT, int ROWT, int VPT, bool Q8>
__global__ void __launch_bounds__(ROWT < 256 ? 256 : ROWT) norm_kernel(const NormArgs a) {
    constexpr int NT = ROWT < 256 ? 256 : ROWT;
    __shared__ float shared[16];
    const int t = threadIdx.x % ROWT;
    // two grid dimensions: a launch counts its threads in 32 bits along one
    const long long row = ((long long)blockIdx.y * gridDim.x + blockIdx.x) * (NT / ROWT) + threadIdx.x / ROWT;
    const bool live = row < a.M;
    const long long rw = live ? row : a.M - 1;          // idle threads of the last workgroup follow its last row
    float h[VPT][8], ss = 0.f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (k * ROWT + t) * 8;
        row8<DT>(a.x, rw * a.ldx, c, a.N, h[k]);
        if (a.r) {
            float r[8];
            row8<DT>(a.r, rw * a.ldr, c, a.N, r);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[k][j] += r[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(h[k][j], h[k][j], ss);
    }
    ss = row_sum<ROWT>(ss, shared);
    const float rstd = 1.f / sqrtf(ss / (float)a.N + a.eps);
    if (live && a.h) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * ROWT + t) * 8;
            if (c < a.N) put8<DT>(a.h, row * a.ldh, c, a.N, h[k]);
        }
    }
    if (live && a.rstd && t == 0) a.rstd[row] = rstd;
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (k * ROWT + t) * 8;
        float w[8];
        row8<DT>(a.w, 0, c, a.N, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            h[k][j] = h[k][j] * rstd * w[j];
            if constexpr (Q8) {
                const unsigned b = c + j < a.N ? __float_as_uint(h[k][j]) & 0x7fffffffu : 0u;
                top = b > top ? b : top;
            }
        }
        if constexpr (!Q8) {
            if (live && c < a.N) put8<DT>(a.y, row * a.ldy, c, a.N, h[k]);
        }
    }
    if constexpr (Q8) {
        top = row_max<ROWT>(top, shared);
        float s = __uint_as_float(top) / E4M3_MAX;
        s = s < SCALE_MIN ? SCALE_MIN : s;
        const float inv = 1.f / s;
        if (live && t == 0) a.scale[row] = s;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * ROWT + t) * 8;
            unsigned lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[k][0] * inv, h[k][1] * inv, 0, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(h[k][2] * inv, h[k][3] * inv, lo, true);
            unsigned hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[k][4] * inv, h[k][5] * inv, 0, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(h[k][6] * inv, h[k][7] * inv, hi, true);
            unsigned char* o = a.q + row * a.ldq + c;
            if (live && c + 8 <= a.N) {
                const uint2 v = make_uint2(lo, hi);
                __builtin_memcpy(o, &v, 8);
            } else if (live) {
#pragma unroll
                for (int j = 0; j < 8; ++j) if (c + j < a.N) o[j] = (unsigned char)((j < 4 ? lo : hi) >> (8 * (j & 3)));
            }
        }
    }
}

// Persistent workgroups walk the rows with the columns' dw sums in registers; a column's sums over the rows that one
// workgroup holds side by side meet in LDS at the end, those of the workgroups in part_sum, always in the same order.
template <int DT, int ROWT, int VPT>
__global__ void __launch_bounds__(ROWT < 256 ? 256 : ROWT) norm_grad_kernel(const NormGradArgs a) {
    constexpr int NT = ROWT < 256 ? 256 : ROWT, ROWS = NT / ROWT;
    __shared__ float shared[16];
    __shared__ float sums[ROWS > 1 ? ROWS * ROWT * VPT * 8 : 1];
    const int t = threadIdx.x % ROWT, mine = threadIdx.x / ROWT;
    float dw[VPT][8] = {};
    for (long long first = (long long)blockIdx.x * ROWS; first < a.M; first += (long long)gridDim.x * ROWS) {
        const long long row = first + mine;
        const bool live = row < a.M;
        const long long rw = live ? row : a.M - 1;
        const float rstd = a.rstd[rw];
        // everything the row needs is asked for at once, and stays as it came (packed, for 16-bit types) until used
        Raw<DT> h[VPT], gy[VPT], gh[VPT], w[VPT];
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * ROWT + t) * 8;
            h[k].get(a.h, rw * a.ldh, c, a.N);
            gy[k].get(a.gy, rw * a.ldgy, c, a.N);
            if (a.gh) gh[k].get(a.gh, rw * a.ldgh, c, a.N);
            w[k].get(a.w, 0, c, a.N);
        }
        float dot = 0.f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float hv[8], gv[8], wv[8];
            h[k].put(hv);
            gy[k].put(gv);
            w[k].put(wv);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float hn = hv[j] * rstd;
                if (live) dw[k][j] = fmaf(gv[j], hn, dw[k][j]);
                dot = fmaf(gv[j] * wv[j], hn, dot);
            }
        }
        dot = row_sum<ROWT>(dot, shared) / (float)a.N;
        if (!a.dx) continue;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * ROWT + t) * 8;
            float hv[8], gv[8], wv[8], g[8] = {};
            h[k].put(hv);
            gy[k].put(gv);
            w[k].put(wv);
            if (a.gh) gh[k].put(g);
#pragma unroll
            for (int j = 0; j < 8; ++j) g[j] = fmaf(rstd, fmaf(-dot, hv[j] * rstd, gv[j] * wv[j]), g[j]);
            if (live && c < a.N) put8<DT>(a.dx, row * a.lddx, c, a.N, g);
        }
    }
    if (!a.dw_part && !a.dw) return;
    if constexpr (ROWS == 1) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (k * ROWT + t) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (c + j >= a.N) continue;
                if (a.dw) st_elem(a.dw, c + j, dw[k][j], DT);
                else a.dw_part[(long long)blockIdx.x * a.N + c + j] = dw[k][j];
            }
        }
    } else {
        constexpr int COLS = ROWT * VPT * 8;
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[mine * COLS + (k * ROWT + t) * 8 + j] = dw[k][j];
        __syncthreads();
        for (int c = threadIdx.x; c < COLS && c < a.N; c += NT) {
            float s = 0.f;
            for (int r = 0; r < ROWS; ++r) s += sums[r * COLS + c];
            if (a.dw) st_elem(a.dw, c, s, DT);
            else a.dw_part[(long long)blockIdx.x * a.N + c] = s;
        }
    }
}

constexpr int NORM_MAX = 32768;      // 1024 threads x 4 x 8 columns

// Threads per row: the fewest that hold it in at most four 8-column pieces each.
#define NERF_NORM_SWITCH(N, CALL)                                  \
    do {                                                           \
        if ((N) <= 32) { CALL(4, 1); }                             \
        else if ((N) <= 128) { CALL(16, 1); }                      \
        else if ((N) <= 512) { CALL(64, 1); }                      \
        else if ((N) <= 1024) { CALL(64, 2); }                     \
        else if ((N) <= 2048) { CALL(256, 1); }                    \
        else if ((N) <= 4096) { CALL(256, 2); }                    \
        else if ((N) <= 8192) { CALL(1024, 1); }                   \
        else if ((N) <= 16384) { CALL(1024, 2); }                  \
        else { CALL(1024, 4); }                                    \
    } while (0)

static int norm_rows(int N) { return N <= 32 ? 64 : N <= 128 ? 16 : N <= 1024 ? 4 : 1; }
static long long norm_grad_blocks(long long M, int N) {
    const long long all = (M + norm_rows(N) - 1) / norm_rows(N);
    const long long most = N <= 2048 ? 1024 : 512;
    return all < most ? all : most;
}

template <int DT>
static int norm_launch(const NormArgs& a, hipStream_t s) {
#define NERF_CALL(T, V)                                                                                                   \
    {                                                                                                                     \
        constexpr int NT = T < 256 ? 256 : T;                                                                             \
        const long long groups = (a.M + NT / T - 1) / (NT / T), wide = groups < (1ll << 20) ? groups : 1ll << 20;          \
        const dim3 grid((unsigned)wide, (unsigned)((groups + wide - 1) / wide));                                          \
        if (a.q) hipLaunchKernelGGL((norm_kernel<DT, T, V, true>), grid, dim3(NT), 0, s, a);                              \
        else hipLaunchKernelGGL((norm_kernel<DT, T, V, false>), grid, dim3(NT), 0, s, a);                                 \
    }
    NERF_NORM_SWITCH(a.N, NERF_CALL);
#undef NERF_CALL
    NERF_LAUNCH_CHECK();
    return NERF_OK;
}
template <int DT>
static int norm_grad_launch(NormGradArgs a, void* dw, hipStream_t s) {
    const long long blocks = norm_grad_blocks(a.M, a.N);
    if (blocks == 1) {
        a.dw = dw;
        a.dw_part = nullptr;
    }
    if (blocks > 0) {
#define NERF_CALL(T, V) hipLaunchKernelGGL((norm_grad_kernel<DT, T, V>), dim3((unsigned)blocks), dim3(T < 256 ? 256 : T), 0, s, a)
        NERF_NORM_SWITCH(a.N, NERF_CALL);
#undef NERF_CALL
        NERF_LAUNCH_CHECK();
    }
    return dw && blocks != 1 ? part_sum(DT, a.dw_part, (int)blocks, 1, a.N, dw, a.N, s) : NERF_OK;
}

}  // namespace lin
}  // namespace nerf

using namespace nerf;
using namespace nerf::lin;

extern "C" int nerf_add_rms_norm(int dtype, const void* x, long long ldx, const void* residual, long long ldr, const void* w,
                                 float eps, void* h, long long ldh, void* y, long long ldy, void* q, long long ldq,
                                 float* scale, float* rstd, long long M, int N, void* stream) {
    NERF_REQUIRE(dtype == F32 || dtype == BF16 || dtype == F16, "nerf_add_rms_norm: unknown type %d", dtype);
    NERF_REQUIRE(M >= 0 && M < (1ll << 31) && N >= 1 && N <= NORM_MAX, "nerf_add_rms_norm: bad sizes M=%lld N=%d (at most %d columns)", M, N, NORM_MAX);
    if (M == 0) return NERF_OK;      // before the pointers: empty tensors have none
    NERF_REQUIRE(x && w && ((y != nullptr) != (q != nullptr)) && (!q || scale), "nerf_add_rms_norm: needs x, w and either y or q with scale");
    NERF_REQUIRE(ldx >= N && (!residual || ldr >= N) && (!h || ldh >= N) && (!y || ldy >= N) && (!q || ldq >= N),
                 "nerf_add_rms_norm: a row stride is below its row's length");
    NERF_REQUIRE(eps >= 0.f, "nerf_add_rms_norm: eps must not be negative");
    const NormArgs a = {x, residual, w, h, y, static_cast<unsigned char*>(q), scale, rstd, ldx, ldr, ldh, ldy, ldq, M, N, eps};
    hipStream_t s = as_stream(stream);
    switch (dtype) {
        case F32: return norm_launch<F32>(a, s);
        case BF16: return norm_launch<BF16>(a, s);
        default: return norm_launch<F16>(a, s);
    }
}

extern "C" size_t nerf_add_rms_norm_backward_workspace_bytes(long long M, int N) {
    if (M < 0 || M >= (1ll << 31) || N < 1 || N > NORM_MAX) return 0;
    return (size_t)norm_grad_blocks(M, N) * N * 4;
}

extern "C" int nerf_add_rms_norm_backward(int dtype, const void* gy, long long ldgy, const void* gh, long long ldgh,
                                          const void* h, long long ldh, const void* w, const float* rstd, void* dx,
                                          long long lddx, void* dw, long long M, int N, void* workspace,
                                          size_t workspace_bytes, void* stream) {
    NERF_REQUIRE(dtype == F32 || dtype == BF16 || dtype == F16, "nerf_add_rms_norm_backward: unknown type %d", dtype);
    NERF_REQUIRE(M >= 0 && M < (1ll << 31) && N >= 1 && N <= NORM_MAX, "nerf_add_rms_norm_backward: bad sizes M=%lld N=%d (at most %d columns)", M, N, NORM_MAX);
    NERF_REQUIRE(M == 0 || (gy && h && w && rstd && (dx || dw)), "nerf_add_rms_norm_backward: null pointer");
    NERF_REQUIRE(ldgy >= N && (!gh || ldgh >= N) && ldh >= N && (!dx || lddx >= N), "nerf_add_rms_norm_backward: a row stride is below its row's length");
    const size_t need = dw ? (size_t)norm_grad_blocks(M, N) * N * 4 : 0;
    NERF_REQUIRE(workspace_bytes >= need && (need == 0 || workspace), "nerf_add_rms_norm_backward: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    const NormGradArgs a = {gy, gh, h, w, rstd, dx, dw ? static_cast<float*>(workspace) : nullptr, nullptr, ldgy, ldgh, ldh, lddx, M, N};
    hipStream_t s = as_stream(stream);
    switch (dtype) {
        case F32: return norm_grad_launch<F32>(a, dw, s);
        case BF16: return norm_grad_launch<BF16>(a, dw, s);
        default: return norm_grad_launch<F16>(a, dw, s);
    }
}
