// Layer norm over the channels of each row (a pixel or a token), summed over the branches of a block, and its backward pass.
//
//   xhat_b[r][c] = (z_b[r][c] - mean_c z_b[r]) / sqrt(var_c z_b[r] + eps)            (biased variance)
//   y[r][c]      = act( sum_b xhat_b[r][c] * gamma_b[c] + beta_b[c] )                 act: identity or ReLU
//   u = dy (ReLU: 0 where y <= 0),  w_b = u * gamma_b
//   dz_b         = (w_b - mean_c w_b - xhat_b * mean_c (w_b * xhat_b)) / sqrt(var + eps)
//   dgamma_b[c]  = sum_r u * xhat_b,   dbeta[c] = sum_r u   (the same for every branch)
//
// One branch without ReLU is the plain layer norm.  Sums, statistics and weights are fp32; activations fp32 or bf16, rounded
// once on the way out.  The variance is the mean of (z - mean)^2: rows far from zero lose nothing.  Statistics are not handed
// from forward to backward: the backward has the row at hand and computes them again, 8 bytes per row and branch less in both.
// NaN stays NaN through the ReLU, and passes gradient, as in torch.
#include "common.h"

constexpr int LN_MAXB = 8;

struct LnArgs {
    const void* z[LN_MAXB];
    void* dz[LN_MAXB];                  // dense [M][C]
    const float* gamma[LN_MAXB];        // NULL: 1
    const float* beta[LN_MAXB];         // NULL: 0
    int ldz[LN_MAXB];
    int nb, C;
    long long M;
    float eps;
};

// ---------------------------------------------------------------------------------------------
// Any width: one wave per row, elements strided over the lanes, the row read once per pass (the passes after the first hit L2).

template <typename T>
__device__ __forceinline__ void ln_row_stats(const T* z, int C, float eps, float& mean, float& rstd) {
    const int lane = threadIdx.x & 63;
    float s = 0.f;
    for (int c = lane; c < C; c += 64) s += to_f32(z[c]);
    mean = wave_sum64(s) / (float)C;
    float q = 0.f;
    for (int c = lane; c < C; c += 64) { const float d = to_f32(z[c]) - mean; q += d * d; }
    rstd = 1.f / sqrtf(wave_sum64(q) / (float)C + eps);
}

template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_rows_kernel(LnArgs a, T* __restrict__ y, int ldy, int relu) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.M; r += (long long)gridDim.x * 4) {
        float mean[LN_MAXB], rstd[LN_MAXB];
#pragma unroll
        for (int b = 0; b < LN_MAXB; ++b)
            if (b < a.nb) ln_row_stats((const T*)a.z[b] + r * a.ldz[b], a.C, a.eps, mean[b], rstd[b]);
        for (int c = lane; c < a.C; c += 64) {
            float o = 0.f;
#pragma unroll
            for (int b = 0; b < LN_MAXB; ++b) {
                if (b < a.nb) {
                    const float x = (to_f32(((const T*)a.z[b])[r * a.ldz[b] + c]) - mean[b]) * rstd[b];
                    o += x * (a.gamma[b] ? a.gamma[b][c] : 1.f) + (a.beta[b] ? a.beta[b][c] : 0.f);
                }
            }
            if (relu && o < 0.f) o = 0.f;
            y[r * ldy + c] = from_f32<T>(o);
        }
    }
}

// u with the ReLU mask applied; y == NULL: no ReLU
template <typename T>
__device__ __forceinline__ float ln_u(const T* dy, const T* y, long long i, long long j) {
    const float u = to_f32(dy[i]);
    return y != nullptr && to_f32(y[j]) <= 0.f ? 0.f : u;
}

// dz of every branch; stats [nb][M][2] = (mean, rstd) for the column pass
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_rows_kernel(LnArgs a, const T* __restrict__ dy, int lddy, const T* __restrict__ y, int ldy,
                                                          float* __restrict__ stats) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.M; r += (long long)gridDim.x * 4) {
        for (int b = 0; b < a.nb; ++b) {
            const T* z = (const T*)a.z[b] + r * a.ldz[b];
            const float* gamma = a.gamma[b];
            float mean, rstd;
            ln_row_stats(z, a.C, a.eps, mean, rstd);
            float s1 = 0.f, s2 = 0.f;
            for (int c = lane; c < a.C; c += 64) {
                const float w = ln_u(dy, y, r * lddy + c, r * ldy + c) * (gamma ? gamma[c] : 1.f);
                s1 += w;
                s2 += w * ((to_f32(z[c]) - mean) * rstd);
            }
            const float m1 = wave_sum64(s1) / (float)a.C, m2 = wave_sum64(s2) / (float)a.C;
            T* dz = (T*)a.dz[b] + r * a.C;
            for (int c = lane; c < a.C; c += 64) {
                const float w = ln_u(dy, y, r * lddy + c, r * ldy + c) * (gamma ? gamma[c] : 1.f);
                const float x = (to_f32(z[c]) - mean) * rstd;
                dz[c] = from_f32<T>(rstd * (w - m1 - x * m2));
            }
            if (lane == 0) { stats[((size_t)b * a.M + r) * 2] = mean; stats[((size_t)b * a.M + r) * 2 + 1] = rstd; }
        }
    }
}

// blockIdx.x: 64 columns, blockIdx.y: a run of rows -> part[blockIdx.y][nb + 1][C] (q < nb: sum u*xhat_q, q == nb: sum u)
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols_kernel(LnArgs a, const T* __restrict__ dy, int lddy, const T* __restrict__ y, int ldy,
                                                          const float* __restrict__ stats, long long rows_per, float* __restrict__ part) {
    __shared__ float red[4][LN_MAXB + 1][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * 64 + lane;
    const long long r0 = (long long)blockIdx.y * rows_per;
    const long long r1 = r0 + rows_per < a.M ? r0 + rows_per : a.M;
    float acc[LN_MAXB + 1];
#pragma unroll
    for (int q = 0; q <= LN_MAXB; ++q) acc[q] = 0.f;
    if (c < a.C) {
        for (long long r = r0 + wave; r < r1; r += 4) {
            const float u = ln_u(dy, y, r * lddy + c, r * ldy + c);
            acc[LN_MAXB] += u;
#pragma unroll
            for (int b = 0; b < LN_MAXB; ++b) {
                if (b < a.nb) {
                    const float* st = stats + ((size_t)b * a.M + r) * 2;
                    acc[b] += u * ((to_f32(((const T*)a.z[b])[r * a.ldz[b] + c]) - st[0]) * st[1]);
                }
            }
        }
    }
#pragma unroll
    for (int q = 0; q <= LN_MAXB; ++q) red[wave][q][lane] = acc[q];
    __syncthreads();
    for (int i = threadIdx.x; i < (a.nb + 1) * 64; i += 256) {
        const int q = i >> 6, l = i & 63, src = q == a.nb ? LN_MAXB : q;
        if (blockIdx.x * 64 + l < a.C)
            part[((size_t)blockIdx.y * (a.nb + 1) + q) * a.C + blockIdx.x * 64 + l] =
                (red[0][src][l] + red[1][src][l]) + (red[2][src][l] + red[3][src][l]);
    }
}

struct LnGrads {
    float* dgamma[LN_MAXB];
    float* dbeta[LN_MAXB];
};

// part [rows][nb + 1][C] -> dgamma_b, dbeta_b: one thread per column and quantity, fp64 sums in row order (no atomics: the same
// bits every time)
__global__ __launch_bounds__(256) void ln_bwd_finalize_kernel(const float* __restrict__ part, int rows, int nb, int C, LnGrads g) {
    const int c = blockIdx.x * 256 + threadIdx.x, q = blockIdx.y;
    if (c >= C) return;
    double s = 0.0;
    for (int r = 0; r < rows; ++r) s += (double)part[((size_t)r * (nb + 1) + q) * C + c];
    if (q < nb) {
        if (g.dgamma[q]) g.dgamma[q][c] = (float)s;
    } else {
        for (int b = 0; b < nb; ++b)
            if (g.dbeta[b]) g.dbeta[b][c] = (float)s;
    }
}

// ---------------------------------------------------------------------------------------------------

static inline int ln_parts(long long M) {
    const long long n = (M + 63) / 64;
    return (int)(n < 256 ? n : 256);
}

static int ln_args(LnArgs& a, const char* what, int dtype, int nb, const void* const* z, const int* ldz, const int* zoff,
                   const float* const* gamma, const float* const* beta, long long M, int C, float eps) {
    UNET_CHECK(dtype == UNET_F32 || dtype == UNET_BF16, "%s: bad dtype %d", what, dtype);
    UNET_CHECK(nb >= 1 && nb <= LN_MAXB, "%s: 1..%d branches (got %d)", what, LN_MAXB, nb);
    UNET_CHECK(M >= 0 && M < (1LL << 40) && C >= 1 && C <= (1 << 24), "%s: bad shape (%lld rows of %d channels)", what, M, C);
    UNET_CHECK(eps >= 0.f, "%s: eps must not be negative", what);
    UNET_CHECK(z && ldz && zoff, "%s: null argument", what);
    const size_t size = dtype == UNET_BF16 ? 2 : 4;
    a.nb = nb; a.C = C; a.M = M; a.eps = eps;
    for (int b = 0; b < nb; ++b) {
        UNET_CHECK(z[b] || M == 0, "%s: branch %d is null", what, b);
        UNET_CHECK(zoff[b] >= 0 && (long long)zoff[b] + C <= ldz[b], "%s: branch %d: channel slice outside the buffer", what, b);
        a.z[b] = (const char*)z[b] + (size_t)zoff[b] * size;
        a.ldz[b] = ldz[b];
        a.gamma[b] = gamma ? gamma[b] : nullptr;
        a.beta[b] = beta ? beta[b] : nullptr;
        a.dz[b] = nullptr;
    }
    for (int b = nb; b < LN_MAXB; ++b) { a.z[b] = nullptr; a.dz[b] = nullptr; a.gamma[b] = a.beta[b] = nullptr; a.ldz[b] = 0; }
    return 0;
}

static inline int ln_grid(long long M, int rows_per_wg) {
    const long long n = (M + rows_per_wg - 1) / rows_per_wg;
    return (int)(n < 8192 ? n : 8192);
}

extern "C" int unet_layer_norm_fwd(int dtype, int relu, int nb, const void* const* z, const int* ldz, const int* zoff,
                                   const float* const* gamma, const float* const* beta, void* y, int ldy, int yoff,
                                   long long M, int C, float eps, void* stream) {
    LnArgs a;
    const int rc = ln_args(a, "layer_norm_fwd", dtype, nb, z, ldz, zoff, gamma, beta, M, C, eps);
    if (rc) return rc;
    UNET_CHECK(y || M == 0, "layer_norm_fwd: null output");
    UNET_CHECK(yoff >= 0 && (long long)yoff + C <= ldy, "layer_norm_fwd: output slice outside the buffer");
    if (M == 0) return 0;
    hipStream_t s = (hipStream_t)stream;
    if (dtype == UNET_BF16)
        hipLaunchKernelGGL((ln_fwd_rows_kernel<__bf16>), dim3(ln_grid(M, 4)), dim3(256), 0, s, a, (__bf16*)y + yoff, ldy, relu);
    else
        hipLaunchKernelGGL((ln_fwd_rows_kernel<float>), dim3(ln_grid(M, 4)), dim3(256), 0, s, a, (float*)y + yoff, ldy, relu);
    UNET_LAUNCH_CHECK();
    return 0;
}

extern "C" int unet_layer_norm_bwd_ws(int dtype, int nb, long long M, int C) {
    if (nb < 1 || nb > LN_MAXB || M < 0 || C < 1) return -1;
    const double n = 2.0 * nb * (double)M + (double)ln_parts(M) * (nb + 1) * C;
    return n > 2147483647.0 ? -1 : (int)n;
}

extern "C" int unet_layer_norm_bwd(int dtype, int nb, const void* dy, int lddy, int dyoff, const void* y, int ldy, int yoff,
                                   const void* const* z, const int* ldz, const int* zoff, const float* const* gamma,
                                   void* const* dz, float* const* dgamma, float* const* dbeta, float* ws, int ws_size,
                                   long long M, int C, float eps, void* stream) {
    LnArgs a;
    const int rc = ln_args(a, "layer_norm_bwd", dtype, nb, z, ldz, zoff, gamma, nullptr, M, C, eps);
    if (rc) return rc;
    UNET_CHECK(dy || M == 0, "layer_norm_bwd: null gradient");
    UNET_CHECK(dyoff >= 0 && (long long)dyoff + C <= lddy, "layer_norm_bwd: gradient slice outside the buffer");
    UNET_CHECK(!y || (yoff >= 0 && (long long)yoff + C <= ldy), "layer_norm_bwd: output slice outside the buffer");
    UNET_CHECK(dz, "layer_norm_bwd: null argument");
    const int need = unet_layer_norm_bwd_ws(dtype, nb, M, C);
    UNET_CHECK(need >= 0 && ws_size >= need && (ws || need == 0), "layer_norm_bwd: workspace too small (%d of %d floats)", ws_size, need);
    LnGrads g;
    for (int b = 0; b < LN_MAXB; ++b) {
        UNET_CHECK(b >= nb || dz[b] || M == 0, "layer_norm_bwd: branch %d has no output", b);
        a.dz[b] = b < nb ? dz[b] : nullptr;
        g.dgamma[b] = b < nb && dgamma ? dgamma[b] : nullptr;
        g.dbeta[b] = b < nb && dbeta ? dbeta[b] : nullptr;
    }
    hipStream_t s = (hipStream_t)stream;
    const int parts = ln_parts(M);
    float* part = ws + 2 * (size_t)nb * M;
    if (M > 0) {
        const dim3 cg((C + 63) / 64, parts);
        const long long per = (M + parts - 1) / parts;
        if (dtype == UNET_BF16) {
            const __bf16 *d = (const __bf16*)dy + dyoff, *o = y ? (const __bf16*)y + yoff : nullptr;
            hipLaunchKernelGGL((ln_bwd_rows_kernel<__bf16>), dim3(ln_grid(M, 4)), dim3(256), 0, s, a, d, lddy, o, ldy, ws);
            UNET_LAUNCH_CHECK();
            hipLaunchKernelGGL((ln_bwd_cols_kernel<__bf16>), cg, dim3(256), 0, s, a, d, lddy, o, ldy, ws, per, part);
        } else {
            const float *d = (const float*)dy + dyoff, *o = y ? (const float*)y + yoff : nullptr;
            hipLaunchKernelGGL((ln_bwd_rows_kernel<float>), dim3(ln_grid(M, 4)), dim3(256), 0, s, a, d, lddy, o, ldy, ws);
            UNET_LAUNCH_CHECK();
            hipLaunchKernelGGL((ln_bwd_cols_kernel<float>), cg, dim3(256), 0, s, a, d, lddy, o, ldy, ws, per, part);
        }
        UNET_LAUNCH_CHECK();
    }
    if (dgamma || dbeta) {
        hipLaunchKernelGGL(ln_bwd_finalize_kernel, dim3((C + 255) / 256, nb + 1), dim3(256), 0, s, part, parts, nb, C, g);
        UNET_LAUNCH_CHECK();
    }
    return 0;
}
