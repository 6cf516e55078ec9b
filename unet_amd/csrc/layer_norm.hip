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
// A row in registers.  L lanes share a row, each with V vectors of 16 bytes (vector k*L + l of the row); L <= 64: a wave holds
// 64/L rows; WG: the workgroup holds one row and L is its size.  EXACT: C = L*V*EPV, nothing to mask; otherwise a lane's last
// vector may end inside, or lie behind, the row.  16-byte accesses need no alignment here.

template <typename T> __device__ __forceinline__ uint4 ln_load(const T* p, int n) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (n >= TT<T>::EPV) {
        __builtin_memcpy(&v, p, 16);
    } else if (n > 0) {
        T e[TT<T>::EPV];
        for (int i = 0; i < TT<T>::EPV; ++i) e[i] = i < n ? p[i] : (T)0.f;
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}
template <typename T> __device__ __forceinline__ void ln_store(T* p, const float* f, int n) {
    const uint4 v = Vec16<T>::pack(f);
    if (n >= TT<T>::EPV) {
        __builtin_memcpy(p, &v, 16);
    } else if (n > 0) {
        for (int i = 0; i < TT<T>::EPV; ++i) if (i < n) p[i] = from_f32<T>(f[i]);
    }
}

__device__ __forceinline__ float ln_swap16(float v) {       // + the lane 16 away
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float ln_swap32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Each s[i] becomes its sum over the L lanes of the row (L: wave-uniform power of two up to 64, or the workgroup).  In a
// workgroup the waves meet in red[buf]; two buffers in turn, so one barrier per sum is enough.
template <int N, bool WG>
__device__ __forceinline__ void ln_row_sum(float (&s)[N], int L, float (*red)[16][N], int& buf) {
#pragma unroll
    for (int i = 0; i < N; ++i) if (WG || L > 1) s[i] += dpp_f32<0xB1>(s[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) if (WG || L > 2) s[i] += dpp_f32<0x4E>(s[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) if (WG || L > 4) s[i] += dpp_f32<0x141>(s[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) if (WG || L > 8) s[i] += dpp_f32<0x140>(s[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) if (WG || L > 16) s[i] = ln_swap16(s[i]);
#pragma unroll
    for (int i = 0; i < N; ++i) if (WG || L > 32) s[i] = ln_swap32(s[i]);
    if constexpr (WG) {
        const int wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < N; ++i) red[buf][wave][i] = s[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = 0.f;
            for (int w = 0; w < waves; ++w) t += red[buf][w][i];
            s[i] = t;
        }
        buf ^= 1;
    }
}

// s / C from inv = 1/C with one correction step: a constant row's mean is that constant (s * inv alone may be a unit off, which
// a row with no variance multiplies by 1/sqrt(eps))
__device__ __forceinline__ float ln_mean(float s, int C, float inv) {
    const float q = s * inv;
    return fmaf(fmaf(-q, (float)C, s), inv, q);
}

// Forward.  V = 1: all branches at once (NB >= a.nb); V > 1: one after another (NB = 1).
template <typename T, int NB, int V, bool EXACT, bool WG>
__global__ __launch_bounds__(WG ? 512 : 256) void ln_fwd_kernel(LnArgs a, T* __restrict__ y, int ldy, int relu, int L) {
    constexpr int EPV = TT<T>::EPV;
    __shared__ float red[WG ? 2 : 1][16][NB];
    int buf = 0;
    const int l = WG ? threadIdx.x : threadIdx.x & (L - 1);
    const int rpi = WG ? 1 : 256 / L, sub = WG ? 0 : threadIdx.x / L;
    const float inv = 1.f / (float)a.C;
    int cnt[V];
#pragma unroll
    for (int k = 0; k < V; ++k) { const int left = a.C - (k * L + l) * EPV; cnt[k] = EXACT ? EPV : left < 0 ? 0 : left < EPV ? left : EPV; }
    float g[V == 1 ? NB : 1][EPV], h[EPV];      // V = 1 (all branches at once): the weights stay in registers, the biases summed
    if constexpr (V == 1) {
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
            const int c = l * EPV + e;
            h[e] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const bool there = b < a.nb && (EXACT || e < cnt[0]);
                g[b][e] = there && a.gamma[b] ? a.gamma[b][c] : 1.f;
                h[e] += there && a.beta[b] ? a.beta[b][c] : 0.f;
            }
        }
    }
    for (long long base = (long long)blockIdx.x * rpi; base < a.M; base += (long long)gridDim.x * rpi) {
        const long long r = base + sub;
        const bool in = WG || r < a.M;
        float o[V][EPV];
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < EPV; ++e) o[k][e] = V == 1 ? h[e] : 0.f;
        for (int b0 = 0; b0 < (V == 1 ? 1 : a.nb); ++b0) {
            float d[NB][V][EPV], s[NB];
            uint4 raw[NB][V];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    raw[b][k] = b0 + b < a.nb && in
                        ? ln_load<T>((const T*)a.z[b0 + b] + (size_t)r * a.ldz[b0 + b] + (size_t)(k * L + l) * EPV, cnt[k]) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                s[b] = 0.f;
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    Vec16<T>::unpack(raw[b][k], d[b][k]);
#pragma unroll
                    for (int e = 0; e < EPV; ++e) s[b] += d[b][k][e];
                }
            }
            ln_row_sum<NB, WG>(s, L, red, buf);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const float mean = ln_mean(s[b], a.C, inv);
                s[b] = 0.f;
#pragma unroll
                for (int k = 0; k < V; ++k)
#pragma unroll
                    for (int e = 0; e < EPV; ++e) {
                        const float x = EXACT || e < cnt[k] ? d[b][k][e] - mean : 0.f;
                        d[b][k][e] = x;
                        s[b] = fmaf(x, x, s[b]);
                    }
            }
            ln_row_sum<NB, WG>(s, L, red, buf);
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                if (b0 + b >= a.nb) break;
                const float rstd = 1.f / sqrtf(fmaf(s[b], inv, a.eps));
                if constexpr (V == 1) {
#pragma unroll
                    for (int e = 0; e < EPV; ++e) o[0][e] = fmaf(d[b][0][e] * rstd, g[b][e], o[0][e]);
                } else {
                    const float *gp = a.gamma[b0], *bp = a.beta[b0];
#pragma unroll
                    for (int k = 0; k < V; ++k)
#pragma unroll
                        for (int e = 0; e < EPV; ++e) {
                            const int c = (k * L + l) * EPV + e;
                            const float gc = gp && (EXACT || e < cnt[k]) ? gp[c] : 1.f, bc = bp && (EXACT || e < cnt[k]) ? bp[c] : 0.f;
                            o[k][e] += fmaf(d[b][k][e] * rstd, gc, bc);
                        }
                }
            }
        }
        if (in) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                if (relu) {
#pragma unroll
                    for (int e = 0; e < EPV; ++e) o[k][e] = o[k][e] < 0.f ? 0.f : o[k][e];
                }
                ln_store<T>(y + (size_t)r * ldy + (size_t)(k * L + l) * EPV, o[k], cnt[k]);
            }
        }
    }
}

// Backward: dz and, per workgroup, the partial sums of dgamma_b and dbeta over its rows: part[blockIdx.x][nb + 1][C].  A lane
// keeps its channels' sums in registers over all its rows.  NB = 1 with several branches: blockIdx.y is the branch.
template <typename T, int NB, int V, bool EXACT, bool WG>
__global__ __launch_bounds__(WG ? 512 : 256) void ln_bwd_kernel(LnArgs a, const T* __restrict__ dy, int lddy, const T* __restrict__ y, int ldy,
                                                                 float* __restrict__ part, int L) {
    constexpr int EPV = TT<T>::EPV;
    __shared__ float red1[WG ? 2 : 1][16][NB];
    __shared__ float red3[WG ? 2 : 1][16][3 * NB];
    __shared__ float cols[WG ? 1 : 4][WG ? 1 : 64 * EPV];
    int buf1 = 0, buf3 = 0;
    const int b0 = NB == 1 ? blockIdx.y : 0, nb = NB == LN_MAXB ? a.nb : NB;
    const int l = WG ? threadIdx.x : threadIdx.x & (L - 1);
    const int rpi = WG ? 1 : 256 / L, sub = WG ? 0 : threadIdx.x / L;
    const float inv = 1.f / (float)a.C;
    int cnt[V];
    float g[NB][V][EPV], accg[NB][V][EPV], accb[V][EPV];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int c = (k * L + l) * EPV, left = a.C - c;
        cnt[k] = EXACT ? EPV : left < 0 ? 0 : left < EPV ? left : EPV;
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
            accb[k][e] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                accg[b][k][e] = 0.f;
                g[b][k][e] = b < nb && a.gamma[b0 + b] && (EXACT || e < cnt[k]) ? a.gamma[b0 + b][c + e] : 1.f;
            }
        }
    }
    for (long long base = (long long)blockIdx.x * rpi; base < a.M; base += (long long)gridDim.x * rpi) {
        const long long r = base + sub;
        const bool in = WG || r < a.M;
        uint4 raw[NB][V], rdy[V], ry[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const size_t c = (size_t)(k * L + l) * EPV;
            rdy[k] = in ? ln_load<T>(dy + (size_t)r * lddy + c, cnt[k]) : make_uint4(0, 0, 0, 0);
            if (y != nullptr) ry[k] = in ? ln_load<T>(y + (size_t)r * ldy + c, cnt[k]) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int b = 0; b < NB; ++b)
                raw[b][k] = b < nb && in ? ln_load<T>((const T*)a.z[b0 + b] + (size_t)r * a.ldz[b0 + b] + c, cnt[k]) : make_uint4(0, 0, 0, 0);
        }
        float u[V][EPV], d[NB][V][EPV], s[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            s[b] = 0.f;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                Vec16<T>::unpack(raw[b][k], d[b][k]);
#pragma unroll
                for (int e = 0; e < EPV; ++e) s[b] += d[b][k][e];
            }
        }
        ln_row_sum<NB, WG>(s, L, red1, buf1);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            Vec16<T>::unpack(rdy[k], u[k]);
            if (y != nullptr) {
                float o[EPV];
                Vec16<T>::unpack(ry[k], o);
#pragma unroll
                for (int e = 0; e < EPV; ++e) u[k][e] = o[e] <= 0.f ? 0.f : u[k][e];
            }
#pragma unroll
            for (int e = 0; e < EPV; ++e) accb[k][e] += u[k][e];
        }
        float t[3 * NB];                    // sums of d^2, w, w*d
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const float mean = ln_mean(s[b], a.C, inv);
            t[3 * b] = t[3 * b + 1] = t[3 * b + 2] = 0.f;
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    const float x = EXACT || e < cnt[k] ? d[b][k][e] - mean : 0.f, w = u[k][e] * g[b][k][e];
                    d[b][k][e] = x;
                    t[3 * b] = fmaf(x, x, t[3 * b]);
                    t[3 * b + 1] += w;
                    t[3 * b + 2] = fmaf(w, x, t[3 * b + 2]);
                }
        }
        ln_row_sum<3 * NB, WG>(t, L, red3, buf3);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (b >= nb) break;
            const float rstd = in ? 1.f / sqrtf(fmaf(t[3 * b], inv, a.eps)) : 0.f;
            const float m1 = t[3 * b + 1] * inv, m2 = t[3 * b + 2] * inv * rstd;      // means of w and w*xhat
#pragma unroll
            for (int k = 0; k < V; ++k) {
                float o[EPV];
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    const float x = d[b][k][e] * rstd;
                    accg[b][k][e] = fmaf(u[k][e], x, accg[b][k][e]);
                    o[e] = rstd * (fmaf(u[k][e], g[b][k][e], -m1) - x * m2);
                }
                if (in) ln_store<T>((T*)a.dz[b0 + b] + (size_t)r * a.C + (size_t)(k * L + l) * EPV, o, cnt[k]);
            }
        }
    }
    // the workgroup's sums: rows of one wave by rotations inside 16 lanes and the two swaps, then the waves through LDS
    float* out = part + (size_t)blockIdx.x * (a.nb + 1) * a.C;
    auto write = [&](float (&acc)[V][EPV], int q) {
        if constexpr (WG) {
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e)
                    if (EXACT || e < cnt[k]) out[(size_t)q * a.C + (k * L + l) * EPV + e] = acc[k][e];
        } else {
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
            for (int k = 0; k < V; ++k) {
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    float v = acc[k][e];
                    if (L <= 8) v += dpp_f32<0x128>(v);
                    if (L <= 4) v += dpp_f32<0x124>(v);
                    if (L <= 2) v += dpp_f32<0x122>(v);
                    if (L <= 1) v += dpp_f32<0x121>(v);
                    if (L <= 16) v = ln_swap16(v);
                    if (L <= 32) v = ln_swap32(v);
                    if (lane < L) cols[wave][lane * EPV + e] = v;
                }
                __syncthreads();
                for (int i = threadIdx.x; i < L * EPV; i += 256) {
                    const int c = k * L * EPV + i;
                    if (c < a.C) out[(size_t)q * a.C + c] = (cols[0][i] + cols[1][i]) + (cols[2][i] + cols[3][i]);
                }
                __syncthreads();
            }
        }
    };
#pragma unroll
    for (int b = 0; b < NB; ++b)
        if (b < nb) write(accg[b], b0 + b);
    if (b0 == 0) write(accb, a.nb);
}

// ---------------------------------------------------------------------------------------------
// Rows too wide for registers: one wave per row, elements strided over the lanes, the row read once per pass (the passes after the first hit L2).

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

// part [rows][nb + 1][C] -> dgamma_b, dbeta_b: 16 columns of one quantity per workgroup, 16 row lanes, fp64 sums in a fixed
// order (no atomics: the same bits every time)
__global__ __launch_bounds__(256) void ln_bwd_finalize_kernel(const float* __restrict__ part, int rows, int nb, int C, LnGrads g) {
    __shared__ double red[16][17];
    const int q = blockIdx.y, col = threadIdx.x & 15, rl = threadIdx.x >> 4;
    const int c = blockIdx.x * 16 + col;
    double s = 0.0;
    if (c < C) {
        const float* p = part + (size_t)q * C + c;
        const size_t ld = (size_t)(nb + 1) * C;
        int r = rl;
        for (; r + 48 < rows; r += 64) {
            const float v0 = p[r * ld], v1 = p[(r + 16) * ld], v2 = p[(r + 32) * ld], v3 = p[(r + 48) * ld];
            s += ((double)v0 + (double)v1) + ((double)v2 + (double)v3);
        }
        for (; r < rows; r += 16) s += (double)p[r * ld];
    }
    red[rl][col] = s;
    __syncthreads();
    if (rl == 0 && c < C) {
        s = 0.0;
        for (int i = 0; i < 16; ++i) s += red[i][col];
        if (q < nb) {
            if (g.dgamma[q]) g.dgamma[q][c] = (float)s;
        } else {
            for (int b = 0; b < nb; ++b)
                if (g.dbeta[b]) g.dbeta[b][c] = (float)s;
        }
    }
}

// ---------------------------------------------------------------------------------------------------

// How a shape is laid out over lanes; wide = too wide for registers (the row kernels).
struct LnPlan { bool wide, wg, exact; int nb, V, L; };

static LnPlan ln_plan(int dtype, int nb, int C, bool bwd) {
    const int epv = dtype == UNET_BF16 ? 8 : 4, nvec = (C + epv - 1) / epv;
    LnPlan p = {false, false, false, nb <= 3 || nb == 6 ? nb : 8, 1, 1};    // NB of the kernel: nb itself, or 8 and a bound at run time
    if (nvec <= 64) {                                   // a wave holds whole rows
        while (p.L < nvec) p.L <<= 1;
    } else if (nb > 1 && nvec <= 512) {                 // a workgroup per row, every branch at once
        p.wg = true; p.L = (nvec + 63) / 64 * 64;
    } else if (nvec <= 2048) {                          // branch by branch
        p.nb = 1;
        p.V = nvec <= 64 ? 1 : nvec <= 128 ? 2 : 4;
        p.wg = nvec > 256;
        p.L = p.wg ? (nvec + 64 * p.V - 1) / (64 * p.V) * 64 : 64;
    } else {
        p.wide = true;
    }
    p.exact = C == p.L * p.V * epv;
    return p;
}

static inline int ln_rows_per_wg(const LnPlan& p) { return p.wide ? 4 : p.wg ? 1 : 256 / p.L; }

// rows of partial sums of the backward = its workgroups
static inline int ln_parts(const LnPlan& p, long long M) {
    const long long n = p.wide ? (M + 63) / 64 : (M + ln_rows_per_wg(p) - 1) / ln_rows_per_wg(p);
    const int most = p.wide ? 256 : p.wg ? 512 : 768;
    return (int)(n < most ? n : most);
}

static int ln_args(LnArgs& a, const char* what, int dtype, int nb, const void* const* z, const int* ldz, const int* zoff,
                   const float* const* gamma, const float* const* beta, long long M, int C, float eps) {
    UNET_CHECK(dtype == UNET_F32 || dtype == UNET_BF16, "%s: bad dtype %d", what, dtype);
    UNET_CHECK(nb >= 1 && nb <= LN_MAXB, "%s: 1..%d branches (got %d)", what, LN_MAXB, nb);
    UNET_CHECK(M >= 0 && M < (1LL << 31) && C >= 1 && C <= (1 << 24), "%s: bad shape (%lld rows of %d channels)", what, M, C);
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

template <typename T, int NB, int V, bool WG>
static void ln_launch_fwd(const LnPlan& p, const LnArgs& a, int grid, T* y, int ldy, int relu, hipStream_t s) {
    const dim3 blk(WG ? p.L : 256);
    if (p.exact) hipLaunchKernelGGL((ln_fwd_kernel<T, NB, V, true, WG>), dim3(grid), blk, 0, s, a, y, ldy, relu, p.L);
    else hipLaunchKernelGGL((ln_fwd_kernel<T, NB, V, false, WG>), dim3(grid), blk, 0, s, a, y, ldy, relu, p.L);
}

template <typename T>
static void ln_fwd(const LnPlan& p, const LnArgs& a, T* y, int ldy, int relu, hipStream_t s) {
    const long long n = (a.M + ln_rows_per_wg(p) - 1) / ln_rows_per_wg(p);
    const int grid = (int)(n < 4096 ? n : 4096);
    if (p.wide) hipLaunchKernelGGL((ln_fwd_rows_kernel<T>), dim3(grid), dim3(256), 0, s, a, y, ldy, relu);
    else if (p.V == 2) ln_launch_fwd<T, 1, 2, false>(p, a, grid, y, ldy, relu, s);
    else if (p.V == 4) p.wg ? ln_launch_fwd<T, 1, 4, true>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, 1, 4, false>(p, a, grid, y, ldy, relu, s);
    else if (p.nb == 1) ln_launch_fwd<T, 1, 1, false>(p, a, grid, y, ldy, relu, s);
    else if (p.nb == 2) p.wg ? ln_launch_fwd<T, 2, 1, true>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, 2, 1, false>(p, a, grid, y, ldy, relu, s);
    else if (p.nb == 3) p.wg ? ln_launch_fwd<T, 3, 1, true>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, 3, 1, false>(p, a, grid, y, ldy, relu, s);
    else if (p.nb == 6) p.wg ? ln_launch_fwd<T, 6, 1, true>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, 6, 1, false>(p, a, grid, y, ldy, relu, s);
    else p.wg ? ln_launch_fwd<T, 8, 1, true>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, 8, 1, false>(p, a, grid, y, ldy, relu, s);
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
    const LnPlan p = ln_plan(dtype, nb, C, false);
    if (dtype == UNET_BF16) ln_fwd<__bf16>(p, a, (__bf16*)y + yoff, ldy, relu, (hipStream_t)stream);
    else ln_fwd<float>(p, a, (float*)y + yoff, ldy, relu, (hipStream_t)stream);
    UNET_LAUNCH_CHECK();
    return 0;
}

extern "C" int unet_layer_norm_bwd_ws(int dtype, int nb, long long M, int C) {
    if ((dtype != UNET_F32 && dtype != UNET_BF16) || nb < 1 || nb > LN_MAXB || M < 0 || C < 1) return -1;
    const LnPlan p = ln_plan(dtype, nb, C, true);
    const double n = (p.wide ? 2.0 * nb * (double)M : 0.0) + (double)ln_parts(p, M) * (nb + 1) * C;
    return n > 2147483647.0 ? -1 : (int)n;
}

template <typename T, int NB, int V, bool WG>
static void ln_launch_bwd(const LnPlan& p, const LnArgs& a, int parts, const T* dy, int lddy, const T* y, int ldy, float* part, hipStream_t s) {
    const dim3 grid(parts, NB == 1 ? a.nb : 1), blk(WG ? p.L : 256);
    if (p.exact) hipLaunchKernelGGL((ln_bwd_kernel<T, NB, V, true, WG>), grid, blk, 0, s, a, dy, lddy, y, ldy, part, p.L);
    else hipLaunchKernelGGL((ln_bwd_kernel<T, NB, V, false, WG>), grid, blk, 0, s, a, dy, lddy, y, ldy, part, p.L);
}

template <typename T>
static int ln_bwd(const LnPlan& p, const LnArgs& a, int parts, const T* dy, int lddy, const T* y, int ldy, float* ws, float* part, hipStream_t s) {
    if (p.wide) {
        hipLaunchKernelGGL((ln_bwd_rows_kernel<T>), dim3((unsigned)((a.M + 3) / 4 < 8192 ? (a.M + 3) / 4 : 8192)), dim3(256), 0, s, a, dy, lddy, y, ldy, ws);
        UNET_LAUNCH_CHECK();
        hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3((a.C + 63) / 64, parts), dim3(256), 0, s, a, dy, lddy, y, ldy, ws, (a.M + parts - 1) / parts, part);
    } else if (p.V == 2) ln_launch_bwd<T, 1, 2, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.V == 4) p.wg ? ln_launch_bwd<T, 1, 4, true>(p, a, parts, dy, lddy, y, ldy, part, s) : ln_launch_bwd<T, 1, 4, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 1) ln_launch_bwd<T, 1, 1, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 2) p.wg ? ln_launch_bwd<T, 2, 1, true>(p, a, parts, dy, lddy, y, ldy, part, s) : ln_launch_bwd<T, 2, 1, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 3) p.wg ? ln_launch_bwd<T, 3, 1, true>(p, a, parts, dy, lddy, y, ldy, part, s) : ln_launch_bwd<T, 3, 1, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 6) p.wg ? ln_launch_bwd<T, 6, 1, true>(p, a, parts, dy, lddy, y, ldy, part, s) : ln_launch_bwd<T, 6, 1, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    else p.wg ? ln_launch_bwd<T, 8, 1, true>(p, a, parts, dy, lddy, y, ldy, part, s) : ln_launch_bwd<T, 8, 1, false>(p, a, parts, dy, lddy, y, ldy, part, s);
    UNET_LAUNCH_CHECK();
    return 0;
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
    const LnPlan p = ln_plan(dtype, nb, C, true);
    const int parts = ln_parts(p, M);
    float* part = ws + (p.wide ? 2 * (size_t)nb * M : 0);
    if (M > 0) {
        const int e = dtype == UNET_BF16
            ? ln_bwd<__bf16>(p, a, parts, (const __bf16*)dy + dyoff, lddy, y ? (const __bf16*)y + yoff : nullptr, ldy, ws, part, s)
            : ln_bwd<float>(p, a, parts, (const float*)dy + dyoff, lddy, y ? (const float*)y + yoff : nullptr, ldy, ws, part, s);
        if (e) return e;
    }
    if (dgamma || dbeta) {
        hipLaunchKernelGGL(ln_bwd_finalize_kernel, dim3((C + 15) / 16, nb + 1), dim3(256), 0, s, part, parts, nb, C, g);
        UNET_LAUNCH_CHECK();
    }
    return 0;
}
