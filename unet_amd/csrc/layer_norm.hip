// Layer norm over the channels of each row (a pixel or a token), summed over the branches of a block, and its backward pass.
//
//   xhat_b[r][c] = (z_b[r][c] - mean_c z_b[r]) / sqrt(var_c z_b[r] + eps)            (biased variance)
//   y[r][c]      = act( sum_b xhat_b[r][c] * gamma_b[c] + beta_b[c] )                 act: identity or ReLU
//   u = dy (ReLU: 0 where y <= 0),  w_b = u * gamma_b
//   dz_b         = (w_b - mean_c w_b - xhat_b * mean_c (w_b * xhat_b)) / sqrt(var + eps)
//   dgamma_b[c]  = sum_r u * xhat_b,   dbeta[c] = sum_r u   (the same for every branch)
//
// One branch without ReLU is the plain layer norm.  Sums, statistics and weights are fp32; activations fp32 or bf16, rounded
// once on the way out.  The variance is the mean of (z - mean)^2, and the mean of an fp32 row comes in two parts (ln_two_steps):
// rows far from zero lose nothing.  Statistics are not handed from forward to backward: the backward has the row at hand and
// computes them again, 8 bytes per row and branch less in both.  NaN stays NaN through the ReLU, and passes gradient, as in torch.
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
// A row in registers: every tensor is read once and written once, and HBM is the bound (one MI355X; in brackets a kernel that only
// streams the same bytes): forward 2.1 M rows x 64 channels x 6 branches bf16 362 us = 5.2 TB/s (300), 8192 x 4096 28 us (22), 50001 x
// 333 fp32 28 us (22); backward 2.1 M x 64 x 6 726 us = 5.2 TB/s (708), 8192 x 1024 x 6 57 us (42), 4099 x 5120 39 us (21: half of the
// time is arithmetic, waves wait for each other at every row, and partial sums are 1/6 of the data).  Below about 1 MB the launch is.
//
// L lanes share a row, each with V vectors of 16 bytes (vector k*L + l of the row).  Either L is a power
// of two up to 64 and a wave holds 64/L rows, or (WG) L is a multiple of 64 and a workgroup holds blockDim/L rows.  Branches
// are worked off one after another; the next row's vectors of a branch are requested as soon as this row's are unpacked, so
// every wave has a whole row in flight.
//
// EXACT: C = L*V*EPV.  Otherwise the last vector of a row starts EPV channels before its end: it overlaps its neighbour, the
// doubled channels count once in every sum, and both lanes store the same bits.  16-byte accesses need no alignment here.

// NT: streaming access.  Activations pass once: forward 2.1 M x 64 x 6 bf16 398 -> 365 us with it, backward 777 -> 736; what is
// read again soon (dy and y of a second group of branches, the rows of a few wide tensors) goes without: 4099 x 5120 43 against 46.
typedef __attribute__((ext_vector_type(4), aligned(2))) uint32_t ln_u32x4;

template <typename T, bool NT> __device__ __forceinline__ uint4 ln_load(const T* p) {
    const ln_u32x4 v = NT ? __builtin_nontemporal_load((const ln_u32x4*)p) : *(const ln_u32x4*)p;
    return make_uint4(v.x, v.y, v.z, v.w);
}
template <typename T, bool NT> __device__ __forceinline__ void ln_store(T* p, const float* f) {
    const uint4 w = Vec16<T>::pack(f);
    const ln_u32x4 v = {w.x, w.y, w.z, w.w};
    if (NT) __builtin_nontemporal_store(v, (ln_u32x4*)p);
    else *(ln_u32x4*)p = v;
}

// first channel of vector `slot`, and in lo how many of its channels belong to the vector before (all: no such vector)
template <int EPV>
__device__ __forceinline__ int ln_channel(int slot, int C, int& lo) {
    const int c0 = slot * EPV, c = c0 + EPV <= C ? c0 : C - EPV;
    lo = c0 < C ? c0 - c : EPV;
    return c;
}

__device__ __forceinline__ float ln_swap16(float v) {       // + the lane 16 away
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float ln_swap32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

constexpr int LN_BLOCK = 512;                               // workgroup of wide rows, as a rule
// threads at most of a forward workgroup that holds whole rows
constexpr int ln_fwd_most(size_t size, int nb, bool mem) { return size == 4 || mem ? LN_BLOCK : nb <= 4 ? 2 * LN_BLOCK : 768; }
constexpr size_t LN_LDS = 156 << 10;                        // dynamic LDS of a workgroup: all but what LnMeet takes
constexpr int LN_ROWS = 8;                                  // so rows of a workgroup, where a row takes two waves or more

// Each s[i] becomes its sum over the lanes that the wave has of a row: all L, at most 64 of them.
template <int N, int LC>
__device__ __forceinline__ void ln_row_sum(float (&s)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        s[i] += dpp_f32<0xB1>(s[i]);
        if (LC == 0 || LC > 2) s[i] += dpp_f32<0x4E>(s[i]);
        if (LC == 0 || LC > 4) s[i] += dpp_f32<0x141>(s[i]);
        if (LC == 0 || LC > 8) s[i] += dpp_f32<0x140>(s[i]);
        if (LC == 0 || LC > 16) s[i] = ln_swap16(s[i]);
        if (LC == 0 || LC > 32) s[i] = ln_swap32(s[i]);
    }
}

// s / n from inv = 1/n with one correction step: s * inv alone may be a unit off, which a row with no variance multiplies by
// 1/sqrt(eps)
__device__ __forceinline__ float ln_mean(float s, float n, float inv) {
    const float q = s * inv;
    return fmaf(fmaf(-q, n, s), inv, q);
}

// Whether a row's mean takes two steps: the mean of what the first one leaves is taken off too.  bf16 rows do without: values with 8
// bits of mantissa add up exactly in fp32 as long as they are close to each other (a constant row's mean is that constant).  fp32
// values do not: a constant row of 1000 channels at 974.7 came out as 0.08 instead of 0, a rounded sum times 1/sqrt(eps).
template <typename T> constexpr bool ln_two_steps = sizeof(T) == 4;

// d, a row, less the mean that its rounded sum gave and the mean of what that leaves; returns the latter.  (The differences of a row
// far from zero have few bits: their sum is exact.)
template <int LC, bool EXACT, int V, int EPV>
__device__ __forceinline__ float ln_centre(float (&d)[V][EPV], const int (&lo)[V], float mean, float n, float inv) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
            d[k][e] -= mean;
            s[0] += EXACT || e >= lo[k] ? d[k][e] : 0.f;
        }
    ln_row_sum<1, LC>(s);
    const float rest = ln_mean(s[0], n, inv);
#pragma unroll
    for (int k = 0; k < V; ++k)
#pragma unroll
        for (int e = 0; e < EPV; ++e) d[k][e] -= rest;
    return rest;
}

// Where the waves of a row meet (rows of several waves).  Each wave brings the mean m of its n channels, their sum of (z - m)^2 and
// in the backward the sums of w and w*(z - m); with m0 = the first wave's mean
//   mean = m0 + sum(n*(m - m0))/C,   e = m - mean,
//   sum (z - mean)^2 = sum over waves (z - m)^2 + n*e^2,   sum w*(z - mean) = sum over waves w*(z - m) + e*w
// All terms of a sum of squares are positive: nothing is lost, however far the waves' means are apart.  16 slots a row, the unused
// ones zero; two buffers in turn, so that one barrier a row is enough (with the mean first and a second meeting for the sums:
// backward 4099 x 5120 bf16 42.4 us).
template <bool> struct LnMore {};
template <> struct LnMore<true> { float more[2][LN_ROWS * 16]; };
template <int N, bool REST> struct LnMeet : LnMore<REST && (N > 1)> {       // N: sums besides the mean; REST: the mean comes in two
    float4 slot[2][LN_ROWS * 16];                                           // parts (the second one: more, N = 1: slot's third number)
    __device__ __forceinline__ void clear() {               // (a barrier has to follow)
        for (int i = threadIdx.x; i < 2 * LN_ROWS * 16; i += blockDim.x) {
            (&slot[0][0])[i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if constexpr (REST && N > 1) (&this->more[0][0])[i] = 0.f;
        }
    }
    // t becomes the row's sums; returns the wave's mean minus the row's.  mean + rest: the wave's mean, n: channels of the wave whose
    // slot this lane reads (0: none), at: first slot of the row, wave: which of the row's.
    __device__ __forceinline__ float join(float (&t)[N], float mean, float rest, float n, int at, int wave, float C, float inv, int& buf) {
        if ((threadIdx.x & 63) == 0) {
            slot[buf][at + wave] = make_float4(mean, t[0], N > 1 ? t[N > 1 ? 1 : 0] : rest, N > 1 ? t[N > 1 ? 2 : 0] : 0.f);
            if constexpr (REST && N > 1) this->more[buf][at + wave] = rest;
        }
        __syncthreads();
        const float4 v = slot[buf][at + (threadIdx.x & 15)];
        const float m0 = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v.x)));
        float e = v.x - m0;
        if constexpr (REST && N > 1) e += this->more[buf][at + (threadIdx.x & 15)];
        else if constexpr (REST) e += v.z;
        float f[1] = {n * e};
        buf ^= 1;
        ln_row_sum<1, 16>(f);
        f[0] = REST ? ln_mean(f[0], C, inv) : f[0] * inv;
        e -= f[0];
        t[0] = fmaf(n * e, e, v.y);
        if constexpr (N > 1) { t[1] = v.z; t[2] = fmaf(e, v.z, v.w); }
        ln_row_sum<N, 16>(t);
        return (REST ? (mean - m0) + rest : mean - m0) - f[0];
    }
};
template <bool REST> struct LnMeet<0, REST> { __device__ __forceinline__ void clear() {} };

// how many of a row's channels wave `wave` of it has (vector k*L + l, lanes of the wave l = 64*wave ..)
template <int EPV, int V>
__device__ __forceinline__ float ln_share(int wave, int L, int C) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int first = (k * L + 64 * wave) * EPV, left = C - first;
        n += left < 0 ? 0 : left < 64 * EPV ? left : 64 * EPV;
    }
    return (float)(wave < L >> 6 ? n : 0);
}

// 1/sqrt(v) by the hardware's instruction (1 unit in the last place), which takes numbers under 2^-126 for zero: small ones are
// scaled first.  No branch: it would let the compiler move the branches' arithmetic together (123 registers became 256).
__device__ __forceinline__ float ln_rstd(float v) {
    const bool small = v < 0x1p-64f;
    return __builtin_amdgcn_rsqf(v * (small ? 0x1p64f : 1.f)) * (small ? 0x1p32f : 1.f);
}

// Weights of all branches: in registers, or from LDS for every row where they would take too many
template <int NB, int W, bool WG> struct LnInLds { static constexpr bool value = NB * W > 32 || WG; };

template <int EPV>
__device__ __forceinline__ void ln_gamma_to_lds(float* gl, const LnArgs& a, int b0, int nb, int slots) {
    for (int b = 0; b < nb; ++b)
        for (int i = threadIdx.x; i < slots * EPV; i += blockDim.x) {
            int lo;
            const int c = ln_channel<EPV>(i / EPV, a.C, lo) + i % EPV;
            gl[b * slots * EPV + i] = a.gamma[b0 + b] ? a.gamma[b0 + b][c] : 1.f;
        }
    __syncthreads();
}

// EPV weights, 16 bytes at a time
template <int EPV> __device__ __forceinline__ void ln_weights(float (&w)[EPV], const float* gamma, int c) {
#pragma unroll
    for (int q = 0; q < EPV; q += 4) {
        uint4 v = make_uint4(0x3f800000u, 0x3f800000u, 0x3f800000u, 0x3f800000u);
        if (gamma != nullptr) v = ln_load<float, false>(gamma + c + q);
        w[q] = __uint_as_float(v.x); w[q + 1] = __uint_as_float(v.y); w[q + 2] = __uint_as_float(v.z); w[q + 3] = __uint_as_float(v.w);
    }
}

// Rows behind the last one read the last one: no load is conditional, so that the compiler can count them.  (Row numbers fit 32
// bits, offsets do not.)
template <typename T, bool NT, int V>
__device__ __forceinline__ void ln_request(uint4 (&v)[V], const void* p, int ld, uint32_t r, uint32_t M, const int (&ch)[V]) {
    const T* row = (const T*)p + (size_t)(r < M ? r : M - 1) * (uint32_t)ld;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = ln_load<T, NT>(row + ch[k]);
}

// Between two branches: their arithmetic is not interleaved (it would take every branch's registers at once), and gl is read
// again for every row instead of staying in registers: forward with six branches 78 registers instead of 158.
#define LN_NEXT_BRANCH(apart) do { if (apart) { asm volatile("" ::: "memory"); __builtin_amdgcn_sched_barrier(0); } } while (0)

// NB branches, at most where BOUND.  LC: L as a constant, 0 for a row per L threads of the workgroup (L a multiple of 64).
// MEM (forward): weights read from memory for every row, where LDS does not hold them.
template <typename T, int NB, bool BOUND, int V, int LC, bool EXACT, bool MEM>
__global__ __launch_bounds__(LC == 0 ? ln_fwd_most(sizeof(T), NB, MEM) : LN_BLOCK) void ln_fwd_kernel(LnArgs a, T* __restrict__ y, int ldy, int relu, int Lrt) {
    constexpr int EPV = TT<T>::EPV;
    constexpr bool WG = LC == 0, GL = !MEM && LnInLds<NB, V * EPV, false>::value, TWO = ln_two_steps<T>;
    __shared__ LnMeet<WG ? 1 : 0, TWO> meet;
    extern __shared__ __attribute__((aligned(16))) float gl[];      // GL: [NB][V*L*EPV]
    int buf = 0;
    const int L = WG ? Lrt : LC, nb = BOUND ? a.nb : NB;
    const int sub = threadIdx.x / L, l = threadIdx.x - sub * L, rpi = blockDim.x / L;
    const uint32_t M = (uint32_t)a.M, stride = gridDim.x * rpi, mine = WG ? sub * gridDim.x : sub;
    const float C = (float)a.C, inv = 1.f / C;
    // the wave's share of the row, and the share of the wave whose slot this lane reads (WG)
    const float n = WG ? ln_share<EPV, V>(l >> 6, L, a.C) : C, ninv = WG ? 1.f / n : inv, nslot = WG ? ln_share<EPV, V>(threadIdx.x & 15, L, a.C) : 0.f;
    int ch[V], lo[V];
    float g[GL || MEM ? 1 : NB][V][EPV], h[V][EPV];               // h: the biases' sum
#pragma unroll
    for (int k = 0; k < V; ++k) {
        ch[k] = ln_channel<EPV>(k * L + l, a.C, lo[k]);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
            h[k][e] = 0.f;
            if constexpr (!GL && !MEM) {
#pragma unroll
                for (int b = 0; b < NB; ++b) g[b][k][e] = b < nb && a.gamma[b] ? a.gamma[b][ch[k] + e] : 1.f;
            }
        }
    }
#pragma unroll 1
    for (int b = 0; b < nb; ++b) {
        if (a.beta[b] == nullptr) continue;
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < EPV; ++e) h[k][e] += a.beta[b][ch[k] + e];
    }
    uint4 raw[NB][V];
    // (rows of several waves: a workgroup's are `mine` apart, so that the rows left over for the last round go to all of them)
    uint32_t base = WG ? blockIdx.x : blockIdx.x * rpi;
#pragma unroll
    for (int b = 0; b < NB; ++b) if (!BOUND || b < nb) ln_request<T, true, V>(raw[b], a.z[b], a.ldz[b], base + mine, M, ch);
    meet.clear();
    if constexpr (GL) ln_gamma_to_lds<EPV>(gl, a, 0, nb, V * L);
    else if constexpr (WG) __syncthreads();
    for (; base < M; base += stride) {
        const uint32_t r = base + mine;
        float o[V][EPV];
#pragma unroll
        for (int k = 0; k < V; ++k)
#pragma unroll
            for (int e = 0; e < EPV; ++e) o[k][e] = h[k][e];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (BOUND && b >= nb) break;
            LN_NEXT_BRANCH(GL || MEM);
            float d[V][EPV], w[V][EPV], s[1] = {0.f};
            if constexpr (MEM) {
#pragma unroll
                for (int k = 0; k < V; ++k) ln_weights<EPV>(w[k], a.gamma[b], ch[k]);
            }
#pragma unroll
            for (int k = 0; k < V; ++k) {
                Vec16<T>::unpack(raw[b][k], d[k]);
#pragma unroll
                for (int e = 0; e < EPV; ++e) s[0] += EXACT || e >= lo[k] ? d[k][e] : 0.f;
            }
            ln_request<T, true, V>(raw[b], a.z[b], a.ldz[b], r + stride, M, ch);
            ln_row_sum<1, LC>(s);
            const float mean = ln_mean(s[0], n, ninv);
            float rest = 0.f;
            if constexpr (TWO) rest = ln_centre<LC, EXACT>(d, lo, mean, n, ninv);
            s[0] = 0.f;
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    if constexpr (!TWO) d[k][e] -= mean;
                    const float x = EXACT || e >= lo[k] ? d[k][e] : 0.f;
                    s[0] = fmaf(x, x, s[0]);
                }
            ln_row_sum<1, LC>(s);
            float off = 0.f;
            if constexpr (WG) off = meet.join(s, mean, rest, nslot, sub * 16, l >> 6, C, inv, buf);
            const float rstd = ln_rstd(fmaf(s[0], inv, a.eps));
            off *= rstd;
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    if constexpr (!MEM) w[k][e] = GL ? gl[((b * V + k) * L + l) * EPV + e] : g[GL ? 0 : b][k][e];
                    o[k][e] = fmaf(WG ? fmaf(d[k][e], rstd, off) : d[k][e] * rstd, w[k][e], o[k][e]);
                }
        }
        if (relu) {
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e) o[k][e] = o[k][e] < 0.f ? 0.f : o[k][e];
        }
        if (r < M) {
#pragma unroll
            for (int k = 0; k < V; ++k) if (EXACT || lo[k] < EPV) ln_store<T, true>(y + (size_t)r * (uint32_t)ldy + ch[k], o[k]);
        }
    }
}

// Workgroup -> (rows, group of branches).  The groups of the same rows are 8 apart, on one XCD at about the same time: the second
// finds dy and y in its L2.
__device__ __forceinline__ int2 ln_block(int groups, int parts) {
    const int id = blockIdx.x, whole = (parts & ~7) * groups;
    if (groups == 1) return make_int2(id, 0);
    if (id < whole) return make_int2(id / (8 * groups) * 8 + (id & 7), id / 8 % groups);
    return make_int2((parts & ~7) + (id - whole) / groups, (id - whole) % groups);
}

// Backward: dz and, per workgroup, the partial sums of dgamma_b and dbeta over its rows: part[block][a.nb + 1][C].  A lane
// keeps its channels' sums in registers over all its rows (at most 64: with six branches of 16 channels they spilled, so such
// rows go to two waves with three branches each; 8192 x 1024 x 6: 59 us, as two rounds of workgroups 70).
template <typename T, int NB, bool BOUND, int V, int LC, bool EXACT>
__global__ __launch_bounds__(LC == 0 ? 2 * LN_BLOCK : V == 1 ? 256 : LN_BLOCK)
void ln_bwd_kernel(LnArgs a, const T* __restrict__ dy, int lddy, const T* __restrict__ y, int ldy, float* __restrict__ part, int parts, int Lrt) {
    constexpr int EPV = TT<T>::EPV;
    constexpr bool WG = LC == 0, GL = LnInLds<NB, V * EPV, WG>::value, NT = !WG, NTU = NT && (V == 1 || NB == 1), TWO = ln_two_steps<T>;
    __shared__ LnMeet<WG ? 3 : 0, TWO> meet;
    extern __shared__ __attribute__((aligned(16))) float gl[];      // GL: [NB][V*L*EPV]; at the end [rows or waves][L*EPV]
    int buf = 0;
    // several groups of NB branches: other workgroups (WG), or other waves of this one
    const int groups = (a.nb + NB - 1) / NB, gt = WG ? blockDim.x : blockDim.x / groups;       // threads to a group
    const int2 where = WG ? ln_block(groups, parts) : make_int2(blockIdx.x, __builtin_amdgcn_readfirstlane(threadIdx.x / gt));
    const int L = WG ? Lrt : LC, block = where.x, b0 = where.y * NB, nb = BOUND && a.nb - b0 < NB ? a.nb - b0 : NB;
    const int t = WG ? threadIdx.x : threadIdx.x - where.y * gt, sub = t / L, l = t - sub * L, rpi = gt / L;
    const uint32_t M = (uint32_t)a.M, stride = parts * rpi, mine = WG ? sub * parts : sub;
    const float C = (float)a.C, inv = 1.f / C;
    // the wave's share of the row, and the share of the wave whose slot this lane reads (WG)
    const float n = WG ? ln_share<EPV, V>(l >> 6, L, a.C) : C, ninv = WG ? 1.f / n : inv, nslot = WG ? ln_share<EPV, V>(threadIdx.x & 15, L, a.C) : 0.f;
    int ch[V], lo[V];
    float g[GL ? 1 : NB][V][EPV], accg[NB][V][EPV], accb[V][EPV];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        ch[k] = ln_channel<EPV>(k * L + l, a.C, lo[k]);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
            accb[k][e] = 0.f;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                accg[b][k][e] = 0.f;
                if constexpr (!GL) g[b][k][e] = b < nb && a.gamma[b0 + b] ? a.gamma[b0 + b][ch[k] + e] : 1.f;
            }
        }
    }
    uint4 raw[NB][V], rdy[V], ry[V];
    uint32_t base = WG ? block : block * rpi;
    ln_request<T, NTU, V>(rdy, dy, lddy, base + mine, M, ch);
    if (y != nullptr) ln_request<T, NTU, V>(ry, y, ldy, base + mine, M, ch);
#pragma unroll
    for (int b = 0; b < NB; ++b) if (!BOUND || b < nb) ln_request<T, NT, V>(raw[b], a.z[b0 + b], a.ldz[b0 + b], base + mine, M, ch);
    meet.clear();
    if constexpr (GL) ln_gamma_to_lds<EPV>(gl, a, WG ? b0 : 0, WG ? nb : a.nb, V * L);      // (always, where WG)
    const float* gb = gl + (WG ? 0 : b0) * V * L * EPV;             // gamma of this group's first branch
    for (; base < M; base += stride) {
        const uint32_t r = base + mine;
        const bool in = r < M;
        float u[V][EPV];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            if (!in) rdy[k] = make_uint4(0, 0, 0, 0);
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
        ln_request<T, NTU, V>(rdy, dy, lddy, r + stride, M, ch);
        if (y != nullptr) ln_request<T, NTU, V>(ry, y, ldy, r + stride, M, ch);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (BOUND && b >= nb) break;
            LN_NEXT_BRANCH(GL);
            auto weight = [&](int k, int e) { return GL ? gb[((b * V + k) * L + l) * EPV + e] : g[GL ? 0 : b][k][e]; };
            float d[V][EPV], s[1] = {0.f}, t[3] = {0.f, 0.f, 0.f};        // t: sums of d^2, w, w*d
#pragma unroll
            for (int k = 0; k < V; ++k) {
                Vec16<T>::unpack(raw[b][k], d[k]);
#pragma unroll
                for (int e = 0; e < EPV; ++e) s[0] += EXACT || e >= lo[k] ? d[k][e] : 0.f;
            }
            ln_request<T, NT, V>(raw[b], a.z[b0 + b], a.ldz[b0 + b], r + stride, M, ch);
            ln_row_sum<1, LC>(s);
            const float mean = ln_mean(s[0], n, ninv);
            float rest = 0.f;
            if constexpr (TWO) rest = ln_centre<LC, EXACT>(d, lo, mean, n, ninv);
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    if constexpr (!TWO) d[k][e] -= mean;
                    const float x = EXACT || e >= lo[k] ? d[k][e] : 0.f, w = u[k][e] * weight(k, e);
                    t[0] = fmaf(x, x, t[0]);
                    t[1] += EXACT || e >= lo[k] ? w : 0.f;
                    t[2] = fmaf(w, x, t[2]);
                }
            ln_row_sum<3, LC>(t);
            float off = 0.f;
            if constexpr (WG) off = meet.join(t, mean, rest, nslot, sub * 16, l >> 6, C, inv, buf);
            const float rstd = ln_rstd(fmaf(t[0], inv, a.eps));
            off *= rstd;
            // dz = rstd*w - (rstd*mean(w) + xhat*rstd*mean(w*xhat)).  (w is the value that the sums took: formed again from weights
            // in LDS, those stay in registers too, 128 -> spills, one row to a workgroup.)
            const float m1 = rstd * (t[1] * inv), m2 = rstd * (t[2] * inv * rstd);
#pragma unroll
            for (int k = 0; k < V; ++k)
#pragma unroll
                for (int e = 0; e < EPV; ++e) {
                    const float x = WG ? fmaf(d[k][e], rstd, off) : d[k][e] * rstd;
                    accg[b][k][e] = fmaf(u[k][e], x, accg[b][k][e]);
                    d[k][e] = fmaf(u[k][e] * weight(k, e), rstd, -fmaf(x, m2, m1));
                }
            if (in) {
#pragma unroll
                for (int k = 0; k < V; ++k) if (EXACT || lo[k] < EPV) ln_store<T, NT>((T*)a.dz[b0 + b] + (size_t)r * (uint32_t)a.C + ch[k], d[k]);
            }
        }
    }
    // the workgroup's sums: the rows of one wave by rotations inside 16 lanes and the two swaps, then the group's waves (or the
    // rows of the workgroup) through LDS
    float* out = part + (size_t)block * (a.nb + 1) * a.C;
    float* cols = gl;
    if (GL) __syncthreads();                    // (the last row's reads of gl)
    const int lane = threadIdx.x & 63, per = WG ? rpi : gt >> 6, at = WG ? sub : threadIdx.x >> 6;
    auto write = [&](float (&acc)[V][EPV], int b, bool beta) {      // b: the branch in its group
#pragma unroll
        for (int k = 0; k < V; ++k) {
#pragma unroll
            for (int e = 0; e < EPV; ++e) {
                float v = acc[k][e];
                if (!WG && LC <= 2) v += dpp_f32<0x122>(v);
                if (!WG && LC <= 4) v += dpp_f32<0x124>(v);
                if (!WG && LC <= 8) v += dpp_f32<0x128>(v);
                if (!WG && LC <= 16) v = ln_swap16(v);
                if (!WG && LC <= 32) v = ln_swap32(v);
                if (WG || lane < L) cols[(at * L + (WG ? l : lane)) * EPV + e] = v;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < (WG || beta ? 1 : groups) * L * EPV; i += blockDim.x) {
                const int grp = i / (L * EPV), j = i - grp * L * EPV, q = beta ? a.nb : (WG ? b0 : grp * NB) + b;
                int lo;
                const int c = ln_channel<EPV>(k * L + j / EPV, a.C, lo) + j % EPV;
                if (j % EPV >= lo && (beta || q < a.nb)) {
                    float v = 0.f;
                    for (int w = 0; w < per; ++w) v += cols[(grp * per + w) * L * EPV + j];
                    out[(size_t)q * a.C + c] = v;
                }
            }
            __syncthreads();
        }
    };
#pragma unroll
    for (int b = 0; b < NB; ++b) write(accg[b], b, false);
    if (!WG || b0 == 0) write(accb, 0, true);
}

// ---------------------------------------------------------------------------------------------
// Any other width (too wide for registers, or narrower than a vector): one wave per row, elements strided over the lanes, the
// row read once per pass (the passes after the first hit L2).

struct LnStats {
    float mean, rest, rstd;             // the mean in two parts, as in ln_centre
    template <typename T> __device__ __forceinline__ float centred(T z) const { return (to_f32(z) - mean) - rest; }
};

template <typename T>
__device__ __forceinline__ LnStats ln_row_stats(const T* z, int C, float eps) {
    const int lane = threadIdx.x & 63;
    LnStats t = {0.f, 0.f, 0.f};
    float q = 0.f;
    if constexpr (ln_two_steps<T>) {    // (a sum in fp64 instead of a second pass: 20 % less time)
        double s = 0.0;
        for (int c = lane; c < C; c += 64) s += (double)z[c];
        s = wave_sum64d(s) / C;
        t.mean = (float)s;
        t.rest = (float)(s - (double)t.mean);
    } else {
        float s = 0.f;
        for (int c = lane; c < C; c += 64) s += to_f32(z[c]);
        t.mean = wave_sum64(s) / (float)C;
    }
    for (int c = lane; c < C; c += 64) { const float d = t.centred(z[c]); q += d * d; }
    t.rstd = 1.f / sqrtf(wave_sum64(q) / (float)C + eps);
    return t;
}

template <typename T>
__global__ __launch_bounds__(256) void ln_fwd_rows_kernel(LnArgs a, T* __restrict__ y, int ldy, int relu) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.M; r += (long long)gridDim.x * 4) {
        LnStats t[LN_MAXB];
#pragma unroll
        for (int b = 0; b < LN_MAXB; ++b)
            if (b < a.nb) t[b] = ln_row_stats((const T*)a.z[b] + r * a.ldz[b], a.C, a.eps);
        for (int c = lane; c < a.C; c += 64) {
            float o = 0.f;
#pragma unroll
            for (int b = 0; b < LN_MAXB; ++b) {
                if (b < a.nb) {
                    const float x = t[b].centred(((const T*)a.z[b])[r * a.ldz[b] + c]) * t[b].rstd;
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

// dz of every branch; stats [nb][M] for the column pass
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_rows_kernel(LnArgs a, const T* __restrict__ dy, int lddy, const T* __restrict__ y, int ldy,
                                                          LnStats* __restrict__ stats) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.M; r += (long long)gridDim.x * 4) {
        for (int b = 0; b < a.nb; ++b) {
            const T* z = (const T*)a.z[b] + r * a.ldz[b];
            const float* gamma = a.gamma[b];
            const LnStats t = ln_row_stats(z, a.C, a.eps);
            float s1 = 0.f, s2 = 0.f;
            for (int c = lane; c < a.C; c += 64) {
                const float w = ln_u(dy, y, r * lddy + c, r * ldy + c) * (gamma ? gamma[c] : 1.f);
                s1 += w;
                s2 += w * (t.centred(z[c]) * t.rstd);
            }
            const float m1 = wave_sum64(s1) / (float)a.C, m2 = wave_sum64(s2) / (float)a.C;
            T* dz = (T*)a.dz[b] + r * a.C;
            for (int c = lane; c < a.C; c += 64) {
                const float w = ln_u(dy, y, r * lddy + c, r * ldy + c) * (gamma ? gamma[c] : 1.f);
                const float x = t.centred(z[c]) * t.rstd;
                dz[c] = from_f32<T>(t.rstd * (w - m1 - x * m2));
            }
            if (lane == 0) stats[(size_t)b * a.M + r] = t;
        }
    }
}

// blockIdx.x: 64 columns, blockIdx.y: a run of rows -> part[blockIdx.y][nb + 1][C] (q < nb: sum u*xhat_q, q == nb: sum u)
template <typename T>
__global__ __launch_bounds__(256) void ln_bwd_cols_kernel(LnArgs a, const T* __restrict__ dy, int lddy, const T* __restrict__ y, int ldy,
                                                          const LnStats* __restrict__ stats, long long rows_per, float* __restrict__ part) {
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
                    const LnStats t = stats[(size_t)b * a.M + r];
                    acc[b] += u * (t.centred(((const T*)a.z[b])[r * a.ldz[b] + c]) * t.rstd);
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

// part [rows][nb + 1][C] -> dgamma_b, dbeta_b: 32 columns of one quantity per workgroup, 8 row lanes, fp64 sums in a fixed
// order (no atomics: the same bits every time)
__global__ __launch_bounds__(256) void ln_bwd_finalize_kernel(const float* __restrict__ part, int rows, int nb, int C, LnGrads g) {
    __shared__ double red[8][33];
    const int q = blockIdx.y, col = threadIdx.x & 31, rl = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + col;
    double s = 0.0;
    if (c < C) {
        const float* p = part + (size_t)q * C + c;
        const size_t ld = (size_t)(nb + 1) * C;
        int r = rl;
        for (; r + 56 < rows; r += 64) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[(r + 8 * i) * ld];
#pragma unroll
            for (int i = 0; i < 8; ++i) s += (double)v[i];
        }
        for (; r < rows; r += 8) s += (double)p[r * ld];
    }
    red[rl][col] = s;
    __syncthreads();
    if (rl == 0 && c < C) {
        s = 0.0;
        for (int i = 0; i < 8; ++i) s += red[i][col];
        if (q < nb) {
            if (g.dgamma[q]) g.dgamma[q][c] = (float)s;
        } else {
            for (int b = 0; b < nb; ++b)
                if (g.dbeta[b]) g.dbeta[b][c] = (float)s;
        }
    }
}

// ---------------------------------------------------------------------------------------------------

// How a shape is laid out over lanes; rows: by the row kernels.
struct LnPlan { bool rows, wg, mem, exact; int nb, V, L, block, grid, groups; };

static LnPlan ln_plan(int dtype, int nb, long long M, int C, bool bwd) {
    const int epv = dtype == UNET_BF16 ? 8 : 4, nvec = (C + epv - 1) / epv, wide = 16 / epv;    // at most 16 channels a lane and branch
    // NB of the kernel: nb itself where a RepUNet has so many (one, two kernel sizes) or a plain layer norm, else 4 or 8 and a bound
    // at run time
    LnPlan p = {C < epv || C > 16 * LN_BLOCK, false, false, false, nb == 1 || nb == 3 || nb == 6 ? nb : nb <= 4 ? 4 : 8, 1, 1, 256, 0, 1};
    if (nvec > 64) p.V = wide;
    const int lanes = (nvec + p.V - 1) / p.V;
    if (lanes <= 64) {                                  // a wave holds whole rows
        p.L = p.V > 1 ? 32 : 2;
        while (p.L < lanes) p.L <<= 1;
        if (p.V > 1) {                                  // (fewer, larger workgroups: fewer rows of partial sums)
            if (bwd) p.groups = (nb + 2) / 3;           // three branches to a wave: their sums take 64 registers
            p.block = LN_BLOCK / 64 / p.groups * 64 * p.groups;
        }
    } else {                                            // several waves do (backward: one branch to a workgroup)
        p.wg = true;
        if (bwd) p.V = 2;                               // (1024 threads of 128 registers: 32 bytes of each tensor a thread)
        p.L = (nvec + 64 * p.V - 1) / (64 * p.V) * 64;
        // Forward, threads: bf16 with a tenth of the lanes or more idle as many as fit (us, 512 | 1024 threads: 58181 x 1100 94 | 67,
        // 41666 x 1536 62 | 55, 14222 x 4500 63 | 57), with full lanes about 512 (32000 x 2000 54 | 58, 15625 x 4096 50 | 55); fp32 at
        // most 512 (16000 x 2000 50 | 53).  Several branches: weights in LDS where they fit and 16 rows a workgroup share them
        // (from memory | from LDS: 8000 x 2000 x 3 bf16 34 | 31, 30000 x 8192 x 3 420 | 354; 2666 x 6000 x 3 38 | 44, 300 x 8192 x 3 13 | 19).
        p.mem = !bwd && nb > 1 && (M < 16 * 256 || (size_t)nb * p.L * 64 > LN_LDS);
        const int most = bwd ? 2 * LN_BLOCK : ln_fwd_most(dtype == UNET_BF16 ? 2 : 4, nb, p.mem);
        const int near = (LN_BLOCK + p.L / 2) / p.L * p.L;
        p.block = !bwd && 10 * nvec >= 9 * p.L * p.V && near <= most ? near : most / p.L * p.L;
    }
    p.exact = C == p.L * p.V * epv;
    // Workgroups: few, so that weights are loaded and partial sums written seldom, and as many as fit at once (no second round).
    // Measured (us): V > 1: forward 8192 x 4096 bf16 192: 34.6, 256: 30.2, 384: 34.7, 512: 33.0, backward 8192 x 1024 x 6 192: 64,
    // 256: 59, 384: 74, 512: 72; V = 1: forward 2.1 M x 64 x 6 1024: 373, 1280: 367, 1536: 386, 2048: 372, 2.1 M x 64 x 3 fp32 1024: 408,
    // 1280: 406, 2048: 435; backward, six branches on 16 lanes and more, 0.5 M x 128 x 6 512: 355, 768: 376; 8 lanes, 2.1 M x 64 x 6
    // 512: 782, 768: 760; 1 M x 64 x 3 fp32 512: 390, 768: 385, 1024: 415; 2.1 M x 64 x 1 512: 142, 768: 140, 1024: 150.  A row of
    // several waves has a workgroup per branch: 256 of them over all branches (256 rows of partial sums instead): 2048 x 8192 x 2
    // 49 (64), 4096 x 2048 x 3 40 (50), 20000 x 1536 x 8 297 (346), 512 x 8192 x 2 fp32 33 (46).
    if (p.rows) p.grid = bwd ? 256 : 8192;
    else if (p.wg && bwd) p.grid = 256 / nb;
    else if (p.V > 1) p.grid = 256;
    else if (!bwd) p.grid = 1280;
    else p.grid = nb >= 6 && p.L > 8 ? 512 : 768;
    return p;
}

static inline int ln_rows_per_wg(const LnPlan& p) { return p.rows ? 4 : p.block / p.groups / p.L; }

// The backward's row kernels take that many rows at a time: their workspace has a bound, and no fp32 sum of the column pass runs over
// more than 1024 rows.
constexpr long long LN_CHUNK = 1 << 20;

// rows of partial sums of the backward = its workgroups (the row kernels: of each chunk)
static inline int ln_parts(const LnPlan& p, long long M) {
    const int rows = p.rows ? 64 : ln_rows_per_wg(p);
    if (p.rows && M > LN_CHUNK) M = LN_CHUNK;
    const long long n = (M + rows - 1) / rows;
    return (int)(n < p.grid ? n : p.grid);
}
static inline int ln_chunks(const LnPlan& p, long long M) { return p.rows ? (int)((M + LN_CHUNK - 1) / LN_CHUNK) : 1; }
// floats of the row kernels' statistics
static inline size_t ln_stats(const LnPlan& p, int nb, long long M) { return p.rows ? 3 * (size_t)nb * (M < LN_CHUNK ? M : LN_CHUNK) : 0; }

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


template <auto KERNEL, typename T>
static int ln_run_fwd(const LnPlan& p, const LnArgs& a, int grid, size_t lds, T* y, int ldy, int relu, hipStream_t s) {
    static DynLdsOnce once;                             // (one for each kernel)
    if (lds > 65536) {
        const int rc = ensure_dyn_lds(once, (const void*)KERNEL, (int)LN_LDS);
        if (rc) return rc;
    }
    hipLaunchKernelGGL(KERNEL, dim3(grid), dim3(p.block), lds, s, a, y, ldy, relu, p.L);
    UNET_LAUNCH_CHECK();
    return 0;
}

template <typename T, int NB, int V, int LC, bool MEM = false>
static int ln_launch_fwd(const LnPlan& p, const LnArgs& a, int grid, T* y, int ldy, int relu, hipStream_t s) {
    constexpr bool BOUND = NB == 4 || NB == 8;          // (a bounded kernel serves exact widths too, there is no second one)
    const size_t lds = !MEM && NB * V * TT<T>::EPV > 32 ? (size_t)a.nb * p.L * V * TT<T>::EPV * 4 : 0;
    if constexpr (!BOUND) {
        if (p.exact) return ln_run_fwd<ln_fwd_kernel<T, NB, BOUND, V, LC, true, MEM>>(p, a, grid, lds, y, ldy, relu, s);
    }
    return ln_run_fwd<ln_fwd_kernel<T, NB, BOUND, V, LC, false, MEM>>(p, a, grid, lds, y, ldy, relu, s);
}

template <typename T, int NB>
static int ln_fwd_waves(const LnPlan& p, const LnArgs& a, int grid, T* y, int ldy, int relu, hipStream_t s) {
    constexpr int VW = 16 / TT<T>::EPV;
    if (p.V > 1) return p.L == 32 ? ln_launch_fwd<T, NB, VW, 32>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, NB, VW, 64>(p, a, grid, y, ldy, relu, s);
    if (p.L == 2) return ln_launch_fwd<T, NB, 1, 2>(p, a, grid, y, ldy, relu, s);
    if (p.L == 4) return ln_launch_fwd<T, NB, 1, 4>(p, a, grid, y, ldy, relu, s);
    if (p.L == 8) return ln_launch_fwd<T, NB, 1, 8>(p, a, grid, y, ldy, relu, s);
    if (p.L == 16) return ln_launch_fwd<T, NB, 1, 16>(p, a, grid, y, ldy, relu, s);
    if (p.L == 32) return ln_launch_fwd<T, NB, 1, 32>(p, a, grid, y, ldy, relu, s);
    return ln_launch_fwd<T, NB, 1, 64>(p, a, grid, y, ldy, relu, s);
}

template <typename T>
static int ln_fwd(const LnPlan& p, const LnArgs& a, T* y, int ldy, int relu, hipStream_t s) {
    constexpr int VW = 16 / TT<T>::EPV;
    const long long n = (a.M + ln_rows_per_wg(p) - 1) / ln_rows_per_wg(p);
    const int grid = (int)(n < p.grid ? n : p.grid);
    if (p.rows) {
        hipLaunchKernelGGL((ln_fwd_rows_kernel<T>), dim3(grid), dim3(256), 0, s, a, y, ldy, relu);
        UNET_LAUNCH_CHECK();
        return 0;
    }
    if (p.wg) {             // (bounded kernels also for three and six branches: those of exactly so many spill)
        if (a.nb == 1) return ln_launch_fwd<T, 1, VW, 0>(p, a, grid, y, ldy, relu, s);
        if (p.mem) return ln_launch_fwd<T, 8, VW, 0, true>(p, a, grid, y, ldy, relu, s);
        return a.nb <= 4 ? ln_launch_fwd<T, 4, VW, 0>(p, a, grid, y, ldy, relu, s) : ln_launch_fwd<T, 8, VW, 0>(p, a, grid, y, ldy, relu, s);
    }
    if (p.nb == 1) return ln_fwd_waves<T, 1>(p, a, grid, y, ldy, relu, s);
    if (p.nb == 3) return ln_fwd_waves<T, 3>(p, a, grid, y, ldy, relu, s);
    if (p.nb == 4) return ln_fwd_waves<T, 4>(p, a, grid, y, ldy, relu, s);
    if (p.nb == 6) return ln_fwd_waves<T, 6>(p, a, grid, y, ldy, relu, s);
    return ln_fwd_waves<T, 8>(p, a, grid, y, ldy, relu, s);
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
    const LnPlan p = ln_plan(dtype, nb, M, C, false);
    return dtype == UNET_BF16 ? ln_fwd<__bf16>(p, a, (__bf16*)y + yoff, ldy, relu, (hipStream_t)stream)
                              : ln_fwd<float>(p, a, (float*)y + yoff, ldy, relu, (hipStream_t)stream);
}

extern "C" int unet_layer_norm_bwd_ws(int dtype, int nb, long long M, int C) {
    if ((dtype != UNET_F32 && dtype != UNET_BF16) || nb < 1 || nb > LN_MAXB || M < 0 || C < 1) return -1;
    const LnPlan p = ln_plan(dtype, nb, M, C, true);
    const double n = (double)ln_stats(p, nb, M) + (double)ln_parts(p, M) * ln_chunks(p, M) * (nb + 1) * C;
    return n > 2147483647.0 ? -1 : (int)n;
}

template <typename T, int NB, bool BOUND, int V, int LC>
static void ln_launch_bwd(const LnPlan& p, const LnArgs& a, int parts, const T* dy, int lddy, const T* y, int ldy, float* part, hipStream_t s) {
    constexpr int W = V * TT<T>::EPV;
    const dim3 grid(LC == 0 ? parts * ((a.nb + NB - 1) / NB) : parts);
    const size_t weights = LC == 0 ? (size_t)NB * p.L * W * 4 : NB * W > 32 ? (size_t)(a.nb > NB ? a.nb : NB) * p.L * W * 4 : 0;
    const size_t sums = (size_t)(LC == 0 ? p.block : p.block / 64 * p.L) * TT<T>::EPV * 4;
    const size_t lds = weights > sums ? weights : sums;
    if (p.exact && !BOUND) hipLaunchKernelGGL((ln_bwd_kernel<T, NB, BOUND, V, LC, !BOUND>), grid, dim3(p.block), lds, s, a, dy, lddy, y, ldy, part, parts, p.L);
    else hipLaunchKernelGGL((ln_bwd_kernel<T, NB, BOUND, V, LC, false>), grid, dim3(p.block), lds, s, a, dy, lddy, y, ldy, part, parts, p.L);
}

template <typename T, int NB>
static void ln_bwd_waves(const LnPlan& p, const LnArgs& a, int parts, const T* dy, int lddy, const T* y, int ldy, float* part, hipStream_t s) {
    constexpr bool B = NB == 4 || NB == 8;
    if (p.L == 2) ln_launch_bwd<T, NB, B, 1, 2>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.L == 4) ln_launch_bwd<T, NB, B, 1, 4>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.L == 8) ln_launch_bwd<T, NB, B, 1, 8>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.L == 16) ln_launch_bwd<T, NB, B, 1, 16>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.L == 32) ln_launch_bwd<T, NB, B, 1, 32>(p, a, parts, dy, lddy, y, ldy, part, s);
    else ln_launch_bwd<T, NB, B, 1, 64>(p, a, parts, dy, lddy, y, ldy, part, s);
}

// 16 channels a lane: three branches to a wave
template <typename T, int LC>
static void ln_bwd_wide(const LnPlan& p, const LnArgs& a, int parts, const T* dy, int lddy, const T* y, int ldy, float* part, hipStream_t s) {
    constexpr int VW = 16 / TT<T>::EPV;
    if (a.nb == 1) ln_launch_bwd<T, 1, false, VW, LC>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (a.nb % 3 == 0) ln_launch_bwd<T, 3, false, VW, LC>(p, a, parts, dy, lddy, y, ldy, part, s);
    else ln_launch_bwd<T, 3, true, VW, LC>(p, a, parts, dy, lddy, y, ldy, part, s);
}

template <typename T>
static int ln_bwd(const LnPlan& p, const LnArgs& a, int parts, const T* dy, int lddy, const T* y, int ldy, float* ws, float* part, hipStream_t s) {
    if (p.rows) {
        LnArgs c = a;
        for (long long r = 0; r < a.M; r += LN_CHUNK) {
            c.M = a.M - r < LN_CHUNK ? a.M - r : LN_CHUNK;
            for (int b = 0; b < a.nb; ++b) {
                c.z[b] = (const T*)a.z[b] + r * a.ldz[b];
                c.dz[b] = (T*)a.dz[b] + r * a.C;
            }
            const T *dyr = dy + r * lddy, *yr = y ? y + r * ldy : nullptr;
            hipLaunchKernelGGL((ln_bwd_rows_kernel<T>), dim3((unsigned)((c.M + 3) / 4 < 8192 ? (c.M + 3) / 4 : 8192)), dim3(256), 0, s, c, dyr, lddy, yr, ldy, (LnStats*)ws);
            UNET_LAUNCH_CHECK();
            hipLaunchKernelGGL((ln_bwd_cols_kernel<T>), dim3((a.C + 63) / 64, parts), dim3(256), 0, s, c, dyr, lddy, yr, ldy, (const LnStats*)ws, (c.M + parts - 1) / parts,
                               part + r / LN_CHUNK * parts * (a.nb + 1) * a.C);
            UNET_LAUNCH_CHECK();
        }
    } else if (p.wg) ln_launch_bwd<T, 1, false, 2, 0>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.V > 1) p.L == 32 ? ln_bwd_wide<T, 32>(p, a, parts, dy, lddy, y, ldy, part, s) : ln_bwd_wide<T, 64>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 1) ln_bwd_waves<T, 1>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 3) ln_bwd_waves<T, 3>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 4) ln_bwd_waves<T, 4>(p, a, parts, dy, lddy, y, ldy, part, s);
    else if (p.nb == 6) ln_bwd_waves<T, 6>(p, a, parts, dy, lddy, y, ldy, part, s);
    else ln_bwd_waves<T, 8>(p, a, parts, dy, lddy, y, ldy, part, s);
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
    const LnPlan p = ln_plan(dtype, nb, M, C, true);
    const int parts = ln_parts(p, M);
    float* part = ws + ln_stats(p, nb, M);
    if (M > 0) {
        const int e = dtype == UNET_BF16
            ? ln_bwd<__bf16>(p, a, parts, (const __bf16*)dy + dyoff, lddy, y ? (const __bf16*)y + yoff : nullptr, ldy, ws, part, s)
            : ln_bwd<float>(p, a, parts, (const float*)dy + dyoff, lddy, y ? (const float*)y + yoff : nullptr, ldy, ws, part, s);
        if (e) return e;
    }
    if (dgamma || dbeta) {
        hipLaunchKernelGGL(ln_bwd_finalize_kernel, dim3((C + 31) / 32, nb + 1), dim3(256), 0, s, part, parts * ln_chunks(p, M), nb, C, g);
        UNET_LAUNCH_CHECK();
    }
    return 0;
}
