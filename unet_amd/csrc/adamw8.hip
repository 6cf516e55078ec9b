// AdamW over many tensors whose moments are held in 8 bits each, 64 consecutive elements to a block.
//
//   g = coef * g;  p *= 1 - lr*wd;  m = m + (g - m)*(1 - beta1);  v = beta2*v + ((1 - beta2)*g)*g
//   p -= lr/(1 - beta1^t) * m / (sqrt(v)/sqrt(1 - beta2^t) + eps)
// in fp32 with m and v as just computed; what is stored of them is rounded to 8 bits.
//
// A block keeps one biased exponent e = (bits(max |x|) + 0xfffff) >> 23, at least 32: no rounding of its values leaves the
// code range.  Relative to it a first moment is sign | 4 exponent bits | 3 mantissa bits, a second moment, never negative,
// 5 exponent bits | 3 mantissa bits, both with subnormals:
//   code = (bits(|x| * 2^(X - e)) + dither) >> 20,   value = float(code << 20) * 2^(e - X),   X = 15 / 31
// Rounding is stochastic (dither: the middle of one of 2^16 equal parts of a code step, 16 bits of a hash of the step's key and the
// element's index in its tensor, so a step is reproducible whatever the launch looks like): beta2*v changes v by 0.1 % a step, less than half a code step, which
// rounding to nearest would throw away at every step.  A second moment that is not zero never gets code 0: its smallest value,
// 2^-33 of the block's scale, is the square of 2^-16.5, the first moment's smallest is 2^-17, so an element that is all
// rounding noise moves by about lr at most.  Probabilities come in units of 2^-16: a stored moment's mean is off by at most 2^-17 of
// a code step a step, 2^-17/(1 - beta) in the long run (0.008 code steps at beta2 = 0.999), and a change under 2^-17 of a code step is
// always rounded away; 1 - beta under 2^-17 is refused, where the smallest codes would never move.  e = 255: the block held a value that is not finite (or above 1.875 * 2^127),
// and every value of it reads as NaN.
#include "common.h"

constexpr int A8_BLOCK = 64;
constexpr int A8_MAX = 112;             // tensors per launch: the table stays under 4 KB of kernel arguments
constexpr int A8_CHUNK = 4096;          // elements per workgroup
constexpr int A8_TOP_M = 15, A8_TOP_V = 31;
constexpr double A8_LEAST = 0x1p-17;    // of 1 - beta

struct A8Table {
    int n;
    int blk_end[A8_MAX];                // running end of each tensor's workgroup range inside this launch
    uint32_t first[A8_MAX];             // the tensor's first block in the moments' buffers
    long long numel[A8_MAX];
    float* p[A8_MAX];
    float* g[A8_MAX];
};
struct A8State {
    uint8_t* m;
    uint8_t* v;
    uint8_t* em;
    uint8_t* ev;
};

struct A8Scalars { float decay, omb1, b2, omb2, inv_bc2, eps, step_size; uint32_t key; int precise; };

__device__ __forceinline__ uint32_t a8_abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// the block's exponent from the largest |x| bits in it
__device__ __forceinline__ int a8_exponent(uint32_t maxbits) {
    const int e = (int)((maxbits + 0xfffffu) >> 23);
    return e < 32 ? 32 : e > 255 ? 255 : e;
}

template <int TOP>
__device__ __forceinline__ uint32_t a8_encode(float x, int e, uint32_t dither) {
    if (e == 255) return 0;
    const uint32_t c = (__float_as_uint(ldexpf(fabsf(x), TOP - e)) + dither) >> 20;
    if (TOP == A8_TOP_V) return c == 0 && x > 0.f ? 1 : c;
    return x < 0.f ? c | 128u : c;
}

template <int TOP>
__device__ __forceinline__ float a8_decode(uint32_t c, int e) {
    if (e == 255) return __uint_as_float(0x7fc00000u);
    const float mag = ldexpf(__uint_as_float((TOP == A8_TOP_V ? c : c & 127u) << 20), e - TOP);
    return TOP == A8_TOP_M && (c & 128u) ? -mag : mag;
}

__device__ __forceinline__ uint32_t wave_max64(uint32_t v) {
    for (int o = 1; o < 64; o <<= 1) { const uint32_t w = (uint32_t)__shfl_xor((int)v, o); v = v > w ? v : w; }
    return v;
}

// Four consecutive elements.  16-byte accesses need no alignment beyond that of a float.
typedef __attribute__((ext_vector_type(4), aligned(4))) float a8_f32x4;

struct A8Quad {
    float x[4];
    __device__ __forceinline__ void load(const float* p, int n) {
        if (n >= 4) {
            const a8_f32x4 v = *(const a8_f32x4*)p;
            x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = j < n ? p[j] : 0.f;
        }
    }
    __device__ __forceinline__ void store(float* p, int n) const {
        if (n >= 4) {
            const a8_f32x4 v = {x[0], x[1], x[2], x[3]};
            *(a8_f32x4*)p = v;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) if (j < n) p[j] = x[j];
        }
    }
};

// the largest of the 16 lanes of a block
__device__ __forceinline__ uint32_t a8_max16(uint32_t v) {
    auto step = [](uint32_t a, int b) { return a > (uint32_t)b ? a : (uint32_t)b; };
    v = step(v, __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
    v = step(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
    v = step(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));
    v = step(v, __builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xf, 0xf, true));
    return v;
}

template <int TOP>
__device__ __forceinline__ void a8_decode4(uint32_t word, int e, float (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t c = word >> (8 * j);
        const float mag = ldexpf(__uint_as_float((c & (TOP == A8_TOP_V ? 255u : 127u)) << 20), e - TOP);
        x[j] = TOP == A8_TOP_V ? mag : __uint_as_float(__float_as_uint(mag) | ((c & 128u) << 24));
    }
    if (e == 255) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __uint_as_float(0x7fc00000u);
    }
}

template <int TOP>
__device__ __forceinline__ uint32_t a8_encode4(const float (&x)[4], int e, const uint32_t (&dither)[4]) {
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t c = (__float_as_uint(ldexpf(fabsf(x[j]), TOP - e)) + dither[j]) >> 20;
        if (TOP == A8_TOP_V) c = c == 0 && x[j] > 0.f ? 1u : c;
        else c |= x[j] < 0.f ? 128u : 0u;
        word |= c << (8 * j);
    }
    return e == 255 ? 0u : word;
}

// 16 lanes share a block, 4 elements a lane; a wave takes 4 runs of 256 elements, whose loads are all requested first.  Bound by
// HBM: 16.06 bytes an element (p 4 + 4, g 4, codes 2 + 2, exponents), 99 us for 31 M parameters and 488 us for 160 M on one
// MI355X = 5.0-5.3 TB/s, where a kernel that only streams these bytes takes 79 and 404 us; one element a lane (byte-wide code accesses) took 197 and 1068 us.  The
// arithmetic, about 80 instructions an element, fits under that with the hardware's root and reciprocal (1 unit in the last
// place each, in the parameter's update alone; the moments are bit for bit those of single-rounded fp32 operations).
__global__ __launch_bounds__(256) void adamw8_kernel(A8Table tb, A8State st, const float* __restrict__ clip, int write_g, A8Scalars k,
                                                     const float* __restrict__ veto) {
    if (veto != nullptr && veto[0] > 0.f) return;
    const int lane = threadIdx.x & 63;
    // the tensor: how many of the ranges end at or before this workgroup
    const int t = __popcll(__ballot((int)blockIdx.x >= tb.blk_end[lane])) +
                  __popcll(__ballot(lane + 64 < A8_MAX && (int)blockIdx.x >= tb.blk_end[lane + 64 < A8_MAX ? lane + 64 : 0]));
    const int chunk = (int)blockIdx.x - (t ? tb.blk_end[t - 1] : 0);
    const long long n = tb.numel[t];
    float *pp = tb.p[t], *pg = tb.g[t];
    const size_t first = tb.first[t];
    const float coef = clip != nullptr ? clip[1] : 1.0f;
    const bool wg = write_g && coef != 1.0f;
    const int sub = lane >> 4;
    constexpr int IT = A8_CHUNK / 1024;             // 256-element runs of a wave
    const long long run0 = (long long)chunk * (A8_CHUNK / 256) + (threadIdx.x >> 6) * IT;
    A8Quad P[IT], G[IT];
    uint32_t mw[IT], vw[IT], me[IT], ve[IT];
    auto left = [&](int j) -> int {                 // elements of run j that are this lane's: 4, fewer at the tensor's end, or none
        const long long r = n - ((run0 + j) * 256 + lane * 4);
        return r >= 4 ? 4 : r > 0 ? (int)r : 0;
    };
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        const int c = left(j);
        const long long i = (run0 + j) * 256 + lane * 4;
        const size_t blk = first + (run0 + j) * 4 + sub;
        mw[j] = vw[j] = me[j] = ve[j] = 0;
        P[j].load(pp + i, c);
        G[j].load(pg + i, c);
        if (c > 0) {
            mw[j] = *(const uint32_t*)(st.m + blk * A8_BLOCK + (lane & 15) * 4);
            vw[j] = *(const uint32_t*)(st.v + blk * A8_BLOCK + (lane & 15) * 4);
            me[j] = st.em[blk];
            ve[j] = st.ev[blk];
        }
    }
#pragma unroll
    for (int j = 0; j < IT; ++j) {
        if ((run0 + j) * 256 >= n) break;
        const int c = left(j);
        const long long i = (run0 + j) * 256 + lane * 4;
        const size_t blk = first + (run0 + j) * 4 + sub;
        float m[4], v[4];
        a8_decode4<A8_TOP_M>(mw[j], (int)me[j], m);
        a8_decode4<A8_TOP_V>(vw[j], (int)ve[j], v);
        uint32_t mx = 0, vx = 0, dm[4], dv[4];
        uint32_t h0 = (uint32_t)i * 0x9E3779B9u + (uint32_t)((unsigned long long)i >> 32) * 0xBB67AE85u + k.key;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float &p = P[j].x[e], &g = G[j].x[e];
            g *= coef;
            p *= k.decay;
            m[e] = m[e] + (g - m[e]) * k.omb1;
            v[e] = v[e] * k.b2 + (k.omb2 * g) * g;
            if (e >= c) m[e] = v[e] = 0.f;          // (behind the tensor's end: nothing that the block's exponent may see)
            const float denom = k.precise ? sqrtf(v[e]) * k.inv_bc2 + k.eps : __builtin_amdgcn_sqrtf(v[e]) * k.inv_bc2 + k.eps;
            p = p - k.step_size * (k.precise ? m[e] / denom : m[e] * __builtin_amdgcn_rcpf(denom));
            const uint32_t mb = a8_abs_bits(m[e]), vb = a8_abs_bits(v[e]);
            mx = mx > mb ? mx : mb;
            vx = vx > vb ? vx : vb;
            uint32_t h = h0 + (uint32_t)e * 0x9E3779B9u;
            h = (h ^ (h >> 15)) * 0x6A09E667u;
            h ^= h >> 16;
            dm[e] = ((h & 0xffffu) << 4) | 8u;
            dv[e] = ((h >> 16) << 4) | 8u;
        }
        const int em = a8_exponent(a8_max16(mx)), ev = a8_exponent(a8_max16(vx));
        if (c > 0) {
            P[j].store(pp + i, c);
            if (wg) G[j].store(pg + i, c);
            *(uint32_t*)(st.m + blk * A8_BLOCK + (lane & 15) * 4) = a8_encode4<A8_TOP_M>(m, em, dm);
            *(uint32_t*)(st.v + blk * A8_BLOCK + (lane & 15) * 4) = a8_encode4<A8_TOP_V>(v, ev, dv);
            if ((lane & 15) == 0) { st.em[blk] = (uint8_t)em; st.ev[blk] = (uint8_t)ev; }
        }
    }
}

template <int TOP>
__global__ __launch_bounds__(256) void moment8_encode_kernel(const float* __restrict__ x, long long n, uint8_t* __restrict__ codes,
                                                             uint8_t* __restrict__ exps) {
    const int lane = threadIdx.x & 63;
    const long long blocks = (n + A8_BLOCK - 1) / A8_BLOCK;
    for (long long b = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); b < blocks; b += (long long)gridDim.x * 4) {
        const long long i = b * A8_BLOCK + lane;
        const float f = i < n ? x[i] : 0.f;
        const int e = a8_exponent(wave_max64(a8_abs_bits(f)));
        if (i < n) codes[i] = (uint8_t)a8_encode<TOP>(f, e, 0x80000u);
        if (lane == 0) exps[b] = (uint8_t)e;
    }
}

// 16 consecutive elements a lane (a quarter of a block): one 16-byte load, 32 or 64 bytes stored
template <int TOP, typename T>
__global__ __launch_bounds__(256) void moment8_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, long long n,
                                                             T* __restrict__ out) {
    typedef __attribute__((ext_vector_type(4), aligned(1))) uint32_t u32x4;
    constexpr int EPV = TT<T>::EPV;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 16; i < n; i += (long long)gridDim.x * 4096) {
        const int e = exps[i / A8_BLOCK];
        if (i + 16 <= n) {
            const u32x4 w = *(const u32x4*)(codes + i);
            float x[16];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float f[4];
                a8_decode4<TOP>(w[q], e, f);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[4 * q + j] = f[j];
            }
#pragma unroll
            for (int q = 0; q < 16 / EPV; ++q) *(uint4*)(out + i + q * EPV) = Vec16<T>::pack(x + q * EPV);
        } else {
            for (int j = 0; i + j < n; ++j) out[i + j] = from_f32<T>(a8_decode<TOP>(codes[i + j], e));
        }
    }
}

// ---------------------------------------------------------------------------------------------------

static uint32_t a8_key(unsigned long long seed, unsigned long long step) {
    unsigned long long x = seed * 0x9E3779B97F4A7C15ull + step * 0x6A09E667F3BCC909ull;
    x = (x ^ (x >> 31)) * 0x9E3779B97F4A7C15ull;
    return (uint32_t)(x >> 32);
}

extern "C" int unet_adamw8_blocks(int nt, const long long* numel) {
    long long n = 0;
    for (int i = 0; i < nt; ++i) n += (numel[i] + A8_BLOCK - 1) / A8_BLOCK;
    return n > 0x7fffffffLL ? -1 : (int)n;
}

extern "C" int unet_adamw8_step(int nt, void* const* params, void* const* grads, const long long* numel, const long long* first_block,
                                void* exp_avg, void* exp_avg_sq, void* exp_avg_e, void* exp_avg_sq_e, long long state_blocks,
                                const float* norm_out, int write_grads, double lr, double beta1, double beta2, double eps,
                                double weight_decay, long long step, long long seed, const float* veto, void* stream) {
    UNET_CHECK(nt >= 0 && (nt == 0 || (params && grads && numel)), "adamw8_step: null argument");
    UNET_CHECK(step >= 1, "adamw8_step: step must be >= 1 (got %lld)", step);
    UNET_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && lr >= 0, "adamw8_step: bad hyper-parameters");
    UNET_CHECK(1 - beta1 >= A8_LEAST && 1 - beta2 >= A8_LEAST, "adamw8_step: bad hyper-parameters (8-bit moments follow a beta up to 1 - 2^-17)");
    UNET_CHECK(state_blocks >= 0 && state_blocks < (1LL << 32), "adamw8_step: too many blocks of state");
    UNET_CHECK(state_blocks == 0 || (exp_avg && exp_avg_sq && exp_avg_e && exp_avg_sq_e), "adamw8_step: null state");
    UNET_CHECK((((size_t)exp_avg | (size_t)exp_avg_sq) & 15) == 0, "adamw8_step: the state buffers must be 16-byte aligned");
    long long at = 0, wgs = 0;
    for (int i = 0; i < nt; ++i) {          // everything is checked before the first launch
        UNET_CHECK(numel[i] >= 0 && numel[i] < (1LL << 38), "adamw8_step: tensor %d has a bad size", i);
        UNET_CHECK(numel[i] == 0 || (params[i] && grads[i]), "adamw8_step: tensor %d has a null pointer", i);
        const long long b0 = first_block ? first_block[i] : at, nblk = (numel[i] + A8_BLOCK - 1) / A8_BLOCK;
        UNET_CHECK(b0 >= 0 && b0 + nblk <= state_blocks, "adamw8_step: tensor %d lies outside the state (blocks %lld..%lld of %lld)", i, b0,
                   b0 + nblk, state_blocks);
        at = b0 + nblk;
        wgs += (numel[i] + A8_CHUNK - 1) / A8_CHUNK;
    }
    UNET_CHECK(wgs < (1LL << 31), "adamw8_step: too many elements");
    A8Scalars k;
    k.decay = (float)(1.0 - lr * weight_decay);
    k.omb1 = (float)(1.0 - beta1);
    k.b2 = (float)beta2;
    k.omb2 = (float)(1.0 - beta2);
    k.inv_bc2 = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)step)));
    k.eps = (float)eps;
    k.step_size = (float)(lr / (1.0 - pow(beta1, (double)step)));
    // the hardware's root takes v under 2^-126 for zero: what is lost, up to 2^-63 * inv_bc2, has to be under half a unit of eps
    // (2^-24 * eps; then no reciprocal is taken of a number that small either)
    k.precise = eps < 0x1p-39 * k.inv_bc2;
    k.key = a8_key((unsigned long long)seed, (unsigned long long)step);
    const A8State st = {(uint8_t*)exp_avg, (uint8_t*)exp_avg_sq, (uint8_t*)exp_avg_e, (uint8_t*)exp_avg_sq_e};
    hipStream_t s = (hipStream_t)stream;
    at = 0;
    for (int i = 0; i < nt;) {
        A8Table tb; tb.n = 0; long long nb = 0;
        for (; i < nt && tb.n < A8_MAX; ++i) {
            const long long b0 = first_block ? first_block[i] : at;
            at = b0 + (numel[i] + A8_BLOCK - 1) / A8_BLOCK;
            if (numel[i] == 0) continue;
            nb += (numel[i] + A8_CHUNK - 1) / A8_CHUNK;
            const int e = tb.n++;
            tb.blk_end[e] = (int)nb; tb.numel[e] = numel[i]; tb.first[e] = (uint32_t)b0;
            tb.p[e] = (float*)params[i]; tb.g[e] = (float*)grads[i];
        }
        if (tb.n == 0) continue;
        for (int e = tb.n; e < A8_MAX; ++e) tb.blk_end[e] = 0x7fffffff;
        hipLaunchKernelGGL(adamw8_kernel, dim3((unsigned)nb), dim3(256), 0, s, tb, st, norm_out, write_grads, k, veto);
        UNET_LAUNCH_CHECK();
    }
    return 0;
}

static inline int a8_grid(long long wgs) { return (int)(wgs < 8192 ? wgs : 8192); }

extern "C" int unet_moment8_encode(int is_signed, const float* x, long long n, void* codes, void* exps, void* stream) {
    UNET_CHECK(n >= 0 && (n == 0 || (x && codes && exps)), "moment8_encode: null argument");
    if (n == 0) return 0;
    const dim3 grid(a8_grid((n + 255) / 256));
    if (is_signed)
        hipLaunchKernelGGL((moment8_encode_kernel<A8_TOP_M>), grid, dim3(256), 0, (hipStream_t)stream, x, n, (uint8_t*)codes, (uint8_t*)exps);
    else
        hipLaunchKernelGGL((moment8_encode_kernel<A8_TOP_V>), grid, dim3(256), 0, (hipStream_t)stream, x, n, (uint8_t*)codes, (uint8_t*)exps);
    UNET_LAUNCH_CHECK();
    return 0;
}

extern "C" int unet_moment8_decode(int is_signed, int dtype, const void* codes, const void* exps, long long n, void* out, void* stream) {
    UNET_CHECK(dtype == UNET_F32 || dtype == UNET_BF16, "moment8_decode: bad dtype %d", dtype);
    UNET_CHECK(n >= 0 && (n == 0 || (out && codes && exps)), "moment8_decode: null argument");
    if (n == 0) return 0;
    UNET_CHECK(((size_t)out & 15) == 0, "moment8_decode: the output must be 16-byte aligned");
    const dim3 grid(a8_grid((n + 4095) / 4096)), blk(256);
    hipStream_t s = (hipStream_t)stream;
    const uint8_t *c = (const uint8_t*)codes, *e = (const uint8_t*)exps;
    if (is_signed && dtype == UNET_F32) hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_M, float>), grid, blk, 0, s, c, e, n, (float*)out);
    else if (is_signed) hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_M, __bf16>), grid, blk, 0, s, c, e, n, (__bf16*)out);
    else if (dtype == UNET_F32) hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_V, float>), grid, blk, 0, s, c, e, n, (float*)out);
    else hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_V, __bf16>), grid, blk, 0, s, c, e, n, (__bf16*)out);
    UNET_LAUNCH_CHECK();
    return 0;
}
