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
// Rounding is stochastic (dither: 20 bits, uniform, from a hash of the step's key and the element's index in its tensor, so a
// step is reproducible whatever the launch looks like): beta2*v changes v by 0.1 % a step, less than half a code step, which
// rounding to nearest would throw away at every step.  A second moment that is not zero never gets code 0: its smallest value,
// 2^-33 of the block's scale, is the square of 2^-16.5, the first moment's smallest is 2^-17, so an element that is all
// rounding noise moves by about lr at most.  e = 255: the block held a value that is not finite (or above 1.875 * 2^127),
// and every value of it reads as NaN.
#include "common.h"

constexpr int A8_BLOCK = 64;
constexpr int A8_MAX = 112;             // tensors per launch: the table stays under 4 KB of kernel arguments
constexpr int A8_CHUNK = 4096;          // elements per workgroup
constexpr int A8_TOP_M = 15, A8_TOP_V = 31;

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

struct A8Scalars { float decay, omb1, b2, omb2, inv_bc2, eps, step_size; uint32_t key; };

__device__ __forceinline__ uint32_t a8_hash(unsigned long long i, uint32_t key) {
    uint32_t h = (uint32_t)i * 0x9E3779B9u + (uint32_t)(i >> 32) * 0xBB67AE85u + key;
    h = (h ^ (h >> 15)) * 0x6A09E667u;
    return h ^ (h >> 16);
}

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

// one wave per block of 64, one element per lane
__global__ __launch_bounds__(256) void adamw8_kernel(A8Table tb, A8State st, const float* __restrict__ clip, int write_g, A8Scalars k,
                                                     const float* __restrict__ veto) {
    if (veto != nullptr && veto[0] > 0.f) return;
    int t = 0;
    while (t < tb.n - 1 && (int)blockIdx.x >= tb.blk_end[t]) ++t;
    const int chunk = (int)blockIdx.x - (t ? tb.blk_end[t - 1] : 0);
    const int lane = threadIdx.x & 63;
    const long long n = tb.numel[t];
    float *pp = tb.p[t], *pg = tb.g[t];
    const float coef = clip != nullptr ? clip[1] : 1.0f;
    const bool wg = write_g && coef != 1.0f;
    for (int j = threadIdx.x >> 6; j < A8_CHUNK / A8_BLOCK; j += 4) {
        const long long b = (long long)chunk * (A8_CHUNK / A8_BLOCK) + j, i = b * A8_BLOCK + lane;
        if (b * A8_BLOCK >= n) break;
        const size_t sb = (size_t)tb.first[t] + b, si = sb * A8_BLOCK + lane;
        const bool in = i < n;
        float p = 0.f, g = 0.f, m = 0.f, v = 0.f;
        if (in) {
            p = pp[i]; g = pg[i] * coef;
            m = a8_decode<A8_TOP_M>(st.m[si], st.em[sb]);
            v = a8_decode<A8_TOP_V>(st.v[si], st.ev[sb]);
            p *= k.decay;
            m = m + (g - m) * k.omb1;
            v = v * k.b2 + (k.omb2 * g) * g;
            p = p - k.step_size * (m / (sqrtf(v) * k.inv_bc2 + k.eps));
        }
        const int em = a8_exponent(wave_max64(a8_abs_bits(m))), ev = a8_exponent(wave_max64(a8_abs_bits(v)));
        if (in) {
            const uint32_t h = a8_hash((unsigned long long)i, k.key);
            pp[i] = p;
            if (wg) pg[i] = g;
            st.m[si] = (uint8_t)a8_encode<A8_TOP_M>(m, em, ((h & 0xffffu) << 4) | 8u);
            st.v[si] = (uint8_t)a8_encode<A8_TOP_V>(v, ev, ((h >> 16) << 4) | 8u);
        }
        if (lane == 0) { st.em[sb] = (uint8_t)em; st.ev[sb] = (uint8_t)ev; }
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

template <int TOP, typename T>
__global__ __launch_bounds__(256) void moment8_decode_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ exps, long long n,
                                                             T* __restrict__ out) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256)
        out[i] = from_f32<T>(a8_decode<TOP>(codes[i], exps[i / A8_BLOCK]));
}

// ---------------------------------------------------------------------------------------------------

static uint32_t a8_key(unsigned long long seed, unsigned long long step) {
    unsigned long long x = seed * 0x9E3779B97F4A7C15ull + step * 0x6A09E667F3BCC909ull;
    x = (x ^ (x >> 31)) * 0x9E3779B97F4A7C15ull;
    return (uint32_t)(x >> 32);
}

extern "C" int unet_adamw8_step(int nt, void* const* params, void* const* grads, const long long* numel, const long long* first_block,
                                void* exp_avg, void* exp_avg_sq, void* exp_avg_e, void* exp_avg_sq_e, long long state_blocks,
                                const float* norm_out, int write_grads, double lr, double beta1, double beta2, double eps,
                                double weight_decay, long long step, long long seed, const float* veto, void* stream) {
    UNET_CHECK(nt >= 0 && (nt == 0 || (params && grads && numel)), "adamw8_step: null argument");
    UNET_CHECK(step >= 1, "adamw8_step: step must be >= 1 (got %lld)", step);
    UNET_CHECK(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0 && lr >= 0, "adamw8_step: bad hyper-parameters");
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
    const dim3 grid(a8_grid((n + 255) / 256)), blk(256);
    hipStream_t s = (hipStream_t)stream;
    const uint8_t *c = (const uint8_t*)codes, *e = (const uint8_t*)exps;
    if (is_signed && dtype == UNET_F32) hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_M, float>), grid, blk, 0, s, c, e, n, (float*)out);
    else if (is_signed) hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_M, __bf16>), grid, blk, 0, s, c, e, n, (__bf16*)out);
    else if (dtype == UNET_F32) hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_V, float>), grid, blk, 0, s, c, e, n, (float*)out);
    else hipLaunchKernelGGL((moment8_decode_kernel<A8_TOP_V, __bf16>), grid, blk, 0, s, c, e, n, (__bf16*)out);
    UNET_LAUNCH_CHECK();
    return 0;
}
