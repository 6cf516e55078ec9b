// What HBM gives a kernel that only streams: R tensors read and W written, 16 bytes a thread and access, U vectors of each in flight.
// Built and run by tools/stream_rates.py.
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

// in: R tensors of n vectors, `gap` vectors apart; out: W tensors likewise
template <int R, int W, int U, bool NT>
__global__ __launch_bounds__(256) void stream_kernel(const u32x4* __restrict__ in, u32x4* __restrict__ out, long long n, long long gap) {
    const long long stride = (long long)gridDim.x * 256 * U;
    for (long long i0 = (long long)blockIdx.x * 256 * U + threadIdx.x; i0 < n; i0 += stride) {
        u32x4 v[U][R];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const long long i = i0 + u * 256 < n ? i0 + u * 256 : n - 1;
                v[u][r] = NT ? __builtin_nontemporal_load(in + r * (n + gap) + i) : in[r * (n + gap) + i];
            }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const long long i = i0 + u * 256;
            if (i >= n) continue;
            u32x4 s = v[u][0];
#pragma unroll
            for (int r = 1; r < R; ++r) s ^= v[u][r];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const u32x4 o = s + (uint32_t)w;
                if (NT) __builtin_nontemporal_store(o, out + w * (n + gap) + i);
                else out[w * (n + gap) + i] = o;
            }
        }
    }
}

template <int R, int W> static int launch(int U, int nt, int grid, const void* in, void* out, long long n, long long gap, hipStream_t s) {
#define LAUNCH(u, x) hipLaunchKernelGGL((stream_kernel<R, W, u, x>), dim3(grid), dim3(256), 0, s, (const u32x4*)in, (u32x4*)out, n, gap)
    if (U == 1) { if (nt) LAUNCH(1, true); else LAUNCH(1, false); }
    else if (U == 2) { if (nt) LAUNCH(2, true); else LAUNCH(2, false); }
    else if (U == 4) { if (nt) LAUNCH(4, true); else LAUNCH(4, false); }
    else return -1;
    return (int)hipGetLastError();
}

extern "C" int stream_run(int R, int W, int U, int nt, int grid, const void* in, void* out, long long n, long long gap, void* stream) {
    if (n < 1 || grid < 1) return -1;
    const hipStream_t s = (hipStream_t)stream;
    if (R == 1 && W == 1) return launch<1, 1>(U, nt, grid, in, out, n, gap, s);
    if (R == 2 && W == 1) return launch<2, 1>(U, nt, grid, in, out, n, gap, s);
    if (R == 3 && W == 1) return launch<3, 1>(U, nt, grid, in, out, n, gap, s);
    if (R == 3 && W == 2) return launch<3, 2>(U, nt, grid, in, out, n, gap, s);
    if (R == 5 && W == 3) return launch<5, 3>(U, nt, grid, in, out, n, gap, s);
    if (R == 6 && W == 1) return launch<6, 1>(U, nt, grid, in, out, n, gap, s);
    if (R == 8 && W == 6) return launch<8, 6>(U, nt, grid, in, out, n, gap, s);
    return -1;
}
