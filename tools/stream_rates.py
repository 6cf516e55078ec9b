"""Rates of a streaming kernel at the sizes and read / write mixes of the layer norm's and the 8-bit AdamW's cases: the best of 48
launch shapes, tensors in turn so that nothing stays in a cache, passes in a graph.

  hipcc --offload-arch=gfx950 -O3 -fPIC -shared -Xclang -target-feature -Xclang -packed-fp32-ops -o tools/libstream_rates.so tools/stream_rates.hip
  python3 tools/stream_rates.py
"""
import ctypes
import os

import torch

CASES = [("ln_fwd_repunet", 6, 1, 1879e6), ("ln_fwd_wide", 1, 1, 134.2e6), ("ln_fwd_odd_f32", 1, 1, 133.2e6), ("ln_bwd_repunet", 8, 6, 3758e6),
         ("ln_bwd_deep", 8, 6, 234.9e6), ("ln_bwd_wide", 2, 1, 125.9e6), ("forward, 3 branches", 3, 1, 134e6), ("forward, 6 branches", 6, 1, 134e6),
         ("backward, 2 branches", 3, 2, 168e6), ("backward, 3 branches, ReLU", 5, 3, 134e6), ("backward, 6 branches, ReLU", 8, 6, 448e6),
         ("adamw8_ragged, step", 2, 1, 80.3e6), ("adamw8_unet, step", 2, 1, 498.6e6), ("adamw8_repunet, step", 2, 1, 2565e6)]
GAP = 256                                            # vectors between tensors: 4 KiB


def main():
    lib = ctypes.CDLL(os.path.join(os.path.dirname(os.path.abspath(__file__)), "libstream_rates.so"))
    lib.stream_run.argtypes = [ctypes.c_int] * 5 + [ctypes.c_void_p] * 2 + [ctypes.c_longlong] * 2 + [ctypes.c_void_p]
    x = torch.zeros(1 << 29, dtype=torch.int64, device="cuda")
    a, b = x.chunk(2)
    t = best_of(lambda: b.copy_(a), 4)
    print(f"torch's copy_, 2 GiB: {4 * 2 ** 30 / t / 1e6:.2f} TB/s", flush=True)
    del x, a, b
    for name, R, W, size in CASES:
        n = int(size) // 16 // (R + W)
        sets = max(1, min(12, int(1.5e9 // size)))
        bufs = [(torch.zeros(R * (n + GAP) * 2, dtype=torch.int64, device="cuda"), torch.zeros(W * (n + GAP) * 2, dtype=torch.int64, device="cuda"))
                for _ in range(sets)]
        found = []
        for nt in (0, 1):
            for U in (1, 2, 4):
                most = -(-n // (256 * U))
                for grid in sorted({min(g, most) for g in (256, 512, 1024, 2048, 4096, 16384, most)}):
                    turn = [0]

                    def one():
                        src, dst = bufs[turn[0] % sets]
                        turn[0] += 1
                        rc = lib.stream_run(R, W, U, nt, grid, src.data_ptr(), dst.data_ptr(), n, GAP, torch.cuda.current_stream().cuda_stream)
                        assert rc == 0, rc
                    found.append((best_of(one, 12), "streaming" if nt else "plain", U, grid))
        t, kind, U, grid = min(found)
        print(f"{name}: {R} read, {W} written, {size / 1e6:.0f} MB: {t:.1f} us, {size / t / 1e6:.2f} TB/s ({kind}, {U} vectors, {grid} workgroups)", flush=True)
        del bufs
        torch.cuda.empty_cache()


def best_of(f, count):
    """us a call: the best of three replays of a graph of `count` calls."""
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(count):
            f()
    graph.replay()
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    best = 1e9
    for _ in range(3):
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b) / count * 1e3)
    return best


if __name__ == "__main__":
    main()
