"""Layer norm forward and backward through the C ABI against fp64 (oracle/layer_norm_ref.py), with error bounds that follow
from the formulas; its refusals; RepUNet with norm="layer"."""
import pytest
import torch

from oracle import layer_norm_ref as ref


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs the MI355X")
    return torch.device("cuda:0")


def make(dev, M, C, nb, dtype, seed=0, pad=0, off=0, shape=None):
    """zs (Acts on the device, slices of wider buffers when pad), gammas, betas."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(seed)
    zs = []
    for b in range(nb):
        buf = (torch.randn((1, 1, M, C + pad), generator=g) * (0.5 + 0.4 * b) + 0.7 * b - 0.5).to(dtype)
        zs.append(ops.Act(buf.to(dev), off, C))
    ws = [[torch.randn(C, generator=g).to(dev) * 0.3 + s for _ in range(nb)] for s in (1.0, 0.0)]
    return zs, ws[0], ws[1], g


def rows(act):
    return act.buf[..., act.off:act.off + act.C].reshape(-1, act.C).cpu()


def cpu(ts):
    return [None if t is None else t.cpu() for t in ts]


def check(got, want, bound, dtype, what):
    half = torch.finfo(dtype).eps / 2
    tol = bound * (1 + half) + half * want.abs() + torch.finfo(torch.float32).tiny
    err = (got.double() - want).abs()
    bad = err > tol
    assert not bad.any(), (what, int(bad.sum()), float((err / tol).max()))


CASES = [(1, 8, 1), (3, 64, 6), (65, 16, 3), (1, 1024, 1), (196, 120, 3), (7, 1, 2), (33, 2, 1), (50, 63, 8), (129, 65, 2), (1000, 333, 1),
         (40, 512, 6), (17, 513, 6), (24, 1000, 8), (64, 1024, 3), (20, 2048, 2), (5, 4100, 1), (9, 5120, 1), (3, 8192, 6), (4, 8200, 1),
         (2, 20000, 2), (3, 40001, 1), (4099, 64, 1), (20011, 8, 3), (2500, 256, 6),
         (30, 72, 4), (9, 700, 5), (6, 2500, 7), (11, 96, 7), (1500, 4096, 1), (600, 1536, 2), (5, 16384, 1), (2, 16385, 3), (3001, 1024, 6), (700, 600, 4), (1111, 1024, 8),
         (777, 24, 8), (1000, 32, 6), (333, 12, 5), (5000, 16, 1), (70001, 9, 2), (70, 4096, 5), (500, 1100, 8), (40, 8192, 4), (300, 8192, 8), (600, 5000, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,C,nb", CASES)
def test_forward_and_backward_match_fp64(dev, M, C, nb, dtype):
    from unet_amd import ops
    relu = (M + C + nb) % 2 == 0
    zs, gammas, betas, g = make(dev, M, C, nb, dtype, seed=M + C)
    y = ops.Act(torch.empty((1, 1, M, C), dtype=dtype, device=dev), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y, relu=relu)
    want, bound = ref.forward([rows(z) for z in zs], cpu(gammas), cpu(betas), relu, 1e-5)
    check(rows(y), want, bound, dtype, "y")
    dy = ops.Act((torch.randn((1, 1, M, C), generator=g) * 0.1).to(dtype).to(dev), 0, C)
    out = ops.layer_norm_bwd(dy, zs, gammas, y=y if relu else None)
    want, (db, e_db) = ref.backward(rows(dy), [rows(z) for z in zs], cpu(gammas), rows(y) if relu else None, 1e-5)
    for b, ((dz, dg, dbeta), (wz, ez, wg, eg)) in enumerate(zip(out, want)):
        check(rows(dz), wz, ez, dtype, f"dz{b}")
        check(dg.cpu(), wg, eg, torch.float32, f"dgamma{b}")
        check(dbeta.cpu(), db, e_db, torch.float32, f"dbeta{b}")
    # the same bits every time
    again = ops.layer_norm_bwd(dy, zs, gammas, y=y if relu else None)
    for o, a in zip(out, again):
        assert torch.equal(o[0].buf, a[0].buf) and torch.equal(o[1], a[1]) and torch.equal(o[2], a[2])
    # every branch has gradients of its own: clipping scales them in place
    ptrs = [t.data_ptr() for o in out for t in (o[0].buf, o[1], o[2])]
    assert len(set(ptrs)) == len(ptrs)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,C,nb", [(4200, 1100, 8), (4096, 2100, 8), (4100, 5000, 5), (5000, 8192, 3), (4097, 1025, 2), (9000, 1536, 1)])
def test_many_wide_rows(dev, M, C, nb, dtype):
    """Wide rows, so many that workgroups hold several branches' weights in LDS (up to 150 KB); a sample of the rows is checked."""
    from unet_amd import ops
    g = torch.Generator(device=dev).manual_seed(C)
    zs = [ops.Act(torch.randn((1, 1, M, C), generator=g, device=dev).to(dtype), 0, C) for _ in range(nb)]
    gammas, betas = ([torch.randn(C, generator=g, device=dev) + s for _ in range(nb)] for s in (1.0, 0.0))
    y = ops.Act(torch.empty((1, 1, M, C), dtype=dtype, device=dev), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y, relu=True)
    some = torch.cat([torch.arange(0, M, 97), torch.arange(M - 9, M)]).to(dev)
    part = [z.buf[0, 0, some].cpu() for z in zs]
    want, bound = ref.forward(part, cpu(gammas), cpu(betas), True, 1e-5)
    check(y.buf[0, 0, some].cpu(), want, bound, dtype, "y")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C,pad,off", [(64, 64, 64), (48, 5, 3), (33, 7, 1), (1024, 8, 8), (1024, 3, 2)])
def test_channel_slices_and_missing_weights(dev, C, pad, off, dtype):
    """Inputs, output and gradients as slices of wider buffers at any offset; the rest of the buffers stays as it was."""
    from unet_amd import ops
    M, nb = 37, 2
    zs, gammas, betas, g = make(dev, M, C, nb, dtype, seed=C, pad=pad, off=off)
    gammas[1], betas[0] = None, None
    ybuf = torch.full((1, 1, M, C + pad), 7.0, dtype=dtype, device=dev)
    y = ops.Act(ybuf, off, C)
    ops.layer_norm_fwd(zs, gammas, betas, y, relu=True, eps=1e-3)
    want, bound = ref.forward([rows(z) for z in zs], cpu(gammas), cpu(betas), True, 1e-3)
    check(rows(y), want, bound, dtype, "y")
    rest = torch.ones(C + pad, dtype=torch.bool)
    rest[off:off + C] = False
    assert bool((ybuf[..., rest.to(dev)] == 7.0).all())
    dy = ops.Act(torch.randn((1, 1, M, C + pad), generator=g).to(dtype).to(dev), off, C)
    out = ops.layer_norm_bwd(dy, zs, gammas, y=y, eps=1e-3)
    want, (db, e_db) = ref.backward(rows(dy), [rows(z) for z in zs], cpu(gammas), rows(y), 1e-3)
    for (dz, dg, dbeta), (wz, ez, wg, eg) in zip(out, want):
        check(rows(dz), wz, ez, dtype, "dz")
        check(dg.cpu(), wg, eg, torch.float32, "dgamma")
        check(dbeta.cpu(), db, e_db, torch.float32, "dbeta")
    y2 = ops.Act(torch.empty((1, 1, M, C), dtype=dtype, device=dev), 0, C)
    ops.layer_norm_fwd(zs[:1], None, None, y2)
    want, bound = ref.forward([rows(zs[0])], [None], [None], False, 1e-5)
    check(rows(y2), want, bound, dtype, "plain")
    one = ops.layer_norm_bwd(dy, zs[:1], None)
    want, _ = ref.backward(rows(dy), [rows(zs[0])], [None], None, 1e-5)
    check(rows(one[0][0]), want[0][0], want[0][1], dtype, "plain dz")


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 100, 3000])
def test_rows_that_are_not_finite_or_constant(dev, C):
    """A NaN or infinite row is NaN (through the ReLU too) and leaves its neighbours alone; a constant row is beta."""
    from unet_amd import ops
    M = 20
    zs, gammas, betas, g = make(dev, M, C, 1, torch.float32, seed=5)
    zs[0].buf[0, 0, 3, C // 2] = float("nan")
    zs[0].buf[0, 0, 7, 0] = float("inf")
    zs[0].buf[0, 0, 11] = 3.25
    y = ops.Act(torch.empty((1, 1, M, C), device=dev), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y, relu=True)
    out = rows(y)
    assert out[3].isnan().all() and out[7].isnan().all()
    assert torch.equal(out[11], betas[0].cpu().clamp_min(0))
    keep = [r for r in range(M) if r not in (3, 7, 11)]
    want, bound = ref.forward([rows(zs[0])[keep]], cpu(gammas), cpu(betas), True, 1e-5)
    check(out[keep], want, bound, torch.float32, "y")
    dy = ops.Act(torch.randn((1, 1, M, C), generator=g).to(dev), 0, C)
    dz, dg, db = ops.layer_norm_bwd(dy, zs, gammas, y=y)[0]
    got = rows(dz)
    assert got[3].isnan().all() and got[7].isnan().all() and got[keep].isfinite().all()
    want, _ = ref.backward(rows(dy)[keep], [rows(zs[0])[keep]], cpu(gammas), out[keep], 1e-5)
    check(got[keep], want[0][0], want[0][1], torch.float32, "dz")
    assert dg.isnan().all()
    # torch's rule for a NaN output of the ReLU: its gradient passes
    u = torch.where(out <= 0, 0.0, rows(dy).double())
    assert (db.cpu().double() - u.sum(0)).abs().max() < 1e-4


@pytest.mark.gpu
def test_far_from_zero(dev):
    """Rows whose mean is 4000 standard deviations: the bound is that of fp32 inputs, not of a difference of squares."""
    from unet_amd import ops
    M, C = 64, 320
    z = ops.Act((torch.randn((1, 1, M, C), generator=torch.Generator().manual_seed(1)) + 4000.0).to(dev), 0, C)
    y = ops.Act(torch.empty((1, 1, M, C), device=dev), 0, C)
    ops.layer_norm_fwd([z], None, None, y)
    want, bound = ref.forward([rows(z)], [None], [None], False, 1e-5)
    check(rows(y), want, bound, torch.float32, "y")
    assert float((rows(y).double() - want).abs().max()) < 5e-3


CONSTANT = [2, 3, 100, 333, 1000, 1024, 3000, 5120, 8192, 8200, 20000]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nb", [1, 3])
@pytest.mark.parametrize("C", CONSTANT)
def test_constant_rows_of_full_mantissas(dev, C, nb, dtype):
    """Rows of one value, whose sum is not exact in fp32: y is beta and dgamma 0 to the bit, and dz = (w - mean w)/sqrt(eps)."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(C)
    some = torch.tensor([865.6096, 974.7146, 0.1, -12345.678, 3141592.7, 1e-3, -3.3e-5, 7.0])
    levels = torch.cat([some, torch.rand(56, generator=g) * 1000 + 1]).view(1, 1, -1, 1)
    M = levels.numel()
    zs = [ops.Act((levels + b).to(dtype).expand(1, 1, M, C).contiguous().to(dev), 0, C) for b in range(nb)]
    gammas, betas = ([(torch.randn(C, generator=g) + s).to(dev) for _ in range(nb)] for s in (1.0, 0.0))
    y = ops.Act(torch.empty((1, 1, M, C), dtype=dtype, device=dev), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y)
    beta = betas[0].cpu()
    for b in betas[1:]:
        beta = beta + b.cpu()
    assert torch.equal(rows(y), beta.to(dtype).expand(M, C))
    dy = ops.Act(torch.randn((1, 1, M, C), generator=g).to(dtype).to(dev), 0, C)
    out = ops.layer_norm_bwd(dy, zs, gammas)
    N = C / 64 + 16                                                  # roundings of a sum over the channels (as in the oracle)
    for (dz, dg, _), gamma in zip(out, gammas):
        assert not dg.any()
        w = rows(dy).double() * gamma.cpu().double()
        m1, rstd = w.mean(-1, keepdim=True), 1e-5 ** -0.5
        want = rstd * (w - m1)
        bound = rstd * ref.U * (5 * w.abs() + 4 * m1.abs() + (N + 2) * w.abs().mean(-1, keepdim=True)) + 6 * ref.U * want.abs()
        check(rows(dz), want, bound, dtype, "dz")


@pytest.mark.gpu
@pytest.mark.parametrize("C", CONSTANT)
def test_rows_of_two_neighbouring_numbers(dev, C):
    """fp32 rows whose channels take two neighbouring numbers in turn: their mean lies between the two, where fp32 has no number."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(C)
    low = torch.rand(40, generator=g) * 90000 + 40000                # the step there: 2^-8 or 2^-7, half of it near sqrt(eps)
    high = torch.nextafter(low, torch.full_like(low, torch.inf))
    z = torch.where(torch.rand((40, C), generator=g) < 0.5, low[:, None], high[:, None]).contiguous()
    zs, y = [ops.Act(z.view(1, 1, 40, C).to(dev), 0, C)], ops.Act(torch.empty((1, 1, 40, C), device=dev), 0, C)
    ops.layer_norm_fwd(zs, None, None, y)
    d = z.double() - z.double().mean(-1, keepdim=True)
    var = (d * d).mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + 1e-5)
    x = d * rstd
    # the differences from the first mean are exact, as is their sum: what is left are the roundings of its quotient, of the sum
    # of squares (C/64 + 16, half of them in the root) and of a few products
    step = (high - low).double()[:, None] * rstd
    bound = ref.U * (8 * step + (C / 128 + 20) * x.abs())
    check(rows(y), x, bound, torch.float32, "y")
    dy = ops.Act(torch.randn((1, 1, 40, C), generator=g).to(dev), 0, C)
    (dz, dg, _), = ops.layer_norm_bwd(dy, zs, None)
    u, N = rows(dy).double(), C / 64 + 16
    m1, m2 = u.mean(-1, keepdim=True), (u * x).mean(-1, keepdim=True)
    want = rstd * (u - m1 - x * m2)
    e2 = (N + 3) * ref.U * (u * x).abs().mean(-1, keepdim=True) + (u.abs() * bound).mean(-1, keepdim=True)
    e = ref.U * 5 * (u.abs() + m1.abs() + (x * m2).abs()) + (N + 2) * ref.U * u.abs().mean(-1, keepdim=True) + x.abs() * e2 + bound * m2.abs()
    check(rows(dz), want, rstd * e + (C / 128 + 20) * ref.U * want.abs(), torch.float32, "dz")
    check(dg.cpu(), (u * x).sum(0), (u.abs() * bound).sum(0) + 41 * ref.U * (u * x).abs().sum(0), torch.float32, "dgamma")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C,step", [(1500, 512), (2049, 2048), (5120, 64), (8191, 1000), (8192, 8100)])
def test_rows_in_steps(dev, C, step, dtype):
    """Parts of a row at levels far apart, with little noise: several waves share such a row, and their means differ by up to
    thousands of times what each of them varies by."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(C)
    M, part = 30, torch.arange(C) // step
    level = torch.randint(-4, 5, (M, int(part[-1]) + 1), generator=g) * 64.0
    z = (level[:, part] + 0.05 * torch.randn((M, C), generator=g)).to(dtype).view(1, 1, M, C).to(dev)
    zs, gammas, betas = [ops.Act(z, 0, C)], [(torch.randn(C, generator=g) + 1).to(dev)], [torch.randn(C, generator=g).to(dev)]
    y = ops.Act(torch.empty_like(z), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y)
    want, bound = ref.forward([rows(zs[0])], cpu(gammas), cpu(betas), False, 1e-5)
    check(rows(y), want, bound, dtype, "y")
    dy = ops.Act(torch.randn((1, 1, M, C), generator=g).to(dtype).to(dev), 0, C)
    (dz, dg, dbeta), = ops.layer_norm_bwd(dy, zs, gammas)
    ((wz, ez, wg, eg),), (db, e_db) = ref.backward(rows(dy), [rows(zs[0])], cpu(gammas), None, 1e-5)
    check(rows(dz), wz, ez, dtype, "dz")
    check(dg.cpu(), wg, eg, torch.float32, "dgamma")
    check(dbeta.cpu(), db, e_db, torch.float32, "dbeta")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("C", [3, 64, 333, 2048])
@pytest.mark.parametrize("scale,eps", [(1e-12, 0.0), (1e-9, 1e-30), (1e-14, 1e-28), (1e-16, 1e-40), (1e12, 1e-5)])
def test_small_and_large_variances(dev, C, scale, eps, dtype):
    """Variances from under 2^-64 to 2^80, eps above, beside and below them."""
    from unet_amd import ops
    g = torch.Generator().manual_seed(C)
    M = 40
    z = (torch.randn((1, 1, M, C), generator=g) * scale).to(dtype).to(dev)
    zs, gammas, betas = [ops.Act(z, 0, C)], [(torch.randn(C, generator=g) + 1).to(dev)], [torch.randn(C, generator=g).to(dev)]
    y = ops.Act(torch.empty_like(z), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y, eps=eps)
    want, bound = ref.forward([rows(zs[0])], cpu(gammas), cpu(betas), False, eps)
    check(rows(y), want, bound, dtype, "y")
    dy = ops.Act(torch.randn((1, 1, M, C), generator=g).to(dtype).to(dev), 0, C)
    (dz, dg, dbeta), = ops.layer_norm_bwd(dy, zs, gammas, eps=eps)
    ((wz, ez, wg, eg),), (db, e_db) = ref.backward(rows(dy), [rows(zs[0])], cpu(gammas), None, eps)
    check(rows(dz), wz, ez, dtype, "dz")
    check(dg.cpu(), wg, eg, torch.float32, "dgamma")
    check(dbeta.cpu(), db, e_db, torch.float32, "dbeta")


@pytest.mark.gpu
def test_gradients_against_differences(dev):
    from unet_amd import ops
    M, C, nb = 12, 40, 3
    zs, gammas, betas, g = make(dev, M, C, nb, torch.float32, seed=9)
    dy = torch.randn((M, C), generator=g)
    y = ops.Act(torch.empty((1, 1, M, C), device=dev), 0, C)
    ops.layer_norm_fwd(zs, gammas, betas, y, relu=True)
    out = ops.layer_norm_bwd(ops.Act(dy.view(1, 1, M, C).to(dev), 0, C), zs, gammas, y=y)
    Z, G, B = [rows(z).double() for z in zs], [t.cpu().double() for t in gammas], [t.cpu().double() for t in betas]

    def f(Z, G, B):
        return float((ref.forward(Z, G, B, True, 1e-5)[0] * dy.double()).sum())
    h = 1e-6
    for b in range(nb):
        for ts, grad in ((Z, out[b][0].buf.view(M, C)), (G, out[b][1]), (B, out[b][2])):
            for _ in range(3):
                d = torch.randn(ts[b].shape, generator=g, dtype=torch.float64)
                old = ts[b]
                ts[b] = old + h * d; hi = f(Z, G, B)
                ts[b] = old - h * d; lo = f(Z, G, B)
                ts[b] = old
                want = float((grad.cpu().double() * d).sum())
                # differences: h^2 of truncation and 1e-16 * |f| / h of rounding, both under 1e-7; the rest is the fp32 gradient
                assert abs((hi - lo) / (2 * h) - want) < 1e-5 * float((grad.cpu().double() * d).abs().sum()) + 1e-6


@pytest.mark.gpu
def test_no_rows_and_offsets_beyond_32_bits(dev):
    from unet_amd import ops
    empty = ops.Act(torch.empty((0, 4, 4, 24), device=dev), 0, 24)
    y = ops.Act(torch.empty((0, 4, 4, 24), device=dev), 0, 24)
    ops.layer_norm_fwd([empty], None, None, y)
    dz, dg, db = ops.layer_norm_bwd(y, [empty], None)[0]
    assert dz.buf.numel() == 0 and not dg.any() and not db.any()
    # 2^25 + 5 rows of 64: element offsets pass 2^31, byte offsets 2^32
    M, C = (1 << 25) + 5, 64
    z = torch.empty((1, 1, M, C), dtype=torch.bfloat16, device=dev)
    z.normal_(generator=torch.Generator(device=dev).manual_seed(3))
    za, ya = ops.Act(z, 0, C), ops.Act(torch.empty_like(z), 0, C)
    gamma, beta = torch.linspace(0.5, 1.5, C, device=dev), torch.linspace(-1, 1, C, device=dev)
    ops.layer_norm_fwd([za], [gamma], [beta], ya, relu=True)
    dz, dg, db = ops.layer_norm_bwd(za, [za], [gamma], y=ya)[0]
    for sl in (slice(0, 100), slice((1 << 24), (1 << 24) + 100), slice(M - 100, M)):
        zc = z[0, 0, sl].cpu()
        want, bound = ref.forward([zc], [gamma.cpu()], [beta.cpu()], True, 1e-5)
        check(ya.buf[0, 0, sl].cpu(), want, bound, torch.bfloat16, "y")
        want, _ = ref.backward(zc, [zc], [gamma.cpu()], ya.buf[0, 0, sl].cpu(), 1e-5)
        check(dz.buf[0, 0, sl].cpu(), want[0][0], want[0][1], torch.bfloat16, "dz")
    # dbeta in fp64 by parts
    s = torch.zeros(C, dtype=torch.float64, device=dev)
    a = torch.zeros(C, dtype=torch.float64, device=dev)
    for r in range(0, M, 1 << 22):
        u = torch.where(ya.buf[0, 0, r:r + (1 << 22)] <= 0, 0.0, z[0, 0, r:r + (1 << 22)].float())
        s += u.sum(0, dtype=torch.float64)
        a += u.abs().sum(0, dtype=torch.float64)
    # sums of M / (workgroups * rows per pass) terms a lane: at most a few thousand roundings of 2^-24
    assert bool(((db.double() - s).abs() <= 4096 * 2.0 ** -24 * a).all())


def test_workspace_of_many_narrow_rows_has_a_bound():
    from unet_amd._lib import lib
    L = lib()
    for dtype, nb, C in ((0, 8, 3), (1, 8, 7), (1, 1, 1)):
        assert 0 < L.unet_layer_norm_bwd_ws(dtype, nb, (1 << 31) - 1, C) < 1 << 28
    assert L.unet_layer_norm_bwd_ws(0, 2, 100000, 3) < L.unet_layer_norm_bwd_ws(0, 2, 1 << 21, 3) < L.unet_layer_norm_bwd_ws(0, 2, (1 << 21) + 1, 3)


def signs(g, dev, M, C, dtype, pad=0):
    """Rows of C/2 ones and C/2 minus ones in random order (C even), behind `pad` channels that are not theirs: mean 0 and variance
    1, xhat with eps = 0 is the row itself."""
    z = torch.empty((1, 1, M, C + pad), dtype=dtype, device=dev)
    order = torch.rand((M, C), generator=g, device=dev).argsort(-1)
    z[0, 0, :, :pad] = 9
    z[0, 0, :, pad:] = torch.where(order < C // 2, 1.0, -1.0).to(dtype)
    return z


@pytest.mark.gpu
@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype,C,pad", [(torch.bfloat16, 6, 3), (torch.float32, 2, 0)])
def test_narrow_rows_in_chunks(dev, dtype, C, pad, relu):
    """More rows than the row kernels take at a time: gradients of rows on both sides of each border, and column sums of whole
    numbers, which fp32 holds exactly."""
    from unet_amd import ops
    nb, M, chunk = 2, 2 * (1 << 20) + 77, 1 << 20
    g = torch.Generator(device=dev).manual_seed(C)
    zs = [ops.Act(signs(g, dev, M, C, dtype, pad), pad, C) for _ in range(nb)]
    dy = ops.Act(torch.randint(-3, 4, (1, 1, M, C + pad), generator=g, device=dev).to(dtype), pad, C)
    y = ops.Act(torch.randint(-1, 3, (1, 1, M, C + pad), generator=g, device=dev).to(dtype), pad, C) if relu else None
    gammas = [torch.rand(C, generator=g, device=dev) + 0.5 for _ in range(nb)]
    out = ops.layer_norm_bwd(dy, zs, gammas, y=y, eps=0.0)
    some = torch.cat([torch.arange(r, r + 40) for r in (0, chunk - 20, 2 * chunk - 20, M - 40)]).to(dev)
    part = lambda a: None if a is None else a.buf[0, 0, some, a.off:].cpu()  # noqa: E731
    want, _ = ref.backward(part(dy), [part(z) for z in zs], cpu(gammas), part(y), 0.0)
    u = dy.buf[0, 0, :, pad:].double()
    u = torch.where(y.buf[0, 0, :, pad:] <= 0, 0.0, u) if relu else u
    for b, (dz, dg, db) in enumerate(out):
        check(dz.buf[0, 0, some].cpu(), want[b][0], want[b][1], dtype, "dz")
        assert torch.equal(db.double(), u.sum(0))
        assert torch.equal(dg.double(), (u * zs[b].buf[0, 0, :, pad:].double()).sum(0))


# One shape per layout of the backward: 2 to 64 lanes a row (bf16 | fp32: 8 | 4 channels a lane, 16 where that is over 64 lanes), one to
# three groups of branches, rows of several waves, row kernels.  Odd row counts, several rows for every lane of every workgroup.
COLUMNS = [(torch.bfloat16, 140003, 16, 1), (torch.bfloat16, 100003, 30, 3), (torch.bfloat16, 120011, 64, 6), (torch.bfloat16, 90007, 100, 2),
           (torch.bfloat16, 30011, 256, 8), (torch.bfloat16, 20011, 512, 6), (torch.bfloat16, 6007, 600, 1), (torch.bfloat16, 6007, 700, 5),
           (torch.bfloat16, 5003, 1024, 6), (torch.bfloat16, 5003, 1024, 8), (torch.bfloat16, 3001, 1100, 3), (torch.bfloat16, 1501, 4096, 5),
           (torch.bfloat16, 701, 8192, 8), (torch.bfloat16, 301, 8200, 2), (torch.bfloat16, 30001, 6, 3),
           (torch.float32, 140003, 8, 1), (torch.float32, 100003, 14, 2), (torch.float32, 120011, 32, 6), (torch.float32, 60013, 64, 3),
           (torch.float32, 30011, 130, 7), (torch.float32, 20011, 256, 4), (torch.float32, 6007, 300, 2), (torch.float32, 6007, 1024, 6),
           (torch.float32, 5003, 1000, 7), (torch.float32, 3001, 1030, 3), (torch.float32, 701, 8192, 8), (torch.float32, 30001, 2, 3)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,M,C,nb", COLUMNS)
def test_every_row_counts_once_in_the_column_sums(dev, dtype, M, C, nb):
    """Gradients of whole numbers: dbeta's sums are exact, so a row that is lost, doubled or shifted shows.  z of +-1 with as many of
    each makes xhat those numbers up to roundings: the same for dgamma, to which every row adds 1 at least."""
    from unet_amd import ops
    g = torch.Generator(device=dev).manual_seed(M + C)
    zs = [ops.Act(signs(g, dev, M, C, dtype), 0, C) for _ in range(nb)]
    dyb = torch.randint(1, 4, (1, 1, M, C), generator=g, device=dev) * (torch.randint(0, 2, (1, 1, M, C), generator=g, device=dev) * 2 - 1)
    out = ops.layer_norm_bwd(ops.Act(dyb.to(dtype), 0, C), zs, None, eps=0.0)
    want = dyb[0, 0].sum(0).double()
    assert float(want.abs().max()) < 2 ** 24
    # Roundings behind an entry of dgamma: 10 in each xhat, one for each row of a lane (rows over how many rows are worked on at a
    # time, at least) and 14 where lanes and waves are joined, all of sums that 3 M bounds
    per = 8 if dtype == torch.bfloat16 else 4
    lanes = -(-C // per)
    at_once = 1024 if C < per or C > 8192 else 512 * 256 // (1 << (lanes - 1).bit_length()) if lanes <= 64 else 256 // nb
    bound = (M / at_once + 1 + 10 + 14) * ref.U * 3 * M
    assert bound < 0.7
    for (_, dg, db), z in zip(out, zs):
        assert torch.equal(db.double(), want)
        assert float((dg.double() - (dyb[0, 0] * z.buf[0, 0].long()).sum(0)).abs().max()) <= bound


@pytest.mark.gpu
@pytest.mark.parametrize("C", [64, 3])
def test_every_row_counts_once_beyond_32_bits(dev, C):
    """2^25 + 5 rows: whole numbers again, whose sums of a workgroup's rows fp32 holds; the sums of all in fp64, rounded once."""
    from unet_amd import ops
    M, g = (1 << 25) + 5, torch.Generator(device=dev).manual_seed(C)
    z = torch.empty((1, 1, M, C), dtype=torch.bfloat16, device=dev).normal_(generator=g)
    dy = torch.empty_like(z).random_(0, 8, generator=g)
    want = sum(dy[0, 0, r:r + (1 << 22)].sum(0, dtype=torch.float64) for r in range(0, M, 1 << 22))
    (_, _, db), = ops.layer_norm_bwd(ops.Act(dy, 0, C), [ops.Act(z, 0, C)], None)
    assert torch.equal(db, want.float())


@pytest.mark.gpu
def test_other_stream_and_graph(dev):
    from unet_amd import ops
    M, C, nb = 300, 96, 3
    zs, gammas, betas, g = make(dev, M, C, nb, torch.bfloat16, seed=2)
    dy = ops.Act(torch.randn((1, 1, M, C), generator=g).bfloat16().to(dev), 0, C)
    y = ops.Act(torch.empty((1, 1, M, C), dtype=torch.bfloat16, device=dev), 0, C)

    def both():
        ops.layer_norm_fwd(zs, gammas, betas, y, relu=True)
        return [t for o in ops.layer_norm_bwd(dy, zs, gammas, y=y) for t in (o[0].buf, o[1], o[2])]
    want = [t.clone() for t in [y.buf] + both()][1:]
    ywant = y.buf.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        y.buf.zero_()
        other = both()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, want)) and torch.equal(y.buf, ywant)
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    with torch.cuda.graph(graph2):                       # a second graph over the same tensors: workspaces of its own
        out2 = both()
    for i in range(4):
        zs[0].buf.copy_((torch.randn((1, 1, M, C), generator=g) + i).bfloat16())
        eager = [t.clone() for t in both()]
        torch.cuda.synchronize()
        for t in out + out2:
            t.zero_()
        graph.replay()
        graph2.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)) and all(torch.equal(a, b) for a, b in zip(out2, eager))


@pytest.mark.gpu
def test_two_streams_at_once(dev):
    """Calls that overlap on two streams have workspaces of their own."""
    from unet_amd import ops
    sets = [make(dev, 20000, 64, 3, torch.bfloat16, seed=s) for s in (1, 2)]
    dys = [ops.Act(torch.randn((1, 1, 20000, 64), generator=s[3]).bfloat16().to(dev), 0, 64) for s in sets]

    def run(k):
        zs, gammas, betas, _ = sets[k]
        y = ops.Act(torch.empty_like(zs[0].buf), 0, 64)
        ops.layer_norm_fwd(zs, gammas, betas, y, relu=True)
        return [y.buf] + [t for o in ops.layer_norm_bwd(dys[k], zs, gammas, y=y) for t in (o[0].buf, o[1], o[2])]
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for i in range(6):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((k, run(k)))
    torch.cuda.synchronize()
    for k, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want[k]))


# ----------------------------------------------------------------------------- refusals (no GPU needed)

def test_the_tensors_device_becomes_the_current_one(monkeypatch):
    from unet_amd import ops
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    assert isinstance(ops._on_device(0), torch.cuda.device) and not isinstance(ops._on_device(1), torch.cuda.device)
    assert not isinstance(ops._on_device(-1), torch.cuda.device)
    from unet_amd._lib import UNetHipError

    class T:
        def __init__(self, d): self.d = d
        def get_device(self): return self.d
    assert ops._one_device("f", T(2), None, T(2)) == 2 and ops._one_device("f", None) == -1
    with pytest.raises(UNetHipError, match="different devices"):
        ops._one_device("f", T(0), T(1))
    with pytest.raises(UNetHipError, match="CPU tensor"):
        ops._one_device("f", T(0), T(-1))


def test_refusals_of_the_wrappers():
    from unet_amd import ops
    from unet_amd._lib import UNetHipError

    def act(M=4, C=8, dtype=torch.float32, ld=None, off=0):
        return ops.Act(torch.zeros((1, 1, M, ld or C), dtype=dtype), off, C)
    with pytest.raises(UNetHipError, match="device tensors"):
        ops.layer_norm_fwd([act()], None, None, act())
    with pytest.raises(UNetHipError, match="device tensors"):
        ops.layer_norm_bwd(act(), [act()], None)


@pytest.mark.gpu
def test_refusals_on_the_device(dev):
    from unet_amd import ops
    from unet_amd._lib import UNetHipError

    def act(M=4, C=8, dtype=torch.float32, ld=None, off=0):
        return ops.Act(torch.zeros((1, 1, M, ld or C), dtype=dtype, device=dev), off, C)
    w = torch.ones(8, device=dev)
    for bad, msg in [
        (lambda: ops.layer_norm_fwd([], None, None, act()), "branches"),
        (lambda: ops.layer_norm_fwd([act()] * 9, None, None, act()), "branches"),
        (lambda: ops.layer_norm_fwd([act(), act(M=5)], None, None, act()), "one shape"),
        (lambda: ops.layer_norm_fwd([act(), act(dtype=torch.bfloat16)], None, None, act()), "one shape"),
        (lambda: ops.layer_norm_fwd([act(dtype=torch.float16)], None, None, act(dtype=torch.float16)), "dtype"),
        (lambda: ops.layer_norm_fwd([act()], [w[:7]], None, act()), "length C"),
        (lambda: ops.layer_norm_fwd([act()], [w.double()], None, act()), "fp32"),
        (lambda: ops.layer_norm_fwd([act()], [w, w], None, act()), "one weight per branch"),
        (lambda: ops.layer_norm_fwd([act()], [w.cpu()], None, act()), "CPU tensor"),
        (lambda: ops.layer_norm_fwd([act()], None, None, act(C=9)), "shape or dtype"),
        (lambda: ops.layer_norm_fwd([act()], None, None, act(dtype=torch.bfloat16)), "shape or dtype"),
        (lambda: ops.layer_norm_fwd([act()], None, None, act(off=1)), "outside the buffer"),
        (lambda: ops.layer_norm_fwd([act()], None, None, act(), eps=-1.0), "eps"),
        (lambda: ops.layer_norm_bwd(act(M=3), [act()], None), "shape or dtype"),
        (lambda: ops.layer_norm_bwd(act(), [act()], None, y=act(C=9)), "shape or dtype"),
    ]:
        with pytest.raises(UNetHipError, match=msg):
            bad()
    x = act(ld=16)
    with pytest.raises(UNetHipError, match="overlaps"):
        ops.layer_norm_fwd([x], None, None, ops.Act(x.buf, 4, 8))
    ops.layer_norm_fwd([x], None, None, ops.Act(x.buf, 8, 8))           # the other half of the same buffer is fine


def test_refusals_of_the_c_entry():
    import ctypes
    from unet_amd._lib import lib
    L = lib()
    PA, IA = ctypes.c_void_p * 1, ctypes.c_int * 1
    z, ld, off = PA(None), IA(8), IA(0)

    def fwd(dtype=0, nb=1, ld=ld, off=off, M=4, C=8, ldy=8, yoff=0, eps=1e-5):
        return L.unet_layer_norm_fwd(dtype, 0, nb, z, ld, off, None, None, None, ldy, yoff, M, C, eps, None), L.unet_last_error().decode()
    for kw, msg in [(dict(dtype=2), "bad dtype"), (dict(nb=0), "branches"), (dict(nb=9), "branches"), (dict(C=0), "bad shape"),
                    (dict(M=-1), "bad shape"), (dict(), "branch 0 is null"), (dict(M=0, off=IA(1)), "outside the buffer"),
                    (dict(M=0, ldy=7), "outside the buffer"), (dict(eps=-1.0), "eps")]:
        rc, text = fwd(**kw)
        assert rc == -1 and msg in text, (kw, text)
    assert fwd(M=0)[0] == 0
    assert L.unet_layer_norm_bwd_ws(0, 9, 4, 8) == -1 and L.unet_layer_norm_bwd_ws(0, 1, -1, 8) == -1
    need = L.unet_layer_norm_bwd_ws(0, 1, 100, 8)
    assert need > 0
    rc = L.unet_layer_norm_bwd(0, 1, 16, 8, 0, None, 0, 0, PA(16), ld, off, None, PA(16), None, None, 16, need - 1, 100, 8, 1e-5, None)
    assert rc == -1 and b"workspace" in L.unet_last_error()


def test_oracle_matches_autograd():
    g = torch.Generator().manual_seed(0)
    M, C, nb = 9, 21, 3
    zs = [torch.randn((M, C), generator=g, dtype=torch.float64).requires_grad_() for _ in range(nb)]
    G = [torch.randn(C, generator=g, dtype=torch.float64).requires_grad_() for _ in range(nb)]
    B = [torch.randn(C, generator=g, dtype=torch.float64).requires_grad_() for _ in range(nb)]
    y = torch.relu(sum(torch.nn.functional.layer_norm(z, (C,), a, b, 1e-5) for z, a, b in zip(zs, G, B)))
    dy = torch.randn((M, C), generator=g, dtype=torch.float64)
    y.backward(dy)
    got, _ = ref.forward([z.detach() for z in zs], [t.detach() for t in G], [t.detach() for t in B], True, 1e-5)
    torch.testing.assert_close(got, y.detach(), rtol=1e-12, atol=1e-12)
    out, (db, _) = ref.backward(dy, [z.detach() for z in zs], [t.detach() for t in G], got, 1e-5)
    for (dz, _, dg, _), z, a, b in zip(out, zs, G, B):
        torch.testing.assert_close(dz, z.grad, rtol=1e-10, atol=1e-12)
        torch.testing.assert_close(dg, a.grad, rtol=1e-10, atol=1e-12)
        torch.testing.assert_close(db, b.grad, rtol=1e-10, atol=1e-12)
