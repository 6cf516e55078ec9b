"""AdamW with 8-bit moments: the format and the step against oracle/adamw8_ref.py (codes bit for bit, parameters within
their fp32 bound), the optimizer around it, its checkpoints and its refusals."""
import copy

import numpy as np
import pytest
import torch

from oracle import adamw8_ref as ref

HYPER = dict(lr=3e-3, b1=0.9, b2=0.999, eps=1e-8, wd=1e-2)


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs the MI355X")
    return torch.device("cuda:0")


# ----------------------------------------------------------------------------- the format (no GPU needed)

def values(n, seed, spread=3.0):
    r = np.random.default_rng(seed)
    return (r.standard_normal(n) * np.exp(spread * r.standard_normal(n))).astype(np.float32)


def test_every_code_stands_for_itself():
    for signed in (True, False):
        c = np.arange(256, dtype=np.uint8)
        e = np.full(4, 140, np.uint8)
        v = ref.decode(c, e, signed)
        assert len(np.unique(v)) == (255 if signed else 256)        # +0 and -0
        # the largest code sets the block's exponent: it and every other code come back from their values
        top = 127 if signed else 255
        for lo in range(0, 256, 63):
            part = np.concatenate([c[lo:lo + 63], [top]]).astype(np.uint8)
            x = ref.decode(part, e[:1], signed)
            assert np.array_equal(x, x.astype(np.float32))
            back, eb = ref.encode(x.astype(np.float32), signed, np.zeros(len(part), np.int64))
            same = (back == part) | (x == 0)                        # (-0 becomes +0)
            assert eb[0] == 140 and same.all()


@pytest.mark.parametrize("signed", [True, False])
def test_rounding_is_unbiased_and_within_a_step(signed):
    x = values(64 * 50, 1, spread=1.5)
    x = x if signed else np.abs(x)
    total = np.zeros(len(x))
    steps = 400
    for t in range(1, steps + 1):
        c, e = ref.encode(x, signed, ref.dither(len(x), 3, t)[0 if signed else 1])
        v = ref.decode(c, e, signed)
        unit = np.repeat(2.0 ** (e.astype(np.float64) - 127 - ref.TOP[signed] - 2), 64)
        assert np.all(np.abs(v - x) < np.maximum(np.abs(x) / 8, unit))
        total += v
    # each rounding is one of two neighbours a step apart (1/8 of the value at most, or the unit): its deviation is at most half a
    # step, and the mean of `steps` of them is within 5 deviations for all 3200 elements
    step = np.maximum(np.abs(x) / 8, unit)
    assert np.all(np.abs(total / steps - x) <= 5 * 0.5 * step / np.sqrt(steps))


def test_blocks_with_extremes():
    x = np.zeros(64 * 6 + 5, np.float32)
    x[64], x[65] = 1e-30, 1e-38                    # tiny values: the scale ends at 2^-95
    x[128:192] = 2.0 ** np.arange(-40, 24)         # 64 binades
    x[200] = np.nan
    x[300] = np.inf
    x[64 * 5 + 3] = 3.3e38
    d = np.full(len(x), ref.NEAREST)
    for signed in (True, False):
        c, e = ref.encode(x, signed, d)
        v = ref.decode(c, e, signed)
        assert not v[:64].any() and e[0] == 32
        assert abs(v[64] - 1e-30) <= 1e-30 / 16 and e[1] == 32 and (v[65] == 0 if signed else 0 < v[65] < 1e-37)
        got = v[128:192]
        big = x[128:192] >= 2.0 ** (23 - (14 if signed else 30))
        assert np.array_equal(got[big], x[128:192][big].astype(np.float64))
        if not signed:
            assert (got > 0).all()                 # a second moment that is not zero stays positive
        assert np.isnan(v[192:256]).all() and np.isnan(v[256:320]).all() and e[3] == e[4] == 255
        assert np.isnan(v[320:384]).all()          # 3.3e38 > 1.875 * 2^127: not representable with its carry
        assert not v[384:].any()


def test_dither_is_uniform():
    a, b = ref.dither(1 << 16, 12345, 7)
    for d in (a, b):
        assert d.min() >= 8 and d.max() <= 0xfffff and abs(d.mean() / 2 ** 20 - 0.5) < 5 / np.sqrt(12 * len(d))
        assert abs(np.corrcoef(d[:-1], d[1:])[0, 1]) < 5 / np.sqrt(len(d))
    assert abs(np.corrcoef(a, b)[0, 1]) < 5 / np.sqrt(len(a))
    assert not np.array_equal(a, ref.dither(1 << 16, 12345, 8)[0]) and not np.array_equal(a, ref.dither(1 << 16, 12346, 7)[0])


def test_second_moment_follows_a_change_of_scale():
    """What stochastic rounding is for: gradients 3 times larger for 2000 steps pull the 8-bit second moment to 9 times its
    value like the fp32 one (1 - 0.999^2000 = 86 % of the way); rounding to nearest leaves it where it was."""
    r = np.random.default_rng(0)
    n, b2 = 64, 0.999
    start = np.full(n, 1e-4, np.float32)
    start[0] = 1.0                                                     # the block's scale is fixed by one element
    near = ref.encode(start, False, np.full(n, ref.NEAREST))
    soft = near
    exact = ref.decode(*near, False)
    for t in range(1, 2001):
        g2 = (9e-4 * r.standard_normal(n) ** 2).astype(np.float32)
        g2[0] = 1.0
        exact = exact * b2 + (1 - b2) * g2
        step = lambda s: (ref.decode(*s, False).astype(np.float32) * np.float32(b2) + np.float32(1 - b2) * g2)  # noqa: E731
        near = ref.encode(step(near), False, np.full(n, ref.NEAREST))
        soft = ref.encode(step(soft), False, ref.dither(n, 0, t)[1])
    mean = lambda s: ref.decode(*s, False)[1:].mean()  # noqa: E731
    # 63 elements, each a random walk whose steps are 1/8 of the value with the chance of a relative change of 1e-3: a spread of
    # about sqrt(1e-3 / 8 * 1000 / 2) = 25 % each, 3 % for the mean
    assert abs(mean(soft) / exact[1:].mean() - 1) < 0.16
    assert mean(near) < 0.5 * exact[1:].mean()


# ----------------------------------------------------------------------------- the step on the GPU

def tensors(numels, seed, scale=1e-2):
    r = np.random.default_rng(seed)
    return [(r.standard_normal(n) * scale * np.exp(r.standard_normal(n))).astype(np.float32) for n in numels]


def flat(parts):
    """Per-tensor codes or exponents -> one buffer of whole blocks."""
    return np.concatenate(parts) if parts else np.zeros(0, np.uint8)


def pad64(c):
    return np.concatenate([c, np.zeros(-len(c) % 64, np.uint8)])


SIZES = [1, 7, 64, 65, 255, 256, 257, 4095, 4096, 4097, 16384, 30001, 3, 128, 1000, 63]


@pytest.mark.gpu
@pytest.mark.parametrize("numels,shift", [(SIZES, 0), (SIZES, 1), (SIZES, 3), ([5] * 130 + [9000, 1], 2), ([300000], 0)])
@pytest.mark.parametrize("coef", [None, 0.3])
def test_step_matches_oracle(dev, numels, shift, coef):
    """Three steps on the same buffers; `shift`: parameters and gradients start that many floats off a 16-byte boundary."""
    from unet_amd import ops
    P, blocks = tensors(numels, 1, 0.1), [-(-n // 64) for n in numels]
    nb = sum(blocks)
    state = [torch.zeros(k, dtype=torch.uint8, device=dev) for k in (nb * 64, nb * 64, nb, nb)]
    M8 = [(np.zeros(n, np.uint8), np.zeros(b, np.uint8)) for n, b in zip(numels, blocks)]
    V8 = list(M8)

    def place(parts):
        out = []
        for x in parts:
            buf = torch.full((len(x) + 8,), -7.0, device=dev)
            view = buf[shift:shift + len(x)]
            view.copy_(torch.from_numpy(x))
            out.append((buf, view))
        return out
    ps = place(P)
    norm = None if coef is None else torch.tensor([123.0, coef], device=dev)
    for t in (1, 2, 3):
        G = tensors(numels, 10 + t)
        gs = place(G)
        ops.adamw8_step([v for _, v in ps], [v for _, v in gs], *state, norm, True, HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"],
                        HYPER["wd"], t, seed=77)
        c = 1.0 if coef is None else coef
        for k, (p, g) in enumerate(zip(P, G)):
            want, bound, M8[k], V8[k] = ref.step(p, g, M8[k], V8[k], c, HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"], HYPER["wd"], t, 77)
            buf, view = ps[k]
            got = view.cpu().numpy()
            assert np.all(np.abs(got - want) <= bound), (k, t, np.max(np.abs(got - want) / bound))
            assert bool((buf[:shift] == -7).all()) and bool((buf[shift + len(p):] == -7).all())
            P[k] = got
            gbuf, gview = gs[k]
            assert np.array_equal(gview.cpu().numpy(), g * np.float32(c))          # clipped gradients are written back
            assert bool((gbuf[:shift] == -7).all()) and bool((gbuf[shift + len(p):] == -7).all())
        for got, per in zip(state, (flat([pad64(m[0]) for m in M8]), flat([pad64(v[0]) for v in V8]),
                                    flat([m[1] for m in M8]), flat([v[1] for v in V8]))):
            assert np.array_equal(got.cpu().numpy(), per)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [1e-8, 1e-10, 1e-12, 2e-15, 2e-18, 1e-20, 0.0])
def test_second_moments_under_the_normal_range(dev, eps):
    """Gradients whose squares are subnormal or vanish, where eps does not hide the root: nothing is taken for zero."""
    from unet_amd import ops
    n, lr, b1, b2 = 640, 1e-3, 0.9, 0.999
    r = np.random.default_rng(5)
    p = np.zeros(n, np.float32)
    dp = torch.zeros(n, device=dev)
    state = [torch.zeros(k, dtype=torch.uint8, device=dev) for k in (n, n, n // 64, n // 64)]
    m8 = v8 = (np.zeros(n, np.uint8), np.zeros(n // 64, np.uint8))
    for t in (1, 2):
        g = (r.standard_normal(n) * np.exp(r.uniform(np.log(3e-19), np.log(3e-15), n))).astype(np.float32)
        ops.adamw8_step([dp], [torch.from_numpy(g).to(dev)], *state, None, False, lr, b1, b2, eps, 0.0, t, seed=3)
        want, bound, m8, v8 = ref.step(p, g, m8, v8, 1.0, lr, b1, b2, eps, 0.0, t, 3)
        p = dp.cpu().numpy()
        assert np.all(np.abs(p - want) <= bound + 2.0 ** -149), (t, np.max(np.abs(p - want) / (bound + 2.0 ** -149)))
        for got, per in zip(state, (m8[0], v8[0], m8[1], v8[1])):
            assert np.array_equal(got.cpu().numpy(), per)


@pytest.mark.gpu
def test_write_grads_veto_and_blocks_of_state(dev):
    from unet_amd import ops
    numels = [100, 64, 1000]
    P, G = tensors(numels, 3), tensors(numels, 4)
    nb, first = 60, [40, 7, 10]                                       # anywhere, in any order, with gaps
    state = [torch.full((k,), 9, dtype=torch.uint8, device=dev) for k in (nb * 64, nb * 64, nb, nb)]
    used = torch.zeros(nb, dtype=torch.bool)
    for f, n in zip(first, numels):
        b = -(-n // 64)
        used[f:f + b] = True
        for s, w in zip(state, (64, 64, 1, 1)):
            s[f * w:(f + b) * w] = 0
    ps, gs = [torch.from_numpy(x).to(dev) for x in P], [torch.from_numpy(x).to(dev) for x in G]
    norm = torch.tensor([1.0, 0.5], device=dev)
    before = [s.clone() for s in state]
    args = (HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"], HYPER["wd"])
    ops.adamw8_step(ps, gs, *state, norm, True, *args, 1, veto=torch.ones(1, device=dev), first_block=first)
    assert all(torch.equal(a, b) for a, b in zip(state, before)) and all(np.array_equal(p.cpu().numpy(), x) for p, x in zip(ps + gs, P + G))
    ops.adamw8_step(ps, gs, *state, norm, False, *args, 1, veto=torch.zeros(1, device=dev), first_block=first)
    for p, g, x, y, f in zip(ps, gs, P, G, first):
        zero = (np.zeros(len(x), np.uint8), np.zeros(-(-len(x) // 64), np.uint8))
        want, bound, m8, v8 = ref.step(x, y, zero, zero, 0.5, *args, 1, 0)
        assert np.all(np.abs(p.cpu().numpy() - want) <= bound) and np.array_equal(g.cpu().numpy(), y)
        assert np.array_equal(state[0][f * 64:f * 64 + len(x)].cpu().numpy(), m8[0])
        assert np.array_equal(state[3][f:f + len(v8[1])].cpu().numpy(), v8[1])
    assert bool((state[2].cpu()[~used] == 9).all()) and bool((state[0].view(-1, 64).cpu()[~used] == 9).all())


@pytest.mark.gpu
def test_gradients_that_are_not_finite(dev):
    """They poison their own block, and nothing else."""
    from unet_amd import ops
    n = 64 * 40
    G = tensors([n], 5)[0]
    G[70], G[64 * 10 + 1], G[64 * 20], G[64 * 30] = np.nan, np.inf, 1e25, 1e-40
    p, g = torch.zeros(n, device=dev), torch.from_numpy(G).to(dev)
    state = [torch.zeros(k, dtype=torch.uint8, device=dev) for k in (n, n, n // 64, n // 64)]
    args = (HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"], 0.0)
    zero = (np.zeros(n, np.uint8), np.zeros(n // 64, np.uint8))
    ops.adamw8_step([p], [g], *state, None, False, *args, 1)
    want, bound, m8, v8 = ref.step(np.zeros(n, np.float32), G, zero, zero, 1.0, *args, 1, 0)
    for got, per in zip(state, (m8[0], v8[0], m8[1], v8[1])):
        assert np.array_equal(got.cpu().numpy(), per)
    got = p.cpu().numpy()
    fine = np.isfinite(want) & (np.arange(n) != 64 * 20)
    assert np.all(np.abs(got - want)[fine] <= bound[fine]) and np.isnan(got[70]) and np.isnan(got[64 * 10 + 1])
    assert got[64 * 20] == 0                                           # v is infinite there
    ops.adamw8_step([p], [g], *state, None, False, *args, 2)
    poisoned = np.isnan(p.cpu().numpy()).reshape(-1, 64).all(1)
    assert poisoned[1] and poisoned[10] and poisoned[20] and poisoned.sum() == 3


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 63, 64, 65, 1000, 64 * 4096 + 17])
@pytest.mark.parametrize("signed", [True, False])
def test_encode_and_decode_match_oracle(dev, n, signed):
    from unet_amd import ops
    x = values(n, n)
    x = x if signed else np.abs(x)
    x[n // 2] = 0.0
    c, e = ops.moment8_encode(torch.from_numpy(x).to(dev), signed)
    wc, we = ref.encode(x, signed, np.full(n, ref.NEAREST))
    assert np.array_equal(c.cpu().numpy(), wc) and np.array_equal(e.cpu().numpy(), we)
    want = ref.decode(wc, we, signed)
    for dtype in (torch.float32, torch.bfloat16):
        got = ops.moment8_decode(c, e, signed, dtype=dtype)
        assert got.dtype == dtype and np.array_equal(got.double().cpu().numpy(), want)
    e[0] = 255
    assert bool(ops.moment8_decode(c, e, signed)[:64].isnan().all())


@pytest.mark.gpu
def test_other_stream_empty_lists_and_capture(dev):
    from unet_amd import ops
    from unet_amd._lib import UNetHipError
    none = [torch.zeros(0, dtype=torch.uint8, device=dev) for _ in range(4)]
    ops.adamw8_step([], [], *none, None, False, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    e = torch.zeros(0, device=dev)
    ops.adamw8_step([e, e], [e, e], *none, None, False, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    assert ops.moment8_encode(e, True)[0].numel() == 0 and ops.moment8_decode(none[0], none[2], True).numel() == 0
    n = 5000
    x = tensors([n], 6)[0]
    nb = -(-n // 64)

    def fresh():
        return torch.zeros(n, device=dev), torch.from_numpy(x).to(dev), [torch.zeros(k, dtype=torch.uint8, device=dev) for k in (nb * 64, nb * 64, nb, nb)]
    a, b = fresh(), fresh()
    ops.adamw8_step([a[0]], [a[1]], *a[2], None, False, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.adamw8_step([b[0]], [b[1]], *b[2], None, False, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a[0], b[0]) and all(torch.equal(p, q) for p, q in zip(a[2], b[2]))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    t = torch.zeros(4, device=dev)
    with torch.cuda.graph(graph):
        t.add_(1)
        with pytest.raises(UNetHipError, match="captured"):
            ops.adamw8_step([b[0]], [b[1]], *b[2], None, False, 1e-3, 0.9, 0.999, 1e-8, 0.0, 2)
    assert torch.equal(a[0], b[0])


def test_betas_that_the_rounding_does_not_resolve():
    """Second moments under steps without gradient: codes 1 to 7 never move where 1 - beta2 is under 2^-17 of what they stand for, and
    follow beta2 at the least 1 - beta2 that is taken."""
    from unet_amd._lib import lib
    from unet_amd.optim import FusedAdamW
    n = 64 * 2048
    x = np.tile(np.arange(64) % 7 + 1.0, 2048).astype(np.float32) * np.float32(2.0) ** -33
    x[63::64] = 1.0                                                   # the block's scale: 2^-33 is the smallest code
    for fall, moves in ((2.0 ** -21, False), (2.0 ** -16, True)):
        v, e = ref.encode(x, False, np.full(n, ref.NEAREST))
        assert np.array_equal(ref.decode(v, e, False)[:63], x[:63].astype(np.float64))
        start, steps = v.copy(), 60
        for t in range(1, steps + 1):
            now = ref.decode(v, e, False).astype(np.float32) * np.float32(1 - fall)
            v, e = ref.encode(now, False, ref.dither(n, 1, t)[1])
            v[63::64] = start[63::64]
        small = np.arange(n) % 64 != 63
        gone = (ref.decode(start, e, False) - ref.decode(v, e, False))[small]
        if not moves:
            assert not gone.any()
        else:                                                         # expected: steps * fall of each value (of those over the floor)
            over = x[small] > 2.0 ** -33
            want = steps * fall * x[small][over].astype(np.float64).mean()
            assert abs(gone[over].mean() - want) < steps * 2.0 ** -17 * 2.0 ** -33 + 5 * 2.0 ** -33 * np.sqrt(steps * fall * 7 / over.sum())
    L, zero = lib(), [None] * 4
    for b1, b2, rc in ((0.9, 1 - 2.0 ** -17, 0), (0.9, 1 - 2.0 ** -18, -1), (1 - 2.0 ** -18, 0.999, -1)):
        assert L.unet_adamw8_step(0, None, None, None, None, *zero, 0, None, 0, 1e-3, b1, b2, 1e-8, 0.0, 1, 0, None, None) == rc
    p = torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="betas"):
        FusedAdamW([p], betas=(0.9, 1 - 1e-6), state_bits=8)
    FusedAdamW([p], betas=(0.9, 1 - 1e-6))


# ----------------------------------------------------------------------------- refusals

def call(dev, ps=None, gs=None, sizes=(64, 64, 1, 1), dtype=torch.uint8, **kw):
    from unet_amd import ops
    ps = [torch.zeros(64, device=dev)] if ps is None else ps
    gs = [torch.zeros(64, device=dev)] if gs is None else gs
    state = [torch.zeros(k, dtype=dtype, device=dev) for k in sizes]
    a = dict(norm_out=None, write_grads=False, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.0, step=1)
    a.update(kw)
    ops.adamw8_step(ps, gs, *state, **a)


def refusals(dev):
    f = lambda n, **k: torch.zeros(n, device=dev, **k)  # noqa: E731
    one = f(64)
    return [
        (dict(gs=[]), "lengths"), (dict(gs=[f(63)]), "sizes differ"), (dict(ps=[f(64, dtype=torch.bfloat16)]), "fp32"),
        (dict(ps=[f((8, 16)).t()[:, :4]], gs=[f(64)]), "contiguous"), (dict(ps=[one, one], gs=[f(64), f(64)], sizes=(128, 128, 2, 2)), "twice"),
        (dict(sizes=(64, 64, 2, 1)), "64 codes"), (dict(sizes=(63, 64, 1, 1)), "64 codes"), (dict(sizes=(128, 128, 2, 2)), "not those"),
        (dict(dtype=torch.int8), "uint8"), (dict(first_block=[0, 1]), "lengths"),
        (dict(ps=[f(64), f(65)], gs=[f(64), f(65)], sizes=(256, 256, 4, 4), first_block=[1, 0]), "share blocks"),
        (dict(norm_out=f(1)), "norm_out two"), (dict(veto=f(1, dtype=torch.float64)), "veto"),
    ]


def test_refusals_without_a_gpu():
    from unet_amd._lib import UNetHipError
    for kw, msg in refusals("cpu") + [({}, "CPU tensor")]:
        with pytest.raises(UNetHipError, match=msg):
            call("cpu", **kw)


@pytest.mark.gpu
def test_refusals_on_the_device(dev):
    from unet_amd._lib import UNetHipError
    for kw, msg in refusals(dev) + [(dict(first_block=[1]), "outside the state"), (dict(first_block=[-1]), "outside the state"), (dict(step=0), "step"),
                                    (dict(beta2=1.0), "hyper"), (dict(eps=-1.0), "hyper"), (dict(veto=torch.zeros(1)), "CPU tensor"),
                                    (dict(gs=[torch.zeros(64)]), "one device")]:
        with pytest.raises(UNetHipError, match=msg):
            call(dev, **kw)


# ----------------------------------------------------------------------------- the optimizer

def params(dev, seed=0, shapes=((3, 5), (16385,), (64, 33, 3, 3), (1,), (40000,))):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g).to(dev)) for s in shapes]


def set_grads(ps, seed, scale=0.3):
    g = torch.Generator().manual_seed(seed)
    for p in ps:
        p.grad = (torch.randn(p.shape, generator=g) * scale).to(p.device)


def test_optimizer_arguments():
    from unet_amd.optim import FusedAdamW
    from unet_amd.utils.builders import get_optim
    from unet_amd._lib import UNetHipError
    p = torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="state_bits"):
        FusedAdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="plain AdamW"):
        FusedAdamW([p], state_bits=8, amsgrad=True)
    opt = get_optim("adamw", [p], lr=1e-3, state_bits=8)
    assert opt.state_bits == 8 and get_optim("adamw", [p], lr=1e-3).state_bits == 32
    p.grad = torch.ones(4)
    with pytest.raises(UNetHipError, match="on the GPU"):
        opt.step()
    assert float(p.detach()[0]) == 1.0 and len(opt.state[p]) == 0
    opt.add_param_group({"params": [torch.nn.Parameter(torch.ones(2))], "maximize": True})
    p.grad = None
    with pytest.raises(UNetHipError, match="plain AdamW"):
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("clip", [None, 1.0])
def test_optimizer_follows_the_oracle(dev, clip):
    """Parameters with and without gradients, late ones, and clipping, all as one oracle run per tensor."""
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=HYPER["lr"], betas=(HYPER["b1"], HYPER["b2"]), eps=HYPER["eps"], weight_decay=HYPER["wd"], state_bits=8, state_seed=5)
    zero = [(np.zeros(p.numel(), np.uint8), np.zeros(-(-p.numel() // 64), np.uint8)) for p in ps]
    M8, V8, steps = list(zero), list(zero), [0] * len(ps)
    for it in range(4):
        set_grads(ps, 100 + it)
        if it < 2:
            ps[4].grad = None                                         # joins later: state of its own
        if it == 2:
            ps[0].grad = None
        P = [p.detach().cpu().numpy().reshape(-1) for p in ps]
        G = [None if p.grad is None else p.grad.cpu().numpy().reshape(-1) for p in ps]
        v0 = ps[1]._version
        if clip is None:
            opt.step()
            coef = 1.0
        else:
            norm = opt.clip_and_step(ps, clip)
            total = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in G if g is not None))
            assert abs(float(norm) - total) < 1e-5 * total
            # the coefficient from the device's own norm
            coef = np.float32(clip) / (np.float32(float(norm)) + np.float32(1e-6))
            assert coef < 1
            for p, g in zip(ps, G):
                assert g is None or np.array_equal(p.grad.cpu().numpy().reshape(-1), g * np.float32(coef))
        assert ps[1]._version > v0
        for k, p in enumerate(ps):
            if G[k] is None:
                continue
            steps[k] += 1
            want, bound, M8[k], V8[k] = ref.step(P[k], G[k], M8[k], V8[k], coef, HYPER["lr"], HYPER["b1"], HYPER["b2"], HYPER["eps"], HYPER["wd"],
                                                 steps[k], 5)
            assert np.all(np.abs(p.detach().cpu().numpy().reshape(-1) - want) <= bound)
            st = opt.state[p]
            assert st["exp_avg"].shape == p.shape and float(st["step"]) == steps[k]
            for key, w in zip(("exp_avg", "exp_avg_e", "exp_avg_sq", "exp_avg_sq_e"), M8[k] + V8[k]):
                assert np.array_equal(st[key].cpu().numpy().reshape(-1), w)


@pytest.mark.gpu
def test_checkpoints_of_both_kinds(dev, tmp_path):
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=8)
    for it in range(3):
        set_grads(ps, it)
        opt.step()
    path = tmp_path / "o.ckpt"
    torch.save(opt.state_dict(), path)
    saved = torch.load(path, map_location="cpu", weights_only=True)
    values = [p.detach().clone() for p in ps]

    def fresh(bits):
        qs = [torch.nn.Parameter(v.clone()) for v in values]
        o = FusedAdamW(qs, lr=1e-3, state_bits=bits)
        o.load_state_dict(copy.deepcopy(saved))            # (torch keeps the step tensors it is given)
        return qs, o
    # 8 -> 8: continues bit for bit
    qs, o8 = fresh(8)
    for it in (3, 4):
        set_grads(ps, it)
        set_grads(qs, it)
        opt.step()
        o8.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        for k in ("exp_avg", "exp_avg_sq", "exp_avg_e", "exp_avg_sq_e"):
            assert torch.equal(opt.state[p][k], o8.state[q][k]) and o8.state[q][k].dtype == torch.uint8
    # 8 -> 32: the values the codes stand for, then the 32-bit step
    qs, o32 = fresh(32)
    set_grads(qs, 3)
    twin = [torch.nn.Parameter(v.clone()) for v in values]
    ot = torch.optim.AdamW(twin, lr=1e-3, foreach=False)
    set_grads(twin, 3)
    for i, q in enumerate(twin):
        s = saved["state"][i]
        ot.state[q] = {"step": s["step"].clone()}
        for k, signed in (("exp_avg", True), ("exp_avg_sq", False)):
            v = ref.decode(s[k].numpy().reshape(-1), s[k + "_e"].numpy(), signed)
            ot.state[q][k] = torch.from_numpy(v.astype(np.float32)).view(q.shape).to(dev)
    o32.step()
    ot.step()
    for q, t in zip(qs, twin):
        torch.testing.assert_close(q, t, rtol=2e-6, atol=2e-7)
        assert o32.state[q]["exp_avg"].dtype == torch.float32 and "exp_avg_e" not in o32.state[q]
    # 32 -> 8: rounded to nearest once
    saved = o32.state_dict()
    moments = [(o32.state[q]["exp_avg"].cpu().numpy().reshape(-1), o32.state[q]["exp_avg_sq"].cpu().numpy().reshape(-1)) for q in qs]
    values = [q.detach().clone() for q in qs]
    qs, o8 = fresh(8)
    set_grads(qs, 9)
    G = [q.grad.cpu().numpy().reshape(-1) for q in qs]
    o8.step()
    for q, v, (m, s), g in zip(qs, values, moments, G):
        near = np.full(len(m), ref.NEAREST)
        want, bound, m8, v8 = ref.step(v.cpu().numpy().reshape(-1), g, ref.encode(m, True, near), ref.encode(s, False, near), 1.0, 1e-3, 0.9, 0.999,
                                       1e-8, 1e-2, 5, 0)
        assert np.all(np.abs(q.detach().cpu().numpy().reshape(-1) - want) <= bound)
        assert np.array_equal(o8.state[q]["exp_avg"].cpu().numpy().reshape(-1), m8[0])


@pytest.mark.gpu
def test_vetoed_step_changes_nothing(dev):
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=8)
    set_grads(ps, 1)
    opt.clip_and_step(ps, 1.0)
    keep = [t.clone() for p in ps for t in (p, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq_e"])]
    set_grads(ps, 2)
    opt.clip_and_step(ps, 1.0, veto=torch.ones(1, device=dev))
    opt.undo_vetoed_step()
    now = [t for p in ps for t in (p, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq_e"])]
    assert all(torch.equal(a, b) for a, b in zip(keep, now)) and float(opt.state[ps[0]]["step"]) == 1.0


@pytest.mark.gpu
def test_gradients_that_hold_a_multiple(dev):
    """Data parallel hands over the ranks' sum with grad_scale = 1/world: the same bits as averaged gradients."""
    from unet_amd.optim import FusedAdamW
    a, b = params(dev), params(dev)
    oa, ob = FusedAdamW(a, lr=1e-3, state_bits=8), FusedAdamW(b, lr=1e-3, state_bits=8)
    for it in range(2):
        set_grads(a, it)
        for p, q in zip(a, b):
            q.grad = p.grad * 4.0                                     # a power of two: exact
        na, nb = oa.clip_and_step(a, 1.0), ob.clip_and_step(b, 1.0, grad_scale=0.25)
        assert torch.equal(na, nb)
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.equal(p.grad, q.grad)
        assert all(torch.equal(oa.state[p][k], ob.state[q][k]) for k in ("exp_avg", "exp_avg_sq", "exp_avg_e", "exp_avg_sq_e"))


@pytest.mark.gpu
def test_refused_steps_leave_everything_alone(dev):
    from unet_amd._lib import UNetHipError
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=8)
    set_grads(ps, 0)
    opt.step()
    keep = [p.detach().clone() for p in ps]
    set_grads(ps, 1)
    torch.cuda.synchronize()
    graph, t = torch.cuda.CUDAGraph(), torch.zeros(4, device=dev)
    with torch.cuda.graph(graph):
        t.add_(1)
        with pytest.raises(UNetHipError, match="captured"):
            opt.clip_and_step(ps, 1.0)
    ps[0].grad = ps[0].grad.t().contiguous().t()                     # the same shape, other strides
    with pytest.raises(UNetHipError, match="contiguous"):
        opt.clip_and_step(ps, 1.0)
    assert all(torch.equal(p, k) for p, k in zip(ps, keep)) and all(float(opt.state[p]["step"]) == 1.0 for p in ps)


@pytest.mark.gpu
def test_state_loaded_before_the_model_moves_to_the_gpu(dev):
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=8)
    set_grads(ps, 0)
    opt.step()
    sd = copy.deepcopy(opt.state_dict())
    qs = [torch.nn.Parameter(p.detach().cpu()) for p in ps]
    o2 = FusedAdamW(qs, lr=1e-3, state_bits=8)
    o2.load_state_dict(sd)                                           # state on the CPU now
    for q in qs:
        q.data = q.data.to(dev)
    set_grads(ps, 1)
    set_grads(qs, 1)
    opt.step()
    o2.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q) and torch.equal(opt.state[p]["exp_avg"], o2.state[q]["exp_avg"]) and o2.state[q]["exp_avg"].is_cuda


def clip_foreign(ps, opt, strange):
    """clip_and_step over this optimizer's parameters and one that it does not own and cannot clip -> what was there and what is."""
    from unet_amd._lib import UNetHipError

    def everything():
        return [t.detach().clone() for p in ps + [strange] for t in (p, p.grad)] + \
               [t.clone() for p in ps for t in opt.state.get(p, {}).values()]
    before = everything()
    with pytest.raises(UNetHipError, match="state_bits=8"):
        opt.clip_and_step(ps + [strange], 0.01, grad_scale=0.5)
    return before, everything()


def test_clipping_a_gradient_of_another_kind_is_refused_before_anything_changes(monkeypatch):
    from unet_amd.optim import FusedAdamW
    monkeypatch.setattr(FusedAdamW, "_tensor_ok", staticmethod(lambda t: t.dtype == torch.float32 and t.is_contiguous()))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for foreach in (False, True):
        ps, strange = params("cpu", shapes=((3, 5), (70,))), torch.nn.Parameter(torch.ones(4, 6))
        set_grads(ps, 1)
        strange.grad = torch.ones(6, 4).t()
        before, now = clip_foreign(ps, FusedAdamW(ps, lr=1e-3, state_bits=8, foreach=foreach), strange)
        assert len(before) == len(now) and all(torch.equal(a, b) for a, b in zip(before, now))


@pytest.mark.gpu
def test_clipping_a_gradient_of_another_kind_on_the_device(dev):
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=8)
    set_grads(ps, 0)
    opt.step()
    transposed, half, host = (torch.nn.Parameter(t) for t in (torch.ones(4, 6, device=dev), torch.ones(8, device=dev, dtype=torch.bfloat16), torch.ones(8)))
    transposed.grad, half.grad, host.grad = torch.ones(6, 4, device=dev).t(), torch.ones_like(half), torch.ones_like(host)
    for strange in (transposed, half, host):
        set_grads(ps, 1)
        before, now = clip_foreign(ps, opt, strange)
        assert len(before) == len(now) and all(torch.equal(a, b) for a, b in zip(before, now))


def test_other_optimizers_refuse_8_bit_state(tmp_path):
    """The codes lie under exp_avg and exp_avg_sq in the parameter's shape: another Adam would train on the bytes as moments."""
    from unet_amd.optim import FusedAdamW
    from unet_amd.utils.builders import get_optim
    ps = params("cpu", shapes=((3, 5), (70,), (1,)))
    o8 = FusedAdamW(ps, lr=1e-3, state_bits=8)
    assert len(o8.state_dict()["param_groups"]) == 1                 # no state yet: nothing to misread
    for p in ps:
        n = p.numel()
        x = values(n, n)
        m, v = (ref.encode(t, signed, np.full(n, ref.NEAREST)) for t, signed in ((x, True), (x * x, False)))
        o8.state[p] = {"step": torch.tensor(3.0), "exp_avg": torch.from_numpy(m[0]).view(p.shape), "exp_avg_sq": torch.from_numpy(v[0]).view(p.shape),
                       "exp_avg_e": torch.from_numpy(m[1]), "exp_avg_sq_e": torch.from_numpy(v[1])}
    torch.save(o8.state_dict(), tmp_path / "o.ckpt")
    saved = torch.load(tmp_path / "o.ckpt", weights_only=True)
    for other in (torch.optim.AdamW(ps, lr=1e-3), get_optim("adam", ps, lr=1e-3), get_optim("sgd", ps, lr=1e-3)):
        with pytest.raises(ValueError, match="number of parameter groups"):
            other.load_state_dict(saved)
        assert not other.state and len(other.param_groups) == 1
    unmarked = {**saved, "param_groups": saved["param_groups"][:-1]}     # as it was written before the mark
    for bits in (8, 32):
        for sd in (saved, unmarked):
            o = FusedAdamW(ps, lr=7.0, state_bits=bits)
            o.load_state_dict(copy.deepcopy(sd))
            assert len(o.param_groups) == 1 and o.param_groups[0]["lr"] == 1e-3 and len(saved["param_groups"]) == 2
            for p in ps:
                assert all(torch.equal(o.state[p][k], o8.state[p][k]) for k in o8.state[p])
            assert o.state_dict()["param_groups"][-1] == {"params": [], "state_bits": 8}


@pytest.mark.gpu
def test_resuming_from_a_checkpoint_file(dev, tmp_path):
    """load_checkpoint maps a file to the GPU, step counts included; the run goes on bit for bit."""
    import types
    from unet_amd.optim import FusedAdamW
    from unet_amd.utils.checkpoint_utils import load_checkpoint, save_checkpoint
    nets = [torch.nn.Linear(33, 70).to(dev) for _ in range(2)]
    opts = [FusedAdamW(n.parameters(), lr=1e-3, state_bits=8) for n in nets]

    def step(k, seed):
        set_grads(list(nets[k].parameters()), seed)
        opts[k].clip_and_step(list(nets[k].parameters()), 1.0)
    step(0, 0)
    step(0, 1)
    save_checkpoint(str(tmp_path), types.SimpleNamespace(model=nets[0], optimizer=opts[0], scheduler=None, scaler=None), 1)
    load_checkpoint(str(tmp_path / "last.ckpt"), nets[1], opts[1])
    for seed in (2, 3):
        step(0, seed)
        step(1, seed)
    for p, q in zip(nets[0].parameters(), nets[1].parameters()):
        assert torch.equal(p, q) and float(opts[1].state[q]["step"]) == 4.0
        assert all(torch.equal(opts[0].state[p][k], opts[1].state[q][k]) for k in opts[0].state[p])


def test_copies_keep_their_state_bits():
    import pickle
    from unet_amd.optim import FusedAdamW
    p = torch.nn.Parameter(torch.ones(70))
    for bits in (8, 32):
        opt = FusedAdamW([p], lr=1e-3, state_bits=bits, state_seed=9)
        opt.state[p] = {"step": torch.tensor(1.0), "exp_avg": torch.full((70,), 3, dtype=torch.uint8), "exp_avg_sq": torch.full((70,), 4, dtype=torch.uint8),
                        "exp_avg_e": torch.full((2,), 120, dtype=torch.uint8), "exp_avg_sq_e": torch.full((2,), 110, dtype=torch.uint8)}
        for twin in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
            assert (twin.state_bits, twin.state_seed) == (bits, 9)
            for again in (False, True):
                (q, st), = twin.state.items()
                assert q is twin.param_groups[0]["params"][0] and all(torch.equal(st[k], v) for k, v in opt.state[p].items())
                assert st["exp_avg"].dtype == torch.uint8 and (bits == 32 or twin.step() is None)      # (no gradients: nothing to do)
                twin.load_state_dict(opt.state_dict())


@pytest.mark.gpu
def test_a_copy_goes_on_like_the_original(dev):
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=8, state_seed=3)
    set_grads(ps, 0)
    opt.clip_and_step(ps, 1.0)
    twin = copy.deepcopy(opt)
    qs = twin.param_groups[0]["params"]
    for seed in (1, 2):
        for o, t in ((opt, ps), (twin, qs)):
            set_grads(t, seed)
            o.clip_and_step(t, 1.0)
    for p, q in zip(ps, qs):
        assert p is not q and torch.equal(p, q) and all(torch.equal(opt.state[p][k], twin.state[q][k]) for k in opt.state[p])


@pytest.mark.parametrize("bits", [8, 32])
def test_a_refused_launch_leaves_the_step_counts(monkeypatch, bits):
    from unet_amd import ops
    from unet_amd._lib import UNetHipError
    from unet_amd.optim import FusedAdamW
    monkeypatch.setattr(FusedAdamW, "_tensor_ok", staticmethod(lambda t: True))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)

    def refuse(*a, **k):
        raise UNetHipError("bad hyper-parameters")
    monkeypatch.setattr(ops, "adamw_step", refuse)
    monkeypatch.setattr(ops, "adamw8_step", refuse)
    ps = params("cpu", shapes=((3, 5), (70,)))
    set_grads(ps, 1)
    opt = FusedAdamW(ps, lr=1e-3, state_bits=bits)
    for _ in range(2):
        with pytest.raises(UNetHipError, match="hyper"):
            opt.step()
    assert all(float(opt.state[p]["step"]) == 0.0 for p in ps)


@pytest.mark.gpu
def test_a_learning_rate_that_is_no_number(dev):
    from unet_amd._lib import UNetHipError
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    opt = FusedAdamW([{"params": ps[:2]}, {"params": ps[2:]}], lr=1e-3, state_bits=8)
    set_grads(ps, 0)
    opt.step()
    keep = [t.clone() for p in ps for t in (p.detach(), p.grad, *opt.state[p].values())]
    opt.param_groups[1]["lr"] = float("nan")                         # the second group's: the first is not stepped either
    with pytest.raises(UNetHipError, match="hyper"):
        opt.clip_and_step(ps, 0.01)
    assert all(torch.equal(a, b) for a, b in zip(keep, [t for p in ps for t in (p.detach(), p.grad, *opt.state[p].values())]))


def test_tensors_that_share_memory_are_refused():
    """Views of one buffer that overlap without starting together; neighbours do not overlap."""
    from unet_amd import ops
    from unet_amd._lib import UNetHipError
    flat, g = torch.zeros(256), torch.zeros(256)
    state = [torch.zeros(k, dtype=torch.uint8) for k in (128, 128, 2, 2)]

    def step(ps, gs, write=False, state=state):
        ops.adamw8_step(ps, gs, *state, None, write, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1)
    apart = [g[:64], g[64:128]]
    for ps, gs, write in (([flat[:64], flat[63:127]], apart, False), ([flat[100:164], flat[40:104]], apart, False), ([flat[:64], flat[:64]], apart, False),
                          ([flat[:64], flat[64:128]], [g[:64], g[32:96]], True)):
        with pytest.raises(UNetHipError, match="share memory"):
            step(ps, gs, write)
    with pytest.raises(UNetHipError, match="different ones"):
        step([flat[:64], flat[64:128]], apart, state=[state[0], state[0], state[2], state[3]])
    for ps, gs, write in (([flat[:64], flat[64:128]], apart, True), ([flat[:64], flat[64:128]], [g[:64], g[32:96]], False),
                          ([flat[:64], flat[10:10], flat[64:128]], apart[:1] + [g[:0]] + apart[1:], True)):
        with pytest.raises(UNetHipError, match="CPU tensor"):            # (gradients that are only read may overlap)
            step(ps, gs, write)


@pytest.mark.gpu
def test_8_bit_state_put_into_a_32_bit_optimizer_by_hand(dev):
    from unet_amd.optim import FusedAdamW
    ps = params(dev)
    o8 = FusedAdamW(ps, lr=1e-3, state_bits=8)
    set_grads(ps, 0)
    o8.step()
    by_hand, loaded = [torch.nn.Parameter(p.detach().clone()) for p in ps], [torch.nn.Parameter(p.detach().clone()) for p in ps]
    oh, ol = FusedAdamW(by_hand, lr=1e-3), FusedAdamW(loaded, lr=1e-3)
    ol.load_state_dict(copy.deepcopy(o8.state_dict()))
    set_grads(by_hand, 1)
    for p, q in zip(ps, by_hand):
        oh.state[q] = {k: v.clone() for k, v in o8.state[p].items()}
    set_grads(loaded, 1)
    oh.step()
    ol.step()
    for q, t in zip(by_hand, loaded):
        assert torch.equal(q, t) and oh.state[q]["exp_avg"].dtype == torch.float32 and torch.equal(oh.state[q]["exp_avg_sq"], ol.state[t]["exp_avg_sq"])
