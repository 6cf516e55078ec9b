"""Layer norm over the last axis, summed over branches, with ReLU, and its gradients: fp64 on the CPU, from the formulas.

Every function also returns what an fp32 evaluation may be off by, element for element, in units that follow from the
formulas: u = 2^-24 per rounding, N roundings on the longest path of a sum over the channels."""
import torch

U = 2.0 ** -24


def _branch(z, eps):
    """xhat, rstd, and the error bounds (absolute for xhat, relative for rstd) of an fp32 evaluation."""
    z = z.double()
    C = z.shape[-1]
    N = C / 64 + 16
    mean = z.mean(-1, keepdim=True)
    d = z - mean
    rstd = 1.0 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    x = d * rstd
    shift = N * U * z.abs().mean(-1, keepdim=True) + U * mean.abs()   # error of the mean, the same for the whole row
    e_rstd = (N / 2 + 4) * U + 0.5 * (shift * rstd) ** 2
    e_x = shift * rstd + (2 * U + e_rstd) * x.abs()
    return x, rstd, e_x, e_rstd


def forward(zs, gammas, betas, relu, eps):
    """-> (y, bound): y in fp64, bound = largest error of an fp32 evaluation before the output's own rounding."""
    y, bound, mag = 0.0, 0.0, 0.0
    for z, g, b in zip(zs, gammas, betas):
        x, _, e_x, _ = _branch(z, eps)
        g = torch.ones(()).double() if g is None else g.double()
        b = torch.zeros(()).double() if b is None else b.double()
        y = y + x * g + b
        bound = bound + e_x * g.abs()
        mag = mag + (x * g).abs() + b.abs()
    bound = bound + (2 * len(zs) + 1) * U * mag
    return (torch.where(y < 0, 0.0, y) if relu else y), bound


def backward(dy, zs, gammas, y, eps):
    """-> [(dz, its bound, dgamma, its bound)], (dbeta, its bound); y: output of the ReLU or None."""
    u = dy.double()
    if y is not None:
        u = torch.where(y.double() <= 0, 0.0, u)
    C = u.shape[-1]
    rows = u.numel() // C
    N, R = C / 64 + 16, rows / 64 + 80
    out = []
    for z, g in zip(zs, gammas):
        x, rstd, e_x, e_rstd = _branch(z, eps)
        w = u * (1.0 if g is None else g.double())
        m1, m2 = w.mean(-1, keepdim=True), (w * x).mean(-1, keepdim=True)
        dz = rstd * (w - m1 - x * m2)
        e1 = (N + 2) * U * w.abs().mean(-1, keepdim=True)
        e2 = (N + 3) * U * (w * x).abs().mean(-1, keepdim=True) + (w.abs() * e_x).mean(-1, keepdim=True)
        e = U * w.abs() + e1 + x.abs() * e2 + e_x * m2.abs() + 4 * U * (w.abs() + m1.abs() + (x * m2).abs())
        e_dz = rstd * e + (e_rstd + U) * dz.abs()
        flat = (-1, C)
        dg = (u * x).reshape(flat).sum(0)
        e_dg = (u.abs() * e_x).reshape(flat).sum(0) + R * U * (u * x).abs().reshape(flat).sum(0) + U * dg.abs()
        out.append((dz, e_dz, dg, e_dg))
    db = u.reshape(-1, C).sum(0)
    return out, (db, R * U * u.abs().reshape(-1, C).sum(0) + U * db.abs())
