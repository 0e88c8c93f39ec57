"""The residual's addition with its norm, 8-bit output and gradients in 64 bits, and how far the kernels' results may be from it.

Bounds: u is half a step of the stream's type, E = 2^-24 that of fp32.  A sum of n numbers in fp32 in any order is off by at most
n E of the sum of magnitudes; other steps round a handful of times.  Everything behind t is computed from t as the kernel gave it:
the norm reads the stream as it is held.
"""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -24


def spread(mod, rows, fill):
    """[M, K] the modulation row of each token, `fill` where it has none."""
    out = torch.full((rows.shape[0], mod.shape[1]), fill, dtype=torch.float64, device=mod.device)
    has = (rows >= 0) & (rows < mod.shape[0])
    out[has] = mod.double()[rows[has]]
    return out


def stream(x, y, gate, rows):
    v = y.double() if gate is None else y.double() * spread(gate, rows, 0.0)
    v = v + x.double()
    return v, U[x.dtype] * v.abs() * (1 + 2.0 ** -9) + (2 * E * v.abs() + 2.0 ** -25)


def normalised(t, weight, eps, shift, scale, rows):
    """(rstd, h before its rounding, how far it may be off)."""
    v, k = t.double(), t.shape[1]
    rstd = (v.square().mean(1, keepdim=True) + eps).rsqrt()
    main = v * rstd * weight.double()
    add = torch.zeros_like(main)
    if scale is not None:
        main, add = main * (1 + spread(scale, rows, 0.0)), spread(shift, rows, 0.0)
    return rstd, main + add, main.abs() * (k / 2 + 12) * E + (main.abs() + add.abs()) * 2 * E


def rotated(h, off):
    """(z, how far it may be off): blocks of 256 times the regular Hadamard matrix / 16."""
    h4 = torch.tensor([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], dtype=torch.float64, device=h.device)
    h16 = torch.kron(h4, h4)
    had = torch.kron(h16, h16) / 16
    m, k = h.shape

    def turn(t, matrix):
        return (t.view(m, k // 256, 256) @ matrix).view(m, k)

    return turn(h, had), turn(off, had.abs()) + 16 * E * turn(h.abs(), had.abs())


def gradients(dt, dh, t, weight, eps, gate, scale, rows):
    """(dx, dy, dw) and bounds."""
    u, k, m = U[t.dtype], t.shape[1], t.shape[0]
    v = t.double()
    rstd = (v.square().mean(1, keepdim=True) + eps).rsqrt()
    n = v * rstd
    g = dh.double()
    if scale is not None:
        g = g * (1 + spread(scale, rows, 0.0))
    p = g * weight.double()
    dot, dots = (p * n).mean(1, keepdim=True), (p * n).abs().mean(1, keepdim=True)
    base = torch.zeros_like(v) if dt is None else dt.double()
    dx = base + rstd * (p - n * dot)
    rough = (k + 16) * E
    tx = rstd * ((p.abs() + n.abs() * dots) * (rough + 8 * E)) + 4 * E * (base.abs() + rstd * (p.abs() + n.abs() * dots))
    dy, ty = dx, tx
    if gate is not None:
        turn = spread(gate, rows, 0.0)
        dy, ty = dx * turn, tx * turn.abs() + 2 * E * (dx * turn).abs()
    dw = (g * n).sum(0)
    tw = (g * n).abs().sum(0) * ((m + 8) * E + rough)
    uw = 2.0 ** -24 if weight.dtype == torch.float32 else U[weight.dtype]
    return (dx, dy, dw), (tx + u * dx.abs() + 2.0 ** -25, ty + u * dy.abs() + 2.0 ** -25, tw + uw * dw.abs() + 2.0 ** -25)


def check(got, want, tol, what=""):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what
    off = (got - want).abs()
    bad = off > tol
    assert not bad.any(), (what, int(bad.sum()), float((off / tol.clamp_min(1e-300)).max()))
