"""Low-rank adapters in 64 bits, and how far the kernels' results may be from it.

Bounds: u is half a step of the operands' type (bf16 2^-8, fp16 2^-11).  A sum of n products in fp32 on the tensor cores, whose additions
may drop bits instead of rounding, is off by at most (n + 16) 2^-23 of the sum of magnitudes.  The hidden row h is rounded once
(u |h|); in fp16 it is scaled so that its largest entry is in [1, 2) first, so that small entries are off by 2^-25 of the
largest instead.  The result is rounded once.
"""
import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gamma(n):
    return (n + 16) * 2.0 ** -23


def groups(rows, adapters):
    for g in range(adapters):
        yield g, (rows == g).nonzero().flatten()


def forward(x, a, b, rows, scales=None, base=None):
    """(out, bound) in 64 bits."""
    u = U[x.dtype]
    x, a, b = x.double(), a.double(), b.double()
    out = torch.zeros(x.shape[0], b.shape[1], dtype=torch.float64, device=x.device) if base is None else base.double()
    tol = torch.zeros_like(out)
    for g, i in groups(rows, a.shape[0]):
        s = 1.0 if scales is None else float(scales[g])
        h, habs = s * x[i] @ a[g].T, abs(s) * x[i].abs() @ a[g].abs().T
        out[i] = out[i] + h @ b[g].T
        low = h.abs() * (u + gamma(a.shape[1])) + habs * gamma(x.shape[1]) * (1 + u)
        low = low + 2.0 ** -25 * h.abs().amax(1, keepdim=True) if u < 2.0 ** -9 and i.numel() else low
        tol[i] = low @ b[g].abs().T
    return out, tol + u * out.abs() + 2.0 ** -24


def backward(do, x, a, b, rows, scales=None):
    """((dx, da, db), (bounds)) in 64 bits."""
    u = U[x.dtype]
    do, x, a, b = do.double(), x.double(), a.double(), b.double()
    dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    tx, ta, tb = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
    for g, i in groups(rows, a.shape[0]):
        if i.numel() == 0:
            continue
        s = 1.0 if scales is None else float(scales[g])
        h, dh = s * x[i] @ a[g].T, s * do[i] @ b[g]
        eh = h.abs() * u + abs(s) * (x[i].abs() @ a[g].abs().T) * gamma(x.shape[1]) * (1 + u)
        ed = dh.abs() * u + abs(s) * (do[i].abs() @ b[g].abs()) * gamma(do.shape[1]) * (1 + u)
        if u < 2.0 ** -9:  # fp16: small next to the row's largest, and next to the largest row that is added up with it
            eh, ed = eh + 2.0 ** -25 * h.abs().max(), ed + 2.0 ** -25 * dh.abs().max()
        n = gamma(i.numel())
        dx[i], da[g], db[g] = dh @ a[g], dh.T @ x[i], do[i].T @ h
        tx[i] = (ed + dh.abs() * gamma(a.shape[1])) @ a[g].abs()
        ta[g] = (ed + dh.abs() * n).T @ x[i].abs()
        tb[g] = do[i].abs().T @ (eh + h.abs() * n)
    return (dx, da, db), tuple(t + u * d.abs() + 2.0 ** -24 for d, t in ((dx, tx), (da, ta), (db, tb)))


def check(got, want, tol, what=""):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    assert torch.isfinite(got).all(), what
    bad = off > tol
    assert not bad.any(), (what, int(bad.sum()), float((off / tol.clamp_min(1e-300)).max()))
