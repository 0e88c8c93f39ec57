"""Cross attention and its gradients from the formulas in 64 bits, with bounds on what a kernel may be off.

The bounds hold for any kernel that takes products of bf16/fp16 operands into fp32 sums, rounds the probabilities P and
the score gradients dS to the operands' type (unit roundoff u) for the second products, and rounds each result once:
    o   u |o| + (u + f) sum_j P |v|                   dv   u |dv| + (u + f) sum_i P |g|
    dS  E = u |dS| + P (u sum_d |g o| + f (|dP| + |delta|))    (delta = g . o may use the rounded o)
    dq  u |dq| + scale E |k|                          dk   u |dk| + scale E' |q|
f = 1e-4 covers the fp32 parts: exp2 of scores whose fp32 error is below 2^-14.  fp16 adds its smallest step times the sums
(probabilities are held relative to the row's largest, at least 2^-8 of it in scale).
"""
import math

import torch

F32 = 1e-4


def unit(dtype):
    return 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -11


def step(dtype):
    """Half the smallest subnormal step of the type."""
    return 0.0 if dtype == torch.bfloat16 else 2.0 ** -25


def key_bias(b, sk, kv_lens, key_mask, device):
    bias = torch.zeros(b, sk, dtype=torch.float64, device=device)
    if key_mask is not None:
        m = key_mask.expand(b, sk)
        bias = torch.where(m, 0.0, -math.inf).double() if m.dtype == torch.bool else m.double()
    if kv_lens is not None:
        bias = bias.masked_fill(torch.arange(sk, device=device) >= kv_lens.view(b, 1), -math.inf)
    if sk:
        top = bias.amax(1, keepdim=True)
        bias = torch.where(bias == -math.inf, bias, bias - torch.where(top == -math.inf, torch.zeros_like(top), top))
    return bias


def cross_ref(q, k, v, kv_lens=None, key_mask=None, scale=None, do=None):
    """dict of results and of bounds ("tol_" + name) for q [B, Sq, Hq, D], k, v [B, Sk, Hkv, D]."""
    b, sq, hq, d = q.shape
    sk, g = k.shape[1], hq // k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    u, st = unit(q.dtype), step(q.dtype)
    bias = key_bias(b, sk, kv_lens, key_mask, q.device).view(b, 1, 1, sk)
    out = bias == -math.inf
    qd = q.double().transpose(1, 2)
    kd, vd = (torch.where(out.view(b, 1, sk, 1), 0.0, t.double().transpose(1, 2)).repeat_interleave(g, 1) for t in (k, v))
    s = (qd @ kd.transpose(2, 3) * scale + torch.where(out, 0.0, bias)).masked_fill(out, -math.inf)
    lse = torch.logsumexp(s, -1) if sk else torch.full((b, hq, sq), -math.inf, dtype=torch.float64, device=q.device)
    p = torch.where(s == -math.inf, 0.0, torch.exp(s - torch.where(lse == -math.inf, 0.0, lse).unsqueeze(-1)))
    o = p @ vd
    r = {"o": o.transpose(1, 2), "lse": lse,
         "tol_o": (u * o.abs() + (u + F32) * (p @ vd.abs()) + st * (1 + vd.abs().sum(2, keepdim=True))).transpose(1, 2)}
    if do is None:
        return r
    gd = do.double().transpose(1, 2)
    dp, delta = gd @ vd.transpose(2, 3), (gd * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e = u * ds.abs() + p * (u * (gd * o).abs().sum(-1, keepdim=True) + F32 * (dp.abs() + delta.abs())) + st

    def keys(t):  # [B, Hq, Sk, D] -> [B, Sk, Hkv, D], shared heads added up
        return t.reshape(b, hq // g, g, sk, d).sum(2).transpose(1, 2)

    tr = lambda t: t.transpose(2, 3)  # noqa: E731
    r["dq"], r["dk"], r["dv"] = (scale * ds @ kd).transpose(1, 2), keys(scale * tr(ds) @ qd), keys(tr(p) @ gd)
    r["tol_dq"] = u * r["dq"].abs() + (scale * e @ kd.abs()).transpose(1, 2) + st
    r["tol_dk"] = u * r["dk"].abs() + keys(scale * tr(torch.where(out, 0.0, e)) @ qd.abs()) + st
    r["tol_dv"] = u * r["dv"].abs() + keys(tr(torch.where(out, 0.0, (u + F32) * p + st)) @ gd.abs()) + st
    return r
