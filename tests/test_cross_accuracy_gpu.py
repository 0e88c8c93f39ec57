"""Cross attention on GPU: digits and bits that depend on the operands' size, on what ran before, and on the exp2 in use."""
import math

import pytest
import torch

from cross_ref import cross_ref
from minimax_h3_turbo_b200.h3 import cross

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, FP = torch.bfloat16, torch.float16


def make(b, sq, sk, hq, hkv, d, dt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(b, s, h, d, generator=g, device=DEV).to(dt) for s, h in ((sq, hq), (sk, hkv), (sk, hkv), (sq, hq))]


@pytest.mark.parametrize("d,dt", [(64, BF), (128, FP)])
@pytest.mark.parametrize("g", [3, 5, 7])
def test_same_bits_whatever_ran_before(g, d, dt):
    """Head groups that do not divide 128 leave rows of a query tile unwritten: what they hold must not reach other rows."""
    q, k, v, do = make(1, 3 * (128 // g), 400, 2 * g, 2, d, dt, seed=g)
    before = make(1, 128 * 148 * 2, 128, 1, 1, d, dt, seed=50)
    results = []
    for size in (0.0, 0.1, 30.0):  # of the scores that were in every SM's shared memory
        cross.cross_attention(before[0] * size, *before[1:3])
        o, lse = cross.cross_attention(q, k, v, return_lse=True)
        cross.cross_attention_backward(before[3] * size, before[0] * size, *before[1:3],
                                       *cross.cross_attention(before[0] * size, *before[1:3], return_lse=True))
        results.append((o, lse, *cross.cross_attention_backward(do, q, k, v, o, lse)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def norm_error(got, want):
    """Relative error over the whole tensor, and that of the exact result rounded to the same type."""
    top = want.norm()
    return float((got.double() - want).norm() / top), float((want.to(got.dtype).double() - want).norm() / top)


# fp16 gradients hold their digits whatever the size of the output's gradient.  P, dS and the o that delta is taken from are
# rounded to 11 bits: each at most 2^-11 of a term, 2^-11 / sqrt(3) = 2.8e-4 root mean square, three of them 5e-4 of the
# result; twice that is asked, beside the rounding of the result itself (which has few digits where it is small).
FP16_LIMIT = 1e-3


@pytest.mark.parametrize("mask", [False, True])
@pytest.mark.parametrize("std", [1.0, 1e-2, 1e-3])
@pytest.mark.parametrize("sq,sk,hq,hkv,d", [(64, 12090, 2, 1, 64), (300, 12090, 1, 1, 128), (17, 57840, 3, 1, 64),
                                            (500, 100, 2, 2, 64)])
def test_small_fp16_gradients_keep_their_digits(sq, sk, hq, hkv, d, std, mask):
    q, k, v, do = make(1, sq, sk, hq, hkv, d, FP, seed=sk)
    do = (do.float() * std).half()
    kw = {"key_mask": torch.zeros(1, sk, device=DEV)} if mask else {}
    r = cross_ref(q, k, v, do=do, **kw)
    o, lse = cross.cross_attention(q, k, v, return_lse=True, **kw)
    for name, got in zip(("dq", "dk", "dv"), cross.cross_attention_backward(do, q, k, v, o, lse, **kw)):
        err, own = norm_error(got, r[name])
        assert err <= own + FP16_LIMIT, (name, err, own)


def test_fp16_rows_of_different_size():
    """Every query's dq has its own digits, next to rows whose gradients are a thousand times larger."""
    q, k, v, do = make(1, 256, 12090, 1, 1, 64, FP, seed=1)
    do[:, ::2] = (do[:, ::2].float() * 1e-3).half()
    r = cross_ref(q, k, v, do=do)
    o, lse = cross.cross_attention(q, k, v, return_lse=True)
    dq = cross.cross_attention_backward(do, q, k, v, o, lse)[0]
    for rows in (slice(0, None, 2), slice(1, None, 2)):
        err, own = norm_error(dq[:, rows], r["dq"][:, rows])
        assert err <= own + FP16_LIMIT, (rows, err, own)


@pytest.mark.parametrize("sk", [3, 200])
def test_large_fp16_gradients_do_not_overflow_inside(sk):
    """dS is past fp16's range, every result is not."""
    q, k, v, do = make(1, 16, sk, 2, 2, 64, FP, seed=2)
    q, k, v, do = q * 0.05, k * 0.05, v * 4, (do.float() * 8000).half()
    m = torch.full((1, sk), -40.0, device=DEV)
    m[:, :3] = 0
    r = cross_ref(q, k, v, do=do, key_mask=m)
    assert all(float(r[n].abs().max()) < 60000 for n in ("dq", "dk", "dv"))
    o, lse = cross.cross_attention(q, k, v, return_lse=True, key_mask=m)
    for name, got in zip(("dq", "dk", "dv"), cross.cross_attention_backward(do, q, k, v, o, lse, key_mask=m)):
        err, own = norm_error(got, r[name])
        assert err <= own + FP16_LIMIT, (name, err, own)


def test_fp16_gradients_do_not_see_what_masked_values_hold():
    """Large finite values in keys that are left out: the same bits as with zeros there."""
    q, k, v, do = make(2, 40, 300, 4, 2, 64, FP, seed=3)
    mask = torch.rand(2, 300, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.7
    lens = torch.tensor([250, 120], device=DEV)
    out = (~mask | (torch.arange(300, device=DEV) >= lens.view(2, 1))).view(2, 300, 1, 1)
    res = []
    for junk in (0.0, 6e4):
        kj, vj = k.masked_fill(out, junk), v.masked_fill(out, junk)
        o, lse = cross.cross_attention(q, kj, vj, key_mask=mask, kv_lens=lens, return_lse=True)
        res.append((o, lse, *cross.cross_attention_backward(do, q, kj, vj, o, lse, key_mask=mask, kv_lens=lens)))
    assert all(torch.equal(a, b) for a, b in zip(*res))


@pytest.mark.parametrize("residue", range(8))
def test_exponentials(residue):
    """The forward pass's exp2 by both units it is taken from (special functions, and a polynomial on the FMA pipe), by the key's place:
    rows whose keys in one residue class mod 8 all score a, the others 60 below: lse = a + log(keys of the class).  lse is
    from sums of unrounded probabilities.  The first tile is taken with maximum 0 where scores are between 0 and 8 (in log2).
    Bounds: 2.7e-6 for the polynomial, 2^-22 for the special function unit, 2^-24 for each of the 16 additions of a thread's
    sum, the score's product, and the log and its two products (4 roundings of a number below 8)."""
    n, d = 2000, 64
    a = (torch.arange(n, device=DEV) * (5.5 / n)).half()  # up to 7.9 in log2
    q = torch.zeros(1, n, 1, d, device=DEV, dtype=FP)
    q[0, :, 0, 0], q[0, :, 0, 1] = a, 1
    for sk in (128, 512):
        k = torch.zeros(1, sk, 1, d, device=DEV, dtype=FP)
        k[0, :, 0, 0] = 1
        k[0, torch.arange(sk, device=DEV) % 8 != residue, 0, 1] = -60
        _, lse = cross.cross_attention(q, k, torch.ones_like(k), scale=1.0, return_lse=True)
        err = (lse[0, 0].double() - a.double() - math.log(sk // 8)).abs().max()
        assert float(err) <= 2.7e-6 + 2.0 ** -22 + 2.0 ** -24 * (16 + 8 + 4 * 16), float(err)


@pytest.mark.parametrize("d,dt", [(64, BF), (128, FP), (128, BF), (64, FP)])
@pytest.mark.parametrize("g,sk,masked", [(3, 100, False), (5, 128, False), (7, 1, False), (7, 90, True)])
def test_few_keys_whatever_ran_before(g, sk, masked, d, dt):
    """All keys in one tile (delta comes from P and dP there), head groups that do not divide 128, numbers that are none left in
    every SM's shared memory: they must not reach any result."""
    q, k, v, do = make(2, 3 * (128 // g) + 1, sk, 2 * g, 2, d, dt, seed=g + sk)
    kw = {"key_mask": torch.arange(sk, device=DEV).view(1, -1) % 3 > 0} if masked else {}
    before = make(1, 128 * 148 * 2, 128, 1, 1, d, dt, seed=51)
    r = cross_ref(q, k, v, do=do, **kw)
    results = []
    for junk in (0.0, float("nan")):
        stale = [t * junk for t in before[:1] + before[3:]]
        cross.cross_attention(stale[0], *before[1:3])
        o, lse = cross.cross_attention(q, k, v, return_lse=True, **kw)
        ob, lb = cross.cross_attention(before[0], *before[1:3], return_lse=True)
        cross.cross_attention_backward(stale[1], stale[0], *before[1:3], ob, lb)
        results.append((o, *cross.cross_attention_backward(do, q, k, v, o, lse, **kw)))
    for name, a, b in zip(("o", "dq", "dk", "dv"), *results):
        assert ((b.double() - r[name]).abs() <= r["tol_" + name]).all(), name
        assert torch.equal(a, b), name
