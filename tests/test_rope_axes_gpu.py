"""The rotary embedding from positions against its formula in 64 bits, on GPU.

Bound: theta is exact up to fp32's roundoff of the reduced angle, so cos and sin are within 4 * 2^-24 of theirs, the two
products and the sum add 3 roundings of fp32: |err| <= u |y| + 8 * 2^-24 (|a| + |b|), u the output type's unit roundoff,
plus its smallest subnormal step."""
import pytest
import torch

from minimax_h3_turbo_b200.h3 import rope

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
UNIT = {BF: 2.0 ** -8, FP: 2.0 ** -11, F32: 2.0 ** -24}


def ref(x, pos, inv_freq, sections, pairing, inverse=False):
    """(y, bound) in 64 bits; x [B, S, H, D], pos [B or 1, S, A]."""
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=DEV)
    ang = pos.double()[..., axis] * inv_freq.double() * (-1 if inverse else 1)
    f = len(axis)
    c, s = ang.cos().unsqueeze(2), ang.sin().unsqueeze(2)
    lo, hi = (slice(0, f), slice(f, 2 * f)) if pairing == "half" else (slice(0, 2 * f, 2), slice(1, 2 * f, 2))
    y = x.double().clone()
    a, b = y[..., lo].clone(), y[..., hi].clone()
    tol = torch.zeros_like(y)
    y[..., lo], y[..., hi] = a * c - b * s, a * s + b * c
    tol[..., lo] = tol[..., hi] = 8 * 2.0 ** -24 * (a.abs() + b.abs())
    return y, tol + UNIT[x.dtype] * y.abs() + (2.0 ** -25 if x.dtype == FP else 0.0)


def check(got, x, pos, inv_freq, sections, pairing, inverse=False):
    y, tol = ref(x, pos, inv_freq, sections, pairing, inverse)
    assert got.shape == x.shape and got.dtype == x.dtype
    err = (got.double() - y).abs()
    assert (err <= tol).all(), float((err - tol).max())
    f = sum(sections)
    assert torch.equal(got[..., 2 * f:], x[..., 2 * f:])  # the channels that are not rotated are copied


def case(b, sq, sk, hq, hkv, d, axes, dt, seed=0, top=500):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = [torch.randn(b, s, h, d, generator=g, device=DEV).to(dt) for s, h in ((sq, hq), (sk, hkv))]
    pos = [torch.randint(-top, top, (b, s, axes), generator=g, device=DEV) for s in (sq, sk)]
    return x, pos


def freqs(sections):
    return torch.cat([10000.0 ** (-torch.arange(n, device=DEV) / max(1, n)) for n in sections]).float()


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
@pytest.mark.parametrize("dt", [BF, FP, F32])
@pytest.mark.parametrize("b,sq,sk,hq,hkv,d,sections", [
    (1, 1, 1, 1, 1, 2, (1,)),
    (8, 1, 1, 56, 56, 128, (16, 16, 16)),       # one token each
    (2, 301, 77, 40, 8, 128, (16, 16, 16)),     # keys of another length and head count
    (1, 130, 33, 3, 1, 128, (8, 28, 28)),       # every channel rotated
    (2, 65, 129, 4, 2, 80, (7, 2, 3, 1)),       # 13 pairs: partners off the 16-byte grid
    (1, 19, 20, 2, 2, 30, (5, 0, 6)),           # odd widths, an axis without pairs
    (3, 9, 0, 5, 5, 17, (8,)),                  # an odd channel left over, no keys
])
def test_against_the_formula(b, sq, sk, hq, hkv, d, sections, dt, pairing):
    (q, k), (pq, pk) = case(b, sq, sk, hq, hkv, d, len(sections), dt)
    inv = freqs(sections)
    for inverse in (False, True):
        yq, yk = rope.rope_axes(q, k, pq, inv, sections, k_positions=pk, pairing=pairing, inverse=inverse)
        check(yq, q, pq, inv, sections, pairing, inverse)
        check(yk, k, pk, inv, sections, pairing, inverse)


@pytest.mark.parametrize("pdt", [torch.float32, torch.int32, torch.int64])
def test_position_types_and_far_positions(pdt):
    (q, _), (pos, _) = case(2, 50, 1, 4, 1, 64, 3, F32, seed=1, top=10_000_000)
    pos = pos.to(pdt)
    inv = freqs((8, 12, 12))
    for p in (pos, pos[:1]):  # a position per entry, one for all
        y, none = rope.rope_axes(q, None, p, inv, (8, 12, 12))
        assert none is None
        check(y, q, p, inv, (8, 12, 12), "half")
    y, _ = rope.rope_axes(q, None, pos[0], inv, (8, 12, 12))  # [S, A]
    check(y, q, pos[:1], inv, (8, 12, 12), "half")


def test_shared_frequencies_are_the_tables_of_the_block():
    """sections=None: the angles of rope_angles; fractional positions too."""
    (q, _), (pos, _) = case(1, 40, 1, 2, 1, 128, 3, BF, seed=2)
    pos = pos[0].float() + 0.25
    inv = 1.0 / (10000 ** (torch.arange(16, device=DEV) / 16))
    y, _ = rope.rope_axes(q[0], None, pos, inv)
    check(y.unsqueeze(0), q, pos.unsqueeze(0), inv.repeat(3), (16, 16, 16), "half")


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_views_and_alignment(pairing):
    (q, k), (pq, pk) = case(2, 60, 44, 6, 6, 64, 2, BF, seed=3)
    sec = (11, 13)
    inv = freqs(sec)
    want = rope.rope_axes(q, k, pq, inv, sec, k_positions=pk, pairing=pairing)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k)]
    wide = [torch.randn(2, t.shape[1], 6 * 64 + 3, device=DEV).to(BF)[..., :384].unflatten(-1, (6, 64)).copy_(t) for t in (q, k)]
    swapped = [t.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1) for t in (q, k)]
    for a, b in (heads_first, odd, wide, swapped):
        got = rope.rope_axes(a, b, pq, inv, sec, k_positions=pk, pairing=pairing)
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_back_and_forth_and_gradients():
    (q, k), (pq, pk) = case(2, 70, 30, 4, 2, 128, 3, F32, seed=4)
    sec = (16, 16, 16)
    inv = freqs(sec)
    y = rope.rope_axes(q, k, pq, inv, sec, k_positions=pk)
    back = rope.rope_axes(*y, pq, inv, sec, k_positions=pk, inverse=True)
    for a, b in zip(back, (q, k)):
        assert (a - b).abs().max() <= 16 * 2.0 ** -24 * 2 * b.abs().max()
    leaves = [t.clone().requires_grad_() for t in (q, k)]
    out = rope.rope_axes(*leaves, pq, inv, sec, k_positions=pk)
    go = [torch.randn_like(t) for t in out]
    got = torch.autograd.grad(out, leaves, go)
    for g, o, p in zip(got, go, (pq, pk)):
        check(g, o, p, inv, sec, "half", inverse=True)
    # <go, R x> along a direction of q: the rotation is linear, a difference of any step is exact up to rounding
    d = torch.randn_like(q)
    f = [(ref(q.double().add(s * d.double()).float(), pq, inv, sec, "half")[0] * go[0].double()).sum() for s in (1, -1)]
    scale = (d.double().abs() * go[0].double().abs()).sum()
    assert abs((f[0] - f[1]) / 2 - (got[0].double() * d.double()).sum()) <= 1e-5 * scale
    # one of the two only
    gq, = torch.autograd.grad(rope.rope_axes(leaves[0], None, pq, inv, sec)[0], leaves[:1], go[0])
    assert torch.equal(gq, got[0])


def test_offsets_past_32_bits():
    base = torch.empty(530, 4_200_000, dtype=BF, device=DEV)
    x = base[:, :128].unflatten(1, (2, 64))
    x.copy_(torch.randn(530, 2, 64, device=DEV))
    pos = torch.arange(530, device=DEV).view(-1, 1)
    inv = freqs((32,))
    y, _ = rope.rope_axes(x, None, pos, inv, (32,))
    assert torch.equal(y, rope.rope_axes(x.contiguous(), None, pos, inv, (32,))[0])


def test_refusals():
    (q, k), (pq, pk) = case(2, 10, 12, 4, 2, 64, 3, BF)
    inv = freqs((8, 8, 8))
    ok = dict(k_positions=pk)
    for bad in (lambda: rope.rope_axes(None, None, pq, inv, (8, 8, 8)),
                lambda: rope.rope_axes(q, k, pq, inv, (8, 8, 8), pairing="thirds", **ok),
                lambda: rope.rope_axes(q, k, pq, inv, (8, 8), **ok),
                lambda: rope.rope_axes(q, k, pq, inv, (8, 8, 9), **ok),
                lambda: rope.rope_axes(q, k, pq, inv, (8, 8, 8)),              # k's length has no positions
                lambda: rope.rope_axes(q, k, pq.double(), inv, (8, 8, 8), **ok),
                lambda: rope.rope_axes(q, k, pq, freqs((12, 12, 12)), (12, 12, 12), **ok),  # 72 channels of 64
                lambda: rope.rope_axes(q, k.half(), pq, inv, (8, 8, 8), **ok),
                lambda: rope.rope_axes(q, k, pq.cpu(), inv, (8, 8, 8), **ok),
                lambda: rope.rope_axes(q, k, pq, inv.cpu(), (8, 8, 8), **ok),
                lambda: rope.rope_axes(q.double(), k.double(), pq, inv, (8, 8, 8), **ok)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        rope.rope_axes(q.cpu(), None, pq.cpu(), inv.cpu(), (8, 8, 8))
