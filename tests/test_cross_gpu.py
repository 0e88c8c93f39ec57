"""Cross attention and its gradients against the formulas in 64 bits (helpers/cross_ref.py derives the bounds), on GPU."""
import math

import pytest
import torch

from cross_ref import cross_ref
from minimax_h3_turbo_b200 import _lib
from minimax_h3_turbo_b200.h3 import cross

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, FP = torch.bfloat16, torch.float16


def make(b, sq, sk, hq, hkv, d, dt, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    rnd = lambda s, h: (torch.randn(b, s, h, d, generator=g, device=DEV) * std).to(dt)  # noqa: E731
    return rnd(sq, hq), rnd(sk, hkv), rnd(sk, hkv), rnd(sq, hq)


def mask_of(kind, b, sk, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 100)
    if kind == "lens":  # a full entry, then shorter ones, an empty one last
        lens = [sk] + [(sk * (b - i)) // b for i in range(1, b)]
        lens[-1] = 0 if b > 1 else max(0, sk - 3)
        return {"kv_lens": torch.tensor(lens, dtype=torch.int32, device=DEV)}
    if kind == "bool":
        m = torch.rand(b, sk, generator=g, device=DEV) < 0.6
        m[-1] = b == 1
        return {"key_mask": m}
    if kind == "bias":
        w = torch.randn(b, sk, generator=g, device=DEV) * 2
        return {"key_mask": torch.where(torch.rand(b, sk, generator=g, device=DEV) < 0.8, w, torch.full_like(w, -math.inf))}
    if kind == "both":
        return {**mask_of("lens", b, sk, seed), "key_mask": torch.rand(1, sk, generator=g, device=DEV) < 0.5}
    return {}


def check(name, got, r):
    want, tol = r[name], r["tol_" + name]
    assert got.shape == want.shape
    bad = ((got.double() - want).abs() > tol) | ~torch.isfinite(got)
    assert not bad.any(), (name, int(bad.sum()), float(((got.double() - want).abs() - tol).max()))


def check_all(q, k, v, do, scale=None, **kw):
    r = cross_ref(q, k, v, do=do, scale=scale, **kw)
    o, lse = cross.cross_attention(q, k, v, return_lse=True, scale=scale, **kw)
    check("o", o, r)
    empty = r["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert torch.allclose(lse[~empty].double(), r["lse"][~empty], rtol=2e-6, atol=1e-4)
    assert not o.transpose(1, 2)[empty].any()
    for name, got in zip(("dq", "dk", "dv"), cross.cross_attention_backward(do, q, k, v, o, lse, scale=scale, **kw)):
        check(name, got, r)
    return o, lse


@pytest.mark.parametrize("kind", ["none", "lens", "bool", "bias", "both"])
@pytest.mark.parametrize("b,sq,sk,hq,hkv,d,dt", [
    (1, 1, 1, 1, 1, 8, BF),        # one token, one key
    (2, 1, 77, 4, 4, 128, BF),     # single queries
    (3, 5, 1000, 14, 2, 128, BF),  # a few queries, seven heads to a key head, a long stream
    (1, 127, 129, 3, 3, 64, FP),   # one under and one over a tile
    (2, 128, 128, 2, 2, 128, FP),
    (2, 129, 127, 2, 1, 128, BF),
    (3, 300, 257, 6, 2, 64, BF),
    (2, 70, 640, 5, 1, 72, BF),    # five heads to a key head: 25 queries fill 125 rows of a tile
    (2, 33, 130, 12, 12, 40, FP),
    (1, 513, 65, 8, 1, 96, BF),
    (1, 3, 200, 128, 1, 16, FP),   # 128 heads to a key head: one query fills a tile
    (1, 1031, 333, 12, 4, 64, FP),
])
def test_against_the_formulas(b, sq, sk, hq, hkv, d, dt, kind):
    q, k, v, do = make(b, sq, sk, hq, hkv, d, dt, seed=sq + sk)
    check_all(q, k, v, do, **mask_of(kind, b, sk))


def test_many_queries_over_few_keys_and_a_long_stream():
    q, k, v, do = make(1, 5000, 200, 4, 4, 128, BF, seed=3)
    check_all(q, k, v, do)
    q, k, v, do = make(1, 4, 20011, 4, 2, 128, BF, seed=4)
    check_all(q, k, v, do)
    check_all(q, k, v, do, kv_lens=torch.tensor([12345], device=DEV))


@pytest.mark.parametrize("lens", [[9000, 5000, 300, 0, 1], [0, 0, 129], [128], [700], [9000], [0], [50] * 39 + [4000]])
@pytest.mark.parametrize("sq,hq,hkv,d,dt", [(1, 4, 4, 128, BF), (5, 14, 2, 64, FP), (70, 5, 1, 72, BF)])
def test_few_queries_over_ragged_lengths(lens, sq, hq, hkv, d, dt):
    b = len(lens)
    q, k, v, do = make(b, sq, 9000 if b < 40 else 4000, hq, hkv, d, dt, seed=b + sq)
    kv = torch.tensor(lens, device=DEV)
    check_all(q, k, v, do, kv_lens=kv)
    check_all(q, k, v, do, key_mask=torch.arange(k.shape[1], device=DEV) < kv.view(b, 1))


@pytest.mark.parametrize("d,dt", [(128, BF), (64, FP)])
@pytest.mark.parametrize("kind", ["none", "lens", "bias"])
def test_more_work_than_ctas(d, dt, kind):
    """Every CTA walks several pairs of query tiles, the last pair of a head is half empty, entries differ in length."""
    q, k, v, do = make(3, 1400, 300, 20, 20, d, dt, seed=13)
    check_all(q, k, v, do, **mask_of(kind, 3, 300))
    q, k, v, do = make(4, 1290, 129, 12, 6, d, dt, seed=14)
    check_all(q, k, v, do, **mask_of(kind, 4, 129))


def test_large_scores_and_own_scale():
    for std, scale in ((6.0, None), (1.0, 0.7), (0.02, None)):  # nearly one-hot rows, an explicit scale, nearly flat rows
        q, k, v, do = make(2, 260, 390, 3, 3, 128, BF, seed=9, std=std)
        check_all(q, k, v, do, scale=scale)
    # the largest score of a row comes late and far above the ones before
    q, k, v, do = make(1, 256, 700, 2, 2, 64, BF, seed=10)
    k = torch.cat([k[:, :600] * 0.1, k[:, 600:] * 8], 1)
    check_all(q, k, v, do)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("shift", [-40.0, -2.0, 2.0, 40.0])
def test_scores_far_from_zero(shift, dt):
    """Every score of a row moved by the same amount, up or down; then only those of the first or of the later keys."""
    for keys in (slice(None), slice(0, 128), slice(128, None), slice(64, 128)):
        q, k, v, do = make(1, 300, 400, 3, 3, 64, dt, seed=21)
        q[..., 0], k[..., 0] = 1, 0
        k[:, keys, :, 0] = shift * 8  # scale 1/8
        check_all(q, k, v, do)


@pytest.mark.parametrize("sq", [3, 300])
def test_masked_keys_may_hold_anything(sq):
    q, k, v, do = make(2, sq, 300, 4, 2, 64, BF, seed=5)
    lens = torch.tensor([300 - 37, 140], dtype=torch.int32, device=DEV)
    mask = torch.rand(2, 300, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV) < 0.7
    out = ~mask | (torch.arange(300, device=DEV) >= lens.view(2, 1))
    clean = check_all(q, k, v, do, kv_lens=lens, key_mask=mask)
    grads = cross.cross_attention_backward(do, q, k, v, *clean, kv_lens=lens, key_mask=mask)
    for junk in (math.nan, math.inf, -math.inf):
        kj, vj = (t.masked_fill(out.view(2, 300, 1, 1), junk) for t in (k, v))
        o, lse = cross.cross_attention(q, kj, vj, kv_lens=lens, key_mask=mask, return_lse=True)
        assert torch.equal(o, clean[0]) and torch.equal(lse, clean[1])
        again = cross.cross_attention_backward(do, q, kj, vj, o, lse, kv_lens=lens, key_mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(again, grads))
        assert not again[1][out].any() and not again[2][out].any()


def test_additive_masks_of_large_negative_values():
    q, k, v, do = make(2, 40, 200, 2, 2, 64, BF, seed=6)
    for low in (-1e4, -1e9, torch.finfo(torch.float32).min, -math.inf):
        m = torch.zeros(2, 200, device=DEV)
        m[0, 150:] = low
        m[1] = low  # every key of the second entry carries the value: taken off, it weighs nothing (unless -inf)
        check_all(q, k, v, do, key_mask=m)
    m = torch.zeros(2, 200, device=DEV, dtype=BF)
    m[:, 77:] = torch.finfo(BF).min
    a = cross.cross_attention(q, k, v, key_mask=m)
    assert torch.equal(a, cross.cross_attention(q, k[:, :77].contiguous(), v[:, :77].contiguous())) or \
        torch.allclose(a.float(), cross.cross_attention(q, k[:, :77], v[:, :77]).float(), rtol=2 ** -7, atol=2 ** -9)


def test_empty_lengths():
    q, k, v, do = make(2, 9, 0, 4, 2, 64, BF)
    o, lse = check_all(q, k, v, do)
    assert not o.any() and (lse == -math.inf).all()
    q, k, v, do = make(2, 0, 9, 4, 2, 64, BF)
    o, lse = cross.cross_attention(q, k, v, return_lse=True)
    dq, dk, dv = cross.cross_attention_backward(do, q, k, v, o, lse)
    assert o.shape == q.shape and dq.shape == q.shape and not dk.any() and not dv.any()
    q, k, v, _ = make(0, 5, 9, 4, 2, 64, BF)
    assert cross.cross_attention(q, k, v).shape == q.shape
    # lengths outside 0 .. Sk are taken as the nearest of them
    q, k, v, do = make(2, 9, 30, 4, 2, 64, BF)
    a = cross.cross_attention(q, k, v, kv_lens=torch.tensor([-3, 99], device=DEV))
    assert torch.equal(a, cross.cross_attention(q, k, v, kv_lens=torch.tensor([0, 30], device=DEV)))


def test_views_orders_and_alignment():
    b, sq, sk, h, d = 2, 150, 210, 4, 64
    q, k, v, do = make(b, sq, sk, h, h, d, BF, seed=7)
    want, lse = cross.cross_attention(q, k, v, return_lse=True)
    grads = cross.cross_attention_backward(do, q, k, v, want, lse)

    def same(qq, kk, vv, dd):
        o, l2 = cross.cross_attention(qq, kk, vv, return_lse=True)
        assert torch.equal(o, want) and torch.equal(l2, lse)
        assert all(torch.equal(x, y) for x, y in zip(cross.cross_attention_backward(dd, qq, kk, vv, o, l2), grads))

    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do)]
    same(*heads_first)
    kv = torch.cat([k.reshape(b, sk, h * d), v.reshape(b, sk, h * d)], -1)  # one projection's output, split
    kk, vv = (t.view(b, sk, h, d) for t in kv.split(h * d, -1))
    same(q, kk, vv, do)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t) for t in (q, k, v, do)]
    same(*odd)  # 2-byte aligned
    swapped = [t.permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1) for t in (q, k, v, do)]
    same(*swapped)  # channels not contiguous
    out = torch.empty(b, h, sq, d, dtype=BF, device=DEV).transpose(1, 2)
    assert cross.cross_attention(q, k, v, out=out) is out and torch.equal(out, want)
    # no batch dimension; keys shared by the whole batch (stride 0)
    o1 = cross.cross_attention(q[0], k[0], v[0])
    assert o1.shape == (sq, h, d) and torch.equal(o1, want[0])
    assert torch.equal(cross.cross_attention(q, k[:1].expand(b, -1, -1, -1), v[:1].expand(b, -1, -1, -1))[0], want[0])


def test_strides_of_extents_of_one():
    """Views with one query, one key, one head or one entry: whatever the stride of that extent is, it is not used."""
    base = torch.randn(3, 5, 7, 72, device=DEV, dtype=BF)[..., :64]
    one_q, one_h = base.as_strided((3, 1, 7, 64), (2520, 3, 72, 1)), base.as_strided((3, 5, 1, 64), (2520, 504, 5, 1))
    one_b = base.as_strided((1, 5, 7, 64), (9, 504, 72, 1))
    check_all(one_q, base, base, torch.randn_like(one_q))
    check_all(base, one_q, one_q, torch.randn_like(base))
    check_all(base, one_h, one_h, torch.randn_like(base))
    check_all(one_b, one_b, one_b, torch.randn_like(one_b))


def test_offsets_past_32_bits():
    sk, d = 520, 128
    base = torch.empty(sk, 4_200_000, dtype=BF, device=DEV)  # rows 8.4 MB apart: the last starts past 2^31 elements
    q, k, v, do = make(1, 20, sk, 1, 1, d, BF, seed=8)
    kk, vv = base[:, :d].unflatten(1, (1, d)).unsqueeze(0), base[:, 2048:2048 + d].unflatten(1, (1, d)).unsqueeze(0)
    kk.copy_(k), vv.copy_(v)
    assert kk.stride(1) * (sk - 1) > 2 ** 31
    o, lse = cross.cross_attention(q, kk, vv, return_lse=True)
    w, wl = cross.cross_attention(q, k, v, return_lse=True)
    assert torch.equal(o, w) and torch.equal(lse, wl)
    assert all(torch.equal(a, b) for a, b in zip(cross.cross_attention_backward(do, q, kk, vv, o, lse),
                                                 cross.cross_attention_backward(do, q, k, v, w, wl)))


def test_same_bits_on_another_stream_and_in_a_graph():
    q, k, v, do = make(2, 300, 500, 4, 2, 128, BF, seed=11)
    kw = mask_of("bool", 2, 500)
    o, lse = cross.cross_attention(q, k, v, return_lse=True, **kw)
    grads = cross.cross_attention_backward(do, q, k, v, o, lse, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, l2 = cross.cross_attention(q, k, v, return_lse=True, **kw)
        g2 = cross.cross_attention_backward(do, q, k, v, o2, l2, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2) and torch.equal(lse, l2) and all(torch.equal(a, b) for a, b in zip(grads, g2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o3, l3 = cross.cross_attention(q, k, v, return_lse=True, **kw)
        g3 = cross.cross_attention_backward(do, q, k, v, o3, l3, **kw)
    graph.replay()
    assert torch.equal(o, o3) and torch.equal(lse, l3) and all(torch.equal(a, b) for a, b in zip(grads, g3))


def test_autograd_and_differences():
    q, k, v, do = make(2, 37, 150, 4, 2, 64, FP, seed=12)
    kw = mask_of("bias", 2, 150)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    o, lse = cross.cross_attention(*leaves, return_lse=True, **kw)
    got = torch.autograd.grad(o, leaves, do)
    want = cross.cross_attention_backward(do, q, k, v, o.detach(), lse, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # the loss <do, o> along a direction of each input: central differences of the formula in 64 bits
    r = cross_ref(q, k, v, do=do, **kw)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(want[i].shape, generator=torch.Generator(device=DEV).manual_seed(i), device=DEV, dtype=torch.float64)
        h = 1e-5
        f = []
        for sgn in (1, -1):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + sgn * h * d
            f.append(float((cross_ref(*x, **kw)["o"] * do.double()).sum()))
        diff = (f[0] - f[1]) / (2 * h)
        have = float((want[i].double() * d).sum())
        assert abs(have - diff) <= float((r["tol_" + name] * d.abs()).sum()) + 1e-5 * abs(diff)


def test_refusals():
    q, k, v, do = make(2, 9, 30, 4, 2, 64, BF)
    with pytest.raises(RuntimeError):
        cross.cross_attention(q.float(), k.float(), v.float())
    with pytest.raises(RuntimeError):
        cross.cross_attention(q, k.half(), v)
    with pytest.raises(RuntimeError):
        cross.cross_attention(q.cpu(), k.cpu(), v.cpu())
    for bad in (dict(kv_lens=torch.ones(3, dtype=torch.int32, device=DEV)), dict(kv_lens=torch.ones(2, device=DEV)),
                dict(key_mask=torch.ones(2, 29, dtype=torch.bool, device=DEV)), dict(scale=0.0), dict(scale=-1.0),
                dict(key_mask=torch.ones(2, 30, dtype=torch.int32, device=DEV)), dict(scale=math.nan),
                dict(key_mask=torch.ones(2, 30, dtype=torch.bool)),
                dict(out=torch.empty(2, 9, 4, 63, dtype=BF, device=DEV))):
        with pytest.raises(ValueError):
            cross.cross_attention(q, k, v, **bad)
    with pytest.raises(ValueError):
        cross.cross_attention(q[:, :, :3], k, v)  # 3 query heads over 2 key heads
    with pytest.raises(ValueError):
        cross.cross_attention(q, k, v[:, :20])
    with pytest.raises(ValueError):
        cross.cross_attention(q[..., :60].contiguous(), k[..., :60].contiguous(), v[..., :60].contiguous())  # 60 channels
    big = torch.zeros(1, 2, 1, 136, dtype=BF, device=DEV)
    with pytest.raises(ValueError):
        cross.cross_attention(big, big, big)
    o, lse = cross.cross_attention(q, k, v, return_lse=True)
    with pytest.raises(ValueError):
        cross.cross_attention_backward(do, q, k, v, o, lse.half())
    with pytest.raises(ValueError):
        cross.cross_attention_backward(do[:, :8], q, k, v, o, lse)
    assert _lib.lib().h3b_device_error(0) == 0
