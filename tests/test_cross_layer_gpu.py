"""The cross-attention layer: with W4A8 linears the same bits as its operators called one by one; with dense linears within
bf16 rounding of the layer in 64 bits.

The bound: a bf16 rounding has a relative error of about 1.1e-3 (root mean square).  h, q and the turned q (three), k and the
turned k (two) put 2.5e-3 of their size on the scores, whose spread is below 3 here: 7e-3 on the probabilities and so on the
attention output; v, P, o and the last linear add one each.  Together 8e-3 of the update's norm; three times that is asked."""
import math

import pytest
import torch

from minimax_h3_turbo_b200.h3 import block as blk
from minimax_h3_turbo_b200.h3 import cross
from minimax_h3_turbo_b200.h3 import qlinear as ql
from minimax_h3_turbo_b200.h3 import rope
from minimax_h3_turbo_b200.h3.synth import synthetic_activation, synthetic_w4a8

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
HID, CTX, HEADS, KVH, HD = 512, 256, 4, 2, 128


def weights(dense=False):
    g = torch.Generator(device=DEV).manual_seed(1)
    shapes = {"q": (HEADS * HD, HID), "kv": (2 * KVH * HD, CTX), "out": (HID, HEADS * HD)}
    if dense:
        w = {n: (torch.randn(s, generator=g, device=DEV) / math.sqrt(s[1])).bfloat16() for n, s in shapes.items()}
    else:
        w = {n: synthetic_w4a8(*s, seed=i, device=DEV) for i, (n, s) in enumerate(shapes.items())}
    return cross.CrossWeights(**w, norm=(1 + 0.1 * torch.randn(HID, generator=g, device=DEV)).bfloat16())


def case(s, sk, masked):
    g = torch.Generator(device=DEV).manual_seed(0)
    x, ctx = torch.randn(s, HID, generator=g, device=DEV).bfloat16(), torch.randn(sk, CTX, generator=g, device=DEV).bfloat16()
    mod = [torch.randn(2, HID, generator=g, device=DEV).bfloat16() for _ in range(3)]
    pos, kpos = blk.video_audio_positions(5, 6, 9, s - 270, DEV), torch.arange(sk, device=DEV).float().view(-1, 1).expand(sk, 3)
    inv = 1.0 / (10000 ** (torch.arange(16, device=DEV) / 16))
    mask = torch.rand(1, sk, generator=g, device=DEV) < 0.7 if masked else None
    return x, ctx, mod, [(0, 270, 0), (270, s, 1)], pos, kpos, inv, mask


def turned(x, pos, inv):
    """The rotation by the tables of the block (all frequencies per axis), fp32."""
    ang = rope.rope_angles(pos, inv, DEV).unsqueeze(1)
    f = ang.shape[-1]
    a, b = x[..., :f], x[..., f:2 * f]
    return torch.cat([a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos(), x[..., 2 * f:]], -1)


@pytest.mark.parametrize("masked", [False, True])
def test_same_bits_as_its_operators(masked):
    s, sk = 300, 77
    x, ctx, (shift, scale, gate), seg, pos, kpos, inv, mask = case(s, sk, masked)
    w = weights()
    layer = cross.CrossLayer(HEADS, HD, KVH)
    kv = layer.keys_values(ctx, w, kpos, inv)
    y = layer(x.clone(), w, kv, shift, scale, gate, seg, pos, inv, key_mask=mask)
    assert torch.equal(y, layer(x.clone(), w, kv, shift, scale, gate, seg, pos, inv, key_mask=mask))  # many steps, one pair
    q = ql.linear(blk.rms_modulate(x, w.norm, 1e-5, shift, scale, seg), w.q).view(s, HEADS, HD)
    k, v = (t.reshape(sk, KVH, HD) for t in ql.linear(ctx, w.kv).split(KVH * HD, -1))
    q, k = rope.rope_axes(q, k, pos, inv, k_positions=kpos)
    o = cross.cross_attention(q, k, v, key_mask=mask)
    assert torch.equal(y, blk.gate_(x.clone(), gate, ql.linear(o.view(s, -1), w.out), seg))


@pytest.mark.parametrize("masked", [False, True])
def test_against_64_bits(masked):
    s, sk = 300, 77
    x, ctx, (shift, scale, gate), seg, pos, kpos, inv, mask = case(s, sk, masked)
    w = weights(dense=True)
    layer = cross.CrossLayer(HEADS, HD, KVH)
    y = layer(x.clone(), w, layer.keys_values(ctx, w, kpos, inv), shift, scale, gate, seg, pos, inv, key_mask=mask)
    xd, rows = x.double(), torch.tensor([0] * 270 + [1] * (s - 270), device=DEV)
    h = xd * torch.rsqrt(xd.square().mean(-1, keepdim=True) + 1e-5) * w.norm.double()
    h = h * (1 + scale.double()[rows]) + shift.double()[rows]
    q = turned((h @ w.q.double().t()).view(s, HEADS, HD), pos, inv)
    k, v = ((ctx.double() @ w.kv.double().t()).split(KVH * HD, -1))
    k, v = (t.reshape(sk, KVH, HD).repeat_interleave(HEADS // KVH, 1) for t in (k, v))
    a = torch.einsum("qhd,khd->hqk", q, turned(k, kpos, inv)) / math.sqrt(HD)
    assert float(a.std()) < 3
    if masked:
        a = a.masked_fill(~mask.view(1, 1, sk), -math.inf)
    o = torch.einsum("hqk,khd->qhd", a.softmax(-1), v).reshape(s, -1)
    update = (o @ w.out.double().t()) * gate.double()[rows]
    # the residual's own rounding (x + update to bf16) is not the layer's: compare with it added
    rel = float((y.double() - xd - update).norm() / update.norm())
    assert rel < 2.4e-2 + 2.0 ** -9 * float((xd + update).norm() / update.norm()), rel


def test_no_positions_and_refusals():
    w = weights()
    x, ctx = synthetic_activation(64, HID, seed=1, device=DEV), synthetic_activation(9, CTX, seed=2, device=DEV)
    layer = cross.CrossLayer(HEADS, HD, KVH)
    zero = torch.zeros(1, HID, device=DEV, dtype=torch.bfloat16)
    y = layer(x.clone(), w, layer.keys_values(ctx, w), zero, zero, zero, [(0, 64, 0)])
    assert torch.equal(y, x)  # a gate of zero
    with pytest.raises(ValueError):
        cross.CrossLayer(4, 128, 3)
    with pytest.raises(ValueError):
        layer.keys_values(synthetic_activation(9, HID, seed=2, device=DEV), w)
