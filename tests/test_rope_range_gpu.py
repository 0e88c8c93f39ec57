"""How far the rotary embedding's angles hold their digits, on GPU.

theta = pos * inv_freq in turns, in fp64: the position (integers past 2^53), the product, 1 / (2 pi) and the product with it
are rounded, 4 * 2^-53 of theta in all; the 64-bit form here adds 2 (position and product) and its cosine's own, counted as one.
The remainder of a turn goes on in fp32, whose bound for cos and sin (8 * 2^-24 with the products) does not depend on theta:
|err| <= u |y| + (8 * 2^-24 + 7 * 2^-53 |theta|) (|a| + |b|).
"""
import pytest
import torch

from minimax_h3_turbo_b200.h3 import rope

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.mark.parametrize("top,pdt", [(2 ** 23, torch.float32), (2 ** 28, torch.float32), (2 ** 28, torch.int32),
                                     (2 ** 31 - 1, torch.int32), (2 ** 31, torch.int64), (2 ** 40, torch.int64),
                                     (2 ** 55, torch.int64)])
def test_angles_of_far_positions(top, pdt):
    g = torch.Generator(device=DEV).manual_seed(1)
    pos = torch.randint(top - top // 4, top, (64, 1), generator=g, device=DEV)
    pos[0] = top - 1
    pos = pos.to(pdt)
    inv = torch.cat([torch.ones(1, device=DEV), torch.rand(31, generator=g, device=DEV)])
    q = torch.randn(64, 2, 64, generator=g, device=DEV)
    y, _ = rope.rope_axes(q, None, pos, inv)
    theta = pos.double() * inv.double()
    c, s = theta.cos().unsqueeze(1), theta.sin().unsqueeze(1)
    a, b = q.double()[..., :32], q.double()[..., 32:]
    want = torch.cat([a * c - b * s, a * s + b * c], -1)
    reach = (8 * 2.0 ** -24 + 7 * 2.0 ** -53 * theta.abs().unsqueeze(1)) * (a.abs() + b.abs())
    assert ((y.double() - want).abs() <= torch.cat([reach, reach], -1) + 2.0 ** -24 * want.abs()).all()
