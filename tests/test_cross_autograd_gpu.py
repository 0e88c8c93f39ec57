"""What autograd may ask of the rotary embedding and of cross attention: what they have is right, what they have not is
refused, never left out without a word."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from minimax_h3_turbo_b200.h3 import cross, rope

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, FP = torch.bfloat16, torch.float16


def make(b, sq, sk, hq, hkv, d, dt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(b, s, h, d, generator=g, device=DEV).to(dt) for s, h in ((sq, hq), (sk, hkv), (sk, hkv), (sq, hq))]


@pytest.mark.parametrize("leaf", [(), (0,), (1, 2)])
def test_a_mask_that_wants_a_gradient_is_refused(leaf):
    ts = make(1, 5, 9, 2, 2, 64, BF)[:3]
    for i in leaf:
        ts[i].requires_grad_()
    mask = torch.zeros(1, 9, device=DEV, requires_grad=True)
    with pytest.raises(ValueError, match="key_mask"):
        cross.cross_attention(*ts, key_mask=mask)
    cross.cross_attention(*ts, key_mask=mask.detach())
    with torch.no_grad():
        cross.cross_attention(*ts, key_mask=mask)


@pytest.mark.parametrize("leaf", [False, True])
def test_rope_refuses_gradients_of_positions_and_frequencies(leaf):
    q = torch.randn(6, 2, 64, device=DEV, requires_grad=leaf)
    pos, inv = torch.rand(6, 1, device=DEV), torch.rand(32, device=DEV)
    for args in ((pos.clone().requires_grad_(), inv, {}), (pos, inv.clone().requires_grad_(), {}),
                 (pos, inv, {"k_positions": pos.clone().requires_grad_()})):
        with pytest.raises(ValueError, match="gradient"):
            rope.rope_axes(q, q.detach(), args[0], args[1], **args[2])
        with torch.no_grad():
            rope.rope_axes(q, q.detach(), args[0], args[1], **args[2])


def test_second_derivatives_of_attention_are_refused():
    q, k, v, do = make(1, 5, 9, 2, 2, 64, FP)
    q.requires_grad_()
    g, = torch.autograd.grad(cross.cross_attention(q, k, v), q, do, create_graph=True)  # the first ones are there
    with torch.no_grad():
        o, lse = cross.cross_attention(q, k, v, return_lse=True)
        assert torch.equal(g, cross.cross_attention_backward(do, q, k, v, o, lse)[0])
    with pytest.raises(RuntimeError, match="second"):
        (g.float().square().sum() + q.float().sum()).backward()
    # gradients of the gradient's own argument too
    w = do.clone().requires_grad_()
    g, = torch.autograd.grad(cross.cross_attention(q, k, v), q, w, create_graph=True)
    with pytest.raises(RuntimeError, match="second"):
        torch.autograd.grad(g.float().sum() + w.float().sum(), w)
    # and those that a direct call of the backward function would lose
    o, lse = cross.cross_attention(q, k, v, return_lse=True)
    dq = cross.cross_attention_backward(do, q, k, v, o, lse)[0]
    with pytest.raises(RuntimeError, match="second"):
        (dq.float().sum() + q.float().sum()).backward()


@pytest.mark.parametrize("pairing", ["half", "adjacent"])
def test_second_derivatives_of_the_rotation(pairing):
    g = torch.Generator(device=DEV).manual_seed(0)
    q, k = (torch.randn(2, s, 2, 64, generator=g, device=DEV).requires_grad_() for s in (7, 5))
    pos = [torch.randint(0, 50, (s, 2), generator=g, device=DEV) for s in (7, 5)]
    inv = torch.rand(24, generator=g, device=DEV)
    call = lambda a, b, **kw: rope.rope_axes(a, b, pos[0], inv, (12, 12), k_positions=pos[1], pairing=pairing, **kw)  # noqa: E731
    yq, yk = call(q, k)
    gq, gk = torch.autograd.grad(yq.pow(3).sum() + yk.pow(3).sum(), (q, k), create_graph=True)
    hq, hk = torch.autograd.grad(gq.pow(2).sum() + gk.pow(2).sum(), (q, k))
    # with y = R x: g = R^T 3 y^2, and the gradient of |g|^2 is R^T (6 y * R 2 g)
    with torch.no_grad():
        ref = call(*(6 * y * 2 * t for y, t in zip((yq, yk), call(gq, gk))), inverse=True)
    for have, want in zip((hq, hk), ref):
        assert torch.allclose(have, want, rtol=1e-5, atol=1e-4 * float(want.abs().max()))


def test_forward_mode_is_refused():
    q, k, v, t = make(1, 5, 9, 2, 2, 64, FP)
    pos, inv = torch.rand(5, 1, device=DEV), torch.rand(32, device=DEV)
    with fwd.dual_level():
        dual = fwd.make_dual(q, t)
        with pytest.raises(RuntimeError, match="forward-mode"):
            cross.cross_attention(dual, k, v)
        with pytest.raises(RuntimeError, match="forward-mode"):
            rope.rope_axes(dual, None, pos, inv)
        cross.cross_attention(q, k, v)  # others pass
        rope.rope_axes(q, None, pos, inv)
        with pytest.raises(RuntimeError, match="forward-mode"):
            cross.cross_attention_backward(dual, q, k, v, q, torch.zeros(1, 2, 5, device=DEV))
