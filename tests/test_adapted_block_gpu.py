"""The DiT block with low-rank adapters of several requests beside its linears, and with the gated residual, norm and quantiser of its
middle in one pass: the operators run together as a batch runs them."""
import pytest
import torch

import test_block_gpu as tb
from minimax_h3_turbo_b200.h3 import adapters as ad
from minimax_h3_turbo_b200.h3 import block as blk
from minimax_h3_turbo_b200.h3 import qlinear as ql
from minimax_h3_turbo_b200.h3 import residual as rs
from minimax_h3_turbo_b200.h3.synth import synthetic_w4a8

pytestmark = pytest.mark.gpu
DEV, HID, FFN, S = tb.DEV, tb.HID, tb.FFN, tb.S
INNER = tb.HEADS * tb.HD


def make_adapters(seed=0, r=16):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def one(n, k):
        return ad.Adapters((torch.randn(2, r, k, generator=g, device=DEV) * k ** -0.5).bfloat16(),
                           (torch.randn(2, n, r, generator=g, device=DEV) * 0.3 * r ** -0.5).bfloat16(),
                           torch.tensor([1.0, 0.5], device=DEV))

    rows = torch.full((S,), -1, device=DEV)
    rows[:110], rows[110:250] = 1, 0
    return rows, ad.BlockAdapters(ad.plan(rows, 2), one(3 * INNER, HID), one(HID, INNER), one(2 * FFN, HID), one(HID, FFN))


def dense_linear(rows, low):
    """The fp32 linear of the reference block with the adapters' products, by the weight it is called with."""
    def lin(t, wt, input_act=None):
        if input_act == "swiglu":
            g, u = t.chunk(2, dim=-1)
            t = torch.nn.functional.silu(g) * u
        y = t @ wt[0].t()
        for i in range(2):
            sel = rows == i
            y[sel] += float(wt[1].scales[i]) * (t[sel] @ wt[1].a[i].float().t()) @ wt[1].b[i].float().t()
        return y

    return lin


@pytest.mark.parametrize("fused", [False, True])
def test_adapted_block_matches_fp32(fused):
    """Int8 noise of about 1 % per linear, as without adapters (whose products are exact to 0.4 % of a part of the output)."""
    x, w, _, seg, cos, sin = tb.make()
    g = torch.Generator(device=DEV).manual_seed(9)
    mod = blk.Modulation(*(torch.randn(2, HID, generator=g, device=DEV) for _ in range(6)))
    rows, low = make_adapters()
    y = blk.DiTBlock(tb.HEADS, tb.HD, fuse_residual=fused)(x.clone(), w, mod, seg, cos, sin, adapters=low)
    _, wd = tb._dense_reference(w)
    wd = type(wd)(**{**wd.__dict__, **{n: (getattr(wd, n), getattr(low, n)) for n in ("qkv", "out", "fc1", "fc2")}})
    ref_block = blk.DiTBlock(tb.HEADS, tb.HD, linear=dense_linear(rows, low), ops=tb.tops.TorchOps())
    want = ref_block(x.float(), wd, mod, seg, cos.float(), sin.float())
    assert torch.isfinite(y.float()).all()
    assert tb._rel(y.float() - x.float(), want - x.float()) < 0.05
    plain = blk.DiTBlock(tb.HEADS, tb.HD, fuse_residual=fused)(x.clone(), w, mod, seg, cos, sin)
    assert tb._rel(y, plain) > 0.02  # the adapters do something


def test_one_pass_and_separate_operators_differ_by_roundings():
    """fc1 reads codes of nearly the same numbers: two 8-bit roundings of a normal row, (amax / 127) / sqrt(12) = 1 % of its
    size each at amax = 4.4, so what follows is at most sqrt(2) of that apart.  The stream itself is rounded twice on each way (after the attention and
    after the MLP): four independent errors of rms 2^-8 |x| / sqrt(3) at most, and with gates of 0.1 the stream is many times
    the update."""
    x, w, mod, seg, cos, sin = tb.make()
    a = blk.DiTBlock(tb.HEADS, tb.HD)(x.clone(), w, mod, seg, cos, sin)
    b = blk.DiTBlock(tb.HEADS, tb.HD, fuse_residual=True)(x.clone(), w, mod, seg, cos, sin)
    xf, af, bf = x.float(), a.float(), b.float()
    assert float((af - bf).norm()) < 0.03 * float((bf - xf).norm()) + 2 * 2.0 ** -8 / 3 ** 0.5 * float(bf.norm())
    with pytest.raises(ValueError, match="fuse_residual"):
        blk.DiTBlock(tb.HEADS, tb.HD, fuse_residual=True, precision="a16")


def test_adapted_linear_and_residual_linear():
    x, w, mod, seg, cos, sin = tb.make(2)
    rows, low = make_adapters(2)
    y = ad.linear(x, w.qkv, low.qkv.a, low.qkv.b, low.plan, scales=low.qkv.scales)
    want = ad.low_rank(x, low.qkv.a, low.qkv.b, low.plan, base=ql.linear(x, w.qkv), scales=low.qkv.scales)
    assert torch.equal(y, want)
    r = rs.residual_norm(x, x.flip(0).contiguous(), w.norm2, 1e-5, gate=mod.gate_a, shift=mod.shift_m, scale=mod.scale_m,
                         segments=seg, hidden=True)
    f = rs.linear(r, w.fc1)
    dense = r.hidden.float() @ ql.dequantize(w.fc1, torch.float32).t()
    assert tb._rel(f, dense) < 0.02  # one 8-bit rounding of the activations, 1 %, and bf16's
    d16 = ql.dequantize(w.fc1, torch.bfloat16)
    assert torch.equal(rs.linear(r, d16), ql.linear(r.hidden, d16))
    with pytest.raises(ValueError, match="codes"):
        rs.linear(rs.residual_norm(x, x, w.norm2, 1e-5, codes=False), w.fc1)
    with pytest.raises(ValueError, match="hidden"):
        rs.linear(rs.residual_norm(x, x, w.norm2, 1e-5), d16)
    xr = x.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient"):
        ad.linear(xr, w.qkv, low.qkv.a, low.qkv.b, low.plan)


def test_training_step_of_adapters_over_a_norm():
    """Loss -> adapters and dense projection -> norm -> stream: every leaf gets the gradient of the composed 64-bit form, up to
    the roundings of the intermediates (bf16: 2^-8 each, at most six on a path)."""
    g = torch.Generator(device=DEV).manual_seed(4)
    m, k, n = 200, 256, 384
    normal = lambda *s, std=1.0: (torch.randn(*s, generator=g, device=DEV) * std).bfloat16()  # noqa: E731
    x, y, wn, wd, gate = normal(m, k), normal(m, k), (1 + 0.1 * torch.randn(k, generator=g, device=DEV)).bfloat16(), \
        normal(n, k, std=k ** -0.5), normal(1, k)
    a, b = normal(2, 8, k, std=k ** -0.5), normal(2, n, 8, std=8 ** -0.5)
    rows = torch.randint(-1, 2, (m,), generator=g, device=DEV)
    do, dt = normal(m, n), normal(m, k)
    leaves = [t.clone().requires_grad_() for t in (x, y, wn, a, b)]
    r = rs.residual_norm(leaves[0], leaves[1], leaves[2], 1e-5, gate=gate, segments=[(0, m, 0)], codes=False, hidden=True)
    out = ad.linear(r.hidden, wd, leaves[3], leaves[4], ad.plan(rows, 2), scales=0.5)
    torch.autograd.backward([out, r.x], [do, dt])
    dd = [t.double().requires_grad_() for t in (x, y, wn, a, b)]
    t = dd[0] + dd[1] * gate.double()
    h = t * (t.square().mean(1, keepdim=True) + 1e-5).rsqrt() * dd[2]
    o = h @ wd.double().t()
    for i in range(2):
        o = o + (rows == i).double().unsqueeze(1) * 0.5 * (h @ dd[3][i].t()) @ dd[4][i].t()
    torch.autograd.backward([o, t], [do.double(), dt.double()])
    for name, got, want in zip("x y w a b".split(), leaves, dd):
        assert tb._rel(got.grad, want.grad) < 6 * 2.0 ** -8, name


@pytest.mark.parametrize("kind", [16, 64, "dense"])
def test_one_pass_with_an_fc1_that_takes_no_codes(kind):
    """An fc1 of another ConvRot block, or a dense one, reads the hidden rows of the same pass: the block still gives what the fp32 block on
    the dequantized weights gives, and the stream is not left halfway."""
    x, w, mod, seg, cos, sin = tb.make(5)
    fc1 = synthetic_w4a8(2 * FFN, HID, seed=8, device=DEV, convrot=256 if kind == "dense" else kind)
    w.fc1 = ql.dequantize(fc1, torch.bfloat16) if kind == "dense" else fc1
    rows, low = make_adapters(5)
    for adapters in (None, low):
        y = blk.DiTBlock(tb.HEADS, tb.HD, fuse_residual=True)(x.clone(), w, mod, seg, cos, sin, adapters=adapters)
        z = blk.DiTBlock(tb.HEADS, tb.HD)(x.clone(), w, mod, seg, cos, sin, adapters=adapters)
        # the bound of test_one_pass_and_separate_operators_differ_by_roundings, whose two 8-bit roundings are here too (or none)
        assert float((y.float() - z.float()).norm()) < 0.03 * float((z.float() - x.float()).norm()) + 2 * 2.0 ** -8 / 3 ** 0.5 * float(z.float().norm())
    r = rs.residual_norm(x, x, w.norm2, 1e-5, codes=False, hidden=True)
    assert torch.equal(rs.linear(r, w.fc1), ql.linear(r.hidden, w.fc1))
    with pytest.raises(ValueError, match="hidden"):
        rs.linear(rs.residual_norm(x, x, w.norm2, 1e-5), w.fc1)


def test_streams_wider_than_the_one_pass_takes_go_separately():
    wide = 16640
    g = torch.Generator(device=DEV).manual_seed(3)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    _, w, _, seg, cos, sin = tb.make(6)
    w.qkv, w.out, w.fc1, w.fc2 = normal(3 * INNER, wide) / 128, normal(wide, INNER) / 16, normal(256, wide) / 128, normal(wide, 128) / 16
    w.norm1, w.norm2 = normal(wide), normal(wide)
    x, mod = normal(S, wide), blk.Modulation(*(normal(2, wide) for _ in range(6)))
    a = blk.DiTBlock(tb.HEADS, tb.HD, fuse_residual=True)(x.clone(), w, mod, seg, cos, sin)
    assert torch.equal(a, blk.DiTBlock(tb.HEADS, tb.HD)(x.clone(), w, mod, seg, cos, sin))
