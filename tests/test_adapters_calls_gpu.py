"""Calls of the low-rank adapters and the residual's norm as programs make them around the kernels: captured plans, other devices'
sizes, gradients that a call cannot give, tensors that autograd has kept."""
import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from minimax_h3_turbo_b200.h3 import adapters as ad
    from minimax_h3_turbo_b200.h3 import residual as rs
DEV = "cuda"


def make(m=50, k=128, n=64, r=8, adapters=3, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device=DEV).bfloat16()  # noqa: E731
    return normal(m, k), normal(adapters, r, k) / k ** 0.5, normal(adapters, n, r) / r ** 0.5, normal(m, n)


def test_plan_of_segments_is_captured():
    """No copy from the host and no wait for the stream: both would end the capture with an error."""
    x, a, b, base = make()
    segments = [(5, 20, 2), (20, 33, 0), (40, 40, 1), (18, 22, 1)]  # later ones win
    rows = torch.full((50,), -1, dtype=torch.int32, device=DEV)
    rows[5:18], rows[18:22], rows[22:33] = 2, 1, 0
    want = ad.low_rank(x, a, b, ad.plan(rows, 3), base=base)
    assert torch.equal(ad.low_rank(x, a, b, ad.plan(iter(segments), 3, count=50, device=DEV), base=base), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ad.low_rank(x, a, b, ad.plan(segments, 3, count=50, device=DEV), base=base)
    out.zero_()
    graph.replay()
    assert torch.equal(out, want)
    none = ad.plan([], 3, count=50, device=DEV)
    assert torch.equal(ad.low_rank(x, a, b, none, base=base), base)


def test_plan_of_segments_does_not_wait_for_the_stream():
    done = torch.cuda.Event()
    big = torch.zeros(1 << 28, device=DEV)
    ad.plan([(0, 4, 0)], 1, count=8, device=DEV)  # the library is loaded, the memory there
    torch.cuda.synchronize()
    for _ in range(200):
        big.add_(1)  # some 60 ms
    done.record()
    p = ad.plan([(0, 4, 0)], 1, count=8, device=DEV)
    assert not done.query()
    torch.cuda.synchronize()
    assert p.rows == 8


def test_bias_beside_a_w4a8_projection_gets_its_gradient_or_an_error():
    from minimax_h3_turbo_b200.h3.synth import synthetic_w4a8

    x, a, b, _ = make(20, 256, 64, 8, 1)
    w = synthetic_w4a8(64, 256, device=DEV)
    bias = torch.zeros(64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    a.requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient for bias"):
        ad.linear(x, w, a, b, None, bias)
    dense = torch.randn(64, 256, device=DEV).bfloat16()
    ad.linear(x, dense, a, b, None, bias).sum().backward()
    assert (bias.grad == 20).all() and a.grad is not None
    with torch.no_grad():
        assert torch.equal(ad.linear(x, w, a, b, None, bias), ad.linear(x, w, a, b))


def norm_operands(m=8, k=256):
    x, _, _, y = make(m, k, k)
    return x, y, torch.ones(k, dtype=torch.bfloat16, device=DEV)


def test_out_that_autograd_has_kept():
    """A value that a backward pass still needs is overwritten: that pass raises, as behind any in-place operation of torch."""
    x, a, b, base = make()
    p = ad.plan(torch.zeros(50, dtype=torch.int32, device=DEV), 3)
    factor = torch.ones(64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    z = base * factor  # keeps base
    ad.low_rank(x, a, b, p, base=base, out=base)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    x, y, w = norm_operands()
    factor = torch.ones(256, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    z = x * factor
    with torch.no_grad():
        rs.residual_norm(x, y, w, 1e-5, out=x[:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    with torch.inference_mode():  # has no such count
        x, a, b, base = make()
        ad.low_rank(x, a, b, p, base=base, out=base)
        x, y, w = norm_operands()
        rs.residual_norm(x, y, w, 1e-5, out=x)


def test_out_that_requires_a_gradient_is_refused():
    x, a, b, base = make()
    p = ad.plan(torch.zeros(50, dtype=torch.int32, device=DEV), 3)
    leaf = torch.zeros_like(base, requires_grad=True)
    with pytest.raises(ValueError, match="out requires a gradient"):
        ad.low_rank(x, a, b, p, base=base, out=leaf)
    with torch.no_grad():
        ad.low_rank(x, a, b, p, base=base, out=leaf)
    x, y, w = norm_operands()
    leaf = torch.zeros_like(x, requires_grad=True)
    with pytest.raises(ValueError, match="out requires a gradient"):
        rs.residual_norm(x, y, w, 1e-5, out=leaf)


def test_out_over_what_every_row_reads_is_refused():
    x, y, w = norm_operands()
    mods = torch.randn(2, 256, device=DEV).bfloat16()
    kw = dict(gate=mods, shift=mods, scale=mods, segments=[(0, 8, 1)])
    flat = torch.cat([x.reshape(-1), w, mods.reshape(-1)])
    t, wf, mf = flat[:2048].view(8, 256), flat[2048:2304], flat[2304:].view(2, 256)
    want = rs.residual_norm(x, y, w, 1e-5, **kw)
    for bad in (dict(gate=t[:2]), dict(shift=t[3:5], scale=mods), dict(shift=mods, scale=t[6:])):
        with pytest.raises(ValueError, match="must not overlap"):
            rs.residual_norm(x, y, w, 1e-5, out=t, segments=[(0, 8, 1)], **bad)
    with pytest.raises(ValueError, match="must not overlap"):
        rs.residual_norm(x, y, t[2], 1e-5, out=t)
    # beside one another in one tensor, before it and behind it, and in columns of its own
    got = rs.residual_norm(t, y, wf, 1e-5, out=t, gate=mf, shift=mf, scale=mf, segments=[(0, 8, 1)])
    assert torch.equal(got.x, want.x) and torch.equal(got.codes, want.codes)
    wide = torch.zeros(8, 1024, dtype=x.dtype, device=DEV)
    wide[:, :256], wide[1, 256:512], wide[2:4, 512:768] = x, w, mods
    m2 = wide[2:4, 512:768]
    got = rs.residual_norm(wide[:, :256], y, wide[1, 256:512], 1e-5, out=wide[:, :256], gate=m2, shift=m2, scale=m2, segments=[(0, 8, 1)])
    assert torch.equal(got.x, want.x) and torch.equal(got.codes, want.codes)


def test_bias_behind_codes_gets_no_gradient_and_says_so():
    from minimax_h3_turbo_b200.h3.synth import synthetic_w4a8

    x, y, w = norm_operands()
    q = synthetic_w4a8(64, 256, device=DEV)
    bias = torch.zeros(64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    r = rs.residual_norm(x, y, w, 1e-5)
    with pytest.raises(RuntimeError, match="no gradient for bias"):
        rs.linear(r, q, bias)
    with torch.no_grad():
        assert torch.equal(rs.linear(r, q, bias), rs.linear(r, q))
