"""The residual's addition with its norm and 8-bit output against the 64-bit form (helpers/residual_ref.py), its gradients."""
import math

import pytest
import torch

import residual_ref as ref

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from minimax_h3_turbo_b200.h3 import residual as rs
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]
EPS = 1e-5


def make(m, k, mods, dtype, seed=0, w_dtype=None, m_dtype=None):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0, dt=dtype):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dt)

    w = (1 + 0.1 * torch.randn(k, generator=g, device=DEV)).to(w_dtype or dtype)
    md = m_dtype or dtype
    mod = [normal(mods, k, std=s, dt=md) if mods else None for s in (0.5, 0.2, 0.2)]
    return normal(m, k), normal(m, k), w, *mod


def dealt(kind, m, mods):
    """(segments, modulation row of each token)."""
    rows = torch.full((m,), -1, dtype=torch.long, device=DEV)
    if mods == 0 or kind == "none":
        return [], rows
    if kind == "tokens":
        rows = torch.randint(-1, mods, (m,), device=DEV, generator=torch.Generator(device=DEV).manual_seed(9))
        return [(0, m, rows)], rows
    n = 20 if kind == "many" else mods
    cuts = [m * i // (n + 1) for i in range(n + 1)]
    segs = [(a, b, i % mods) for i, (a, b) in enumerate(zip(cuts, cuts[1:]))]
    for a, b, r in segs:
        rows[a:b] = r
    return segs, rows


CASES = [(1, 256, 1, "runs"), (2, 512, 0, "none"), (7, 5120, 2, "runs"), (8, 5376, 3, "tokens"), (33, 1280, 4, "many"),
         (65, 16384, 2, "runs"), (130, 8448, 1, "tokens"), (257, 768, 2, "none"), (1031, 1280, 3, "runs"), (5000, 256, 2, "runs"),
         (3, 14336, 0, "none"), (2100, 2560, 2, "tokens"), (70, 6144, 2, "runs"), (39, 8192, 2, "tokens"), (150, 4096, 3, "runs"),
         (41, 8704, 2, "runs"), (29, 11264, 3, "many"), (150, 14080, 2, "runs"), (2, 7936, 0, "none")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,mods,kind", CASES)
def test_forward(m, k, mods, kind, dtype):
    x, y, w, gate, shift, scale = make(m, k, mods, dtype)
    segs, rows = dealt(kind, m, mods)
    kw = dict(gate=gate, shift=shift, scale=scale, segments=segs)
    r = rs.residual_norm(x, y, w, EPS, codes=True, hidden=True, **kw)
    ref.check(r.x, *ref.stream(x, y, gate, rows), "t")
    if gate is not None:
        assert torch.equal(r.x[rows < 0], x[rows < 0])
    rstd, h, off = ref.normalised(r.x, w, EPS, shift, scale, rows)
    ref.check(r.rstd, rstd.view(-1), rstd.view(-1) * (k / 2 + 8) * ref.E, "rstd")
    ref.check(r.hidden, h, off + ref.U[dtype] * h.abs() + 2.0 ** -25, "h")
    z, offz = ref.rotated(h, off)
    top, step = z.abs().amax(1, keepdim=True), r.scales.double()
    ref.check(r.scales, top / 127, (offz.amax(1, keepdim=True) + 4 * ref.E * top) / 127, "scales")
    ref.check(r.codes.double() * step, z, step / 2 + offz + 256 * ref.E * step, "codes")
    # each output by itself is the same
    for c, hid in ((True, False), (False, True), (False, False)):
        part = rs.residual_norm(x, y, w, EPS, codes=c, hidden=hid, **kw)
        for a, b in zip(part, r):
            assert a is None or torch.equal(a, b)
        assert (part.codes is not None) == c and (part.hidden is not None) == hid
    for target in (0, 1):
        xs = [x.clone(), y.clone()]
        again = rs.residual_norm(*xs, w, EPS, codes=True, out=xs[target], **kw)
        assert again.x is xs[target] and torch.equal(again.x, r.x) and torch.equal(again.codes, r.codes)


GRADS = [(1, 8, 1, "runs"), (3, 136, 0, "none"), (17, 1288, 2, "runs"), (130, 5376, 3, "tokens"), (517, 1288, 0, "none"),
         (600, 16384, 1, "runs"), (2050, 640, 4, "many"), (300, 8200, 2, "none"), (40, 264, 2, "tokens"),
         (70, 6400, 2, "runs"), (90, 6152, 3, "tokens"), (33, 13568, 2, "runs")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,mods,kind", GRADS)
def test_gradients(m, k, mods, kind, dtype):
    x, y, w, gate, shift, scale = make(m, k, mods, dtype, 1)
    dt, dh = make(m, k, 0, dtype, 2)[:2]
    segs, rows = dealt(kind, m, mods)
    kw = dict(gate=gate, scale=scale, segments=segs)
    r = rs.residual_norm(x, y, w, EPS, shift=shift, codes=False, hidden=True, **kw)
    got = rs.residual_norm_backward(dt, dh, r.x, r.rstd, w, **kw)
    want, tol = ref.gradients(dt, dh, r.x, w, EPS, gate, scale, rows)
    for name, a, b, c in zip(("dx", "dy", "dw"), got, want, tol):
        ref.check(a, b, c, name)
    assert (got[0] is got[1]) == (gate is None)
    again = rs.residual_norm_backward(dt, dh, r.x, r.rstd, w, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    alone = rs.residual_norm_backward(None, dh, r.x, r.rstd, w, need_weight=False, **kw)
    assert alone[2] is None
    ref.check(alone[0], *(v[0] for v in ref.gradients(None, dh, r.x, w, EPS, gate, scale, rows)), "dx without dt")


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_and_differences(dtype):
    m, k = 40, 264
    x, y, w, gate, shift, scale = make(m, k, 2, dtype, 3)
    segs, rows = dealt("runs", m, 2)
    kw = dict(gate=gate, shift=shift, scale=scale, segments=segs)
    leaves = [t.clone().requires_grad_() for t in (x, y, w)]
    r = rs.residual_norm(*leaves, EPS, codes=False, hidden=True, **kw)
    dt, dh = make(m, k, 0, dtype, 4)[:2]
    torch.autograd.backward([r.x, r.hidden], [dt, dh])
    direct = rs.residual_norm_backward(dt, dh, r.x.detach(), r.rstd, w, gate=gate, scale=scale, segments=segs)
    for leaf, g in zip(leaves, direct):
        assert torch.equal(leaf.grad, g)
    only = [t.clone().requires_grad_() for t in (x, y, w)]
    rs.residual_norm(*only, EPS, codes=False, **kw).x.backward(dt)  # through the stream alone
    assert torch.equal(only[0].grad, dt) and not only[2].grad.any()

    # central differences of the 64-bit form, whose gradient the kernels are held to above, along a direction
    def value(ops):
        v = ops[0].double() + ops[1].double() * ref.spread(gate, rows, 0.0)
        n = v * (v.square().mean(1, keepdim=True) + EPS).rsqrt() * ops[2].double()
        h = n * (1 + ref.spread(scale, rows, 0.0)) + ref.spread(shift, rows, 0.0)
        return float((v * dt.double()).sum() + (h * dh.double()).sum())

    for i, leaf in enumerate(leaves):
        d = torch.randn(leaf.shape, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV).double()
        ops = [t.double() for t in (x, y, w)]
        hi, lo = list(ops), list(ops)
        hi[i], lo[i] = ops[i] + 1e-4 * d, ops[i] - 1e-4 * d
        diff = (value(hi) - value(lo)) / 2e-4
        along = leaf.grad.double() * d
        # the gradient's own rounding and that of t (u each, independent, uniform) and the differences' 1e-6
        tol = 6 * ref.U[dtype] / math.sqrt(3) * 3 * float(along.square().sum().sqrt()) + 1e-6 * float(along.abs().sum())
        assert abs(diff - float(along.sum())) <= tol, (i, diff, float(along.sum()))


@pytest.mark.parametrize("w_dtype,m_dtype", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                             (torch.float16, torch.float32)])
def test_weight_and_modulation_types(w_dtype, m_dtype):
    m, k = 50, 512
    x, y, w, gate, shift, scale = make(m, k, 2, torch.bfloat16, 6, w_dtype, m_dtype)
    segs, rows = dealt("runs", m, 2)
    r = rs.residual_norm(x, y, w, EPS, gate=gate, shift=shift, scale=scale, segments=segs, hidden=True)
    ref.check(r.x, *ref.stream(x, y, gate, rows), "t")
    _, h, off = ref.normalised(r.x, w, EPS, shift, scale, rows)
    ref.check(r.hidden, h, off + ref.U[x.dtype] * h.abs(), "h")
    dt, dh = y, x
    got = rs.residual_norm_backward(dt, dh, r.x, r.rstd, w, gate=gate, scale=scale, segments=segs)
    want, tol = ref.gradients(dt, dh, r.x, w, EPS, gate, scale, rows)
    assert got[2].dtype == w_dtype
    for a, b, c in zip(got, want, tol):
        ref.check(a, b, c)
    mixed = rs.residual_norm(x, y, w, EPS, gate=gate.float(), shift=shift, scale=scale, segments=segs, hidden=True)
    assert all(a is None or torch.equal(a, b) for a, b in zip(mixed, r))


def test_rows_without_numbers():
    """Zeros, infinities and NaN stay in their rows; views, empty streams."""
    x, y, w, gate, shift, scale = make(6, 512, 1, torch.bfloat16, 7)
    kw = dict(gate=gate, shift=shift, scale=scale, segments=[(0, 4, 0)], hidden=True)
    want = rs.residual_norm(x, y, w, EPS, **kw)
    x2, y2 = x.clone(), y.clone()
    x2[1, 3], x2[2, 5], x2[5] = float("nan"), float("inf"), 0
    y2[4] = float("nan")  # outside the segments: not read into the row
    r = rs.residual_norm(x2, y2, w, EPS, **kw)
    for i in (0, 3, 4):
        assert torch.equal(r.x[i], want.x[i]) and torch.equal(r.codes[i], want.codes[i]) and r.scales[i] == want.scales[i]
    for i in (1, 2):
        assert not torch.isfinite(r.scales[i]) and not r.codes[i].any() and r.hidden[i].isnan().any()
    assert r.scales[5] == 0 and not r.codes[5].any() and not r.hidden[5].any()
    wide = torch.zeros(6, 1040, dtype=x.dtype, device=DEV)
    wide[:, 8:520], wide[:, 520:1032] = x, y
    again = rs.residual_norm(wide[:, 8:520], wide[:, 520:1032], w, EPS, **kw)
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    odd = torch.zeros(6 * 512 + 1, dtype=x.dtype, device=DEV)[1:].view(6, 512)
    odd.copy_(x)
    assert torch.equal(rs.residual_norm(odd, y, w, EPS, **kw).codes, want.codes)
    e = rs.residual_norm(x[:0], y[:0], w, EPS, **{**kw, "segments": []})
    assert e.codes.shape == (0, 512) and e.scales.shape == (0, 1)
    dx, dy, dw = rs.residual_norm_backward(x[:0], x[:0], x[:0], e.rstd, w, gate=gate, scale=scale, segments=[])
    assert dx.shape == (0, 512) and dy.shape == (0, 512) and not dw.any()


def test_streams_and_graphs():
    x, y, w, gate, shift, scale = make(300, 1280, 2, torch.bfloat16, 8)
    segs, _ = dealt("runs", 300, 2)
    kw = dict(gate=gate, scale=scale, segments=segs)
    want = rs.residual_norm(x, y, w, EPS, shift=shift, hidden=True, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = rs.residual_norm(x, y, w, EPS, shift=shift, hidden=True, **kw)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = rs.residual_norm(xs, y, w, EPS, shift=shift, hidden=True, **kw)
        grads = rs.residual_norm_backward(y, x, r.x, r.rstd, w, **kw)
    xs.copy_(y)
    graph.replay()
    r2 = rs.residual_norm(y, y, w, EPS, shift=shift, hidden=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(r, r2))
    assert all(torch.equal(a, b) for a, b in zip(grads, rs.residual_norm_backward(y, x, r2.x, r2.rstd, w, **kw)))


def test_refusals():
    x, y, w, gate, shift, scale = make(16, 512, 2, torch.bfloat16)
    segs = [(0, 16, 0)]
    for args, kw, err in (((x.float(), y, w), {}, RuntimeError), ((x.cpu(), y, w), {}, RuntimeError), ((x, y[:8], w), {}, ValueError),
                          ((x, y.half(), w), {}, ValueError), ((x, y, w[:8]), {}, ValueError), ((x, y, w), dict(shift=shift), ValueError),
                          ((x, y, w), dict(gate=gate[:, :8], segments=segs), ValueError), ((x, y, w), dict(segments=segs), ValueError),
                          ((x, y, w), dict(gate=gate, segments=[(0, 17, 0)]), ValueError),
                          ((x, y, w), dict(gate=gate, segments=[(0, 16, 2)]), ValueError),
                          ((x[:, :264], y[:, :264], w[:264]), {}, ValueError), ((x[:, :12], y[:, :12], w[:12]), dict(codes=False), ValueError),
                          ((x, y, w), dict(out=x.half()), ValueError), ((x, y, w), dict(out=x.t().contiguous().t()), ValueError),
                          ((x, y, w), dict(gate=gate.clone().requires_grad_(), segments=segs), ValueError)):
        with pytest.raises(err):
            rs.residual_norm(*args, EPS, **kw)
    buf = torch.zeros(17 * 512, dtype=x.dtype, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        rs.residual_norm(buf[:8192].view(16, 512), y, w, EPS, out=buf[512:].view(16, 512))
    with pytest.raises(ValueError, match="gradients"):
        rs.residual_norm(x.clone().requires_grad_(), y, w, EPS)
    r = rs.residual_norm(x, y, w, EPS, codes=False, hidden=True)
    with pytest.raises(ValueError, match="rstd"):
        rs.residual_norm_backward(x, y, r.x, r.rstd[:4], w)
    xr = x.clone().requires_grad_()
    g, = torch.autograd.grad(rs.residual_norm(xr, y, w, EPS, codes=False, hidden=True).hidden.sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


def test_offsets_beyond_32_bits():
    x, y, w, gate, shift, scale = make(140, 512, 2, torch.bfloat16, 12)
    segs, _ = dealt("runs", 140, 2)
    kw = dict(gate=gate, scale=scale, segments=segs)
    want = rs.residual_norm(x, y, w, EPS, shift=shift, hidden=True, **kw)
    far = torch.empty(140, 1 << 24, dtype=x.dtype, device=DEV)  # the last row begins behind 2^31 numbers
    xf, yf, tf = far[:, :512], far[:, 1024:1536], far[:, 2048:2560]
    xf.copy_(x), yf.copy_(y), tf.copy_(want.x)
    got = rs.residual_norm(xf, yf, w, EPS, shift=shift, hidden=True, **kw)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(rs.residual_norm_backward(yf, xf, tf, want.rstd, w, **kw),
                    rs.residual_norm_backward(y, x, want.x, want.rstd, w, **kw)):
        assert torch.equal(a, b)
    assert rs.residual_norm(xf, yf, w, EPS, shift=shift, out=xf, **kw).x.data_ptr() == xf.data_ptr()
    assert torch.equal(xf, want.x)


@pytest.mark.parametrize("m,k", [(3, 1280), (700, 512), (300, 5376)])
def test_calls_in_a_row(m, k):
    """A stream carried through many layers in place (over x, or over y), in two streams at once and captured, against calls with
    a synchronisation behind each."""
    x, y, w, gate, shift, scale = make(m, k, 2, torch.bfloat16, 13)
    segs, _ = dealt("runs", m, 2)
    kw = dict(gate=gate, shift=shift, scale=scale, segments=segs, codes=k % 256 == 0, hidden=True)

    def run(x, sync=False):
        t, out = x.clone(), []
        for i in range(12):
            h = y.clone()
            r = rs.residual_norm(t, h, w, EPS, out=(t, h)[i % 2], **kw)
            t = r.x
            out += [t.clone().float(), r.hidden.float(), r.codes.float()]
            if sync:
                torch.cuda.synchronize()
        return torch.stack(out)

    want, other = run(x, True), run(x.flip(0), True)
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for side, start in zip(sides, (x, x.flip(0))):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(run(start))
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want) and torch.equal(got[1], other)
    graph, xs = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        z = run(xs)
    graph.replay()
    assert torch.equal(z, want)
    xs.copy_(x.flip(0))
    graph.replay()
    assert torch.equal(z, other)


def test_modulation_of_no_rows_is_refused():
    """An empty gate has no address, which would read as no gate at all: y added everywhere where it belongs nowhere."""
    x, y, w, gate, shift, scale = make(4, 512, 2, torch.bfloat16, 14)
    for kw in (dict(gate=gate[:0]), dict(shift=shift[:0], scale=scale[:0])):
        with pytest.raises(ValueError, match="a row at least"):
            rs.residual_norm(x, y, w, EPS, **kw)
    with pytest.raises(ValueError, match="a row at least"):
        rs.residual_norm_backward(x, x, x, torch.ones(4, device=DEV), w, gate=gate[:0])
    assert torch.equal(rs.residual_norm(x, y, w, EPS, gate=gate, codes=False).x, x)  # a gate whose rows no token has


def test_one_modulation_row_and_one_token():
    x, y, w, gate, shift, scale = make(1, 256, 1, torch.float16, 15)
    r = rs.residual_norm(x, y, w, EPS, gate=gate, shift=shift, scale=scale, segments=[(0, 1, 0)], hidden=True)
    wide = [torch.stack([t[0], t[0]])[:1].expand(1, 256) for t in (gate, shift, scale)]
    q = rs.residual_norm(x, y, w, EPS, gate=wide[0], shift=wide[1], scale=wide[2], segments=[(0, 1, 0)], hidden=True)
    assert all(torch.equal(a, b) for a, b in zip(r, q))
    ref.check(r.x, *ref.stream(x, y, gate, torch.zeros(1, dtype=torch.long, device=DEV)), "t")
