"""Low-rank adapters beside a shared projection against their 64-bit form (helpers/adapters_ref.py): ranks, widths, row maps,
strides, gradients."""
import math

import pytest
import torch

import adapters_ref as ref

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from minimax_h3_turbo_b200.h3 import adapters as ad
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16]


def make(m, k, n, r, adapters, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)

    return normal(m, k), normal(adapters, r, k, std=k ** -0.5), normal(adapters, n, r, std=r ** -0.5), normal(m, n), \
        torch.rand(adapters, generator=g, device=DEV) + 0.5


def mapped(kind, m, adapters, seed=0):
    g = torch.Generator().manual_seed(seed)
    if kind == "runs":  # contiguous runs of uneven length, some rows without an adapter between them
        rows = torch.full((m,), -1)
        cuts = sorted(torch.randint(0, m + 1, (2 * adapters,), generator=g).tolist())
        for i in range(adapters):
            rows[cuts[2 * i]:cuts[2 * i + 1]] = i
    elif kind == "mixed":
        rows = torch.randint(-1, adapters, (m,), generator=g)
    elif kind == "one":
        rows = torch.zeros(m, dtype=torch.long)
    elif kind == "none":
        rows = torch.full((m,), -1)
    else:  # each adapter once, then numbers out of range
        rows = torch.arange(m) - 1
    return rows.to(DEV)


CASES = [
    # m, k, n, rank, adapters, map
    (1, 8, 8, 1, 1, "one"), (1, 5120, 1024, 16, 1, "one"), (3, 136, 264, 4, 2, "mixed"), (8, 5120, 136, 64, 8, "each"),
    (9, 256, 2056, 128, 3, "mixed"), (17, 1288, 640, 24, 40, "mixed"), (64, 512, 1536, 33, 64, "each"),
    (127, 200, 328, 5, 2, "runs"), (128, 64, 128, 16, 1, "one"), (129, 640, 72, 48, 2, "runs"), (257, 264, 520, 8, 3, "mixed"),
    (300, 1024, 256, 127, 2, "mixed"), (1031, 1288, 2056, 24, 3, "runs"), (2049, 384, 640, 32, 4, "mixed"),
    (700, 96, 168, 112, 300, "mixed"), (513, 320, 192, 16, 5, "none"), (4100, 136, 4104, 12, 2, "runs"),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,r,adapters,kind", CASES)
def test_forward(m, k, n, r, adapters, kind, dtype):
    x, a, b, base, scales = make(m, k, n, r, adapters, dtype)
    rows = mapped(kind, m, adapters)
    p = ad.plan(rows, adapters)
    ref.check(ad.low_rank(x, a, b, p, base=base, scales=scales), *ref.forward(x, a, b, rows, scales, base), "base")
    got = ad.low_rank(x, a, b, p)
    ref.check(got, *ref.forward(x, a, b, rows), "no base")
    assert not got[(rows < 0) | (rows >= adapters)].any()
    out = base.clone()
    assert ad.low_rank(x, a, b, p, base=out, scales=scales, out=out) is out
    assert torch.equal(out, ad.low_rank(x, a, b, p, base=base, scales=scales))
    with_hidden, _ = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    ref.check(with_hidden, *ref.forward(x, a, b, rows, scales, base), "with hidden rows")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,n,r,adapters,kind", CASES)
def test_gradients(m, k, n, r, adapters, kind, dtype):
    x, a, b, base, scales = make(m, k, n, r, adapters, dtype, 1)
    rows = mapped(kind, m, adapters, 1)
    do = make(m, 8, n, 1, 1, dtype, 2)[3]
    p = ad.plan(rows, adapters)
    _, hidden = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    got = ad.low_rank_backward(do, x, a, b, p, hidden, scales=scales)
    want, tol = ref.backward(do, x, a, b, rows, scales)
    for name, g, w, t in zip(("dx", "da", "db"), got, want, tol):
        ref.check(g, w, t, name)
    again = ad.low_rank_backward(do, x, a, b, p, hidden, scales=scales)
    assert all(torch.equal(g, h) for g, h in zip(got, again))
    for need in ((True, False, False), (False, True, False), (False, False, True)):
        part = ad.low_rank_backward(do, x, a, b, p, hidden, scales=scales, need=need)
        assert [t is not None for t in part] == list(need)
        assert all(t is None or torch.equal(t, g) for t, g in zip(part, got))


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_and_differences(dtype):
    m, k, n, r = 150, 136, 264, 12
    x, a, b, base, scales = make(m, k, n, r, 2, dtype, 3)
    rows = mapped("mixed", m, 2, 3)
    p = ad.plan(rows, 2)
    leaves = [t.clone().requires_grad_() for t in (x, a, b, base)]
    do = make(m, 8, n, 1, 1, dtype, 4)[3]
    y = ad.low_rank(*leaves[:3], p, base=leaves[3], scales=scales)
    y.backward(do)
    _, hidden = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    for leaf, g in zip(leaves, (*ad.low_rank_backward(do, x, a, b, p, hidden, scales=scales), do)):
        assert torch.equal(leaf.grad, g)
    # out is linear in each operand by itself: the difference along a direction is the gradient along it, up to the roundings
    # of two outputs and of the gradient.  Those are independent, uniform to +-u of each term: six standard deviations
    u = ref.U[dtype]
    for i, t in enumerate((x, a, b)):
        d = (torch.randn(t.shape, generator=torch.Generator(device=DEV).manual_seed(5), device=DEV) * t.float().std()).to(dtype)
        moved = [x, a, b]
        moved[i] = (t.float() + d.float()).to(dtype)
        step = moved[i].double() - t.double()
        y0, y1 = (ad.low_rank(*ops, p, scales=scales).double() for ops in ((x, a, b), moved))
        diff = float(((y1 - y0) * do.double()).sum())
        grad = leaves[i].grad.double()
        along = float((grad * step).sum())
        var = sum(float((2 * v * do.double()).square().sum()) for v in (y0, y1)) + float((2 * grad * step).square().sum())
        assert abs(diff - along) <= 6 * u / math.sqrt(3) * math.sqrt(var), (i, diff, along)


def test_strides_leading_dims_and_unaligned_views():
    x, a, b, base, scales = make(60, 256, 384, 16, 2, torch.bfloat16)
    rows = mapped("mixed", 60, 2)
    p = ad.plan(rows, 2)
    want = ad.low_rank(x, a, b, p, base=base, scales=scales)
    wide = torch.zeros(60, 1024, dtype=x.dtype, device=DEV)
    wide[:, 128:384] = x
    assert torch.equal(ad.low_rank(wide[:, 128:384], a, b, p, base=base, scales=scales), want)
    odd = torch.zeros(60 * 256 + 1, dtype=x.dtype, device=DEV)[1:].view(60, 256)
    odd.copy_(x)
    assert torch.equal(ad.low_rank(odd, a, b, p, base=base, scales=scales), want)
    assert torch.equal(ad.low_rank(x.t().contiguous().t(), a, b, p, base=base, scales=scales), want)
    got = ad.low_rank(x.view(3, 20, 256), a, b, p, base=base.view(3, 20, 384), scales=scales)
    assert got.shape == (3, 20, 384) and torch.equal(got.view(60, 384), want)
    big = torch.full((60, 512), 7.0, dtype=x.dtype, device=DEV)
    ad.low_rank(x, a, b, p, base=base, scales=scales, out=big[:, 64:448])
    assert torch.equal(big[:, 64:448], want) and (big[:, :64] == 7).all() and (big[:, 448:] == 7).all()
    at = a.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ad.low_rank(x, at, b, p, base=base, scales=scales), want)
    one = ad.low_rank(x, a[0], b[0], scales=2.0)
    assert torch.equal(one, ad.low_rank(x, a[:1], b[:1], ad.plan(torch.zeros_like(rows), 1),
                                        scales=torch.full((1,), 2.0, device=DEV)))


@pytest.mark.parametrize("m", [20, 200])
def test_a_request_does_not_see_the_others(m):
    """Infinities and NaN of one request's rows and adapter stay with it."""
    x, a, b, base, scales = make(m, 264, 392, 24, 3, torch.bfloat16)
    rows = mapped("mixed", m, 3)
    p = ad.plan(rows, 3)
    do = base.flip(0).contiguous()
    want, hidden = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    grads = ad.low_rank_backward(do, x, a, b, p, hidden, scales=scales)
    bad = rows == 1
    x[bad], do2 = float("inf"), do.clone()
    do2[bad] = float("nan")
    a[1], b[1], base[bad] = float("nan"), float("inf"), float("nan")
    got, hidden = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    assert torch.equal(got[~bad], want[~bad]) and got[bad].isnan().all()
    assert torch.equal(ad.low_rank(x, a, b, p, base=base, scales=scales)[~bad], want[~bad])
    new = ad.low_rank_backward(do2, x, a, b, p, hidden, scales=scales)
    assert torch.equal(new[0][~bad], grads[0][~bad])
    for i in (0, 2):
        assert torch.equal(new[1][i], grads[1][i]) and torch.equal(new[2][i], grads[2][i])


@pytest.mark.parametrize("size", [1e-3, 1.0, 200.0])
def test_fp16_hidden_rows_of_any_size(size):
    """x A^T past 65504 or among fp16's subnormals: the rows are scaled for the second product."""
    m, k, n, r = 200, 512, 264, 16
    x, a, b, base, _ = make(m, k, n, r, 1, torch.float16, 6)
    x = (x.float() * size).half()
    a = (a.float() * 20 * min(size, 30.0)).half()
    b = (b.float() * (1e-4 if size > 1 else 1.0)).half()
    rows = torch.zeros(m, dtype=torch.long, device=DEV)
    p = ad.plan(rows, 1)
    out, hidden = ad.low_rank(x, a, b, p, return_hidden=True)
    ref.check(out, *ref.forward(x, a, b, rows), "forward")
    do = (base.float() * 1e-3).half()
    want, tol = ref.backward(do, x, a, b, rows)
    for name, g, w, t in zip(("dx", "da", "db"), ad.low_rank_backward(do, x, a, b, p, hidden), want, tol):
        assert torch.isfinite(w).all() and w.abs().max() < 65504
        ref.check(g, w, t, name)


def test_segments_plan_and_empty_batches():
    x, a, b, base, scales = make(50, 128, 64, 8, 3, torch.bfloat16)
    rows = torch.full((50,), -1, device=DEV)
    rows[5:20], rows[20:33] = 2, 0
    want = ad.low_rank(x, a, b, ad.plan(rows, 3), base=base, scales=scales)
    p = ad.plan([(5, 20, 2), (20, 33, 0), (40, 40, 1)], 3, count=50, device=DEV)
    assert torch.equal(ad.low_rank(x, a, b, p, base=base, scales=scales), want)
    far = rows.clone()
    far[rows < 0] = 2 ** 40 + 1  # out of range in 64 bits stays so
    assert torch.equal(ad.low_rank(x, a, b, ad.plan(far, 3), base=base, scales=scales), want)
    p0 = ad.plan(rows[:0], 3)
    y, hidden = ad.low_rank(x[:0], a, b, p0, base=base[:0], return_hidden=True)
    assert y.shape == (0, 64)
    dx, da, db = ad.low_rank_backward(base[:0], x[:0], a, b, p0, hidden)
    assert dx.shape == (0, 128) and not da.any() and not db.any()
    xr, ar = x[:0].clone().requires_grad_(), a.clone().requires_grad_()
    ad.low_rank(xr, ar, b, p0).sum().backward()
    assert xr.grad.shape == (0, 128) and not ar.grad.any()


def test_streams_and_graphs():
    x, a, b, base, scales = make(300, 512, 640, 16, 4, torch.bfloat16)
    rows = mapped("mixed", 300, 4)
    p = ad.plan(rows, 4)
    want = ad.low_rank(x, a, b, p, base=base, scales=scales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ad.low_rank(x, a, b, ad.plan(rows, 4), base=base, scales=scales)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph, xs = torch.cuda.CUDAGraph(), x.clone()
    static_rows = rows.to(torch.int32)
    with torch.cuda.graph(graph):  # plan, forward and gradients, replayed on other rows and another map
        q = ad.plan(static_rows, 4)
        y, hidden = ad.low_rank(xs, a, b, q, base=base, scales=scales, return_hidden=True)
        grads = ad.low_rank_backward(base, xs, a, b, q, hidden, scales=scales)
    xs.copy_(x.flip(0))
    static_rows.copy_(rows.flip(0))
    graph.replay()
    p2 = ad.plan(rows.flip(0), 4)
    y2, hidden2 = ad.low_rank(x.flip(0), a, b, p2, base=base, scales=scales, return_hidden=True)
    assert torch.equal(y, y2)
    for g, h in zip(grads, ad.low_rank_backward(base, x.flip(0).contiguous(), a, b, p2, hidden2, scales=scales)):
        assert torch.equal(g, h)


def test_refusals():
    x, a, b, base, scales = make(16, 64, 128, 8, 2, torch.bfloat16)
    p = ad.plan(torch.zeros(16, dtype=torch.int32, device=DEV), 2)
    ok = dict(base=base, scales=scales)
    for args, kw, err in (
            ((x.float(), a, b, p), ok, RuntimeError), ((x, a.half(), b, p), ok, RuntimeError), ((x.cpu(), a, b, p), ok, RuntimeError),
            ((x[:, :56], a, b, p), ok, ValueError), ((x, a, b[:1], p), ok, ValueError), ((x, a[:, :4], b, p), ok, ValueError),
            ((x[:8], a, b, p), dict(), ValueError), ((x, a, b, None), ok, ValueError), ((x, a[:1], b[:1], p), ok, ValueError),
            ((x, a, b, p), dict(base=base[:, :64]), ValueError), ((x, a, b, p), dict(base=base.half()), ValueError),
            ((x, a, b, p), dict(scales=scales[:1]), ValueError), ((x, a, b, p), dict(scales=scales.double()), ValueError),
            ((x, a, b, p), dict(out=base.half()), ValueError), ((x, a, b, p), dict(out=base.t().contiguous().t()), ValueError)):
        with pytest.raises(err):
            ad.low_rank(*args, **kw)
    buf = torch.zeros(17 * 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="overlap"):
        ad.low_rank(x, a, b, p, base=buf[:2048].view(16, 128), out=buf[128:].view(16, 128))
    with pytest.raises(ValueError, match="overlap"):
        ad.low_rank(x, a, b[:, :64].contiguous(), p, out=x)
    with pytest.raises(ValueError, match="scales"):
        ad.low_rank(x, a, b, p, scales=scales.clone().requires_grad_())
    with pytest.raises(ValueError, match="out cannot"):
        ad.low_rank(x.clone().requires_grad_(), a, b, p, out=base)
    with pytest.raises(ValueError, match="hidden"):
        ad.low_rank_backward(base, x, a, b, p, torch.zeros(8, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="adapters"):
        ad.plan(torch.zeros(4, dtype=torch.int32, device=DEV), 0)
    xr = x.clone().requires_grad_()
    g, = torch.autograd.grad(ad.low_rank(xr, a, b, p).sum(), xr, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivatives"):
        g.sum().backward()


@pytest.mark.parametrize("r", [16, 128])  # rows by eights, rows by 128
def test_offsets_beyond_32_bits(r):
    x, a, b, base, scales = make(140, 256, 384, r, 3, torch.bfloat16)
    p = ad.plan(mapped("mixed", 140, 3), 3)
    want, hidden = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    far = torch.empty(140, 1 << 24, dtype=x.dtype, device=DEV)  # the last row begins behind 2^31 numbers
    xf, bf = far[:, :256], far[:, 512:896]
    xf.copy_(x), bf.copy_(base)
    assert torch.equal(ad.low_rank(xf, a, b, p, base=bf, scales=scales), want)
    for u, v in zip(ad.low_rank_backward(bf, xf, a, b, p, hidden, scales=scales),
                    ad.low_rank_backward(base, x, a, b, p, hidden, scales=scales)):
        assert torch.equal(u, v)
    assert ad.low_rank(x, a, b, p, base=bf, scales=scales, out=bf).data_ptr() == bf.data_ptr()
    assert torch.equal(bf, want)


@pytest.mark.parametrize("m,r", [(4, 64), (40, 16), (300, 64)])
def test_calls_in_a_row(m, r):
    """Each call reads what the one before wrote, and workspaces pass from call to call: as many as a decoder's layers, in a
    stream, in two streams at once and captured, give what calls with a synchronisation behind each give."""
    x, a, b, _, scales = make(m, 512, 512, r, 4, torch.bfloat16)
    b, p = b / 8, ad.plan(mapped("mixed", m, 4), 4)

    def run(x, sync=False):
        out = []
        for _ in range(24):
            x = ad.low_rank(x, a, b, p, base=x, scales=scales)
            y = x.clone()
            out += [x, ad.low_rank(x, a, b, p, base=y, scales=scales, out=y)]
            if sync:
                torch.cuda.synchronize()
        return torch.stack(out)

    want, other = run(x, True), run(x.flip(0), True)
    assert torch.isfinite(want).all()
    assert torch.equal(run(x), want)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for side, start in zip(sides, (x, x.flip(0))):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(run(start))
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want) and torch.equal(got[1], other)
    graphs, xs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], x.clone()
    got = []
    for graph in graphs:  # of two in one pool, replayed in turn
        with torch.cuda.graph(graph, pool=graphs[0].pool() if got else None):
            got.append(run(xs))
    for graph, y in zip(graphs, got):
        graph.replay()
        assert torch.equal(y, want)
    xs.copy_(x.flip(0))
    for graph, y in zip(graphs, got):
        graph.replay()
        assert torch.equal(y, other)


def test_one_plan_for_many_projections_and_no_hidden_rows():
    x, a, b, base, scales = make(50, 256, 384, 16, 3, torch.float16)
    p = ad.plan(mapped("runs", 50, 3), 3)
    first = ad.low_rank(x, a, b, p, base=base, scales=scales)
    x2, a2, b2, base2, _ = make(50, 520, 136, 40, 3, torch.float16)
    second = ad.low_rank(x2, a2, b2, p, base=base2)
    assert torch.equal(first, ad.low_rank(x, a, b, p, base=base, scales=scales))
    assert torch.equal(second, ad.low_rank(x2, a2, b2, ad.plan(mapped("runs", 50, 3), 3), base=base2))
    with pytest.raises(ValueError, match="hidden"):
        ad.low_rank_backward(base, x, a, b, p, None, scales=scales)


def test_columns_of_one_tensor_as_input_and_output():
    x, a, b, base, scales = make(30, 256, 384, 16, 3, torch.bfloat16)
    p = ad.plan(mapped("mixed", 30, 3), 3)
    both = torch.full((30, 648), 7.0, dtype=x.dtype, device=DEV)
    both[:, :256] = x
    ad.low_rank(both[:, :256], a, b, p, base=base, scales=scales, out=both[:, 256:640])
    assert torch.equal(both[:, 256:640], ad.low_rank(x, a, b, p, base=base, scales=scales))
    assert torch.equal(both[:, :256], x) and (both[:, 640:] == 7).all()
    for out in (both[:, 248:632], both[:, 264:]):
        with pytest.raises(ValueError, match="overlap"):
            ad.low_rank(both[:, :256] if out.data_ptr() < both[:, 256:].data_ptr() else both[:, 392:], a, b, p, out=out)
    with pytest.raises(ValueError, match="overlap"):  # a row further, half a row back
        flat = torch.zeros(31 * 512, dtype=x.dtype, device=DEV)
        ad.low_rank(flat[:30 * 512].view(30, 512)[:, :256], a, b, p, out=flat[384:384 + 30 * 512].view(30, 512)[:, :384])


@pytest.mark.parametrize("r", [1, 7, 24, 127])
def test_gradients_of_single_rows_and_of_none(r):
    """An adapter of one row, one of none, one of some: the first's gradients are outer products, the second's zeros."""
    x, a, b, base, scales = make(9, 136, 264, r, 3, torch.float16)
    rows = torch.tensor([2, 0, 2, 2, -1, 2, 2, 5, 2], device=DEV)
    p = ad.plan(rows, 3)
    _, hidden = ad.low_rank(x, a, b, p, base=base, scales=scales, return_hidden=True)
    dx, da, db = ad.low_rank_backward(base, x, a, b, p, hidden, scales=scales)
    want, tol = ref.backward(base, x, a, b, rows, scales)
    for name, u, v, t in zip(("dx", "da", "db"), (dx, da, db), want, tol):
        ref.check(u, v, t, name)
    assert not da[1].any() and not db[1].any() and not dx[4].any() and not dx[7].any()
