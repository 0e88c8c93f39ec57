"""Low-rank adapters whose rows, ranks and other operands have sizes of their own, up to 2^20 apart and the other way round: each
result is held to the sum of its own terms' magnitudes, whatever larger numbers stand beside it in a row or in a rank.

Bounds: u is half a step of the type that a hidden number is an operand in, 2^-8 in bf16 and 2^-11 beside fp16, relative to that
number.  A sum of n products in fp32 on the tensor cores is off by at most (n + 16) 2^-23 of the sum of magnitudes.  The result is
rounded once: half a step, in fp16 at least 2^-25."""
import pytest
import torch

from adapters_ref import U, check, gamma, groups

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from minimax_h3_turbo_b200.h3 import adapters as ad
DEV = "cuda"


def powers(shape, most, g):
    return torch.randint(-most, most + 1, shape, generator=g, device=DEV).double().exp2()


def spread(m, k, n, r, adapters, dtype, seed):
    """Rows of x up to 2^10 from 1 either way and do's the other way, ranks of A the same and B's the other way."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    row, rank = powers((m, 1), 10, g), powers((adapters, r, 1), 10, g)

    def normal(*shape):
        return torch.randn(shape, generator=g, device=DEV).double()

    x, a = normal(m, k) * row, normal(adapters, r, k) * k ** -0.5 * rank
    b, do = normal(adapters, n, r) * r ** -0.5 / rank.transpose(1, 2), normal(m, n) * n ** -0.5 / row
    rows = torch.randint(-1, adapters, (m,), generator=g, device=DEV)
    return *(t.to(dtype) for t in (x, a, b, do)), rows


def results(x, a, b, do, rows, s):
    """(out, dx, da, db) in 64 bits and bounds."""
    u = U[x.dtype]
    x, a, b, do = (t.double() for t in (x, a, b, do))
    out, dx = torch.zeros(x.shape[0], b.shape[1], device=DEV).double(), torch.zeros_like(x)
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    to, tx, ta, tb = (torch.zeros_like(t) for t in (out, dx, da, db))
    for g, i in groups(rows, a.shape[0]):
        if i.numel() == 0:
            continue
        h, dh = s * x[i] @ a[g].T, s * do[i] @ b[g]
        # the sum's own error is rounded along with it
        eh = u * h.abs() + (1 + u) * gamma(x.shape[1]) * s * x[i].abs() @ a[g].abs().T
        ed = u * dh.abs() + (1 + u) * gamma(do.shape[1]) * s * do[i].abs() @ b[g].abs()
        r, m = gamma(a.shape[1]), gamma(i.numel())
        out[i], to[i] = h @ b[g].T, (eh + r * (h.abs() + eh)) @ b[g].abs().T
        dx[i], tx[i] = dh @ a[g], (ed + r * (dh.abs() + ed)) @ a[g].abs()
        da[g], ta[g] = dh.T @ x[i], (ed + m * (dh.abs() + ed)).T @ x[i].abs()
        db[g], tb[g] = do[i].T @ h, do[i].abs().T @ (eh + m * (h.abs() + eh))
    return (out, dx, da, db), tuple(t + u * (v.abs() + t) + 2.0 ** -25 for v, t in ((out, to), (dx, tx), (da, ta), (db, tb)))


# rows by eights and by 128; gradients of whole units and of units whose parts are added up; ranks that are no multiples of 8
CASES = [(5, 136, 264, 8, 2), (20, 264, 392, 24, 3), (60, 512, 136, 128, 4), (300, 264, 392, 24, 3), (700, 512, 640, 64, 2),
         (130, 136, 264, 33, 1), (2300, 136, 264, 128, 2), (2300, 264, 136, 16, 40), (640, 256, 128, 72, 64)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n,r,adapters", CASES)
def test_sizes_apart(m, k, n, r, adapters, dtype):
    x, a, b, do, rows = spread(m, k, n, r, adapters, dtype, m + r)
    p = ad.plan(rows, adapters)
    out, hidden = ad.low_rank(x, a, b, p, scales=0.75, return_hidden=True)
    got = (out, *ad.low_rank_backward(do, x, a, b, p, hidden, scales=0.75))
    want, tol = results(x, a, b, do, rows, 0.75)
    for name, g, w, t in zip(("out", "dx", "da", "db"), got, want, tol):
        check(g, w, t, name)
    assert torch.equal(ad.low_rank(x, a, b, p, scales=0.75), out)


@pytest.mark.parametrize("m", [2, 200, 4000])  # adapters of one and of many units
def test_small_rows_beside_large_ones(m):
    """A hidden row 2^-26 of another's size whose other operand is 2^27 of its: all numbers and sums are exact."""
    x, do = torch.zeros(m, 8, dtype=torch.float16, device=DEV), torch.zeros(m, 8, dtype=torch.float16, device=DEV)
    x[0, 0], x[m - 1, 0], do[0, 0], do[m - 1, 0] = 2.0 ** -12, 2.0 ** 15, 2.0 ** 13, 2.0 ** -13
    a, b = torch.zeros(1, 1, 8, dtype=torch.float16, device=DEV), torch.zeros(1, 8, 1, dtype=torch.float16, device=DEV)
    a[0, 0, 0], b[0, 0, 0] = 2.0 ** -10, 2.0 ** -13
    p = ad.plan(torch.zeros(m, dtype=torch.int32, device=DEV), 1)
    _, hidden = ad.low_rank(x, a, b, p, return_hidden=True)
    dx, da, db = ad.low_rank_backward(do, x, a, b, p, hidden)
    assert float(da[0, 0, 0]) == 2.0 ** -12 + 2.0 ** -11  # dh = 1, 2^-26
    assert float(db[0, 0, 0]) == 2.0 ** -9 + 2.0 ** -8  # h = 2^-22, 2^5
    assert float(dx[0, 0]) == 2.0 ** -10 and not da[0, 0, 1:].any() and not db[0, 1:].any()


@pytest.mark.parametrize("m", [3, 200])
def test_small_ranks_beside_large_ones(m):
    """Ranks 2^-30 of another's size, each with channels of its own behind it: out and dx are exact."""
    x, do = torch.zeros(m, 16, dtype=torch.float16, device=DEV), torch.zeros(m, 16, dtype=torch.float16, device=DEV)
    x[:, 0], x[:, 1], do[:, 0], do[:, 1] = 2.0 ** 10, 2.0 ** -8, 2.0 ** 10, 2.0 ** -8
    a, b = torch.zeros(1, 2, 16, dtype=torch.float16, device=DEV), torch.zeros(1, 16, 2, dtype=torch.float16, device=DEV)
    a[0, 0, 0], a[0, 1, 1], b[0, 0, 0], b[0, 1, 1] = 2.0 ** 4, 2.0 ** -8, 2.0 ** -8, 2.0 ** 6  # h = 2^14, 2^-16
    p = ad.plan(torch.zeros(m, dtype=torch.int32, device=DEV), 1)
    out, hidden = ad.low_rank(x, a, b, p, return_hidden=True)
    assert (out[:, 0] == 2.0 ** 6).all() and (out[:, 1] == 2.0 ** -10).all() and not out[:, 2:].any()
    dx, _, _ = ad.low_rank_backward(do, x, a, b, p, hidden)  # dh = 2^2, 2^-2
    assert (dx[:, 0] == 2.0 ** 6).all() and (dx[:, 1] == 2.0 ** -10).all()
    do[:, 0], b[0, 0, 0] = 2.0 ** 15, 2.0 ** -1  # dh = 2^14, 2^-2
    x[:, 0] = 2.0 ** -2  # h = 2^2
    out, hidden = ad.low_rank(x, a, b, p, return_hidden=True)
    do[:, 1] = 2.0 ** -14
    a[0, 0, 0], a[0, 1, 1] = 2.0 ** -4, 2.0 ** 4
    dx, _, _ = ad.low_rank_backward(do, x, a, b, p, hidden)  # dh = 2^14, 2^-8
    assert (dx[:, 0] == 2.0 ** 10).all() and (dx[:, 1] == 2.0 ** -4).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("r", [1, 8, 24, 33, 120])
def test_infinities_of_positive_numbers(r, m, dtype):
    """Sums of positive numbers of which one is infinite are infinite, whatever the rank is filled up to; other rows keep theirs."""
    g = torch.Generator(device=DEV).manual_seed(r)
    x, a, b, do = ((torch.rand(s, generator=g, device=DEV) + 0.5).to(dtype) for s in ((m, 40), (2, r, 40), (2, 72, r), (m, 72)))
    rows = torch.arange(m, device=DEV) % 2
    p = ad.plan(rows, 2)
    inf = float("inf")
    for first in (True, False):  # of x, then of the output's gradient, both in row 1
        xi, doi = x.clone(), do.clone()
        (xi if first else doi)[1, 5] = inf
        out, hidden = ad.low_rank(xi, a, b, p, return_hidden=True)
        assert torch.equal(ad.low_rank(xi, a, b, p), out)
        dx, da, db = ad.low_rank_backward(doi, xi, a, b, p, hidden)
        others = torch.arange(m, device=DEV) != 1
        assert out[others].isfinite().all() and dx[others].isfinite().all() and da[0].isfinite().all() and db[0].isfinite().all()
        if first:  # h is infinite, dh is not
            assert (out[1] == inf).all() and dx.isfinite().all() and (db[1] == inf).all()
            assert (da[1, :, 5] == inf).all() and da[1, :, :5].isfinite().all() and da[1, :, 6:].isfinite().all()
        else:
            assert out.isfinite().all() and (dx[1] == inf).all() and (da[1] == inf).all()
            assert (db[1, 5] == inf).all() and db[1, :5].isfinite().all() and db[1, 6:].isfinite().all()


@pytest.mark.parametrize("r", [16, 128])  # rows by eights, rows by 128
def test_offsets_beyond_32_bits(r):
    x, a, b, do, rows = spread(140, 256, 384, r, 3, torch.float16, 5)
    p = ad.plan(rows, 3)
    want, hidden = ad.low_rank(x, a, b, p, base=do, return_hidden=True)
    far = torch.empty(140, 1 << 24, dtype=x.dtype, device=DEV)  # the last row begins behind 2^31 numbers
    xf, df = far[:, :256], far[:, 512:896]
    xf.copy_(x), df.copy_(do)
    assert torch.equal(ad.low_rank(xf, a, b, p, base=df), want)
    for u, v in zip(ad.low_rank_backward(df, xf, a, b, p, hidden), ad.low_rank_backward(do, x, a, b, p, hidden)):
        assert torch.equal(u, v)
    assert ad.low_rank(x, a, b, p, base=df, out=df).data_ptr() == df.data_ptr() and torch.equal(df, want)


@pytest.mark.parametrize("m,r,adapters", [(12, 40, 3), (300, 16, 4), (300, 128, 2), (2500, 72, 1)])
def test_training_steps_captured_and_in_two_streams(m, r, adapters):
    """The gradients of several steps, each on what the one before left, replayed and side by side, as they come one by one."""
    x, a, b, do, rows = spread(m, 264, 264, r, adapters, torch.float16, 6)
    p = ad.plan(rows, adapters)

    def steps(x, sync=False):
        results = []
        for _ in range(6):
            out, hidden = ad.low_rank(x, a, b, p, base=x, scales=0.5, return_hidden=True)
            results += [out, *ad.low_rank_backward(do, x, a, b, p, hidden, scales=0.5)]
            x = (x + out) / 2
            if sync:
                torch.cuda.synchronize()
        return results

    want, other = steps(x, True), steps(x.flip(0), True)
    sides, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for side, start in zip(sides, (x, x.flip(0))):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got.append(steps(start))
    for side in sides:
        torch.cuda.current_stream().wait_stream(side)
    graph, xs = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        captured = steps(xs)
    graph.replay()
    same = lambda u, v: all(torch.equal(s, t) for s, t in zip(u, v))  # noqa: E731
    assert same(got[0], want) and same(got[1], other) and same(captured, want)
    xs.copy_(x.flip(0))
    graph.replay()
    assert same(captured, other)


@pytest.mark.parametrize("m,k,n,r,adapters", [(1, 136, 264, 33, 1), (5, 136, 264, 8, 2), (8, 520, 136, 64, 8), (20, 264, 392, 24, 3),
                                              (60, 512, 136, 128, 8), (200, 256, 264, 16, 2)])
def test_few_bf16_rows_have_hidden_rows_of_11_digits(m, k, n, r, adapters):
    """Rows by eights: beside bf16 operands too, what is rounded to 8 digits is the result alone."""
    x, a, b, _, rows = spread(m, k, n, r, adapters, torch.bfloat16, m)
    out = torch.zeros(m, n, device=DEV).double()
    tol = torch.zeros_like(out)
    for g, i in groups(rows, adapters):
        xi, ag, bg = x[i].double(), a[g].double(), b[g].double()
        h = xi @ ag.T
        eh = 2.0 ** -11 * h.abs() + (1 + 2.0 ** -11) * gamma(k) * xi.abs() @ ag.abs().T
        out[i], tol[i] = h @ bg.T, (eh + gamma(r) * (h.abs() + eh)) @ bg.abs().T
    check(ad.low_rank(x, a, b, ad.plan(rows, adapters)), out, tol + 2.0 ** -8 * (out.abs() + tol) + 2.0 ** -133, "out")
