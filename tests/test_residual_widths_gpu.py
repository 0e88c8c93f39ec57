"""The residual's norm without codes at widths that are no multiples of 256: the last block of a row, or of a split row's second half,
ends inside.  Bounds: helpers/residual_ref.py."""
import pytest
import torch

import residual_ref as ref
from test_residual_gpu import DEV, EPS, TYPES, dealt, make

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from minimax_h3_turbo_b200.h3 import residual as rs

WIDTHS = [(1, 8, 0, "none"), (5, 8, 2, "runs"), (3, 248, 1, "tokens"), (7, 264, 2, "runs"), (33, 1288, 3, "tokens"), (601, 1288, 2, "runs"),
          (517, 1288, 0, "none"), (2051, 136, 4, "many"), (9, 6152, 2, "runs"), (150, 6400, 2, "tokens"), (11, 8184, 2, "runs"),
          (5, 8200, 2, "runs"), (301, 8200, 3, "tokens"), (4, 8448, 0, "none"), (13, 8712, 2, "many"), (3, 14088, 2, "runs"),
          (7, 16376, 2, "tokens"), (160, 16376, 1, "runs"), (2, 16384, 0, "none")]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k,mods,kind", WIDTHS)
def test_stream_and_hidden_rows(m, k, mods, kind, dtype):
    x, y, w, gate, shift, scale = make(m, k, mods, dtype, 21)
    segs, rows = dealt(kind, m, mods)
    forms = [dict(gate=gate, shift=shift, scale=scale, segments=segs)]
    if mods:  # each by itself
        forms += [dict(gate=gate, segments=segs), dict(shift=shift, scale=scale, segments=segs)]
    for kw in forms:
        g, h0, s0 = (kw.get(n) for n in ("gate", "shift", "scale"))
        wide = torch.full((m + 1, k + 8), 3.0, dtype=dtype, device=DEV)  # what lies behind each row, and behind the last, stays
        r = rs.residual_norm(x, y, w, EPS, codes=False, hidden=True, out=wide[:m, :k], **kw)
        assert (wide[:m, k:] == 3).all() and (wide[m] == 3).all()
        ref.check(r.x, *ref.stream(x, y, g, rows), "t")
        if g is not None:
            assert torch.equal(r.x[rows < 0], x[rows < 0])
        rstd, h, off = ref.normalised(r.x, w, EPS, h0, s0, rows)
        ref.check(r.rstd, rstd.view(-1), rstd.view(-1) * (k / 2 + 8) * ref.E, "rstd")
        ref.check(r.hidden, h, off + ref.U[dtype] * h.abs() + 2.0 ** -25, "h")
        for target in (0, 1):
            xs = [x.clone(), y.clone()]
            again = rs.residual_norm(*xs, w, EPS, codes=False, hidden=True, out=xs[target], **kw)
            assert again.x is xs[target] and torch.equal(again.x, r.x) and torch.equal(again.hidden, r.hidden)
            assert torch.equal(xs[1 - target], (y, x)[target])


@pytest.mark.parametrize("w_dtype,m_dtype", [(torch.float32, torch.float32), (torch.float16, torch.float32),
                                             (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("k", [264, 1288, 8200])
def test_types_of_weight_and_modulation(k, w_dtype, m_dtype):
    m = 19
    x, y, w, gate, shift, scale = make(m, k, 2, torch.bfloat16, 22, w_dtype, m_dtype)
    segs, rows = dealt("runs", m, 2)
    r = rs.residual_norm(x, y, w, EPS, gate=gate, shift=shift, scale=scale, segments=segs, codes=False, hidden=True)
    ref.check(r.x, *ref.stream(x, y, gate, rows), "t")
    _, h, off = ref.normalised(r.x, w, EPS, shift, scale, rows)
    ref.check(r.hidden, h, off + ref.U[x.dtype] * h.abs() + 2.0 ** -25, "h")
