"""Arguments of the low-rank adapters that must come back as an error before anything is launched, and the 64-bit form's
gradients against differences."""
import ctypes

import pytest
import torch

import adapters_ref as ref
from minimax_h3_turbo_b200 import _lib
from minimax_h3_turbo_b200.h3 import adapters as ad


def pointer(n=1 << 14):
    buf = ctypes.create_string_buffer(n)
    return buf, ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256


def error(rc):
    return rc, _lib.lib().h3b_last_error().decode()


GOOD = dict(ldx=64, ldbase=128, ldo=128, dtype=_lib.BF16, M=4, K=64, N=128, rank=8, R=2)


def forward(p, **kw):
    a = {**GOOD, "x": p, "a": p, "b": p, "base": p, "out": p, "scales": p, "plan": p, "hidden": None, "ws": None, "n": 0, **kw}
    return error(_lib.lib().h3b_low_rank(a["x"], a["ldx"], a["a"], a["b"], a["base"], a["ldbase"], a["out"], a["ldo"], a["dtype"],
                                         a["M"], a["K"], a["N"], a["rank"], a["R"], a["scales"], a["plan"], a["hidden"], a["ws"],
                                         a["n"], None))


def backward(p, **kw):
    a = {**GOOD, "go": p, "ldgo": 128, "x": p, "a": p, "b": p, "hidden": p, "dx": p, "lddx": 64, "da": p, "db": p, "scales": p,
         "plan": p, "ws": None, "n": 0, **kw}
    return error(_lib.lib().h3b_low_rank_backward(a["go"], a["ldgo"], a["x"], a["ldx"], a["a"], a["b"], a["hidden"], a["dx"],
                                                  a["lddx"], a["da"], a["db"], a["dtype"], a["M"], a["K"], a["N"], a["rank"], a["R"],
                                                  a["scales"], a["plan"], a["ws"], a["n"], None))


SIZES = [(dict(dtype=_lib.FP32), "bf16 or fp16"), (dict(M=-1), "multiples of 8"), (dict(K=60), "multiples of 8"),
         (dict(N=0), "multiples of 8"), (dict(rank=0), "rank"), (dict(rank=129), "rank"), (dict(R=0), "adapters"),
         (dict(R=65536), "adapters"), (dict(ldx=56), "rows"), (dict(ldx=68), "rows"), (dict(plan=None), "plan"),
         (dict(a=None), "null"), (dict(b=None), "null"), (dict(x=None), "rows")]


@pytest.mark.parametrize("kw,msg", SIZES + [(dict(ldo=120), "rows"), (dict(ldbase=0), "rows"), (dict(out=None), "rows")])
def test_forward_refusals(kw, msg):
    buf, p = pointer()
    rc, text = forward(p, **kw)
    assert rc == _lib.ERR_ARG and msg in text, text
    rc, text = forward(p)  # everything else is in order: only the workspace is missing
    assert rc == _lib.ERR_ARG and "workspace" in text


@pytest.mark.parametrize("kw,msg", SIZES + [(dict(ldgo=64), "rows"), (dict(lddx=8), "rows"), (dict(hidden=None), "hidden")])
def test_backward_refusals(kw, msg):
    buf, p = pointer()
    rc, text = backward(p, **kw)
    assert rc == _lib.ERR_ARG and msg in text, text
    rc, text = backward(p)
    assert rc == _lib.ERR_ARG and "workspace" in text


def test_misaligned_pointers_are_refused():
    buf, p = pointer()
    for name in ("x", "a", "b", "base", "out"):
        rc, text = forward(p, **{name: p + 8})
        assert rc == _lib.ERR_ARG and "aligned" in text, name
    for kw in (dict(scales=p + 2), dict(plan=p + 4), dict(hidden=p + 16), dict(ws=p + 16, n=1 << 20), dict(ws=p, n=16)):
        rc, text = forward(p, **kw)
        assert rc == _lib.ERR_ARG and "aligned" in text, kw
    for name in ("go", "dx", "da", "db"):
        rc, text = backward(p, **{name: p + 8})
        assert rc == _lib.ERR_ARG and "aligned" in text, name


def test_sizes_of_refused_problems_are_none():
    lib = _lib.lib()
    assert lib.h3b_adapter_plan_ints(10, 0) == 0 and lib.h3b_adapter_plan_ints(-1, 1) == 0 and lib.h3b_adapter_plan_ints(10, 3) > 10
    assert lib.h3b_low_rank_hidden_bytes(10, 0) == 0 and lib.h3b_low_rank_hidden_bytes(10, 129) == 0
    assert lib.h3b_low_rank_hidden_bytes(2 ** 40, 8) == 0 and lib.h3b_low_rank_hidden_bytes(10, 9) >= 10 * 16 * 2
    for bad in ((-1, 64, 64, 8, 1), (4, 4, 64, 8, 1), (4, 64, 60, 8, 1), (4, 64, 64, 200, 1), (4, 64, 64, 8, 0)):
        assert lib.h3b_low_rank_workspace_bytes(*bad, 1) == 0 and lib.h3b_low_rank_workspace_bytes(*bad, 0) == 0


def test_plan_refusals():
    lib = _lib.lib()
    buf, p = pointer()
    for args in ((p, 4, 0, p, 100), (p, 4, 70000, p, 100), (None, 4, 1, p, 100), (p, 4, 1, None, 100), (p, 4, 1, p + 4, 100),
                 (p, 4, 1, p, 3)):
        assert lib.h3b_adapter_plan(*args, None) == _lib.ERR_ARG, args
    for args, kw in (((torch.zeros(4, 1, dtype=torch.int32), 1), {}), ((torch.zeros(4), 1), {}), (([(0, 1, 0)], 1), {}),
                     (([(0, 9, 0)], 1), dict(count=4, device="cuda")), (([(0, 2, 1)], 1), dict(count=4, device="cuda")),
                     ((torch.zeros(4, dtype=torch.int32), 0), {}), ((torch.zeros(4, dtype=torch.int32), 1), dict(count=4))):
        with pytest.raises(ValueError):
            ad.plan(*args, **kw)
    with pytest.raises(RuntimeError, match="CUDA"):
        ad.plan(torch.zeros(4, dtype=torch.int32), 1)


def test_cpu_tensors_are_refused():
    x, a, b = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(16, 8, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ad.low_rank(x, a, b)


def test_formulas_against_differences():
    """The gradients of the 64-bit form are those of its outputs: out is linear in x, a and b each."""
    g = torch.Generator().manual_seed(0)
    x, a, b, do = (torch.randn(s, generator=g).to(torch.bfloat16) for s in ((20, 16), (2, 4, 16), (2, 24, 4), (20, 24)))
    rows = torch.randint(-1, 2, (20,), generator=g)
    scales = torch.tensor([0.5, 2.0])
    (dx, da, db), _ = ref.backward(do, x, a, b, rows, scales)
    for i, grad in enumerate((dx, da, db)):
        d = torch.randn(grad.shape, generator=g).to(torch.bfloat16)
        ops = [x, a, b]
        y0, _ = ref.forward(*ops, rows, scales)
        moved = list(ops)
        moved[i] = d
        y1, _ = ref.forward(*moved, rows, scales)  # linear: the value at d is the difference along d
        assert abs(float((y1 * do.double()).sum()) - float((grad * d.double()).sum())) < 1e-9 * float((y1 * do.double()).abs().sum())
