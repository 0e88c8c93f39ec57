"""Rules that the cross-attention kernels' sources keep, read as text."""
import re
from pathlib import Path

import numpy as np
import pytest

CSRC = Path(__file__).resolve().parent.parent / "minimax-h3-turbo_b200" / "csrc"
FILES = sorted(CSRC.glob("cross_*.cuh"))


def code(path):
    return re.sub(r"//.*", "", path.read_text())


@pytest.mark.parametrize("path", FILES, ids=lambda p: p.name)
def test_no_read_only_loads_where_a_launch_begins_early(path):
    """These kernels begin while the one before them may still write what they read: the read-only path is not theirs."""
    assert not re.search(r"__ldg|ld\.global\.nc|__restrict__", code(path))


def test_every_kernel_that_begins_early_waits():
    text = "".join(code(p) for p in FILES)
    launched = set(re.findall(r'cross_launch_after\("(\w+)"', text))
    assert len(launched) >= 7
    for name in launched:
        body = text[re.search(r"__global__[^;{]*\b%s\(" % name, text).end():]
        assert "after_previous()" in body[:body.index("\n}\n")], name


def exp2_of_the_fma_pipe(x, tail):
    """f2_exp2 of cross_common.cuh step by step in fp32, with its own coefficients (a fused multiply-add is a product and a sum in
    fp64, rounded once: the sum of two fp64 roundings is far below half a step of fp32)."""
    f32 = np.float32
    text = code(CSRC / "cross_common.cuh")
    body = text[text.index("f2_exp2(float xa"):]
    coef = [f32(a) for a, b in re.findall(r"f2\(([0-9.]+)f, ([0-9.]+)f\)", body[:body.index("f2_split")])
            if float(a) <= 1 and a == b]
    assert len(coef) == 5
    fma = lambda a, b, c: (a.astype(np.float64) * np.float64(b) + np.asarray(c, np.float64)).astype(f32)  # noqa: E731
    with np.errstate(invalid="ignore"):
        x = np.maximum(x, f32(-127 if tail else -126))  # NaN stays (with a tail)
        t = x + f32(12582912)
        f = fma(t - f32(12582912), -1.0, x)
        p = fma(f, coef[0], coef[1])
        for c in coef[2:]:
            p = (p.astype(np.float64) * f.astype(np.float64) + np.float64(c)).astype(f32)
        n = t.view(np.int32) << 23
        if tail:
            return p * (n + np.int32(127 << 23)).view(f32)
        return (p.view(np.int32) + n).view(f32)


@pytest.mark.parametrize("tail", [False, True])
def test_exp2_polynomial(tail):
    """Within the 2.7e-6 that the bounds of the numerics tests count, over the range in use (up to 16) and at the steps of it."""
    x = np.concatenate([np.linspace(-126, 16, 2_000_001), np.arange(-126, 16, 0.5), np.arange(-126, 16, 0.5) + 1e-6,
                        np.arange(-125, 17, 0.5) - 1e-6]).astype(np.float32)
    want = np.exp2(x.astype(np.float64))
    rel = np.abs(exp2_of_the_fma_pipe(x, tail).astype(np.float64) / want - 1)
    assert rel[x > -125.9].max() <= 2.7e-6
    assert rel.max() <= (1.0 if tail else 2.7e-6)  # the last half step may be 0 with a tail
    low = np.array([-126.6, -127, -128, -1000, -np.inf], np.float32)
    got = exp2_of_the_fma_pipe(low, tail)
    assert (got == 0).all() if tail else ((got > 0) & (got <= 2.0 ** -125.9)).all()
    if tail:
        assert np.isnan(exp2_of_the_fma_pipe(np.array([np.nan], np.float32), True)).all()
