"""Rules that the cross-attention kernels' sources keep, read as text."""
import re
from pathlib import Path

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
