"""Arguments of the cross-attention entry points that must come back as an error: checks that need no device."""
import ctypes
import subprocess
import sys

import pytest

from minimax_h3_turbo_b200 import _lib


def workspace_bytes(*args):
    """h3b_cross_attention_workspace_bytes in a process of its own (a signal in there is a result, not the end of the tests)."""
    code = ("import ctypes, sys; f = ctypes.CDLL(sys.argv[1]).h3b_cross_attention_workspace_bytes; f.restype = ctypes.c_size_t; "
            "f.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_int] * 5; print(f(*map(int, sys.argv[2:])))")
    path = _lib.lib()._name
    run = subprocess.run([sys.executable, "-c", code, path, *map(str, args)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run
    return int(run.stdout)


@pytest.mark.parametrize("hq,hkv", [(129, 1), (1, 2), (3, 2), (0, 1), (1, 0), (65537, 65537)])
@pytest.mark.parametrize("backward", [0, 1])
def test_workspace_of_refused_heads_is_none(hq, hkv, backward):
    assert workspace_bytes(1, 4, 8, hq, hkv, 64, 0, backward) == 0


def test_workspace_of_refused_sizes_is_none():
    for sizes in ((-1, 4, 8, 1, 1, 64), (1, -4, 8, 1, 1, 64), (1, 4, -8, 1, 1, 64), (1, 4, 8, 1, 1, 0), (1, 4, 8, 1, 1, 60),
                  (1, 4, 8, 1, 1, 136), (1, 2 ** 40, 8, 1, 1, 64), (1, 4, 2 ** 40, 1, 1, 64), (2 ** 33, 4, 8, 1, 1, 64),
                  (0, 4, 8, 1, 1, 64)):
        assert workspace_bytes(*sizes, _lib.MASK_BIAS, 1) == 0, sizes
    assert workspace_bytes(1, 4, 8, 128, 1, 64, 0, 1) > 0
