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


def tensor(p, b, s, h):
    return (ctypes.c_int64 * 4)(p, b, s, h)


def call(tensors, sizes, p, lens=None, mask=None, lse=None):
    """The forward call for four tensors, the backward call for eight (in the entry's order), with an additive mask and without
    the workspace that it needs: nothing is ever launched."""
    a = [ctypes.addressof(t) for t in tensors]
    rest = (_lib.BF16, *sizes, 0.125, lens, p if mask is None else mask, _lib.MASK_BIAS, 0)
    lse = p if lse is None else lse
    if len(a) == 4:
        rc = _lib.lib().h3b_cross_attention(*a, *rest, lse, None, 0, None)
    else:
        rc = _lib.lib().h3b_cross_attention_backward(*a[:5], lse, *a[5:], *rest, None, 0, None)
    assert rc == _lib.ERR_ARG
    return _lib.lib().h3b_last_error().decode()


@pytest.mark.parametrize("n", [4, 8])
def test_strides_of_zero_and_outputs_that_fold_are_refused(n):
    buf = ctypes.create_string_buffer(1 << 16)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    sizes = (2, 200, 200, 2, 2, 64)  # every extent above one
    fits = (200 * 128, 128, 64)
    assert "workspace" in call([tensor(p, *fits)] * n, sizes, p)
    assert "workspace" in call([tensor(p, 0, 0, 0)] * n, (1, 1, 1, 1, 1, 64), p)  # extents of one
    written = (3,) if n == 4 else (5, 6, 7)
    for i in range(n):
        for axis in range(3):
            for bad in (0, -64, 4) + ((56,) if i in written else ()):
                st = list(fits)
                st[axis] = bad
                ts = [tensor(p, *fits) for _ in range(n)]
                ts[i] = tensor(p, *st)
                assert "strides" in call(ts, sizes, p), (i, axis, bad)


@pytest.mark.parametrize("n", [4, 8])
def test_misaligned_vectors_are_refused(n):
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    ts, sizes = [tensor(p, 0, 64, 0)] * n, (1, 4, 8, 1, 1, 64)
    assert "workspace" in call(ts, sizes, p, lens=p + 4, mask=p + 4, lse=p + 4)
    for kw in (dict(lens=p + 2), dict(mask=p + 1), dict(lse=p + 2)):
        assert "4-byte aligned" in call(ts, sizes, p, **kw), kw


def test_misaligned_rope_pointers_are_refused():
    buf = ctypes.create_string_buffer(1 << 12)
    p = ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256
    sec = (ctypes.c_int32 * 1)(8)

    def call_rope(x, y, pos, inv, dtype, pos_dtype, second):
        op = (ctypes.c_int64 * 13)(x, y, pos, 4, 0, 128, 64, 0, 128, 64, 0, 1, 2)
        at = ctypes.addressof(op)
        rc = _lib.lib().h3b_rope_axes(None if second else at, at if second else None, dtype, 1, 64, inv, sec, 1, pos_dtype, 0,
                                      0, None)
        return rc, _lib.lib().h3b_last_error().decode()

    for second in (False, True):
        for dtype, size in ((_lib.BF16, 2), (_lib.FP16, 2), (_lib.FP32, 4)):
            for bad in ((p + size // 2, p, p, p), (p, p + size // 2, p, p), (p, p, p + 2, p), (p, p, p, p + 2)):
                rc, msg = call_rope(*bad, dtype, _lib.FP32, second)
                assert rc == _lib.ERR_ARG and "aligned" in msg, (dtype, bad, rc, msg)
            rc, msg = call_rope(p, p, p + 4, p, dtype, _lib.INT64, second)
            assert rc == _lib.ERR_ARG and "aligned" in msg
