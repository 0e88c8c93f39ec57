"""Argument checks of the rotary embedding from positions and of cross attention that need no device."""
import ctypes
import math

import pytest
import torch

from minimax_h3_turbo_b200 import _lib
from minimax_h3_turbo_b200.h3 import cross, rope


def err(rc):
    return rc, _lib.lib().h3b_last_error().decode()


def buffer(n):
    buf = ctypes.create_string_buffer(n + 256)
    return buf, ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256


def rope_operand(p, s=4, heads=2):
    return (ctypes.c_int64 * 13)(p, p, p, s, 0, 128, 64, 0, 128, 64, 0, 3, heads)


def call_rope(q, k=None, dtype=_lib.BF16, b=1, d=64, sections=(8, 8, 8), pos=_lib.FP32, pairing=0, inv=1):
    sec = (ctypes.c_int32 * max(1, len(sections)))(*sections)
    return err(_lib.lib().h3b_rope_axes(ctypes.addressof(q) if q else None, ctypes.addressof(k) if k else None, dtype, b, d,
                                        inv, sec, len(sections), pos, pairing, 0, None))


def test_rope_axes_argument_errors():
    keep, p = buffer(4096)
    q = rope_operand(p)
    for kw, word in ((dict(q=None), "both null"), (dict(q=q, dtype=_lib.FP8_E4M3), "dtype"), (dict(q=q, pos=_lib.FP16), "positions"),
                     (dict(q=q, pairing=2), "pairing"), (dict(q=q, sections=()), "axes"), (dict(q=q, sections=(1,) * 9), "axes"),
                     (dict(q=q, sections=(-1, 8)), "negative"), (dict(q=q, sections=(33,)), "sections"), (dict(q=q, b=-1), "sections"),
                     (dict(q=q, inv=None), "inv_freq"), (dict(q=rope_operand(p, s=-1)), "S >= 0"), (dict(q=rope_operand(0)), "null"),
                     (dict(q=rope_operand(p, heads=0)), "heads")):
        rc, msg = call_rope(**kw)
        assert rc == _lib.ERR_ARG and word in msg, (kw, rc, msg)
    assert call_rope(q=q, b=0)[0] == _lib.OK  # nothing to do
    assert call_rope(q=rope_operand(0, s=0))[0] == _lib.OK


def call_cross(p, dtype=_lib.BF16, sizes=(1, 4, 8, 2, 1, 64), scale=0.125, mask=None, kind=0, stride=64, ws=None, nws=0, base=None):
    t = (ctypes.c_int64 * 4)(p if base is None else base, 0, stride, 64)
    a = ctypes.addressof(t)
    return err(_lib.lib().h3b_cross_attention(a, a, a, a, dtype, *sizes, scale, None, mask, kind, 8, None, ws, nws, None))


def test_cross_attention_argument_errors():
    keep, p = buffer(4096)
    for kw, word in ((dict(dtype=_lib.FP32), "bf16 or fp16"), (dict(sizes=(1, 4, 8, 3, 2, 64)), "key heads"),
                     (dict(sizes=(1, 4, 8, 129, 1, 64)), "128 times"), (dict(sizes=(1, -4, 8, 2, 1, 64)), "negative"),
                     (dict(sizes=(1, 4, 8, 2, 1, 60)), "multiple of 8"), (dict(sizes=(1, 4, 8, 2, 1, 136)), "at most 128"),
                     (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
                     (dict(kind=7), "mask kind"), (dict(kind=_lib.MASK_BOOL), "mask"), (dict(stride=60), "strides"),
                     (dict(base=p + 8), "aligned"), (dict(kind=_lib.MASK_BIAS, mask=p), "workspace")):
        rc, msg = call_cross(p, **kw)
        assert rc == _lib.ERR_ARG and word in msg, (kw, rc, msg)
    assert call_cross(p, sizes=(0, 4, 8, 2, 1, 64))[0] == _lib.OK
    assert call_cross(p, sizes=(1, 0, 8, 2, 1, 64))[0] == _lib.OK


def test_cross_backward_needs_lse():
    keep, p = buffer(4096)
    t = (ctypes.c_int64 * 4)(p, 0, 64, 64)
    a = ctypes.addressof(t)
    L = _lib.lib()
    n = L.h3b_cross_attention_workspace_bytes(1, 4, 8, 2, 1, 64, 0, 1)
    assert n > 0
    hold, w = buffer(n)
    rc, msg = err(L.h3b_cross_attention_backward(a, a, a, a, a, None, a, a, a, _lib.BF16, 1, 4, 8, 2, 1, 64, 0.125, None, None,
                                                 0, 0, w, n, None))
    assert rc == _lib.ERR_ARG and "lse" in msg


def test_python_layer_refuses_cpu_tensors_and_bad_names():
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        cross.cross_attention(q, q, q)
    with pytest.raises(RuntimeError):
        rope.rope_axes(q, None, torch.zeros(4, 3), torch.ones(16))
    with pytest.raises(ValueError):
        rope.rope_axes(None, None, None, torch.ones(16))
    with pytest.raises(ValueError):
        rope.rope_axes(q, None, torch.zeros(4, 3), torch.ones(16), pairing="thirds")
