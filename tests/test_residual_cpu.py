"""Arguments of the residual's norm that must come back as an error before anything is launched."""
import ctypes

import pytest
import torch

from minimax_h3_turbo_b200 import _lib
from minimax_h3_turbo_b200.h3 import residual as rs


def pointer(n=1 << 14):
    buf = ctypes.create_string_buffer(n)
    return buf, ctypes.addressof(buf) + (-ctypes.addressof(buf)) % 256


def forward(p, **kw):
    """Every call here carries something that is refused: nothing is ever launched."""
    a = {"x": p, "ldx": 512, "y": p, "ldy": 512, "dtype": _lib.BF16, "M": 4, "K": 512, "w": p, "wd": _lib.BF16, "gate": p, "shift": p,
         "scale": p, "ldm": 512, "rows": 2, "md": _lib.BF16, "segs": None, "n": 0, "tok": None, "t": p, "ldt": 512, "h": p, "ldh": 512,
         "codes": p, "ldc": 512, "scales": p, "rstd": p, **kw}
    segs = None if a["segs"] is None else (ctypes.c_int32 * len(a["segs"]))(*a["segs"])
    rc = _lib.lib().h3b_residual_norm(a["x"], a["ldx"], a["y"], a["ldy"], a["dtype"], a["M"], a["K"], a["w"], a["wd"], 1e-5, a["gate"],
                                      a["shift"], a["scale"], a["ldm"], a["rows"], a["md"], segs, a["n"], a["tok"], a["t"], a["ldt"],
                                      a["h"], a["ldh"], a["codes"], a["ldc"], a["scales"], a["rstd"], None, 0, None)
    return rc, _lib.lib().h3b_last_error().decode()


def backward(p, **kw):
    a = {"dt": p, "lddt": 512, "dh": p, "lddh": 512, "t": p, "ldt": 512, "rstd": p, "dtype": _lib.BF16, "M": 4, "K": 512, "w": p,
         "wd": _lib.BF16, "gate": p, "scale": p, "ldm": 512, "rows": 2, "md": _lib.BF16, "segs": None, "n": 0, "tok": None, "dx": p,
         "lddx": 512, "dy": p, "lddy": 512, "dw": p, **kw}
    rc = _lib.lib().h3b_residual_norm_backward(a["dt"], a["lddt"], a["dh"], a["lddh"], a["t"], a["ldt"], a["rstd"], a["dtype"], a["M"],
                                               a["K"], a["w"], a["wd"], a["gate"], a["scale"], a["ldm"], a["rows"], a["md"], None,
                                               a["n"], a["tok"], a["dx"], a["lddx"], a["dy"], a["lddy"], a["dw"], None, 0, None)
    return rc, _lib.lib().h3b_last_error().decode()


COMMON = [(dict(dtype=_lib.FP32), "bf16 or fp16"), (dict(M=-1), "width"), (dict(K=0), "width"), (dict(K=12), "width"),
          (dict(w=None), "weight"), (dict(wd=_lib.FP8_E4M3), "weight"), (dict(md=_lib.INT32), "gate"), (dict(rows=0), "gate"),
          (dict(ldm=504), "rows"), (dict(n=17), "segments"), (dict(n=1), "segments"), (dict(t=None), "rows"), (dict(ldt=508), "rows")]


@pytest.mark.parametrize("kw,msg", COMMON + [
    (dict(shift=None), "together"), (dict(x=None), "rows"), (dict(ldy=8), "rows"), (dict(K=264, ldm=264), "256"),
    (dict(ldc=520), "codes"), (dict(scales=None), "codes"), (dict(segs=[0, 4, 2], n=1), "segment"),
    (dict(segs=[-1, 4, 0], n=1), "segment"), (dict(segs=[3, 2, 0], n=1), "segment")])
def test_forward_refusals(kw, msg):
    buf, p = pointer()
    rc, text = forward(p, **kw)
    assert rc == _lib.ERR_ARG and msg in text, text


@pytest.mark.parametrize("kw,msg", COMMON + [
    (dict(dh=None), "rows"), (dict(lddt=8), "rows"), (dict(rstd=None), "rstd"), (dict(gate=None), "gate")])
def test_backward_refusals(kw, msg):
    buf, p = pointer()
    rc, text = backward(p, **kw)
    assert rc == _lib.ERR_ARG and msg in text, text


def test_misaligned_pointers_and_wide_rows_are_refused():
    buf, p = pointer()
    for name in ("x", "y", "w", "gate", "shift", "scale", "t", "h", "codes"):
        rc, text = forward(p, **{name: p + 8})
        assert rc == _lib.ERR_ARG and "aligned" in text, name
    for name in ("scales", "rstd", "tok"):
        rc, text = forward(p, **{name: p + 2})
        assert rc == _lib.ERR_ARG and "aligned" in text, name
    for name in ("dt", "dh", "t", "dx", "dy", "dw"):
        rc, text = backward(p, **{name: p + 8})
        assert rc == _lib.ERR_ARG and "aligned" in text, name
    for call in (forward, backward):
        assert call(p, K=16640)[0] == _lib.ERR_UNSUPPORTED and call(p, M=2 ** 31)[0] == _lib.ERR_UNSUPPORTED
    assert _lib.lib().h3b_residual_norm_workspace_bytes(4, 12, 1) == 0 and _lib.lib().h3b_residual_norm_workspace_bytes(-1, 8, 1) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        rs.residual_norm(x, x, x[0], 1e-5)


def test_workspace_is_of_the_device_that_the_call_runs_on(monkeypatch):
    """GPUs with other numbers of SMs take other workspaces: the size is asked with the stream's device current, and kept for it alone."""
    import contextlib
    import types

    current, asked, passed = [0], [], []

    @contextlib.contextmanager
    def device(d):
        before, current[0] = current[0], d.index
        yield
        current[0] = before

    def size(m, k, backward):
        asked.append(current[0])
        return 1000 * (current[0] + 1)

    monkeypatch.setattr(rs._lib, "lib", lambda: types.SimpleNamespace(h3b_residual_norm_workspace_bytes=size))
    monkeypatch.setattr(rs._lib, "raw_stream", lambda index: 0)
    monkeypatch.setattr(rs.torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(rs.torch.cuda, "device", device)
    empty = torch.empty
    monkeypatch.setattr(rs.torch, "empty", lambda n, dtype, device: empty(n, dtype=dtype))
    rs._workspace_bytes.cache_clear()
    for index in (0, 1, 1, 0):
        p = rs._Problem.__new__(rs._Problem)
        p.m, p.k, p.dev = 16, 512, types.SimpleNamespace(index=index)
        p.launch(lambda ws, n, stream: passed.append(n) or 0, (), True)
    rs._workspace_bytes.cache_clear()
    assert passed == [1000, 2000, 2000, 1000] and asked == [0, 1]
