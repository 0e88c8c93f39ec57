"""Per-head q/k RMSNorm + split-half rotary embedding (h3turbo/h3/layout.py:265-356).

`norm_rope_` keeps the reference's signature and runs the fused kernel `h3b_qk_norm_rope`, which is bit-identical to the
reference's "torch" form of comfy_kitchen's fused op (rms_norm_fused_order, layout.py:309-326, then the fp32 rotation):
impl "auto", "b200", "ck" and "torch" all mean that kernel.  ComfyUI's portable "eager" formula (other roundings) is not
built, and neither is a CPU or fp32 path: such calls raise RuntimeError.

`rope_axes` is the rotary embedding alone, from positions on several axes instead of cos/sin tables: out of place, for q
and k of different lengths and head counts, bf16/fp16/fp32, in both directions (kernel `h3b_rope_axes`).
"""
from __future__ import annotations

import ctypes
from array import array
from typing import Optional, Sequence, Tuple

import torch
from torch.autograd import forward_ad

from .. import _lib


def rope_angles(position_ids: torch.Tensor, inv_freq: torch.Tensor, device) -> torch.Tensor:
    """[S, 3] positions -> [S, 3 F] fp32 angles: all t frequencies, then h, then w (layout.py:265-273)."""
    pos = position_ids.to(torch.float32).to(device)
    ang = pos.unsqueeze(-1) * inv_freq.to(device=device, dtype=torch.float32).view(1, 1, -1)
    return ang.reshape(pos.shape[0], -1)


def _kernel_ok(x: torch.Tensor) -> bool:
    d = x.shape[-1]
    return x.is_cuda and x.dtype in (torch.bfloat16, torch.float16) and d in (32, 64, 128, 256)


def _fused(q: Optional[torch.Tensor], k: Optional[torch.Tensor], wq, wk, eps: float, cos: torch.Tensor,
           sin: torch.Tensor) -> None:
    ref = q if q is not None else k
    s, heads, d = ref.shape
    for t in (q, k):
        if t is not None and (t.shape != ref.shape or t.dtype != ref.dtype or t.stride(2) != 1 or t.stride(1) != d):
            raise ValueError("q and k must be [S, heads, D] views with contiguous heads and the same shape/dtype")
    half = cos.shape[1]
    if sin.shape != cos.shape or cos.shape[0] != s or cos.stride(1) != 1 or sin.stride() != cos.stride():
        raise ValueError("cos/sin must be [S, half] with unit column stride and equal strides")
    if cos.device != ref.device:
        raise ValueError("cos/sin must be on the q/k device")
    ws = [None if w is None else w.contiguous() for w in (wq, wk)]
    wdt = _lib.act_code((ws[0] if ws[0] is not None else ws[1]).dtype)
    if ws[0] is not None and ws[1] is not None and ws[0].dtype != ws[1].dtype:
        ws[1] = ws[1].to(ws[0].dtype)
    L = _lib.lib()
    _lib.check(L.h3b_qk_norm_rope(_lib.ptr(q), 0 if q is None else q.stride(0), _lib.ptr(k), 0 if k is None else k.stride(0),
                                  _lib.act_code(ref.dtype), s, heads, d, _lib.ptr(ws[0]), _lib.ptr(ws[1]), wdt, float(eps),
                                  cos.data_ptr(), sin.data_ptr(), cos.stride(0), _lib.act_code(cos.dtype), half,
                                  _lib.stream_ptr(ref.device)), "qk_norm_rope")


@torch.no_grad()
def norm_rope_(q: torch.Tensor, k: torch.Tensor, wq: torch.Tensor, wk: torch.Tensor, eps: float, cos: torch.Tensor,
               sin: torch.Tensor, impl: str = "auto", table=None, chunk: int = 1024) -> None:
    """In place on [S, heads, D] views: per-head RMSNorm, then split-half rotation of the leading 2 * half dims
    (layout.py:329-356; `table` and `chunk` are accepted for the reference's signature and ignored)."""
    if impl not in ("auto", "b200", "ck", "torch", "eager"):
        raise ValueError(f"rope_impl must be auto/b200/ck/torch/eager, got {impl!r}")
    if impl == "eager":
        raise RuntimeError("rope_impl 'eager' (ComfyUI's portable formula) is not built; 'torch' / 'b200' run the fused "
                           "kernel, bit-identical to the reference's 'torch' form")
    if not all(t is None or _kernel_ok(t) for t in (q, k)):
        raise RuntimeError("the fused q/k norm+RoPE kernel needs bf16/fp16 CUDA tensors with head_dim 32/64/128/256 "
                           "(there is no CPU or fp32 path)")
    _fused(q, k, wq, wk, eps, cos, sin)


# ------------------------------------------------------------------------------------------- rotary from positions
_POS_CODES = {torch.float32: _lib.FP32, torch.int32: _lib.INT32, torch.int64: _lib.INT64}


def no_tangents(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """Raises where one of these carries a forward-mode tangent (requires_grad does not tell): the kernels would lose it."""
    if getattr(forward_ad, "_current_level", 0) >= 0 and \
            any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivatives")


_section_tables = {}  # tuple of sections -> the C table of it


def _section_table(sections: Tuple[int, ...]):
    t = _section_tables.get(sections)
    if t is None:
        if len(_section_tables) > 256:
            _section_tables.clear()
        t = _section_tables[sections] = (ctypes.c_int32 * max(1, len(sections)))(*sections)
    return t


def _rope_operand(arg: array, x: torch.Tensor, pos: Optional[torch.Tensor], axes: int, name: str, keep: list) -> torch.Tensor:
    """Appends struct h3b_rope_operand of one side, x [B, S, heads, D] or [S, heads, D], to `arg` and copies it had to make
    to `keep`; the output."""
    if x.dim() == 4:
        b, s, h, d = x.shape
        sb, ss, sh, sd = x.stride()
    elif x.dim() == 3:
        b, sb = 1, 0
        s, h, d = x.shape
        ss, sh, sd = x.stride()
    else:
        raise ValueError(f"{name} must be [B, S, heads, D] or [S, heads, D], got {tuple(x.shape)}")
    if pos is None or pos.device != x.device or pos.dtype not in _POS_CODES:
        raise ValueError(f"{name}: positions must be fp32, int32 or int64 on {x.device}")
    if pos.dim() == 3:
        pn, n, pa = pos.shape
        pb, ps, stride = pos.stride()
    elif pos.dim() == 2:
        pn, pb = 1, 0
        n, pa = pos.shape
        ps, stride = pos.stride()
    else:
        pn = n = pa = stride = -1
    if pn not in (1, b) or n != s or pa != axes:
        raise ValueError(f"{name}: positions must be [{s}, {axes}] or [{b}, {s}, {axes}], got {tuple(pos.shape)}")
    if stride != 1 and axes > 1:
        pos = pos.contiguous()
        keep.append(pos)
        pb, ps = s * axes, axes
    if sd != 1 and d > 1:
        x = x.contiguous()
        keep.append(x)
        sb, ss, sh = s * h * d, h * d, d
    y = torch.empty_like(x) if x.is_contiguous() else torch.empty_like(x, memory_format=torch.contiguous_format)
    arg.extend((x.data_ptr(), y.data_ptr(), pos.data_ptr(), s, sb if b > 1 else 0, ss, sh, s * h * d, h * d, d,
                pb if pn > 1 else 0, ps, h))
    return y


def _rope_axes(q, k, q_pos, k_pos, inv_freq, sections, pairing, inverse):
    ref = q if q is not None else k
    if not ref.is_cuda or (k is not None and not k.is_cuda):
        raise RuntimeError("rope_axes: CUDA tensors only (there is no CPU path)")
    dev, dt = ref.device, ref.dtype
    code = _lib.act_code(dt)
    if inv_freq.dim() != 1 or inv_freq.device != dev:
        raise ValueError(f"rope_axes: inv_freq must be 1-D on {dev}")
    first = q_pos if q is not None else k_pos
    axes = first.shape[-1] if first is not None and first.dim() in (2, 3) else 0
    if sections is None:  # every axis turns by all the frequencies, axis after axis
        sections, inv_freq = (inv_freq.shape[0],) * axes, inv_freq.repeat(axes)
    sections = tuple(sections)
    if len(sections) != axes or sum(sections) != inv_freq.shape[0]:
        raise ValueError(f"rope_axes: {axes} axes with {inv_freq.shape[0]} frequencies do not match sections {sections}")
    if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
        inv_freq = inv_freq.to(torch.float32).contiguous()
    arg, keep = array("q"), []
    yq = yk = None
    if q is not None:
        if k is not None:
            if k.dtype != dt or k.device != dev or k.dim() != q.dim() or k.shape[-1] != q.shape[-1] or \
                    (q.dim() == 4 and k.shape[0] != q.shape[0]):
                raise ValueError(f"rope_axes: q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} do not match")
            if k_pos is not None and first is not None and k_pos.dtype != first.dtype:
                raise ValueError("rope_axes: positions of q and k must have one dtype")
        yq = _rope_operand(arg, q, q_pos, axes, "q", keep)
    if k is not None:
        yk = _rope_operand(arg, k, k_pos, axes, "k", keep)
    at = arg.buffer_info()[0]
    args = (at if q is not None else None, None if k is None else at + 104 if q is not None else at, code,
            ref.shape[0] if ref.dim() == 4 else 1, ref.shape[-1], inv_freq.data_ptr(), _section_table(sections), axes,
            _POS_CODES[first.dtype], _lib.PAIRING[pairing], int(inverse))
    lib = _lib.lib()
    if dev.index == torch.cuda.current_device():
        rc = lib.h3b_rope_axes(*args, _lib.raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            rc = lib.h3b_rope_axes(*args, _lib.raw_stream(dev.index))
    if rc:
        _lib.check(rc, "rope_axes")
    return yq, yk


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_pos, k_pos, inv_freq, sections, pairing, inverse):
        ctx.save_for_backward(q_pos, k_pos, inv_freq)
        ctx.rest = (sections, pairing, inverse)
        return _rope_axes(q, k, q_pos, k_pos, inv_freq, sections, pairing, inverse)

    @staticmethod
    def backward(ctx, gq, gk):
        (q_pos, k_pos, inv_freq), (sections, pairing, inverse) = ctx.saved_tensors, ctx.rest
        if gq is None and gk is None:
            return (None,) * 8
        # where autograd records (second derivatives), the rotation back is one of its own
        turn = _RopeAxes.apply if torch.is_grad_enabled() else _rope_axes
        dq, dk = turn(gq, gk, q_pos, k_pos, inv_freq, sections, pairing, not inverse)
        return dq, dk, None, None, None, None, None, None


def rope_axes(q: Optional[torch.Tensor], k: Optional[torch.Tensor], positions: Optional[torch.Tensor],
              inv_freq: torch.Tensor, sections: Optional[Sequence[int]] = None, *,
              k_positions: Optional[torch.Tensor] = None, pairing: str = "half", inverse: bool = False
              ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Rotary embedding from positions on several axes (time, height, width), out of place -> (q', k').

    q, k: [B, S, heads, D] or [S, heads, D], one of them may be None; lengths and head counts may differ.  positions:
    [S, A] or [B, S, A] fp32, int32 or int64 for q (and for k, unless k_positions gives k's own).  Pair j of a head turns by
    positions[axis(j)] * inv_freq[j]: sections (n_0, ..., n_{A-1}) deals the sum(sections) frequencies out to the axes in
    order; None lets every axis turn by all of inv_freq, as rope_angles does.  pairing "half": channels (j, j + F), F the
    number of pairs, as norm_rope_ rotates; "adjacent": (2j, 2j + 1).  Channels >= 2 F are copied.  inverse=True turns back:
    the gradient's direction.  bf16, fp16 or fp32 (rounded once); differentiable in q and k (not in positions or inv_freq)."""
    if q is None and k is None:
        raise ValueError("rope_axes: q and k are both None")
    if pairing not in _lib.PAIRING:
        raise ValueError(f"pairing must be 'half' or 'adjacent', got {pairing!r}")
    k_positions = positions if k_positions is None else k_positions
    no_tangents("rope_axes", q, k, positions, k_positions, inv_freq)
    if torch.is_grad_enabled():
        if inv_freq.requires_grad or (positions is not None and positions.requires_grad) or \
                (k_positions is not None and k_positions.requires_grad):
            raise ValueError("rope_axes: positions and inv_freq have no gradient; detach them")
        if (q is not None and q.requires_grad) or (k is not None and k.requires_grad):
            return _RopeAxes.apply(q, k, positions, k_positions, inv_freq, sections, pairing, inverse)
    return _rope_axes(q, k, positions, k_positions, inv_freq, sections, pairing, inverse)
