"""The residual's addition with its root-mean-square norm and 8-bit output for the next W4A8 linear, with gradients.

    t = x + gate y  (the stream, rounded to its type)    h = t rsqrt(mean t^2 + eps) w (1 + scale) + shift
    codes, scales = h rotated by blocks of 256 in 8 bits, a scale per row

One pass over the stream where `block.gate_` and `block.prenorm_linear` take two (the end of one sub-layer and the entry of the
next: _gate_, _rms, _scale_shift_ and the activation half of the linear, h3turbo/h3/model.py:64-66, 106-115, 239-241,
qlinear.py:267-303).  Everything between t and the outputs is held in 32 bits, so the results are not bit for bit those of the two
passes, which round to the stream's type after every step.  Kernels: h3b_residual_norm and h3b_residual_norm_backward
(include/h3b.h).  bf16/fp16 CUDA tensors only; there is no CPU path.
"""
from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from .. import _lib
from . import block as blk
from . import qlinear as ql
from .adapters import _overlap, _written
from .rope import no_tangents
from .types import W4A8Weight, Weight


class ResidualNorm(NamedTuple):
    """What `residual_norm` gives: the stream t, and what was asked for (else None)."""

    x: torch.Tensor                   # [M, K] t
    rstd: Optional[torch.Tensor]      # [M] fp32, with hidden: the row factors rsqrt(mean t^2 + eps), which the gradients take
    hidden: Optional[torch.Tensor]    # [M, K] h
    codes: Optional[torch.Tensor]     # [M, K] int8, of h rotated
    scales: Optional[torch.Tensor]    # [M, 1] fp32


@lru_cache(maxsize=4096)
def _workspace_bytes(m: int, k: int, backward: bool, device: int) -> int:
    """Asked with `device` current: the number of SMs counts."""
    return _lib.lib().h3b_residual_norm_workspace_bytes(m, k, backward)


def _rows(t: torch.Tensor) -> torch.Tensor:
    """t itself when the kernels can read its rows in place, or a copy."""
    if t.is_contiguous():  # rows of multiples of 8
        return t if t.data_ptr() % 16 == 0 else t.clone()
    if t.stride(1) == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (t.stride(0) % 8 == 0 and t.stride(0) >= t.shape[1])):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ld(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _code(t: Optional[torch.Tensor]) -> int:
    return _lib.BF16 if t is None else _lib.act_code(t.dtype)


_tables = {}  # (segments, rows, modulation rows) -> the C table of them and its length


def _segments(segments, m: int, n_rows: int, device):
    """block._segment_args, its tables of plain numbers kept (a table is a few numbers by value; making one takes microseconds)."""
    try:
        key = (tuple(segments), m, n_rows)
        found = _tables.get(key)
    except TypeError:  # per-token rows
        return blk._segment_args(segments, m, n_rows, device)
    if found is None:
        table, n, rows = blk._segment_args(segments, m, n_rows, device)
        if rows is not None or any(type(v) is not int for seg in key[0] for v in seg):
            return table, n, rows
        if len(_tables) > 256:
            _tables.clear()
        found = _tables[key] = (table, n)
    return (*found, None)


class _Problem:
    """Checked stream, weight and modulation of one call."""

    def __init__(self, x, weight, gate, shift, scale, segments):
        if not x.is_cuda or x.dtype not in (torch.bfloat16, torch.float16):
            raise RuntimeError(f"residual_norm: the b200 kernels take bf16/fp16 CUDA rows, got {x.dtype} on {x.device} (there is "
                               "no CPU or fp32 path)")
        if x.dim() != 2 or x.shape[1] % 8 or not 8 <= x.shape[1] <= _lib.MAX_RESIDUAL:
            raise ValueError(f"residual_norm: the stream must be [M, K] with K a multiple of 8 up to {_lib.MAX_RESIDUAL}, got "
                             f"{tuple(x.shape)}")
        self.shape = x.shape
        self.m, self.k = x.shape
        self.dev, self.dt, self.code = x.device, x.dtype, _lib.act_code(x.dtype)
        if weight.shape != (self.k,) or weight.device != self.dev:
            raise ValueError(f"residual_norm: weight must be [{self.k}] on {self.dev}, got {tuple(weight.shape)} on {weight.device}")
        self.w = weight.contiguous()
        if self.w.data_ptr() % 16:
            self.w = self.w.clone()
        self.w_code = _lib.act_code(self.w.dtype)
        self.gate, self.shift, self.scale = gate, shift, scale
        first = gate if gate is not None else shift if shift is not None else scale
        if first is None:
            self.mod_args = (0, 0, _lib.BF16, None, 0, None)
            return
        n_rows, dt, ld = first.shape[0] if first.dim() == 2 else -1, first.dtype, _ld(first) if first.dim() == 2 else 0
        alike = True  # read as they are
        for t in (gate, shift, scale):
            if t is None:
                continue
            if t.dim() != 2 or t.shape[1] != self.k or t.shape[0] != n_rows or n_rows < 1 or t.device != self.dev:
                raise ValueError(f"residual_norm: gate, shift and scale must be [rows, {self.k}] alike on {self.dev}, of a row at least")
            alike = alike and t.dtype is dt and t.is_contiguous() and t.data_ptr() % 16 == 0
        if not alike:
            mods = [t for t in (gate, shift, scale) if t is not None]
            if any(t.dtype != dt for t in mods):
                dt, mods = torch.float32, [t.float() for t in mods]
            mods = [_rows(t) for t in mods]
            ld = _ld(mods[0])
            if any(_ld(t) != ld for t in mods):
                mods = [_rows(t.contiguous()) for t in mods]
                ld = self.k
            it = iter(mods)
            self.gate, self.shift, self.scale = (None if t is None else next(it) for t in (gate, shift, scale))
        table, n_seg, self.token_rows = _segments(segments or (), self.m, n_rows, self.dev)
        self.mod_args = (ld, n_rows, _lib.act_code(dt), table, n_seg, _lib.ptr(self.token_rows))

    def rows(self, t: torch.Tensor, name: str) -> torch.Tensor:
        if t.shape != self.shape or t.dtype is not self.dt or t.device != self.dev:
            raise ValueError(f"residual_norm: {name} must be {(self.m, self.k)} {self.dt} on {self.dev}, got {tuple(t.shape)} "
                             f"{t.dtype} on {t.device}")
        return _rows(t)

    def launch(self, fn, args, backward: bool) -> None:
        if self.dev.index == torch.cuda.current_device():
            rc = self._call(fn, args, backward)
        else:
            with torch.cuda.device(self.dev):
                rc = self._call(fn, args, backward)
        if rc:
            _lib.check(rc, "residual_norm")

    def _call(self, fn, args, backward: bool) -> int:
        index = self.dev.index
        n = _workspace_bytes(self.m, self.k, backward, index) if backward else 0
        ws = torch.empty(n, dtype=torch.uint8, device=self.dev) if n else None
        return fn(*args, _lib.ptr(ws), n, _lib.raw_stream(index))


def _forward(p: _Problem, x, y, eps, codes, hidden, out) -> ResidualNorm:
    x, y = p.rows(x, "x"), p.rows(y, "y")
    m, k, dev = p.m, p.k, p.dev
    t, ldt = (torch.empty(m, k, dtype=p.dt, device=dev), k) if out is None else (out, _ld(out))
    h = rstd = q = s = None
    if hidden:
        h = torch.empty_like(t, memory_format=torch.contiguous_format)
        rstd = torch.empty(m, dtype=torch.float32, device=dev)
    if codes:
        q = torch.empty(m, k, dtype=torch.int8, device=dev)
        s = torch.empty(m, 1, dtype=torch.float32, device=dev)
    if m:
        ptr = _lib.ptr
        p.launch(_lib.lib().h3b_residual_norm,
                 (x.data_ptr(), _ld(x), y.data_ptr(), _ld(y), p.code, m, k, p.w.data_ptr(), p.w_code, eps, ptr(p.gate),
                  ptr(p.shift), ptr(p.scale), *p.mod_args, t.data_ptr(), ldt, ptr(h), k, ptr(q), k, ptr(s), ptr(rstd)), False)
    return ResidualNorm(t, rstd, h, q, s)


def _backward(dt, dh, t, rstd, weight, gate, scale, segments, need_w):
    p = _Problem(t, weight, gate, None, scale, segments)
    t, dh = p.rows(t, "x"), p.rows(dh, "dh")
    dt = None if dt is None else p.rows(dt, "dt")
    if rstd is None or rstd.shape != (p.m,) or rstd.dtype != torch.float32 or rstd.device != p.dev:
        raise ValueError(f"residual_norm: rstd must be fp32 [{p.m}] on {p.dev} (residual_norm gives it with hidden=True)")
    rstd = rstd.contiguous()
    dx = torch.empty(p.m, p.k, dtype=p.dt, device=p.dev)
    dy = torch.empty_like(dx) if gate is not None else dx
    dw = torch.empty(p.k, dtype=p.w.dtype, device=p.dev) if need_w else None
    if p.m or need_w:
        p.launch(_lib.lib().h3b_residual_norm_backward,
                 (_lib.ptr(dt), _ld(dt), dh.data_ptr(), _ld(dh), t.data_ptr(), _ld(t), rstd.data_ptr(), p.code, p.m, p.k,
                  p.w.data_ptr(), p.w_code, _lib.ptr(p.gate), _lib.ptr(p.scale), *p.mod_args, dx.data_ptr(), p.k,
                  None if dy is dx else dy.data_ptr(), p.k, _lib.ptr(dw)), True)
    return dx, dy, dw


class _ResidualNormGrads(torch.autograd.Function):
    """The gradients where autograd records: they have no derivatives of their own, and say so when one is asked for."""

    @staticmethod
    def forward(ctx, *args):
        dx, dy, dw = _backward(*args)
        return dx, dx.clone() if dy is dx else dy, dw

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("residual_norm has no second derivatives")


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, weight, eps, gate, shift, scale, segments):
        r = _forward(_Problem(x, weight, gate, shift, scale, segments), x, y, eps, False, True, None)
        ctx.save_for_backward(r.x, r.rstd, weight, gate, scale)
        ctx.segments = segments
        ctx.mark_non_differentiable(r.rstd)
        ctx.set_materialize_grads(False)
        return r.x, r.rstd, r.hidden

    @staticmethod
    def backward(ctx, dt, _, dh):
        t, rstd, weight, gate, scale = ctx.saved_tensors
        if dt is None and dh is None:
            return (None,) * 8
        dh = torch.zeros_like(t) if dh is None else dh
        args = (dt, dh, t, rstd, weight, gate, scale, ctx.segments, ctx.needs_input_grad[2])
        dx, dy, dw = (_ResidualNormGrads.apply if torch.is_grad_enabled() else _backward)(*args)
        return dx, dy, dw, None, None, None, None, None


def _constants(gate, shift, scale) -> None:
    if (gate is not None and gate.requires_grad) or (shift is not None and shift.requires_grad) or \
            (scale is not None and scale.requires_grad):
        raise ValueError("residual_norm: gate, shift and scale have no gradient; detach them")


def residual_norm(x: torch.Tensor, y: torch.Tensor, weight: torch.Tensor, eps: float, *, gate: Optional[torch.Tensor] = None,
                  shift: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                  segments: Optional[Sequence[blk.Segment]] = None, codes: bool = True, hidden: bool = False,
                  out: Optional[torch.Tensor] = None) -> ResidualNorm:
    """t = x + gate y, h = t rsqrt(mean t^2 + eps) weight (1 + scale) + shift, and h's codes: see ResidualNorm.

    x, y: [M, K] bf16 or fp16, K a multiple of 8 up to 16384 (of 256 with codes).  gate, shift, scale: [rows, K] modulation rows
    that `segments` deals out to the tokens as `block.rms_modulate` takes them (ints, or per-token row tensors; numbers
    outside the rows: none).  Without a gate y is added everywhere; with one a token outside every segment keeps x.  Without
    shift and scale (they go together) h is the norm alone.  codes: int8 codes and scales of h rotated, as the W4A8 linears
    take them (`linear`); hidden: h itself.  out: a [M, K] tensor for t, which may be x or y and overlaps nothing else
    (not with gradients).
    Differentiable in x, y and weight through x and hidden of the result; with gradients the codes, which have none, are
    refused."""
    no_tangents("residual_norm", x, y, weight, gate, shift, scale)
    if (shift is None) != (scale is None):
        raise ValueError("residual_norm: shift and scale go together")
    if segments is not None and len(segments) and gate is None and shift is None:
        raise ValueError("residual_norm: segments without gate, shift or scale")
    if codes and x.shape[-1] % 256:
        raise ValueError(f"residual_norm: codes need a width that is a multiple of 256, got {x.shape[-1]}")
    if torch.is_grad_enabled():
        _constants(gate, shift, scale)
        if out is not None and out.requires_grad:
            raise ValueError("residual_norm: out requires a gradient, which what is written there does not have; detach it")
        if x.requires_grad or y.requires_grad or weight.requires_grad:
            if out is not None or codes:
                raise ValueError("residual_norm: out and codes cannot be asked for where gradients are recorded")
            t, rstd, h = _ResidualNorm.apply(x, y, weight, float(eps), gate, shift, scale, segments)
            return ResidualNorm(t, rstd, h if hidden else None, None, None)
    p = _Problem(x, weight, gate, shift, scale, segments)
    if out is not None:
        if p.rows(out, "out").data_ptr() != out.data_ptr():
            raise ValueError("residual_norm: out needs contiguous channels, a 16-byte aligned base and a row stride that is a multiple of 8")
        if out.numel() and any(t.data_ptr() != out.data_ptr() or _ld(t) != _ld(out) for t in (x, y) if _overlap(t, out)):
            raise ValueError("residual_norm: out may be x or y, and overlaps them in no other way")
        # the weight and the modulation are read for every row, also behind those that are written
        w = p.w.as_strided((1, p.k), (_ld(out), 1))  # a row, told apart from columns beside it
        if any(t is not None and _overlap(t, out) for t in (w, p.gate, p.shift, p.scale)):
            raise ValueError("residual_norm: out must not overlap weight, gate, shift or scale")
    r = _forward(p, x, y, float(eps), codes, hidden, out)
    if out is not None:
        _written(out)
    return r


def residual_norm_backward(dt: Optional[torch.Tensor], dh: torch.Tensor, t: torch.Tensor, rstd: torch.Tensor,
                           weight: torch.Tensor, *, gate: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                           segments: Optional[Sequence[blk.Segment]] = None, need_weight: bool = True
                           ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Gradients (dx, dy, dweight) of residual_norm from those of its x (dt, None: zeros) and hidden (dh); t and rstd as it gave
    them for the same arguments.  Without a gate dy is dx itself.  The same call gives the same bits.  No second derivatives."""
    no_tangents("residual_norm", dt, dh, t, weight, gate, scale)
    if torch.is_grad_enabled():
        _constants(gate, None, scale)
        if (dt is not None and dt.requires_grad) or dh.requires_grad or t.requires_grad or weight.requires_grad:
            return _ResidualNormGrads.apply(dt, dh, t, rstd, weight, gate, scale, segments, need_weight)
    return _backward(dt, dh, t, rstd, weight, gate, scale, segments, need_weight)


def reads_codes(w: Weight) -> bool:
    """Whether `linear` takes this weight's input as codes (W4A8, ConvRot 256) or as hidden rows (any other)."""
    return isinstance(w, W4A8Weight) and w.convrot == 256


def linear(r: ResidualNorm, w: Weight, bias: Optional[torch.Tensor] = None, *, quant_mode: str = "ck") -> torch.Tensor:
    """The linear that reads h: a W4A8 weight of ConvRot 256 from the codes, any other from hidden."""
    if reads_codes(w):
        if torch.is_grad_enabled() and bias is not None and bias.requires_grad:
            raise RuntimeError("residual.linear: a W4A8 projection has no gradient for bias; add it outside, or use a dense weight")
        if r.codes is None:
            raise ValueError("residual.linear: a W4A8 weight of ConvRot 256 reads the codes; ask residual_norm for them")
        if w.q.shape[1] * 2 != r.codes.shape[1]:
            raise ValueError(f"residual.linear: the codes are of {r.codes.shape[1]} channels, the weight takes {w.q.shape[1] * 2}")
        return ql._gemm_codes(r.codes, r.scales, w, bias, out_dtype=r.x.dtype, quant_mode=quant_mode)
    if r.hidden is None:
        raise ValueError("residual.linear: a dense weight, or one of another ConvRot than 256, reads hidden; ask residual_norm for it")
    return ql.linear(r.hidden, w, bias, quant_mode=quant_mode)
