"""Low-rank adapters of many requests beside a shared projection, with their gradients.  No reference counterpart.

    out_i = base_i + s_g (x_i A_g^T) B_g^T          g the adapter of row i; rows without one keep base_i

A batch holds rows of several requests, each with an adapter (A_g [rank, K], B_g [N, rank]) of its own or none, beside one
projection that they share (a W4A8 linear, qlinear.linear).  `plan` says once per batch which rows an adapter has, in any order;
`low_rank` runs on it for every projection of every layer, from one row per request to whole prompts; `linear` is the shared
projection and its adapters in one call.  Kernels: h3b_adapter_plan, h3b_low_rank, h3b_low_rank_backward (include/h3b.h).
bf16/fp16 CUDA tensors only, as the block's operators; there is no CPU path.
"""
from __future__ import annotations

from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _lib
from . import qlinear as ql
from .rope import no_tangents
from .types import Weight

Scales = Union[None, float, torch.Tensor]
Rows = Union[torch.Tensor, Sequence[Tuple[int, int, int]]]
_CODES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}


@dataclass(frozen=True)
class AdapterPlan:
    """Which rows of a batch each adapter has (from `plan`): opaque, valid for any projection of that batch."""

    table: Optional[torch.Tensor]  # int32, as h3b_adapter_plan writes it; None without rows
    rows: int
    adapters: int
    device: torch.device


def plan(rows: Rows, adapters: int, *, count: Optional[int] = None, device=None) -> AdapterPlan:
    """The plan of a batch for `adapters` adapters.  rows: an int32 or int64 CUDA tensor [M], the adapter of each row, any
    number outside 0 .. adapters - 1 for none; or segments [(first row, end row, adapter)] with the number of rows `count` and
    their device (rows outside every segment have none, later segments win).  Does not synchronise; the kernels that
    build it run on the current stream (a fill per segment; of hundreds of them, pass a tensor), and may be captured."""
    if not 1 <= adapters <= _lib.MAX_ADAPTERS:
        raise ValueError(f"adapters.plan: 1 to {_lib.MAX_ADAPTERS} adapters, got {adapters}")
    if not isinstance(rows, torch.Tensor):
        if count is None or device is None:
            raise ValueError("adapters.plan: segments need the number of rows and their device")
        segments = list(rows)
        for first, end, g in segments:
            if not 0 <= first <= end <= count or not 0 <= g < adapters:
                raise ValueError(f"adapters.plan: segment {(first, end, g)} is out of range for {count} rows and {adapters} adapters")
        if torch.device(device).type != "cuda":
            raise RuntimeError("adapters.plan: CUDA tensors only (there is no CPU path)")
        rows = torch.full((count,), -1, dtype=torch.int32, device=device)
        for first, end, g in segments:  # filled on the device: a copy from the host would wait for the stream
            if end > first:
                rows[first:end].fill_(g)
    elif count is not None or device is not None:
        raise ValueError("adapters.plan: count and device go with segments, not with a tensor of rows")
    if rows.dim() != 1 or rows.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"adapters.plan: rows must be int32 or int64 [M], got {tuple(rows.shape)} {rows.dtype}")
    if not rows.is_cuda:
        raise RuntimeError("adapters.plan: CUDA tensors only (there is no CPU path)")
    if rows.dtype == torch.int64:  # before they lose their upper half
        rows = rows.clamp(-1, adapters).to(torch.int32)
    rows, m, dev = rows.contiguous(), rows.shape[0], rows.device
    if m == 0:
        return AdapterPlan(None, 0, adapters, dev)
    lib = _lib.lib()
    n = lib.h3b_adapter_plan_ints(m, adapters)
    table = torch.empty(n, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.check(lib.h3b_adapter_plan(rows.data_ptr(), m, adapters, table.data_ptr(), n, _lib.raw_stream(dev.index)),
                   "adapters.plan")
    return AdapterPlan(table, m, adapters, dev)


@lru_cache(maxsize=4096)
def _sizes(m: int, k: int, n: int, rank: int, adapters: int, backward: bool) -> Tuple[int, int]:
    """(workspace, hidden) bytes: numbers per problem size, kept since they take a microsecond of a short call."""
    lib = _lib.lib()
    return lib.h3b_low_rank_workspace_bytes(m, k, n, rank, adapters, backward), lib.h3b_low_rank_hidden_bytes(m, rank)


def _readable(t: torch.Tensor) -> torch.Tensor:
    """[M, width] rows the kernels can read in place (contiguous channels, 16-byte aligned rows that do not overlap), or a copy."""
    if t.is_contiguous():  # rows of multiples of 8
        return t if t.data_ptr() % 16 == 0 else t.clone()
    m, width = t.shape
    st = t.stride()
    if (st[1] == 1 or width == 1) and (m <= 1 or (st[0] % 8 == 0 and st[0] >= width)) and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _weight(t: torch.Tensor) -> torch.Tensor:
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


class _Problem:
    """Checked sizes and operands of one call, forward or backward."""

    __slots__ = ("x", "a", "b", "m", "k", "n", "rank", "adapters", "dev", "dt", "code", "scales", "plan", "lead")

    def __init__(self, x, a, b, pl, scales):
        dt, dev = x.dtype, x.device
        if not x.is_cuda:
            raise RuntimeError("low_rank: CUDA tensors only (there is no CPU path)")
        code = _CODES.get(dt)
        if code is None or a.dtype != dt or b.dtype != dt:
            raise RuntimeError(f"low_rank: x, a and b must be bf16 or fp16, all of one type, got {dt}, {a.dtype}, {b.dtype} "
                               "(there is no fp32 path)")
        if a.device != dev or b.device != dev:
            raise ValueError("low_rank: x, a and b must be on one device")
        if a.dim() == 2 and b.dim() == 2:
            a, b = a.unsqueeze(0), b.unsqueeze(0)
        if a.dim() != 3 or b.dim() != 3 or a.shape[0] != b.shape[0] or a.shape[1] != b.shape[2]:
            raise ValueError(f"low_rank: a must be [adapters, rank, K] and b [adapters, N, rank] (or without adapters), got "
                             f"{tuple(a.shape)} and {tuple(b.shape)}")
        if x.dim() < 1 or x.shape[-1] != a.shape[2]:
            raise ValueError(f"low_rank: x must be [..., {a.shape[2]}], got {tuple(x.shape)}")
        self.adapters, self.rank, self.k = a.shape
        self.n = b.shape[1]
        if self.k % 8 or self.n % 8 or self.k == 0 or self.n == 0:
            raise ValueError(f"low_rank: widths must be positive multiples of 8, got {self.k} and {self.n}")
        if not 1 <= self.rank <= _lib.MAX_RANK or not 1 <= self.adapters <= _lib.MAX_ADAPTERS:
            raise ValueError(f"low_rank: a rank of 1 to {_lib.MAX_RANK} and 1 to {_lib.MAX_ADAPTERS} adapters, got {self.rank} "
                             f"and {self.adapters}")
        self.lead = x.shape[:-1]
        x = x if x.dim() == 2 else x.reshape(self.lead.numel(), self.k)
        self.m, self.dev, self.dt, self.code = x.shape[0], dev, dt, code
        if pl is None:
            if self.adapters != 1:
                raise ValueError(f"low_rank: {self.adapters} adapters need a plan of their rows")
            pl = _whole(self.m, dev)
        if pl.rows != self.m or pl.adapters != self.adapters or pl.device != dev:
            raise ValueError(f"low_rank: the plan is of {pl.rows} rows and {pl.adapters} adapters on {pl.device}, the call of "
                             f"{self.m} and {self.adapters} on {dev}")
        self.plan = pl
        if scales is None or isinstance(scales, torch.Tensor):
            if scales is not None and (scales.shape != (self.adapters,) or scales.dtype != torch.float32 or scales.device != dev):
                raise ValueError(f"low_rank: scales must be a number or fp32 [{self.adapters}] on {dev}")
        else:
            scales = torch.full((self.adapters,), float(scales), dtype=torch.float32, device=dev)
        self.scales = None if scales is None else scales.contiguous()
        self.x, self.a, self.b = _readable(x), _weight(a), _weight(b)

    def rows(self, t: torch.Tensor, width: int, name: str) -> torch.Tensor:
        if t.shape != (*self.lead, width) or t.dtype != self.dt or t.device != self.dev:
            raise ValueError(f"low_rank: {name} must be {(*self.lead, width)} {self.dt} on {self.dev}, got {tuple(t.shape)} "
                             f"{t.dtype} on {t.device}")
        return t if t.dim() == 2 else t.reshape(self.m, width)

    def launch(self, fn, head, tail, backward: bool, what: str) -> None:
        """Workspace and the call: fn(*head, workspace, its bytes, stream) with the sizes that both entry points share in between."""
        n = _sizes(self.m, self.k, self.n, self.rank, self.adapters, backward)[0]
        ws = torch.empty(n, dtype=torch.uint8, device=self.dev) if n else None
        args = (*head, self.code, self.m, self.k, self.n, self.rank, self.adapters, _lib.ptr(self.scales), _lib.ptr(self.plan.table),
                *tail, _lib.ptr(ws), n)
        index = self.dev.index
        if index == torch.cuda.current_device():
            rc = fn(*args, _lib.raw_stream(index))
        else:
            with torch.cuda.device(self.dev):
                rc = fn(*args, _lib.raw_stream(index))
        if rc:
            _lib.check(rc, what)


@dataclass(frozen=True)
class Adapters:
    """The adapters beside one projection: a [adapters, rank, K], b [adapters, N, rank], scales a number or fp32 [adapters]."""

    a: torch.Tensor
    b: torch.Tensor
    scales: Scales = None


@dataclass(frozen=True)
class BlockAdapters:
    """The adapters of one DiT block (None: that projection has none) and the plan of the batch's rows.  fc2's read what fc2
    reads: swiglu of fc1's output."""

    plan: AdapterPlan
    qkv: Optional[Adapters] = None
    out: Optional[Adapters] = None
    fc1: Optional[Adapters] = None
    fc2: Optional[Adapters] = None


def _whole(m: int, dev: torch.device) -> AdapterPlan:
    """All rows have the one adapter."""
    return plan(torch.zeros(m, dtype=torch.int32, device=dev), 1)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two tensors share memory.  Rows with the same stride (columns of one wider tensor) are told apart; of other
    strided tensors the stretches from their first to their last number count."""
    if a.numel() == 0 or b.numel() == 0:
        return False

    def span(t):
        return t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))

    (a0, a1), (b0, b1) = span(a), span(b)
    if a0 >= b1 or b0 >= a1:
        return False
    if a.dim() == b.dim() == 2 and a.dtype == b.dtype and a.stride() == b.stride() and a.stride(1) == 1:
        size, width = a.element_size(), a.stride(0) * a.element_size()
        if width >= max(a.shape[1], b.shape[1]) * size:
            at = (b0 - a0) % width  # of b's rows behind a's
            return at < a.shape[1] * size or at + b.shape[1] * size > width
    return True


def _written(out: torch.Tensor) -> None:
    """Tells autograd that a kernel has written out, as torch's own in-place operations do: a backward pass that kept its old values
    then raises instead of using the new ones."""
    if not out.is_inference():
        torch.autograd.graph.increment_version(out)


def _forward(p: _Problem, base, out, want_hidden: bool):
    y = torch.empty(p.m, p.n, dtype=p.dt, device=p.dev) if out is None else out
    base = None if base is None else base if base is out else _readable(base)
    hidden = None
    if want_hidden:
        hidden = torch.empty(_sizes(p.m, p.k, p.n, p.rank, p.adapters, False)[1], dtype=torch.uint8, device=p.dev)
    if p.m:
        p.launch(_lib.lib().h3b_low_rank, (p.x.data_ptr(), _ld(p.x), p.a.data_ptr(), p.b.data_ptr(), _lib.ptr(base),
                                           0 if base is None else _ld(base), y.data_ptr(), p.n if out is None else _ld(y)),
                 (_lib.ptr(hidden),), False, "low_rank")
    return y, hidden


def _backward(do, x, a, b, pl, hidden, scales, need):
    p = _Problem(x, a, b, pl, scales)
    do = _readable(p.rows(do, p.n, "do"))
    m, k, dev = p.m, p.k, p.dev
    size = _sizes(m, k, p.n, p.rank, p.adapters, True)[1]
    if hidden is None or hidden.dtype is not torch.uint8 or hidden.dim() != 1 or hidden.shape[0] != size or \
            hidden.device != dev or not hidden.is_contiguous() or hidden.data_ptr() % 256:
        raise ValueError(f"low_rank: hidden must be what low_rank(..., return_hidden=True) gave, {size} bytes on {dev}")
    dx = da = db = None
    if need[0]:
        dx = torch.empty(m, k, dtype=p.dt, device=dev)
    if need[1]:
        da = torch.empty_like(p.a)
    if need[2]:
        db = torch.empty_like(p.b)
    if need[0] or need[1] or need[2]:
        p.launch(_lib.lib().h3b_low_rank_backward,
                 (do.data_ptr(), _ld(do), p.x.data_ptr(), _ld(p.x), p.a.data_ptr(), p.b.data_ptr(), hidden.data_ptr(), _lib.ptr(dx), k,
                  _lib.ptr(da), _lib.ptr(db)), (), True, "low_rank_backward")
    if x.dim() != 2 and dx is not None:
        dx = dx.view(x.shape)
    if a.dim() != 3:
        da, db = None if da is None else da[0], None if db is None else db[0]
    return dx, da, db


class _LowRankGrads(torch.autograd.Function):
    """The gradients where autograd records: they have no derivatives of their own, and say so when one is asked for."""

    @staticmethod
    def forward(ctx, *args):
        return _backward(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("low_rank has no second derivatives")


class _LowRank(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, base, pl, scales):
        p = _Problem(x, a, b, pl, scales)
        y, hidden = _forward(p, None if base is None else p.rows(base, p.n, "base"), None, True)
        ctx.save_for_backward(x, a, b, hidden, scales if isinstance(scales, torch.Tensor) else None)
        ctx.rest = (p.plan, scales)
        ctx.mark_non_differentiable(hidden)
        return y.view(*p.lead, p.n), hidden

    @staticmethod
    def backward(ctx, do, _):
        x, a, b, hidden, scales = ctx.saved_tensors
        pl, s = ctx.rest
        need = ctx.needs_input_grad
        dx = da = db = None
        if any(need[:3]):
            args = (do, x, a, b, pl, hidden, s if scales is None else scales, need[:3])
            dx, da, db = (_LowRankGrads.apply if torch.is_grad_enabled() else _backward)(*args)
        return dx, da, db, do if need[3] else None, None, None


def low_rank(x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: Optional[AdapterPlan] = None, *,
             base: Optional[torch.Tensor] = None, scales: Scales = None,
             out: Optional[torch.Tensor] = None, return_hidden: bool = False):
    """out_i = base_i + s_g (x_i A_g^T) B_g^T for x [..., K] -> [..., N], or (out, hidden) with return_hidden.

    a [adapters, rank, K] and b [adapters, N, rank] (or [rank, K] and [N, rank]: one adapter, which without a plan has every
    row); bf16 or fp16 as x, ranks up to 128, K and N multiples of 8.  Adapters of one call have one rank: lower ones are filled
    up with zeros.  Adapters without rows are not read, but the launches allow for them: pass those in use where there are many.  plan: the batch's, from `plan`.  base [..., N]: what the
    shared projection gave (None: zeros).  scales: a number or fp32 [adapters].  out: a [..., N] tensor to write, which may be
    base itself (its rows without an adapter are then not touched) and overlaps nothing else; not with gradients, its own
    included.
    Differentiable in x, a, b and base (not in scales, nor through hidden); hidden is what low_rank_backward takes."""
    no_tangents("low_rank", x, a, b, base, scales if isinstance(scales, torch.Tensor) else None)
    if torch.is_grad_enabled():
        if isinstance(scales, torch.Tensor) and scales.requires_grad:
            raise ValueError("low_rank: scales have no gradient; detach them")
        if out is not None and out.requires_grad:
            raise ValueError("low_rank: out requires a gradient, which what is written there does not have; detach it")
        if x.requires_grad or a.requires_grad or b.requires_grad or (base is not None and base.requires_grad):
            if out is not None:
                raise ValueError("low_rank: out cannot be given where gradients are recorded")
            y, hidden = _LowRank.apply(x, a, b, base, plan, scales)
            return (y, hidden) if return_hidden else y
    p = _Problem(x, a, b, plan, scales)
    y = None
    base2 = None if base is None else p.rows(base, p.n, "base")
    if out is None:
        y, hidden = _forward(p, base2, None, return_hidden)
        if x.dim() != 2:
            y = y.view(*p.lead, p.n)
        return (y, hidden) if return_hidden else y
    y = p.rows(out, p.n, "out")
    if y.data_ptr() != out.data_ptr() or _readable(y).data_ptr() != y.data_ptr():
        raise ValueError("low_rank: out needs contiguous channels, a 16-byte aligned base and row strides that are multiples of 8")
    if base is not None and (base is out or (base2.data_ptr() == y.data_ptr() and _ld(base2) == _ld(y))):
        base2 = y
    if any(_overlap(y, t) for t in (p.x, p.a, p.b, *([] if base2 is None or base2 is y else [base2]))):
        raise ValueError("low_rank: out must not overlap x, a, b or a part of base")
    _, hidden = _forward(p, base2, y, return_hidden)
    _written(out)
    return (out, hidden) if return_hidden else out


def low_rank_backward(do: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, plan: Optional[AdapterPlan],
                      hidden: torch.Tensor, *, scales: Scales = None,
                      need: Tuple[bool, bool, bool] = (True, True, True)
                      ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """Gradients (dx, da, db) of low_rank's out with respect to x, a and b from the gradient do of out (base's gradient is do
    itself); hidden as low_rank(..., return_hidden=True) gave it for the same arguments; need: which of the three to compute.
    Adapters without rows get zeros.  The same call gives the same bits.  There are no second derivatives."""
    no_tangents("low_rank", do, x, a, b)
    if torch.is_grad_enabled() and (do.requires_grad or x.requires_grad or a.requires_grad or b.requires_grad):
        return _LowRankGrads.apply(do, x, a, b, plan, hidden, scales, need)
    return _backward(do, x, a, b, plan, hidden, scales, need)


def linear(x: torch.Tensor, w: Weight, a: torch.Tensor, b: torch.Tensor, plan: Optional[AdapterPlan] = None,
           bias: Optional[torch.Tensor] = None, *, scales: Scales = None, **kw) -> torch.Tensor:
    """The shared projection and its adapters: qlinear.linear(x, w, bias, **kw) + s_g (x A_g^T) B_g^T.  kw as qlinear.linear
    takes it, without input_act (the adapters read x as it is) and with outputs of x's type.  A W4A8 weight has no gradient
    for x and bias: where one of them requires it, that raises (a dense weight gives both)."""
    if kw.get("input_act") not in (None, "none") or kw.get("out_dtype") not in (None, x.dtype):
        raise ValueError("adapters.linear: input_act and another out_dtype are not taken; apply them outside")
    if torch.is_grad_enabled() and isinstance(w, ql.W4A8Weight):
        if x.requires_grad:
            raise RuntimeError("adapters.linear: a W4A8 projection has no gradient for x; detach x, or use a dense weight")
        if bias is not None and bias.requires_grad:
            raise RuntimeError("adapters.linear: a W4A8 projection has no gradient for bias; add the bias outside, or use a dense weight")
    y = ql.linear(x, w, bias, **kw)
    if torch.is_grad_enabled() and (y.requires_grad or a.requires_grad or b.requires_grad):
        return low_rank(x, a, b, plan, base=y, scales=scales)
    return low_rank(x, a, b, plan, base=y, scales=scales, out=y)
