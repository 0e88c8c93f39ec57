"""Cross attention: queries of one stream attend to the keys and values of another, of another length (video tokens to
audio tokens or to a text encoder's states, audio tokens to the video, one new query to a long stream), with its
gradients.  No reference counterpart: the reference's attention is one stream's own (h3turbo/h3/model.py:196-228).

    s_ij = scale * q_i . k_j + bias_j        o_i = sum_j softmax_j(s_ij) v_j        lse_i = log sum_j exp(s_ij - t)

t is 0, or with an additive mask the largest bias in use of the batch entry: a mask of large negative values keeps the scores'
digits that way, in lse and so in the gradients, which are computed from it.  `full_lse` adds t back.

Kernels: h3b_cross_attention and h3b_cross_attention_backward (include/h3b.h).  bf16/fp16 CUDA tensors only, as the
block's other operators; there is no CPU path.  `CrossLayer` runs them as a residual layer between W4A8 linears, with the
rotary embedding of both streams' positions (rope.rope_axes).
"""
from __future__ import annotations

import math
from array import array
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib
from . import block as blk
from . import qlinear as ql
from .rope import no_tangents, rope_axes
from .types import Weight

_CODES = {torch.bfloat16: _lib.BF16, torch.float16: _lib.FP16}


def _guard(dev: torch.device):
    """The kernels launch on the current device: make it the tensors'."""
    return torch.cuda.device(dev)


def _batched(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() == 4:
        return t
    if t.dim() != 3:
        raise ValueError(f"{name} must be [B, S, heads, D] or [S, heads, D], got {tuple(t.shape)}")
    return t.unsqueeze(0)


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t itself when the kernels can read it in place: channels contiguous, 16-byte aligned base and strides."""
    if t.is_contiguous():
        ok = t.shape[3] % 8 == 0
    else:
        st = t.stride()
        ok = st[3] == 1 or t.shape[3] == 1
        for n, s in zip(t.shape[:3], st[:3]):
            ok = ok and (n <= 1 or (s > 0 and s % 8 == 0))
    if ok and t.data_ptr() % 16 == 0:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _empty(t: torch.Tensor) -> torch.Tensor:
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


@lru_cache(maxsize=4096)
def _workspace_bytes(device: int, sizes: Tuple[int, ...], kind: int, backward: bool) -> int:
    """A number per problem size and device: kept, since it takes a microsecond of a short call."""
    return _lib.lib().h3b_cross_attention_workspace_bytes(*sizes, kind, backward)


class _Problem:
    """Checked sizes and arguments of one call, forward or backward."""

    __slots__ = ("b", "sq", "sk", "hq", "hkv", "d", "scale", "q", "k", "v", "dev", "lens", "mask", "kind", "ldm", "code")

    def __init__(self, q, k, v, kv_lens, key_mask, scale):
        q, k, v = _batched(q, "q"), _batched(k, "k"), _batched(v, "v")
        dev, dt = q.device, q.dtype
        one_device = k.device == dev and v.device == dev
        if not (q.is_cuda and (one_device or (k.is_cuda and v.is_cuda))):
            raise RuntimeError("cross_attention: CUDA tensors only (there is no CPU path)")
        code = _CODES.get(dt)
        if code is None or k.dtype != dt or v.dtype != dt:
            raise RuntimeError(f"cross_attention: q, k and v must be bf16 or fp16, all of one type, got {q.dtype}, {k.dtype}, "
                               f"{v.dtype} (there is no fp32 path)")
        if not one_device:
            raise ValueError("cross_attention: q, k and v must be on one device")
        b, self.sq, hq, d = q.shape
        kb, sk, hkv, kd = k.shape
        if k.shape != v.shape or kb != b or kd != d:
            raise ValueError(f"cross_attention: k and v must be [{b}, Sk, heads, {d}] alike, got {tuple(k.shape)} and "
                             f"{tuple(v.shape)}")
        if hkv == 0 or hq == 0 or hq % hkv:
            raise ValueError(f"cross_attention: {hq} query heads are not a multiple of {hkv} key heads")
        if hq > 128 * hkv:
            raise ValueError(f"cross_attention: at most 128 query heads to a key head, got {hq} to {hkv}")
        self.b, self.sk, self.hq, self.hkv, self.d, self.code, self.dev = b, sk, hq, hkv, d, code, dev
        self.scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
        self.q, self.k, self.v = _readable(q), _readable(k), _readable(v)
        self.lens = self.mask = None
        self.kind, self.ldm = _lib.MASK_NONE, 0
        if kv_lens is not None:
            if kv_lens.shape != (b,) or kv_lens.dtype not in (torch.int32, torch.int64) or kv_lens.device != dev:
                raise ValueError(f"cross_attention: kv_lens must be int32 or int64 [{b}] on {dev}")
            if kv_lens.dtype == torch.int64:  # before they lose their upper half
                kv_lens = kv_lens.clamp(0, sk).to(torch.int32)
            self.lens = kv_lens.contiguous()
        if key_mask is not None:
            self._set_mask(key_mask)

    def _set_mask(self, m):
        if m.dim() != 2 or m.shape[1] != self.sk or m.shape[0] not in (1, self.b) or m.device != self.dev:
            raise ValueError(f"cross_attention: key_mask must be [{self.b}, {self.sk}] (or [1, {self.sk}]) on {self.dev}, got "
                             f"{tuple(m.shape)} on {m.device}")
        if m.dtype == torch.bool:
            self.kind = _lib.MASK_BOOL
        elif m.is_floating_point():
            self.kind = _lib.MASK_BIAS
            if m.dtype != torch.float32:
                m = m.detach().float()
        else:
            raise ValueError(f"cross_attention: key_mask must be bool or floating point, got {m.dtype}")
        self.mask = m if m.stride(1) == 1 or self.sk == 1 else m.contiguous()
        self.ldm = self.mask.stride(0) if self.mask.shape[0] > 1 else 0

    def rows(self, t: torch.Tensor, name: str) -> torch.Tensor:
        t = _batched(t, name)
        if t.shape != self.q.shape or t.dtype != self.q.dtype or t.device != self.dev:
            raise ValueError(f"cross_attention: {name} must be {tuple(self.q.shape)} {self.q.dtype} on {self.dev}, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")
        return t

    def call(self, entry: str, tensors, lse: Optional[torch.Tensor], backward: bool) -> None:
        """Workspace, arguments and the call of one entry point; `tensors` in its order (lse after the fifth, backward)."""
        lib = _lib.lib()
        sizes = (self.b, self.sq, self.sk, self.hq, self.hkv, self.d)
        n = _workspace_bytes(self.dev.index, sizes, self.kind, backward)
        ws = torch.empty(n, dtype=torch.uint8, device=self.dev) if n else None
        arr = array("q")  # struct h3b_attn_tensor, one after the other: pointer, strides of batch, token and head
        for t in tensors:
            arr.append(t.data_ptr())
            arr.extend(t.stride()[:3])
        at = arr.buffer_info()[0]
        ts = range(at, at + 32 * len(tensors), 32)
        mid = (self.code, *sizes, self.scale, _lib.ptr(self.lens), _lib.ptr(self.mask), self.kind, self.ldm)
        tail = (_lib.ptr(ws), n, _lib.raw_stream(self.dev.index))
        if backward:
            rc = lib.h3b_cross_attention_backward(*ts[:5], lse.data_ptr(), *ts[5:], *mid, *tail)
        else:
            rc = lib.h3b_cross_attention(*ts, *mid, _lib.ptr(lse), *tail)
        if rc:
            _lib.check(rc, entry)


def _forward(p: _Problem, want_lse: bool, out: Optional[torch.Tensor]):
    o = _empty(p.q) if out is None else out
    lse = torch.empty(p.b, p.hq, p.sq, dtype=torch.float32, device=p.dev) if want_lse else None
    if p.dev.index == torch.cuda.current_device():
        p.call("cross_attention", (p.q, p.k, p.v, o), lse, False)
    else:
        with _guard(p.dev):
            p.call("cross_attention", (p.q, p.k, p.v, o), lse, False)
    return o, lse


def _backward(do, q, k, v, o, lse, kv_lens, key_mask, scale):
    p = _Problem(q, k, v, kv_lens, key_mask, scale)
    do_, o_ = _readable(p.rows(do, "do")), _readable(p.rows(o, "o"))
    if tuple(lse.shape) != (p.b, p.hq, p.sq) or lse.dtype != torch.float32 or lse.device != p.dev:
        raise ValueError(f"cross_attention: lse must be fp32 {(p.b, p.hq, p.sq)} on {p.dev}")
    lse = lse.contiguous()
    dq, dk, dv = _empty(p.q), _empty(p.k), _empty(p.v)
    tensors = (do_, p.q, p.k, p.v, o_, dq, dk, dv)
    if p.dev.index == torch.cuda.current_device():
        p.call("cross_attention_backward", tensors, lse, True)
    else:
        with _guard(p.dev):
            p.call("cross_attention_backward", tensors, lse, True)
    return tuple(g if t.dim() == 4 else g.view(t.shape) for g, t in ((dq, q), (dk, k), (dv, v)))


class _CrossAttentionGrads(torch.autograd.Function):
    """The gradients where autograd records: they have no derivatives of their own, and say so when one is asked for."""

    @staticmethod
    def forward(ctx, *args):
        return _backward(*args)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("cross_attention has no second derivatives")


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_lens, key_mask, scale):
        p = _Problem(q, k, v, kv_lens, key_mask, scale)
        o, lse = _forward(p, True, None)
        o = o.view(q.shape)
        ctx.save_for_backward(q, k, v, kv_lens, key_mask, o, lse)
        ctx.scale = scale
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    def backward(ctx, do, _):
        q, k, v, kv_lens, key_mask, o, lse = ctx.saved_tensors
        dq, dk, dv = cross_attention_backward(do, q, k, v, o, lse, kv_lens=kv_lens, key_mask=key_mask, scale=ctx.scale)
        return dq, dk, dv, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None, return_lse: bool = False,
                    out: Optional[torch.Tensor] = None):
    """Attention of q [B, Sq, Hq, D] over k, v [B, Sk, Hkv, D] -> o [B, Sq, Hq, D] (without the batch dimension when q has
    none), or (o, lse [B, Hq, Sq] fp32) with return_lse.

    bf16 or fp16, D a multiple of 8 up to 128, any lengths, Hq a multiple of Hkv (query head h reads key head
    h // (Hq // Hkv)); views whose channels are contiguous and whose strides are multiples of 8 elements are read in place,
    others are copied.  kv_lens: int [B], keys in use of each entry of a padded batch.  key_mask: [B, Sk] (or [1, Sk]) bool,
    False leaves a key out; or floating point, added to the scaled scores (a key's log weight), -inf leaves it out; the
    entry's largest value is taken off first, which changes lse (full_lse puts it back) but not o.  A query without keys gets
    0 (lse -inf); what keys that are left out hold never reaches a result.  Differentiable in q, k and v (not in key_mask, nor
    through lse).  out: a [B, Sq, Hq, D] tensor to write (16-byte aligned rows; not with gradients; no part of k or v, which are
    read while it is written)."""
    no_tangents("cross_attention", q, k, v, key_mask)
    if torch.is_grad_enabled():
        if key_mask is not None and key_mask.requires_grad:
            raise ValueError("cross_attention: key_mask has no gradient; detach it")
        if q.requires_grad or k.requires_grad or v.requires_grad:
            if out is not None:
                raise ValueError("cross_attention: out cannot be given where gradients are recorded")
            o, lse = _CrossAttention.apply(q, k, v, kv_lens, key_mask, scale)
            return (o, lse) if return_lse else o
    p = _Problem(q, k, v, kv_lens, key_mask, scale)
    if out is not None:
        if _readable(p.rows(out, "out")).data_ptr() != _batched(out, "out").data_ptr():
            raise ValueError("cross_attention: out needs contiguous channels, a 16-byte aligned base and strides that are "
                             "multiples of 8 elements")
        if out.numel() and out.data_ptr() in (p.k.data_ptr(), p.v.data_ptr()):
            raise ValueError("cross_attention: out must not overlap k or v")
    o, lse = _forward(p, return_lse, None if out is None else _batched(out, "out"))
    if out is not None:
        o = out
    elif q.dim() == 3:
        o = o.view(q.shape)
    return (o, lse) if return_lse else o


def cross_attention_backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                             lse: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                             key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of cross_attention's o with respect to q, k and v, from the gradient do of o; o and lse as
    cross_attention(..., return_lse=True) gave them for the same arguments.  The heads that share a key head add up in dk
    and dv; keys that are left out get zeros.  The same call gives the same bits.  There are no second derivatives: asking
    for them raises RuntimeError."""
    args = (do, q, k, v, o, lse, kv_lens, key_mask, scale)
    no_tangents("cross_attention", *args[:6], key_mask)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or do.requires_grad or o.requires_grad
                                    or lse.requires_grad):
        return _CrossAttentionGrads.apply(*args)
    return _backward(*args)


def full_lse(lse: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None
             ) -> torch.Tensor:
    """The log-sum-exp of the scores with their whole bias, [B, Hq, Sq] fp32, from lse as cross_attention(...,
    return_lse=True) gave it for the same kv_lens and key_mask: adds the largest bias in use of each entry's additive mask.
    This is what results over disjoint sets of keys are merged by (block.AttnMerger); cross_attention_backward takes lse as it
    came."""
    if lse.dim() != 3 or lse.dtype != torch.float32:
        raise ValueError(f"full_lse: lse must be [B, Hq, Sq] fp32, got {tuple(lse.shape)} {lse.dtype}")
    if key_mask is None or key_mask.dtype == torch.bool or key_mask.numel() == 0:
        return lse
    if key_mask.dim() != 2 or key_mask.shape[0] not in (1, lse.shape[0]) or not key_mask.is_floating_point():
        raise ValueError(f"full_lse: key_mask must be [{lse.shape[0]}, Sk] (or [1, Sk]) bool or floating point")
    bias = key_mask.float()
    if kv_lens is not None:
        bias = bias.masked_fill(torch.arange(bias.shape[1], device=bias.device) >= kv_lens.view(-1, 1), -math.inf)
    top = bias.amax(1)
    return lse + top.masked_fill(top == -math.inf, 0.0).view(-1, 1, 1)


@dataclass
class CrossWeights:
    """Weights of one cross-attention layer: W4A8 or dense [N, K] linears and the norm of the residual stream."""

    q: Weight     # [heads * head_dim, hidden]
    kv: Weight    # [2 * kv_heads * head_dim, width of the other stream]: keys, then values
    out: Weight   # [hidden, heads * head_dim]
    norm: torch.Tensor  # [hidden]


class CrossLayer:
    """x += gate * out(attention(rope(q(h)), rope(k), v)),  h = rms(x, norm) * (1 + scale) + shift: the residual stream x
    [S, hidden] attends to another stream's states [Sk, width], with the block's modulation rows and segments.

    The keys and values depend on the other stream only: `keys_values` computes them once for all denoising steps (with
    their rotary embedding); a call takes the pair.  sections / pairing: how rope_axes deals the frequencies out; without
    inv_freq nothing is turned."""

    def __init__(self, heads: int, head_dim: int, kv_heads: Optional[int] = None, norm_eps: float = 1e-5,
                 precision: str = "a8", sections: Optional[Sequence[int]] = None, pairing: str = "half"):
        self.heads, self.head_dim = heads, head_dim
        self.kv_heads = heads if kv_heads is None else kv_heads
        if self.kv_heads < 1 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads are not a multiple of {self.kv_heads} key heads")
        self.norm_eps, self.precision, self.sections, self.pairing = norm_eps, precision, sections, pairing

    def keys_values(self, states: torch.Tensor, w: CrossWeights, positions: Optional[torch.Tensor] = None,
                    inv_freq: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [Sk, kv_heads, head_dim] of the other stream's states [Sk, width], k turned by its positions."""
        inner = self.kv_heads * self.head_dim
        k, v = (t.unflatten(-1, (self.kv_heads, self.head_dim)) for t in
                ql.linear(states, w.kv, precision=self.precision).split(inner, dim=-1))
        if inv_freq is not None:
            _, k = rope_axes(None, k, None, inv_freq, self.sections, k_positions=positions, pairing=self.pairing)
        return k, v

    def __call__(self, x: torch.Tensor, w: CrossWeights, kv: Tuple[torch.Tensor, torch.Tensor], shift: torch.Tensor,
                 scale: torch.Tensor, gate: torch.Tensor, segments: Sequence[blk.Segment],
                 positions: Optional[torch.Tensor] = None, inv_freq: Optional[torch.Tensor] = None, *,
                 kv_lens: Optional[torch.Tensor] = None, key_mask: Optional[torch.Tensor] = None) -> torch.Tensor:
        """x (updated in place and returned); kv from keys_values; kv_lens [1] / key_mask [1, Sk] as in cross_attention."""
        s = x.shape[0]
        pre = blk.Prenorm(x, w.norm, self.norm_eps, shift, scale, segments)
        q = blk.prenorm_linear(pre, w.q, self.precision).view(s, self.heads, self.head_dim)
        if inv_freq is not None:
            q, _ = rope_axes(q, None, positions, inv_freq, self.sections, pairing=self.pairing)
        o = cross_attention(q, *kv, kv_lens=kv_lens, key_mask=key_mask)
        return blk.gate_(x, gate, ql.linear(o.view(s, -1), w.out, precision=self.precision), segments)
