"""Cross attention: queries of one stream attend to the keys and values of another, of another length (video tokens to
audio tokens or to a text encoder's states, audio tokens to the video, one new query to a long stream), with its
gradients.  No reference counterpart: the reference's attention is one stream's own (h3turbo/h3/model.py:196-228).

    s_ij = scale * q_i . k_j + bias_j        o_i = sum_j softmax_j(s_ij) v_j        lse_i = log sum_j exp(s_ij)

Kernels: h3b_cross_attention and h3b_cross_attention_backward (include/h3b.h).  bf16/fp16 CUDA tensors only, as the
block's other operators; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import math
from contextlib import nullcontext
from typing import Optional, Tuple

import torch

from .. import _lib

_DTYPES = (torch.bfloat16, torch.float16)


def _guard(dev: torch.device):
    """The kernels launch on the current device: make it the tensors'."""
    return nullcontext() if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _batched(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() not in (3, 4):
        raise ValueError(f"{name} must be [B, S, heads, D] or [S, heads, D], got {tuple(t.shape)}")
    return t if t.dim() == 4 else t.unsqueeze(0)


def _readable(t: torch.Tensor) -> torch.Tensor:
    """t itself when the kernels can read it in place: channels contiguous, 16-byte aligned base and strides."""
    st = t.stride()
    ok = t.data_ptr() % 16 == 0 and (st[3] == 1 or t.shape[3] == 1)
    for n, s in zip(t.shape[:3], st[:3]):
        ok = ok and (n <= 1 or (s > 0 and s % 8 == 0))
    if ok:
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _arg(t: torch.Tensor) -> _lib.AttnTensor:
    (b, s, h, _), (sb, ss, sh, _) = t.shape, t.stride()
    return _lib.AttnTensor(t.data_ptr(), sb if b > 1 else 0, ss if s > 1 else 0, sh if h > 1 else 0)


class _Problem:
    """Checked sizes and arguments of one call, forward or backward."""

    def __init__(self, q, k, v, kv_lens, key_mask, scale):
        q, k, v = _batched(q, "q"), _batched(k, "k"), _batched(v, "v")
        dev = q.device
        if not (q.is_cuda and k.is_cuda and v.is_cuda):
            raise RuntimeError("cross_attention: CUDA tensors only (there is no CPU path)")
        if q.dtype not in _DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
            raise RuntimeError(f"cross_attention: q, k and v must be bf16 or fp16, all of one type, got {q.dtype}, {k.dtype}, "
                               f"{v.dtype} (there is no fp32 path)")
        if k.device != dev or v.device != dev:
            raise ValueError("cross_attention: q, k and v must be on one device")
        self.b, self.sq, self.hq, self.d = q.shape
        self.sk, self.hkv = k.shape[1], k.shape[2]
        if k.shape != v.shape or k.shape[0] != self.b or k.shape[3] != self.d:
            raise ValueError(f"cross_attention: k and v must be [{self.b}, Sk, heads, {self.d}] alike, got {tuple(k.shape)} "
                             f"and {tuple(v.shape)}")
        if self.hkv == 0 or self.hq == 0 or self.hq % self.hkv:
            raise ValueError(f"cross_attention: {self.hq} query heads are not a multiple of {self.hkv} key heads")
        self.scale = 1.0 / math.sqrt(self.d) if scale is None else float(scale)
        self.q, self.k, self.v, self.dev = _readable(q), _readable(k), _readable(v), dev
        self.lens = self.mask = None
        self.kind, self.ldm = _lib.MASK_NONE, 0
        if kv_lens is not None:
            if tuple(kv_lens.shape) != (self.b,) or kv_lens.dtype not in (torch.int32, torch.int64) or kv_lens.device != dev:
                raise ValueError(f"cross_attention: kv_lens must be int32 or int64 [{self.b}] on {dev}")
            self.lens = kv_lens.to(torch.int32).contiguous()
        if key_mask is not None:
            if key_mask.dim() != 2 or key_mask.shape[1] != self.sk or key_mask.shape[0] not in (1, self.b) or key_mask.device != dev:
                raise ValueError(f"cross_attention: key_mask must be [{self.b}, {self.sk}] (or [1, {self.sk}]) on {dev}, got "
                                 f"{tuple(key_mask.shape)} on {key_mask.device}")
            if key_mask.requires_grad and torch.is_grad_enabled():
                raise ValueError("cross_attention: key_mask has no gradient; detach it")
            if key_mask.dtype == torch.bool:
                self.kind = _lib.MASK_BOOL
            elif key_mask.is_floating_point():
                self.kind, key_mask = _lib.MASK_BIAS, key_mask.detach().float()
            else:
                raise ValueError(f"cross_attention: key_mask must be bool or floating point, got {key_mask.dtype}")
            self.mask = key_mask if key_mask.stride(1) == 1 or self.sk == 1 else key_mask.contiguous()
            self.ldm = self.mask.stride(0) if self.mask.shape[0] > 1 else 0

    def rows(self, t: torch.Tensor, name: str, like: torch.Tensor) -> torch.Tensor:
        t = _batched(t, name)
        if t.shape != like.shape or t.dtype != like.dtype or t.device != like.device:
            raise ValueError(f"cross_attention: {name} must be {tuple(like.shape)} {like.dtype} on {like.device}, got "
                             f"{tuple(t.shape)} {t.dtype} on {t.device}")
        return t

    def sizes(self):
        return self.b, self.sq, self.sk, self.hq, self.hkv, self.d

    def workspace(self, backward: bool) -> Tuple[Optional[torch.Tensor], int]:
        n = _lib.lib().h3b_cross_attention_workspace_bytes(*self.sizes(), self.kind, int(backward))
        return (torch.empty(n, dtype=torch.uint8, device=self.dev) if n else None), n

    def tail(self):
        return (_lib.act_code(self.q.dtype), *self.sizes(), self.scale, _lib.ptr(self.lens), _lib.ptr(self.mask), self.kind,
                self.ldm)


def _forward(p: _Problem, want_lse: bool, out: Optional[torch.Tensor]):
    with _guard(p.dev):
        o = torch.empty(p.b, p.sq, p.hq, p.d, dtype=p.q.dtype, device=p.dev) if out is None else out
        lse = torch.empty(p.b, p.hq, p.sq, dtype=torch.float32, device=p.dev) if want_lse else None
        ws, n = p.workspace(False)
        ref = ctypes.byref
        _lib.check(_lib.lib().h3b_cross_attention(ref(_arg(p.q)), ref(_arg(p.k)), ref(_arg(p.v)), ref(_arg(o)), *p.tail(),
                                                  _lib.ptr(lse), _lib.ptr(ws), n, _lib.stream_ptr(p.dev)), "cross_attention")
    return o, lse


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
    entry's largest value is taken off first, which changes lse but not o.  A query without keys gets 0 (lse -inf); what
    keys that are left out hold never reaches a result.  Differentiable in q, k and v.  out: a [B, Sq, Hq, D] tensor to
    write (16-byte aligned rows; not with gradients)."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        if out is not None:
            raise ValueError("cross_attention: out cannot be given where gradients are recorded")
        o, lse = _CrossAttention.apply(q, k, v, kv_lens, key_mask, scale)
        return (o, lse) if return_lse else o
    p = _Problem(q, k, v, kv_lens, key_mask, scale)
    if out is not None and _readable(p.rows(out, "out", p.q)).data_ptr() != _batched(out, "out").data_ptr():
        raise ValueError("cross_attention: out needs contiguous channels, a 16-byte aligned base and strides that are "
                         "multiples of 8 elements")
    o, lse = _forward(p, return_lse, None if out is None else _batched(out, "out"))
    o = out if out is not None else o.view(q.shape)
    return (o, lse) if return_lse else o


@torch.no_grad()
def cross_attention_backward(do: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor,
                             lse: torch.Tensor, *, kv_lens: Optional[torch.Tensor] = None,
                             key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None
                             ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients (dq, dk, dv) of cross_attention's o with respect to q, k and v, from the gradient do of o; o and lse as
    cross_attention(..., return_lse=True) gave them for the same arguments.  The heads that share a key head add up in dk
    and dv; keys that are left out get zeros.  The same call gives the same bits."""
    p = _Problem(q, k, v, kv_lens, None if key_mask is None else key_mask.detach(), scale)
    do_, o_ = _readable(p.rows(do, "do", p.q)), _readable(p.rows(o, "o", p.q))
    if tuple(lse.shape) != (p.b, p.hq, p.sq) or lse.dtype != torch.float32 or lse.device != p.dev:
        raise ValueError(f"cross_attention: lse must be fp32 {(p.b, p.hq, p.sq)} on {p.dev}")
    with _guard(p.dev):
        lse = lse.contiguous()
        dq = torch.empty(p.b, p.sq, p.hq, p.d, dtype=p.q.dtype, device=p.dev)
        dk, dv = (torch.empty(p.b, p.sk, p.hkv, p.d, dtype=p.q.dtype, device=p.dev) for _ in range(2))
        ws, n = p.workspace(True)
        ref = ctypes.byref
        _lib.check(_lib.lib().h3b_cross_attention_backward(
            ref(_arg(do_)), ref(_arg(p.q)), ref(_arg(p.k)), ref(_arg(p.v)), ref(_arg(o_)), lse.data_ptr(), ref(_arg(dq)),
            ref(_arg(dk)), ref(_arg(dv)), *p.tail(), _lib.ptr(ws), n, _lib.stream_ptr(p.dev)), "cross_attention_backward")
    return dq.view(q.shape), dk.view(k.shape), dv.view(v.shape)
