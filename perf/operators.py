"""Rotary embedding over several position axes, and cross attention to another stream's states: what is measured.

The two operators serve the video + audio + text blocks around the W4A8 linears: queries of one stream (video patches at
(t, y, x), audio frames at (t, 0, 0)) attend to the keys and values of another stream of another length (the audio
frames, the whole video, a text encoder's states).  Three kinds of case:

  rope    q and k rotated by the angles of their positions, or rotated back (the gradient's direction)
  cross   attention output of q over k, v
  train   attention output, then the gradients of q, k and v from the output's gradient

`run` computes them either in plain torch operations in 32 bits (`own` false) or through the package's entry points
(`own` true); `exact` restates the definitions in 64 bits.
"""
import importlib.util
import math
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_DEV = "cuda"
_MAX_MACS = 57840 * 1600 * 40 * 128  # query x key x head x channel products of the largest listed case
_MAX_SCORES = 57840 * 1600 * 40  # and its scores, which the plain form holds at once
_MAX_KV = 57840 * 40 * 128  # elements of the longest listed query and key sequences


def listed():
    return [
        # one new query step against a short prompt: launch latency only
        {"name": "cross_1q_77k", "kind": "cross", "dtype": "bf16", "B": 2, "Sq": 1, "Sk": 77, "Hq": 40, "Hkv": 40,
         "D": 128, "mask": "none"},
        # one query over the 57840 video tokens of the 40 s sequence: all time goes into reading the keys and values
        {"name": "cross_1q_57840k", "kind": "cross", "dtype": "bf16", "B": 1, "Sq": 1, "Sk": 57840, "Hq": 40, "Hkv": 40,
         "D": 128, "mask": "none"},
        # a few queries of three requests with shared key heads over ragged video lengths of the 5 s sequence
        {"name": "cross_5q_12090k_gqa", "kind": "cross", "dtype": "bf16", "B": 3, "Sq": 5, "Sk": 12090, "Hq": 56, "Hkv": 8,
         "D": 128, "mask": "lens"},
        # odd sizes: fp16, 64 channels, shared key heads, a key mask that leaves one batch entry without keys
        {"name": "cross_odd_fp16", "kind": "cross", "dtype": "fp16", "B": 3, "Sq": 1031, "Sk": 333, "Hq": 12, "Hkv": 4,
         "D": 64, "mask": "bool"},
        # the 5 s video's tokens over padded text states (two prompts of different length)
        {"name": "cross_12090q_512k", "kind": "cross", "dtype": "bf16", "B": 2, "Sq": 12090, "Sk": 512, "Hq": 40, "Hkv": 40,
         "D": 128, "mask": "lens"},
        # the 40 s video's tokens over its audio tokens: the largest forward
        {"name": "cross_57840q_1600k", "kind": "cross", "dtype": "bf16", "B": 1, "Sq": 57840, "Sk": 1600, "Hq": 40,
         "Hkv": 40, "D": 128, "mask": "none"},
        # a training step of the odd sizes, keys weighted by an additive bias
        {"name": "train_odd_fp16", "kind": "train", "dtype": "fp16", "B": 3, "Sq": 517, "Sk": 77, "Hq": 12, "Hkv": 4,
         "D": 64, "mask": "bias"},
        # an ordinary training step: 4096 video tokens, padded prompts
        {"name": "train_4096q_512k", "kind": "train", "dtype": "bf16", "B": 2, "Sq": 4096, "Sk": 512, "Hq": 40, "Hkv": 40,
         "D": 128, "mask": "lens"},
        # a training step of the official head count: the 5 s video's tokens over the long audio sequence
        {"name": "train_12090q_1600k", "kind": "train", "dtype": "bf16", "B": 1, "Sq": 12090, "Sk": 1600, "Hq": 56,
         "Hkv": 56, "D": 128, "mask": "none"},
        # one token per request: launch latency only
        {"name": "rope_1token", "kind": "rope", "dtype": "bf16", "B": 8, "Sq": 1, "Sk": 1, "Hq": 56, "Hkv": 56, "D": 128,
         "sections": "16,16,16", "pairing": "half", "inverse": False},
        # gradients of an odd fp32 sequence, adjacent pairs, shared key heads, keys of another length
        {"name": "rope_back_odd_fp32", "kind": "rope", "dtype": "fp32", "B": 2, "Sq": 4093, "Sk": 1601, "Hq": 24, "Hkv": 8,
         "D": 64, "sections": "4,14,14", "pairing": "adjacent", "inverse": True},
        # the whole 40 s sequence
        {"name": "rope_59440tokens", "kind": "rope", "dtype": "bf16", "B": 1, "Sq": 59440, "Sk": 59440, "Hq": 40, "Hkv": 40,
         "D": 128, "sections": "16,16,16", "pairing": "half", "inverse": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["cross", "cross", "train", "rope"])
    if kind == "rope":
        d = rng.choice([32, 64, 80, 128, 128])
        pairs = d // 2
        a = rng.randint(1, 4)
        cuts = sorted(rng.randint(0, pairs) for _ in range(a))
        sections = [max(1, y - x) for x, y in zip([0] + cuts[:-1], cuts)]
        while sum(sections) > pairs:
            sections[sections.index(max(sections))] -= 1
        hkv = rng.choice([1, 2, 8, 24, 40])
        hq = hkv * rng.choice([1, 1, 3, 4]) if hkv <= 24 else hkv
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        b = rng.randint(1, 3)
        top = max(1, min(59440, 59440 * 40 * 128 * 2 * 2 // (b * (hq + hkv) * d * _SIZES[dtype])))
        return {"kind": "rope", "dtype": dtype, "B": b, "Sq": _log_int(rng, 1, top), "Sk": _log_int(rng, 1, top),
                "Hq": hq, "Hkv": hkv, "D": d, "sections": ",".join(str(s) for s in sections),
                "pairing": rng.choice(["half", "adjacent"]), "inverse": rng.random() < 0.5}
    d = rng.choice([40, 64, 64, 96, 128, 128, 128])
    hkv = rng.choice([1, 2, 4, 8, 12, 40])
    hq = hkv * rng.choice([1, 1, 2, 4, 7]) if hkv <= 12 else hkv
    b = rng.randint(1, 4)
    shape = rng.choice(["few", "wide", "wide"])
    # with one or two keys the gradients of q and k are differences of rounding errors: none to compare
    sk = _log_int(rng, 8 if kind == "train" else 1, min(57840, _MAX_KV // (b * hkv * d)))
    if shape == "few":
        sq = rng.randint(1, 32)
    else:
        cap = min(_MAX_MACS // d, _MAX_SCORES) * (2 if kind == "train" else 7) // 7 // (b * hq * sk)
        rows = _MAX_KV // (2 if kind == "train" else 1) // (b * hq * d)
        sq = _log_int(rng, 1, max(1, min(57840, cap, rows)))
    return {"kind": kind, "dtype": rng.choice(["bf16", "bf16", "fp16"]), "B": b, "Sq": sq, "Sk": sk, "Hq": hq, "Hkv": hkv,
            "D": d, "mask": rng.choice(["none", "none", "lens", "bool", "bias"])}


def _lens(case):
    """Keys in use per batch entry of a padded batch: full, then shorter ones, deterministic from the case."""
    sk, b = case["Sk"], case["B"]
    return [sk if i == 0 else max(1, (sk * (b - i)) // b - i) if sk > 1 else i % 2 for i in range(b)]


def _package():
    name = "minimax_h3_turbo_b200"
    if name not in sys.modules:
        root = Path(__file__).resolve().parent.parent / "minimax-h3-turbo_b200"
        spec = importlib.util.spec_from_file_location(name, root / "__init__.py", submodule_search_locations=[str(root)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        spec.loader.exec_module(mod)
    from minimax_h3_turbo_b200.h3 import cross, rope

    return rope, cross


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(shape, generator=g, device=_DEV) * std).to(dt)

    b, sq, sk, hq, hkv, d = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    st = {"case": case, "q": normal(b, sq, hq, d), "k": normal(b, sk, hkv, d)}
    if case["kind"] == "rope":
        sections = tuple(int(s) for s in case["sections"].split(","))

        def grid(s):  # positions of a video walk: the first axis slow, the last fast, an offset per batch entry
            i = torch.arange(s, device=_DEV).view(1, s, 1) + torch.randint(0, 1000, (b, 1, 1), generator=g, device=_DEV)
            side = 20
            return torch.cat([(i // side ** (len(sections) - 1 - a)) % (side if a else 1 << 30) for a in range(len(sections))],
                             -1).to(torch.float32)

        st["pos_q"], st["pos_k"] = grid(sq), grid(sk)
        st["inv_freq"] = torch.cat([10000.0 ** (-torch.arange(n, dtype=torch.float32, device=_DEV) / n) for n in sections])
        st["sections"] = sections
    else:
        st["v"] = normal(b, sk, hkv, d)
        st["kv_lens"] = st["key_mask"] = None
        if case["mask"] == "lens":
            st["kv_lens"] = torch.tensor(_lens(case), dtype=torch.int32, device=_DEV)
        elif case["mask"] == "bool":  # a fifth of the keys is padding anywhere; the last of several entries has none left
            st["key_mask"] = torch.rand(b, sk, generator=g, device=_DEV) < 0.8
            if b > 1:
                st["key_mask"][-1] = False
        elif case["mask"] == "bias":  # log weights of the keys, a tenth of them out
            w = torch.rand(b, sk, generator=g, device=_DEV) * 1.5 + 0.25
            st["key_mask"] = torch.where(torch.rand(b, sk, generator=g, device=_DEV) < 0.9, w.log(),
                                         torch.full_like(w, float("-inf")))
        if case["kind"] == "train":
            st["do"] = normal(b, sq, hq, d)
    if own:
        st["rope"], st["cross"] = _package()
    return st


# ------------------------------------------------------------------------------------------------ plain forms, 32 bits
def _plain_rotate(x, pos, inv_freq, sections, pairing, inverse):
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    ang = pos.index_select(-1, axis) * inv_freq
    c, s = ang.cos().unsqueeze(2), ang.sin().unsqueeze(2)
    if inverse:
        s = -s
    f = sum(sections)
    xf = x.float()
    out = xf.clone()
    if pairing == "half":
        a, b = xf[..., :f], xf[..., f:2 * f]
        out[..., :f] = a * c - b * s
        out[..., f:2 * f] = a * s + b * c
    else:
        a, b = xf[..., 0:2 * f:2], xf[..., 1:2 * f:2]
        out[..., 0:2 * f:2] = a * c - b * s
        out[..., 1:2 * f:2] = a * s + b * c
    return out.to(x.dtype)


def _plain_bias(case, kv_lens, key_mask):
    """[B, Sk] what a key adds to its scores: 0, a given bias, or -inf where it is masked."""
    b, sk = case["B"], case["Sk"]
    bias = torch.zeros(b, sk, device=_DEV)
    if key_mask is not None:
        bias = bias.masked_fill(~key_mask, float("-inf")) if key_mask.dtype == torch.bool else key_mask.float()
    if kv_lens is not None:
        out = torch.arange(sk, device=_DEV).view(1, sk) >= kv_lens.view(b, 1)
        bias = bias.masked_fill(out, float("-inf"))
    return bias


def _plain_probs(qf, kf, bias, scale):
    """[.., rows, Sk] softmax over the keys; a row without keys is all zero."""
    s = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale).add_(bias)
    m = s.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = s.sub_(m).exp_()
    return p.div_(p.sum(-1, keepdim=True).clamp_min_(1e-37))


def _plain_attention(st):
    case = st["case"]
    b, sq, sk, hq, hkv, d = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    g = hq // hkv
    dt, scale = st["q"].dtype, 1.0 / math.sqrt(d)
    bias = _plain_bias(case, st["kv_lens"], st["key_mask"]).view(b, 1, 1, sk)

    def rows(x):  # [B, Sq, Hq, D] -> [B, Hkv, Sq * G, D] in 32 bits
        return x.float().view(b, sq, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, sq * g, d)

    def back(x):
        return x.view(b, hkv, sq, g, d).permute(0, 2, 1, 3, 4).reshape(b, sq, hq, d).to(dt)

    qf, kf, vf = rows(st["q"]), st["k"].float().transpose(1, 2), st["v"].float().transpose(1, 2)
    p = _plain_probs(qf, kf, bias, scale)
    o = torch.matmul(p, vf)
    if case["kind"] == "cross":
        return back(o)
    do = rows(st["do"])
    dv = torch.matmul(p.transpose(-1, -2), do)
    dp = torch.matmul(do, vf.transpose(-1, -2))
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq, dk = torch.matmul(ds, kf), torch.matmul(ds.transpose(-1, -2), qf)
    return [back(o), back(dq), dk.transpose(1, 2).contiguous().to(dt), dv.transpose(1, 2).contiguous().to(dt)]


def run(state):
    st, case = state, state["case"]
    if case["kind"] == "rope":
        args = (st["inv_freq"], st["sections"])
        if own:
            return st["rope"].rope_axes(st["q"], st["k"], st["pos_q"], *args, k_positions=st["pos_k"],
                                        pairing=case["pairing"], inverse=case["inverse"])
        return tuple(_plain_rotate(x, p, *args, case["pairing"], case["inverse"])
                     for x, p in ((st["q"], st["pos_q"]), (st["k"], st["pos_k"])))
    if not own:
        return _plain_attention(st)
    kw = {"kv_lens": st["kv_lens"], "key_mask": st["key_mask"]}
    if case["kind"] == "cross":
        return st["cross"].cross_attention(st["q"], st["k"], st["v"], **kw)
    o, lse = st["cross"].cross_attention(st["q"], st["k"], st["v"], return_lse=True, **kw)
    return [o, *st["cross"].cross_attention_backward(st["do"], st["q"], st["k"], st["v"], o, lse, **kw)]


def work(case):
    b, sq, sk, hq, hkv, d = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    es = _SIZES[case["dtype"]]
    if case["kind"] == "rope":
        f = sum(int(s) for s in case["sections"].split(","))
        axes = len(case["sections"].split(","))
        x = b * (sq * hq + sk * hkv)
        # a product for every angle, four products and two sums for every pair; cos and sin are not counted
        return {"bytes": 2 * x * d * es + b * (sq + sk) * axes * 4 + f * 4, "flops": 6 * x * f + b * (sq + sk) * f}
    keys = sum(_lens(case)) if case["mask"] == "lens" else b * sk
    share = 1.0
    if case["mask"] == "bool":  # masked keys are needed by nobody
        keys, share = (b - 1 if b > 1 else 1) * sk, 0.8
    elif case["mask"] == "bias":
        share = 0.9
    keys *= share
    qn, kn = b * sq * hq * d, int(keys * hkv * d)
    extra = {"none": 0, "lens": 4 * b, "bool": b * sk, "bias": 4 * b * sk}[case["mask"]]
    mm = 2.0 * sq * keys * hq * d  # one product of the scores' size
    if case["kind"] == "cross":
        return {"bytes": es * (2 * qn + 2 * kn) + extra, "flops": int(2 * mm)}
    # q, k, v, do read; o, dq, dk, dv written (gradients of masked keys are written as zeros)
    return {"bytes": es * (4 * qn + 2 * kn + 2 * b * sk * hkv * d) + extra, "flops": int(7 * mm)}


# ------------------------------------------------------------------------------------------------ definitions, 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    b, sq, sk, hq, hkv, d = (case[n] for n in ("B", "Sq", "Sk", "Hq", "Hkv", "D"))
    if case["kind"] == "rope":
        res = []
        for x, pos in ((st["q"], st["pos_q"]), (st["k"], st["pos_k"])):
            y = x.double()
            f, j = sum(st["sections"]), 0
            for a, n in enumerate(st["sections"]):
                for _ in range(n):
                    lo, hi = (j, j + f) if case["pairing"] == "half" else (2 * j, 2 * j + 1)
                    theta = pos[..., a].double() * st["inv_freq"][j].double()
                    z = torch.complex(x[..., lo].double(), x[..., hi].double())
                    turn = torch.polar(torch.ones_like(theta), -theta if case["inverse"] else theta)
                    z = z * turn.unsqueeze(-1)
                    y[..., lo], y[..., hi] = z.real, z.imag
                    j += 1
            res.append(y)
        return tuple(res)
    if 14.0 * b * hq * sq * sk * d > 4e13:
        return None
    train = case["kind"] == "train"
    o = torch.zeros(b, sq, hq, d, dtype=torch.float64, device=_DEV)
    dq = torch.zeros_like(o)
    dk = torch.zeros(b, sk, hkv, d, dtype=torch.float64, device=_DEV)
    dv = torch.zeros_like(dk)
    for i in range(b):  # only the keys that take part, gathered
        keep = torch.ones(sk, dtype=torch.bool, device=_DEV)
        add = torch.zeros(sk, dtype=torch.float64, device=_DEV)
        if st["kv_lens"] is not None:
            keep[int(st["kv_lens"][i]):] = False
        if st["key_mask"] is not None and st["key_mask"].dtype == torch.bool:
            keep &= st["key_mask"][i]
        elif st["key_mask"] is not None:
            add = st["key_mask"][i].double()
            keep &= add != float("-inf")
        idx = keep.nonzero().flatten()
        if idx.numel() == 0:
            continue
        add = add[idx]
        for h in range(hq):
            kk, vv = st["k"][i, idx, h * hkv // hq].double(), st["v"][i, idx, h * hkv // hq].double()
            for r in range(0, sq, 16384):
                rows = slice(r, r + 16384)
                qq = st["q"][i, rows, h].double()
                logits = qq @ kk.T / d ** 0.5 + add
                w = torch.exp(logits - torch.logsumexp(logits, 1, keepdim=True))
                o[i, rows, h] = w @ vv
                if train:
                    gg = st["do"][i, rows, h].double()
                    gw = gg @ vv.T
                    gl = w * (gw - (w * gw).sum(1, keepdim=True)) / d ** 0.5
                    dq[i, rows, h] = gl @ kk
                    dk[i, :, h * hkv // hq].index_add_(0, idx, gl.T @ qq)
                    dv[i, :, h * hkv // hq].index_add_(0, idx, w.T @ gg)
    return [o, dq, dk, dv] if train else o
