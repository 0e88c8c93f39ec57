"""The log-sum-exps of cross attention: results over disjoint sets of keys merge by them, on GPU."""
import math

import pytest
import torch

from cross_ref import cross_ref
from minimax_h3_turbo_b200.h3 import block as blk
from minimax_h3_turbo_b200.h3 import cross

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def case(kind, dt, b=2, sq=33, sk=300):
    """q, k, v, key mask, lengths, and the scores with their whole bias in 64 bits [B, Hq, Sq, Sk]."""
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v = (torch.randn(b, s, h, 64, generator=g, device=DEV).to(dt) for s, h in ((sq, 4), (sk, 2), (sk, 2)))
    mask = lens = None
    if kind in ("bias", "shared"):
        mask = torch.randn(b if kind == "bias" else 1, sk, generator=g, device=DEV) * 3
        mask[:, 200:] -= 5
        mask = mask.masked_fill(torch.rand(mask.shape, generator=g, device=DEV) < 0.2, -math.inf)
    if kind == "bool":
        mask = torch.rand(b, sk, generator=g, device=DEV) < 0.6
    else:
        lens = torch.tensor([290, 130][:b], device=DEV)
    bias = torch.zeros(b, sk, dtype=torch.float64, device=DEV)
    if mask is not None:
        bias = bias + (torch.where(mask, 0.0, -math.inf).double() if mask.dtype == torch.bool else mask.double())
    if lens is not None:
        bias = bias.masked_fill(torch.arange(sk, device=DEV) >= lens.view(b, 1), -math.inf)
    s = torch.einsum("bqhd,bkhd->bhqk", q.double(), k.double().repeat_interleave(2, 2)) / 8 + bias.view(b, 1, 1, sk)
    return q, k, v, mask, lens, s


def shards(q, k, v, mask, lens):
    for a, b in ((0, 130), (130, 300)):
        kw = {"kv_lens": None if lens is None else lens - a, "key_mask": None if mask is None else mask[:, a:b]}
        o, lse = cross.cross_attention(q, k[:, a:b], v[:, a:b], return_lse=True, **kw)
        yield o, cross.full_lse(lse, **kw)


@pytest.mark.parametrize("kind", ["bias", "bool", "lens", "shared"])
def test_shards_of_the_keys_merge(kind):
    """Bounds: lse as elsewhere (fp32 scores); a shard's o is rounded once more than the whole's, by u sum P |v| at most, which
    tol_o has."""
    q, k, v, mask, lens, s = case(kind, torch.float16)
    parts = list(shards(q, k, v, mask, lens))
    lse = torch.logaddexp(parts[0][1], parts[1][1])
    assert torch.allclose(lse.double(), torch.logsumexp(s, -1), rtol=2e-6, atol=1e-4)
    o, whole = cross.cross_attention(q, k, v, key_mask=mask, kv_lens=lens, return_lse=True)
    assert torch.allclose(cross.full_lse(whole, key_mask=mask, kv_lens=lens).double(), torch.logsumexp(s, -1), rtol=2e-6, atol=1e-4)
    merged = sum(torch.exp(p[1] - lse).transpose(1, 2).unsqueeze(-1) * p[0].float() for p in parts)
    r = cross_ref(q, k, v, lens, mask)
    assert ((merged.double() - r["o"]).abs() <= 2 * r["tol_o"]).all()


def test_the_blocks_merger_takes_them():
    """AttnMerger, one entry in bf16: within a rounding (u) of the merged fp32 rows on top of the shards' bounds."""
    q, k, v, mask, lens, _ = case("bias", torch.bfloat16, b=1)
    merger = blk.AttnMerger(4, 33, 64, DEV)
    for i, (o, lse) in enumerate(shards(q, k, v, mask, lens)):
        out = merger.add(o.transpose(1, 2), lse, last=i == 1)
    r = cross_ref(q, k, v, lens, mask)
    bound = 2 * r["tol_o"] + 2.0 ** -8 * (r["o"].abs() + r["tol_o"])
    assert ((out.view(1, 33, 4, 64).double() - r["o"]).abs() <= bound).all()


def test_full_lse():
    inf = math.inf
    m = torch.tensor([[1.0, 5.0, 9.0], [-inf, -inf, -inf], [-1e9, -1e9, -3.0]], device=DEV)
    lse = torch.zeros(3, 2, 4, device=DEV)
    lse[1] = -inf
    row = lambda *a, **kw: cross.full_lse(lse, **kw)[:, 0, 0].tolist()  # noqa: E731
    assert row(key_mask=m) == [9.0, -inf, -3.0]
    assert row(key_mask=m, kv_lens=torch.tensor([2, 3, 2], device=DEV)) == [5.0, -inf, -1e9]
    assert row(key_mask=m.half()) == [9.0, -inf, -3.0]
    assert row(key_mask=m[:1], kv_lens=torch.tensor([1, 0, 2 ** 40], device=DEV)) == [1.0, -inf, 9.0]
    for same in (dict(), dict(key_mask=m > 0), dict(kv_lens=torch.tensor([1, 0, 2], device=DEV)), dict(key_mask=m[:, :0])):
        assert cross.full_lse(lse, **same) is lse
    for bad in (lambda: cross.full_lse(lse[0], key_mask=m), lambda: cross.full_lse(lse.half(), key_mask=m),
                lambda: cross.full_lse(lse, key_mask=m[:2]), lambda: cross.full_lse(lse, key_mask=m.int())):
        with pytest.raises(ValueError):
            bad()
