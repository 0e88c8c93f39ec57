"""Cross attention on GPU: digits and bits that depend on the operands' size, on what ran before, and on the exp2 in use."""
import pytest
import torch

from minimax_h3_turbo_b200.h3 import cross

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF, FP = torch.bfloat16, torch.float16


def make(b, sq, sk, hq, hkv, d, dt, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randn(b, s, h, d, generator=g, device=DEV).to(dt) for s, h in ((sq, hq), (sk, hkv), (sk, hkv), (sq, hq))]


@pytest.mark.parametrize("d,dt", [(64, BF), (128, FP)])
@pytest.mark.parametrize("g", [3, 5, 7])
def test_same_bits_whatever_ran_before(g, d, dt):
    """Head groups that do not divide 128 leave rows of a query tile unwritten: what they hold must not reach other rows."""
    q, k, v, do = make(1, 3 * (128 // g), 400, 2 * g, 2, d, dt, seed=g)
    before = make(1, 128 * 148 * 2, 128, 1, 1, d, dt, seed=50)
    results = []
    for size in (0.0, 0.1, 30.0):  # of the scores that were in every SM's shared memory
        cross.cross_attention(before[0] * size, *before[1:3])
        o, lse = cross.cross_attention(q, k, v, return_lse=True)
        cross.cross_attention_backward(before[3] * size, before[0] * size, *before[1:3],
                                       *cross.cross_attention(before[0] * size, *before[1:3], return_lse=True))
        results.append((o, lse, *cross.cross_attention_backward(do, q, k, v, o, lse)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
