"""Arguments of cross attention that must come back as an error, or as the nearest thing they mean, on GPU."""
import pytest
import torch

from minimax_h3_turbo_b200.h3 import cross

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF = torch.bfloat16


def test_too_many_query_heads_to_a_key_head():
    q, k = torch.zeros(1, 4, 129, 64, dtype=BF, device=DEV), torch.zeros(1, 8, 1, 64, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="128"):
        cross.cross_attention(q, k, k)
    with pytest.raises(ValueError, match="128"):
        cross.cross_attention_backward(q, q, k, k, q, torch.zeros(1, 129, 4, device=DEV))
    with pytest.raises(ValueError, match="128"):
        cross.cross_attention(q.requires_grad_(), k, k)


def test_lengths_past_32_bits():
    q, k, v = (torch.randn(4, s, 2, 64, device=DEV, dtype=BF) for s in (5, 30, 30))
    far = torch.tensor([2 ** 32 + 5, -(2 ** 33) + 7, 2 ** 31, 2 ** 63 - 1], device=DEV)
    near = torch.tensor([30, 0, 30, 30], dtype=torch.int32, device=DEV)
    assert torch.equal(cross.cross_attention(q, k, v, kv_lens=far), cross.cross_attention(q, k, v, kv_lens=near))
    strided = torch.tensor([7, 99, 5, 99, 30, 99, -1, 99], device=DEV)[::2]  # both types, any stride
    want = cross.cross_attention(q, k, v, kv_lens=strided.clamp(min=0).to(torch.int32))
    assert torch.equal(cross.cross_attention(q, k, v, kv_lens=strided), want)
    assert torch.equal(cross.cross_attention(q, k, v, kv_lens=strided.to(torch.int32).repeat_interleave(2)[::2]), want)


def test_out_is_no_part_of_what_is_read():
    q, k, v = (torch.randn(2, 30, 2, 64, device=DEV, dtype=BF) for _ in range(3))
    want = cross.cross_attention(q, k, v)
    for out in (k, v):
        with pytest.raises(ValueError, match="overlap"):
            cross.cross_attention(q, k, v, out=out)
    with pytest.raises(ValueError):  # rows that fold onto one another
        cross.cross_attention(q, k, v, out=torch.empty(10000, dtype=BF, device=DEV).as_strided(q.shape, (3840, 128, 8, 1)))
    both = torch.empty(2, 30, 2, 2, 64, dtype=BF, device=DEV)  # keys and results side by side in one buffer
    both[:, :, 0] = k
    assert torch.equal(cross.cross_attention(q, both[:, :, 0], v, out=both[:, :, 1]), want)
    assert torch.equal(both[:, :, 0], k)
