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
