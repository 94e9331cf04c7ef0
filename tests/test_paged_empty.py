"""Empty batches of the operators over a paged cache: nothing to do, whatever the machine (no GPU)."""
import pytest
import torch

import timestral_b200 as tb


def test_norm_rope_of_no_token_with_a_rotation():
    """An empty positions array has no address: that is not a missing array."""
    q, k = torch.zeros(0, 4, 64, dtype=torch.float16), torch.zeros(0, 2, 64, dtype=torch.float16)
    cos, pos = torch.zeros(8, 32), torch.zeros(0, dtype=torch.int32)
    tb.norm_rope(q, q, cos=cos, sin=cos, positions=pos)
    tb.norm_rope(q, torch.empty_like(q), k, k, q_weight=torch.ones(64), k_weight=torch.ones(64), cos=cos, sin=cos, positions=pos)
    # what is wrong without a token stays refused
    with pytest.raises(tb.TimestralError, match="rope_dim 80"):
        tb.norm_rope(q, q, cos=torch.zeros(8, 40), sin=torch.zeros(8, 40), positions=pos)
    with pytest.raises(tb.TimestralError, match="positions"):
        tb.norm_rope(torch.zeros(3, 4, 64, dtype=torch.float16), torch.zeros(3, 4, 64, dtype=torch.float16), cos=cos, sin=cos)


def test_append_and_attention_of_no_token():
    kv, table = torch.zeros(6, 2, 16, 64, dtype=torch.float16), torch.zeros(2, 3, dtype=torch.int32)
    cache = tb.PagedCache(kv, kv.clone(), table)
    batch = tb.PagedBatch(torch.zeros(3, dtype=torch.int32), torch.tensor([5, 0], dtype=torch.int32), 1, 8)
    q, k = torch.zeros(0, 4, 64, dtype=torch.float16), torch.zeros(0, 2, 64, dtype=torch.float16)
    cos, pos = torch.zeros(8, 32), torch.zeros(0, dtype=torch.int32)
    tb.paged_append(cache, batch, k, k, k_weight=torch.ones(64), cos=cos, sin=cos)
    tb.paged_append(cache, batch, k, k, cos=cos, sin=cos, positions=pos)
    bits = torch.zeros(2, 1, dtype=torch.int32)
    tb.paged_attention(cache, batch, q, q, gate=q, key_valid=bits, self_visible=True, workspace=torch.empty(0, dtype=torch.uint8))
    assert tb.paged_attention_workspace(cache, batch, 0, 4) == 0
