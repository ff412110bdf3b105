"""Calls that would attend over, or sum, something else than was asked for: refused, without a GPU."""
import pytest
import torch


@pytest.mark.parametrize("heads, kv_heads, cached", [(28, 4, 2), (28, 4, 7), (28, 4, 14), (28, 4, 28), (8, 8, 4), (8, 1, 2)])
def test_a_cache_of_other_heads_is_refused(pkg, heads, kv_heads, cached):
    """Also where no keys are written: 28 queries on a cache of 2 (or 7, 14, 28) heads would find some key head each."""
    layer = pkg.PagedAttention(heads, 16, num_kv_heads=kv_heads)
    layer.cache = pkg.PagedKVCache(2, 4, cached, 16, device="cpu")
    x = torch.zeros(2, heads * 16, dtype=torch.bfloat16)
    k = torch.zeros(2, kv_heads * 16, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="heads"):
        layer(x, None, None, None, i[:, None], i)
    with pytest.raises(ValueError, match="heads"):
        layer(x, k, k, i, i[:, None], i)
    with pytest.raises(ValueError, match="heads"):
        layer.forward_quant(x, None, None, None, i[:, None], i, torch.tensor(1.0))
    layer.cache = pkg.PagedKVCache(2, 4, kv_heads, 16, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(x, None, None, None, i[:, None], i)
