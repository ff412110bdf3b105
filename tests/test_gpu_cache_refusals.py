"""Reads of more rows than a call takes: refused in front of the memory for them."""
import pytest
import torch

from helpers import kernels

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [(1 << 30) + 1, 1 << 40, (1 << 62) + 1, -1])
@pytest.mark.parametrize("own", [False, True])
def test_reads_of_too_many_rows(pkg, rows, own):
    c = pkg.PagedKVCache(2, 16, 4, 128)
    tables, cu = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    k_out = torch.empty(4, 4, 128, dtype=torch.bfloat16, device="cuda") if own else None
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError):
        kernels().kv_cache_read(c.k, c.v, tables, cu, rows, k_out=k_out)
    with pytest.raises(ValueError):
        c.read(tables, cu, rows)
    assert torch.cuda.max_memory_allocated() == before


def test_reads_from_caches_of_too_many_heads():
    k = torch.zeros(2, 16, 1, 16, dtype=torch.bfloat16, device="cuda").expand(2, 16, 1 << 30, 16)
    tables, cu = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        kernels().kv_cache_read(k, k, tables, cu, 1 << 30)
