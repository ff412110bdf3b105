"""Writes and reads on both sides of the sizes where they change from one row a thread to several: what is written is the
formula's, and comes back."""
import pytest
import torch

from test_gpu_cache import E4M3, quantised, rows_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kv_heads, dim, tokens", [(16, 128, (1036, 1037, 1184, 1185)), (4, 128, (4144, 4145, 4736, 4737)), (10, 80, (444, 445, 1036, 1037, 1184, 1185)),
                                                   (24, 96, (296, 297, 690, 691, 789, 790)), (12, 64, (888, 889, 2072, 2073, 2368, 2369)), (3, 128, (5180, 5181, 5920, 5921)),
                                                   (64, 256, (64, 65, 74, 75, 150))])
def test_both_sides_of_a_limit(pkg, kv_heads, dim, tokens, e4m3):
    block, most = 16, max(tokens)
    for n in tokens:
        k, v = rows_of(n, kv_heads, dim, seed=n)
        c = pkg.PagedKVCache(-(-most // block) + 1, block, kv_heads, dim, E4M3 if e4m3 else torch.bfloat16)
        pages = torch.randperm(c.k.shape[0], generator=torch.Generator().manual_seed(n)).cuda()
        slots = pages.repeat_interleave(block)[:n] * block + torch.arange(n, device="cuda") % block
        c.write(k, v, slots.to(torch.int32))
        got = c.read(pages[None].to(torch.int32), torch.tensor([0, n], dtype=torch.int32, device="cuda"), n)
        for x, cache, scale, out in ((k, c.k, c.k_scale, got[0]), (v, c.v, c.v_scale, got[1])):
            at, want = (slots // block, slots % block), x
            if e4m3:
                codes, s = quantised(x)
                assert torch.equal(cache[at].view(torch.uint8), codes.view(torch.uint8)) and torch.equal(scale[at], s)
                want = (codes.float() * s[..., None]).to(torch.bfloat16)
            else:
                assert torch.equal(cache[at], x)
            assert torch.equal(out, want)
            rest = cache.clone().view(torch.uint8)
            rest[at] = 0
            assert not rest.any()                               # nothing else was written
