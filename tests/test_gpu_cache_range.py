"""Decode attention over values of very different sizes: no token's part of the result is lost beside a louder token's value."""
import math

import pytest
import torch

from helpers import kernels
from test_gpu_cache import Cache, check, queries

pytestmark = pytest.mark.gpu

HEADS = [(14, 2, 64), (28, 4, 128), (24, 2, 128), (8, 1, 256), (40, 2, 64)]          # one and two groups of eight query heads at a time
LENGTHS = [[64, 65, 400, 401], [16, 3, 33], [9000, 5, 20000]]                        # a warp, some warps, some CTAs for a sequence


def cache_of(lengths, heads, scores, sizes, e4m3, seed=0):
    """(cache, q): token i of sequence b has about the score scores(b, n)[i] in every head, and a value sizes(b, n)[i] times a
    random one.  (Queries are 8 in their first channel; a key has that channel alone, but for noise.)"""
    heads, kv_heads, dim = heads
    q = queries(len(lengths), heads, dim, spread=0.05).clone()
    q[:, :, 0] = 8.0

    def keys(b, n):
        x = torch.zeros(n, kv_heads, dim, device="cuda")
        x[:, :, 0] = scores(b, n)[:, None] * (math.sqrt(dim) / 8.0)
        return x

    def values(b, n):
        g = torch.Generator(device="cuda").manual_seed(seed + b)
        return torch.randn(n, kv_heads, dim, device="cuda", generator=g) * sizes(b, n)[:, None, None]
    return Cache(lengths, kv_heads, dim, 16, e4m3, k=keys, v=values, seed=seed), q


def shuffled(x, b):
    return x[torch.randperm(x.shape[0], generator=torch.Generator().manual_seed(b)).cuda()]


ORDERS = {"rising": lambda x, b: x, "falling": lambda x, b: x.flip(0), "shuffled": shuffled}


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=len)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("order", list(ORDERS))
def test_one_token_takes_all_beside_values_of_any_size(order, at, heads, lengths, e4m3):
    def scores(b, n):
        x = torch.zeros(n, device="cuda")
        x[{"first": 0, "middle": n // 2, "last": n - 1}[at]] = 60.0
        return x
    check(*cache_of(lengths, heads, scores, lambda b, n: ORDERS[order](torch.logspace(-6, 6, n, device="cuda"), b), e4m3))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=len)
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("at", ["first", "middle", "last"])
@pytest.mark.parametrize("louder", [18, 22, 31, 60])
def test_a_loud_value_of_no_weight(louder, at, heads, lengths, e4m3):
    def there(b, n, there, elsewhere):
        x = torch.full((n,), elsewhere, device="cuda")
        x[{"first": 0, "middle": n // 2, "last": n - 1}[at]] = there
        return x
    check(*cache_of(lengths, heads, lambda b, n: there(b, n, -60.0, 0.0), lambda b, n: there(b, n, 2.0 ** louder, 1.0), e4m3))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads", HEADS, ids=str)
@pytest.mark.parametrize("order", list(ORDERS))
@pytest.mark.parametrize("span", [6, 12])
def test_weights_that_undo_the_sizes(span, order, heads, e4m3):
    """Every token has the same part of the result: a small weight of a loud value, a large one of a quiet value."""
    def sizes(b, n):
        return ORDERS[order](torch.logspace(-span, span, n, device="cuda"), b)
    check(*cache_of([64, 401, 4000], heads, lambda b, n: -torch.log(sizes(b, n)), sizes, e4m3))


@pytest.mark.parametrize("heads", HEADS, ids=str)
def test_scales_of_the_callers_own(heads):
    """Scales that the cache's formula does not make: zeros (values of nothing), negative ones, tiny ones, beside scores of any size."""
    c, q = cache_of([64, 65, 400, 401, 30], heads, lambda b, n: torch.linspace(-5, 5, n, device="cuda"), lambda b, n: torch.ones(n, device="cuda"), True)

    def times(b, factor):
        n = c.lengths[b]
        at = torch.tensor(c.pages[b], device="cuda").repeat_interleave(16)[:n], torch.arange(n, device="cuda") % 16
        c.vs[at] *= factor[:, None]
        c.rows[b][1] *= factor.double()[:, None, None]
    times(0, torch.zeros(64, device="cuda"))
    times(1, torch.where(torch.arange(65, device="cuda") % 2 == 0, -1.0, 2.0))
    times(2, torch.full((400,), 2.0 ** -85, device="cuda"))
    times(3, torch.logspace(-25, 25, 401, device="cuda"))
    times(4, torch.where(torch.arange(30, device="cuda") == 7, 0.0, -1e-5))
    out = check(c, q)
    assert not out[0].any()
    for scale in (1e3, -1e8, 1e12):                        # scores beside which the scales' logarithms are rounded away
        check(c, q, scale=scale)
    Kn, s = kernels(), torch.tensor(0.003, device="cuda")
    assert torch.equal(Kn.paged_attention(q, *c.args(), **c.scales(), out_scale=s).view(5, -1), Kn.quantize_activation(out.view(5, -1), s))
