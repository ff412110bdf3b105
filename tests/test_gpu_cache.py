"""The paged cache and the decode attention on the GPU against their definitions in 64 bits."""
import importlib
import math
import threading

import numpy as np
import pytest
import torch

from helpers import kernels

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
BF16_HALF = 2.0 ** -8                 # a rounding to bf16, relative
SUM = 2.0 ** -23                      # an fp32 sum of the tensor core (which may cut off), relative


def quantised(x):
    """(codes, scales) by the formula.  (Divided by a tensor: by a number, torch multiplies with its reciprocal.)"""
    x = x.float()
    s = x.abs().amax(-1).clamp(min=1e-8) / torch.tensor(448.0, device="cuda")
    return (x / s[..., None]).clamp(-448, 448).to(E4M3), s


class Cache:
    """Pages in no order, with everything that no sequence owns (whole pages, slots behind an end, table entries behind the last
    page) set to what must not be read: NaN, and page numbers that do not exist.  ``order``: how the pages lie in memory."""

    def __init__(self, lengths, kv_heads, dim, block, e4m3, seed=0, order="heads", k=None, v=None, spare=2, values=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.kv_heads, self.dim, self.block, self.e4m3 = lengths, kv_heads, dim, block, e4m3
        need = [-(-n // block) for n in lengths]
        blocks = sum(need) + spare
        deal = torch.randperm(blocks, generator=g, device="cuda").cpu().tolist()
        self.pages = [[deal.pop() for _ in range(n)] for n in need]
        width = max(need + [0]) + 1
        self.tables = torch.tensor([p + [-1 - i if i % 2 else 1 << 30 for i in range(width - len(p))] for p in self.pages], dtype=torch.int32).view(len(need), width).cuda()
        self.lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        dtype = torch.uint8 if e4m3 else torch.bfloat16
        shape = (blocks, kv_heads, block, dim) if order == "heads" else (blocks, block, kv_heads, dim)
        if order == "wide":                                   # rows of a wider tensor
            shape = (*shape[:3], dim + 16)
        if order == "heads":
            made = lambda: torch.full(shape, 0x7f if e4m3 else math.nan, dtype=dtype, device="cuda").transpose(1, 2)              # noqa: E731
            scales = lambda: torch.full(shape[:3], math.nan, device="cuda").transpose(1, 2)                                       # noqa: E731
        else:
            made = lambda: torch.full(shape, 0x7f if e4m3 else math.nan, dtype=dtype, device="cuda")[..., :dim]                   # noqa: E731
            scales = lambda: torch.full(shape[:3], math.nan, device="cuda")                                                       # noqa: E731
        self.k, self.v = made(), made()
        self.ks, self.vs = (scales(), scales()) if e4m3 else (None, None)
        self.rows = []
        for b, n in enumerate(lengths):
            pair = []
            for x, cache, scale, given in ((0, self.k, self.ks, k), (1, self.v, self.vs, v)):
                r = given(b, n) if given else torch.randn(n, kv_heads, dim, generator=g, device="cuda") * (1.0 if x == 0 else values)
                r = r.to(torch.bfloat16)
                at = torch.tensor(self.pages[b], dtype=torch.long, device="cuda").repeat_interleave(block)[:n], torch.arange(n, device="cuda") % block
                if e4m3:
                    codes, s = quantised(r)
                    cache[at] = codes.view(torch.uint8)
                    scale[at] = s
                    r = codes.double() * s.double()[..., None]
                else:
                    cache[at] = r
                pair.append(r.double())
            self.rows.append(pair)
        if e4m3:
            self.k, self.v = self.k.view(E4M3), self.v.view(E4M3)

    def args(self):
        return self.k, self.v, self.tables, self.lens

    def scales(self):
        return dict(k_scale=self.ks, v_scale=self.vs)


def definition(c, q, scale):
    """(o, bound): the attention in 64 bits, and how far fp32 sums and one rounding to bf16 may take a kernel from it.

    A score is a sum of D products, off by at most (D + 4) SUM of the sum of their sizes, S; its exponential has that as a
    relative error, and 2^-21 of its own (of the exponential function, and of the argument's rounding: |s| 2^-23).  The weights may be held as
    two bf16 numbers, 2^-16 off at most.  n weighted values are summed, and the n weights: 2 n SUM.  All of it relative to the weighted mean of |v|, A."""
    batch, heads, dim = q.shape
    o, bound = torch.zeros(batch, heads, dim, dtype=torch.float64, device="cuda"), torch.zeros(batch, heads, dim, dtype=torch.float64, device="cuda")
    group = heads // c.kv_heads
    for b, n in enumerate(c.lengths):
        if n == 0:
            continue
        k, v = (t.repeat_interleave(group, 1).transpose(0, 1) for t in c.rows[b])       # [heads, n, dim]
        qb = q[b].double()[:, None]
        s = (qb @ k.transpose(1, 2)) * scale
        w = torch.softmax(s, -1)
        o[b] = (w @ v)[:, 0]
        size = (qb.abs() @ k.abs().transpose(1, 2)).amax((1, 2)) * abs(scale)
        off = 2 * (size * (dim + 4) * SUM + 2.0 ** -21 + s.abs().amax((1, 2)) * SUM) + 2.0 ** -16 + 2 * min(n, 4096) * SUM
        bound[b] = o[b].abs() * BF16_HALF + (w @ v.abs())[:, 0] * off[:, None]
    return o, bound


def queries(batch, heads, dim, seed=1, spread=1.0):
    """A slice of a wider row, as of a qkv projection."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    wide = (torch.randn(batch, heads * dim + 64, generator=g, device="cuda") * spread).to(torch.bfloat16)
    return wide[:, :heads * dim].view(batch, heads, dim)


def check(c, q, scale=None, **kw):
    out = kernels().paged_attention(q, *c.args(), scale=scale, **c.scales(), **kw)
    torch.cuda.synchronize()
    o, bound = definition(c, q, q.shape[2] ** -0.5 if scale is None else scale)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    worst = ((out.double() - o).abs() / bound.clamp(min=1e-300)).max().item() if out.numel() else 0.0
    assert torch.isfinite(out.float()).all() and worst <= 1.0, worst
    return out


LENGTHS = [[1], [0], [15, 16, 17], [0, 3, 0, 129, 1, 0], [300, 5, 1000, 64, 31], [2, 2, 2, 2, 2, 2, 2], [4097]]


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths", LENGTHS, ids=str)
def test_lengths(lengths, e4m3):
    check(Cache(lengths, 4, 128, 16, e4m3, seed=len(lengths)), queries(len(lengths), 28, 128))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads, kv_heads, dim", [(1, 1, 16), (4, 4, 32), (14, 2, 64), (10, 10, 80), (24, 2, 96), (16, 16, 128), (9, 1, 128), (16, 1, 128),
                                                  (17, 1, 128), (40, 2, 64), (6, 2, 144), (3, 1, 192), (8, 1, 256), (33, 1, 256), (5, 5, 240), (71, 1, 64)])
def test_heads(heads, kv_heads, dim, e4m3):
    lengths = [37, 0, 1, 260]
    check(Cache(lengths, kv_heads, dim, 16, e4m3, seed=heads), queries(4, heads, dim, seed=heads))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("order", ["heads", "tokens", "wide"])
@pytest.mark.parametrize("block", [1, 5, 8, 16, 24, 48, 256, 1000])
def test_pages_and_orders(block, order, e4m3):
    check(Cache([1, 250, 33, 511], 2, 64, block, e4m3, seed=block, order=order), queries(4, 14, 64))


@pytest.mark.parametrize("e4m3", [False, True])
def test_long_context_is_split_and_joined(e4m3):
    c = Cache([50001, 3], 2, 128, 256, e4m3, seed=5)
    first = check(c, queries(2, 14, 128, spread=3.0))
    for _ in range(3):                                                  # whatever block comes last
        assert torch.equal(kernels().paged_attention(queries(2, 14, 128, spread=3.0), *c.args(), **c.scales()), first)


@pytest.mark.parametrize("e4m3", [False, True])
def test_many_sequences(e4m3):
    lengths = [(i * 37) % 90 for i in range(700)]                       # more than a block has threads, some empty
    check(Cache(lengths, 2, 64, 16, e4m3, seed=9), queries(700, 14, 64))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("seed", range(12))
def test_batches_of_any_lengths(seed, e4m3):
    """Lengths spread over their logarithm, so that sequences of all sizes share warps and CTAs in all ways; heads and pages at random."""
    r = np.random.default_rng(seed)
    heads, kv_heads, dim = [(28, 4, 128), (14, 2, 64), (16, 16, 128), (20, 1, 128), (12, 12, 64), (24, 2, 96), (8, 1, 256), (32, 8, 128)][seed % 8]
    batch = int(r.choice([1, 2, 5, 17, 33, 70, 150]))
    longest = int(r.choice([40, 400, 4000]) * (1 if batch > 30 else 4))
    lengths = [int(n) for n in np.exp(r.uniform(0, math.log(longest), batch))]
    for i in range(0, batch, 7):
        lengths[i] = 0
    check(Cache(lengths, kv_heads, dim, int(r.choice([3, 8, 16, 24, 64, 256])), e4m3, seed=seed), queries(batch, heads, dim, seed=seed))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("heads, kv_heads, length", [(8, 1, 70000), (20, 1, 33333), (16, 16, 9000), (3, 3, 30000)])
def test_one_sequence_over_many_ctas(heads, kv_heads, length, e4m3):
    """From a few pieces of a head to so many that they are joined in two steps."""
    c, q = Cache([length], kv_heads, 128, 64, e4m3, seed=7), queries(1, heads, 128, spread=2.0)
    first = check(c, q)
    for _ in range(3):
        assert torch.equal(kernels().paged_attention(q, *c.args(), **c.scales()), first)


def test_codes_as_bytes_and_heads_apart():
    """A cache of uint8 codes is one of float8; queries whose heads do not follow one another."""
    c = Cache([100, 37], 2, 64, 16, True)
    wide = torch.randn(2, 6, 3, 64, device="cuda").to(torch.bfloat16)
    q = wide[:, :, 1]
    want = check(c, q)
    k, v = c.k.view(torch.uint8), c.v.view(torch.uint8)
    assert torch.equal(kernels().paged_attention(q, k, v, c.tables, c.lens, **c.scales()), want)
    cu = torch.tensor([0, 100, 137], dtype=torch.int32, device="cuda")
    for x, y in zip(kernels().kv_cache_read(k, v, c.tables, cu, 137, c.ks, c.vs), kernels().kv_cache_read(c.k, c.v, c.tables, cu, 137, c.ks, c.vs)):
        assert torch.equal(x, y)


@pytest.mark.parametrize("e4m3", [False, True])
def test_sequences_that_share_pages(e4m3):
    """A common beginning in the same pages, as of a shared prompt."""
    c = Cache([200, 200], 2, 64, 16, e4m3, seed=8)
    tables = c.tables.clone()
    tables[1, :6] = tables[0, :6]
    q = queries(2, 8, 64)
    c.tables, c.rows[1] = tables, [torch.cat([a[:96], b[96:]]) for a, b in zip(c.rows[0], c.rows[1])]
    check(c, q)


@pytest.mark.parametrize("e4m3", [False, True])
def test_empty_batch_and_all_empty(e4m3):
    assert kernels().paged_attention(queries(0, 14, 64), *Cache([], 2, 64, 16, e4m3).args(), **Cache([], 2, 64, 16, e4m3).scales()).shape == (0, 14, 64)
    c = Cache([0] * 40, 2, 64, 16, e4m3)
    assert not kernels().paged_attention(queries(40, 14, 64), *c.args(), **c.scales()).any()
    c.lens.fill_(-5)                                                    # less than none is none
    assert not kernels().paged_attention(queries(40, 14, 64), *c.args(), **c.scales()).any()


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 1e-30])
def test_scales(scale, e4m3):
    check(Cache([200, 31], 2, 64, 16, e4m3, seed=3), queries(2, 8, 64), scale=scale)


@pytest.mark.parametrize("e4m3", [False, True])
def test_scores_far_apart(e4m3):
    """One token takes everything, late or early; scores of some hundreds; values that differ by orders of magnitude."""
    def keys(b, n):
        x = torch.randn(n, 2, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(b))
        x[(n - 1) if b % 2 else 0] *= 40
        return x

    def values(b, n):
        x = torch.randn(n, 2, 64, device="cuda", generator=torch.Generator(device="cuda").manual_seed(50 + b))
        return x * torch.logspace(-6, 6, n, device="cuda")[:, None, None]
    check(Cache([64, 65, 400, 401], 2, 64, 16, e4m3, k=keys, v=values), queries(4, 14, 64, spread=4.0))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("spread", [1e-20, 1e15])
def test_queries_of_any_size(spread, e4m3):
    """(scores as of ordinary queries: the scale undoes the size)"""
    q = queries(3, 7, 128, spread=spread)
    q[1, 2] = 0
    q[2, 3, 5:] *= 2.0 ** -30                                           # channels that matter little beside the others
    check(Cache([70, 9, 200], 1, 128, 16, e4m3), q, scale=0.1 / spread)


@pytest.mark.parametrize("e4m3", [False, True])
def test_what_is_not_finite_stays_where_it_is(e4m3):
    """A NaN or an infinity among a sequence's own keys reaches that sequence's heads of that key head, one among its values too."""
    c = Cache([40, 40, 40], 2, 64, 16, e4m3, seed=4)
    q = queries(3, 8, 64)
    clean = check(c, q)
    page = c.pages[1][1]
    if e4m3:
        c.ks[page, 3, 0] = math.nan
        c.vs[c.pages[2][0], 2, 1] = math.inf
    else:
        c.k[page, 3, 0, 7] = math.nan
        c.v[c.pages[2][0], 2, 1] = math.inf
    out = kernels().paged_attention(q, *c.args(), **c.scales())
    assert torch.isnan(out[1, :4].float()).all() and torch.equal(out[1, 4:], clean[1, 4:])
    assert not torch.isfinite(out[2, 4:].float()).any() and torch.equal(out[2, :4], clean[2, :4])
    assert torch.equal(out[0], clean[0])


@pytest.mark.parametrize("e4m3", [False, True])
def test_codes_are_those_of_the_quantiser(e4m3):
    Kn = kernels()
    c = Cache([40, 0, 700, 1], 2, 64, 16, e4m3, seed=4)
    q = queries(4, 14, 64)
    s = torch.tensor(0.003, device="cuda")
    codes = Kn.paged_attention(q, *c.args(), **c.scales(), out_scale=s)
    assert codes.dtype == torch.uint8 and codes.shape == q.shape
    assert torch.equal(codes.view(4, -1), Kn.quantize_activation(check(c, q).view(4, -1), s))
    assert (codes.view(E4M3).float().abs() == 448).any()                # (some are clamped)


def test_outputs_of_the_caller():
    Kn = kernels()
    c = Cache([40, 0, 700], 2, 64, 16, True, seed=4)
    q = queries(3, 14, 64)
    want = check(c, q)
    wide = torch.full((5, 14 * 64 + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    got = Kn.paged_attention(q, *c.args(), **c.scales(), out=wide[:3, :14 * 64])
    assert got.data_ptr() == wide.data_ptr() and torch.equal(wide[:3, :14 * 64].reshape(3, 14, 64), want)
    assert (wide[3:] == 7).all() and (wide[:, 14 * 64:] == 7).all()
    out3 = torch.empty(3, 14, 64, dtype=torch.bfloat16, device="cuda")
    assert torch.equal(Kn.paged_attention(q, *c.args(), **c.scales(), out=out3), want)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("lengths", [[7], [5000], [1, 0, 300, 17, 2000, 64], [40 + 7 * i for i in range(200)]], ids=len)
def test_result_in_place_of_the_queries(lengths, e4m3):
    """Every reader of a query has read it when its result is there: the same bits as in memory of its own."""
    heads, kv_heads, dim = 24, 2, 128
    c = Cache(lengths, kv_heads, dim, 16, e4m3)
    q = queries(len(lengths), heads, dim)
    want = kernels().paged_attention(q, *c.args(), **c.scales())
    for _ in range(5):
        own = queries(len(lengths), heads, dim)
        assert kernels().paged_attention(own, *c.args(), out=own, **c.scales()).data_ptr() == own.data_ptr()
        assert torch.equal(own, want)


@pytest.mark.parametrize("e4m3", [False, True])
def test_offsets_beyond_32_bits(e4m3):
    """The last pages of a cache of more than 4 GB."""
    dim, heads, block = 128, 4, 256
    blocks = (5 << 30) // (dim * heads * block * (1 if e4m3 else 2))
    shape = (blocks, heads, block, dim)
    pages = torch.empty((2, *shape), dtype=torch.uint8 if e4m3 else torch.bfloat16, device="cuda").view(E4M3 if e4m3 else torch.bfloat16).transpose(2, 3)
    scales = torch.empty((2, *shape[:3]), device="cuda").transpose(2, 3) if e4m3 else (None, None)
    Kn, n = kernels(), 300
    g = torch.Generator(device="cuda").manual_seed(2)
    k, v = (torch.randn(n, heads, dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    table = torch.tensor([[blocks - 1, blocks - 2]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = (table[0, at // block].long() * block + at % block).to(torch.int32)
    small = Cache([n], heads, dim, block, e4m3, k=lambda b, m: k, v=lambda b, m: v)
    Kn.kv_cache_write(k, v, slots, pages[0], pages[1], scales[0], scales[1])
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    for got, want in zip(Kn.kv_cache_read(pages[0], pages[1], table, cu, n, scales[0], scales[1]), small.rows[0]):
        torch.testing.assert_close(got.double(), want, rtol=BF16_HALF * 1.01, atol=0)
    q = queries(1, 28, dim)
    out = Kn.paged_attention(q, pages[0], pages[1], table, torch.tensor([n], dtype=torch.int32, device="cuda"), k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(out, check(small, q))


# ---- write and read ----------------------------------------------------------------------------------------------------------


def rows_of(tokens, kv_heads, dim, seed=0):
    """Keys and values as slices of one projection's output."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = torch.randn(tokens, 3 * kv_heads * dim, generator=g, device="cuda").to(torch.bfloat16)
    return (qkv[:, i * kv_heads * dim:(i + 1) * kv_heads * dim].view(tokens, kv_heads, dim) for i in (1, 2))


def plain_write(x, block, blocks, slots, e4m3, like):
    """What the cache holds afterwards, and its scales."""
    cache, scales = torch.zeros(like.shape, dtype=torch.uint8 if e4m3 else torch.bfloat16, device="cuda"), torch.zeros(like.shape[:3], device="cuda")
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            r = x[t]
            if e4m3:
                codes, scales[s // block, s % block] = quantised(r)
                r = codes.view(torch.uint8)
            cache[s // block, s % block] = r
    return cache, scales


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("tokens, kv_heads, dim, block", [(1, 1, 16, 1), (3, 4, 128, 16), (65, 2, 64, 5), (130, 16, 128, 16), (31, 3, 80, 24), (17, 1, 256, 256),
                                                          (40, 5, 240, 7), (9, 2, 144, 16), (333, 1, 32, 64)])
def test_write_and_read_back(pkg, tokens, kv_heads, dim, block, e4m3):
    k, v = rows_of(tokens, kv_heads, dim, seed=tokens)
    k[0] *= 1e-12                                                       # below the smallest scale's 1e-8
    v[tokens // 2, 0] = 0
    v[-1, -1] *= 1e30
    blocks = -(-tokens // block) + 2
    slots = torch.randperm(blocks * block)[:tokens].to(torch.int32).cuda()
    slots[::5] = -1
    c = pkg.PagedKVCache(blocks, block, kv_heads, dim, E4M3 if e4m3 else torch.bfloat16)
    c.write(k, v, slots)
    for x, cache, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want, scales = plain_write(x, block, blocks, slots, e4m3, cache)
        assert torch.equal(cache.view(torch.uint8) if e4m3 else cache, want)     # byte for byte
        if e4m3:
            assert torch.equal(scale, scales)
    # back: sequences over the pages in memory order, with an empty one among them
    ends = [0, min(3, blocks * block), min(3, blocks * block), blocks * block]
    tables = torch.full((3, blocks), 99, dtype=torch.int32, device="cuda")
    tables[0, :] = tables[2, :] = torch.arange(blocks, device="cuda")
    got = c.read(tables, torch.tensor(ends, dtype=torch.int32, device="cuda"), ends[-1])
    for out, cache, scale in zip(got, (c.k, c.v), (c.k_scale, c.v_scale)):
        flat = (cache.float() * scale[..., None] if e4m3 else cache).to(torch.bfloat16).reshape(blocks * block, kv_heads, dim)
        assert torch.equal(out, torch.cat([flat[:ends[1]], flat[:ends[3] - ends[2]]]))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("tokens, kv_heads, dim", [(5000, 4, 128), (3001, 3, 80), (700, 40, 64), (2000, 1, 256), (9000, 2, 48), (150, 130, 16), (20000, 10, 80), (9999, 16, 128)])
def test_many_rows_there_and_back(pkg, tokens, kv_heads, dim, e4m3):
    """More than a block's turn, heads that divide it and heads that do not; the formula's codes byte for byte, and many sequences."""
    k, v = rows_of(tokens, kv_heads, dim, seed=dim)
    block = 16
    c = pkg.PagedKVCache(-(-tokens // block), block, kv_heads, dim, E4M3 if e4m3 else torch.bfloat16)
    slots = torch.randperm(c.k.shape[0] * block, generator=torch.Generator().manual_seed(1))[:tokens].cuda()
    c.write(k, v, slots.to(torch.int32))
    ends = sorted(np.random.default_rng(2).integers(0, 3000, 1500).tolist())          # (more than a block keeps at hand)
    ends = [0] + [min(e, 3 * block) for e in ends[:3]] + [3 * block + i // 8 for i in range(1500)]
    tables = torch.arange(c.k.shape[0], dtype=torch.int32, device="cuda").expand(len(ends) - 1, -1).contiguous()
    got = c.read(tables, torch.tensor(ends, dtype=torch.int32, device="cuda"), ends[-1])
    for x, cache, scale, out in ((k, c.k, c.k_scale, got[0]), (v, c.v, c.v_scale, got[1])):
        at = slots // block, slots % block
        if e4m3:
            codes, s = quantised(x)
            assert torch.equal(cache.view(torch.uint8)[at], codes.view(torch.uint8)) and torch.equal(scale[at], s)
        else:
            assert torch.equal(cache[at], x)
        flat = (cache.float() * scale[..., None] if e4m3 else cache).to(torch.bfloat16).reshape(-1, kv_heads, dim)
        assert torch.equal(out, torch.cat([flat[:b - a] for a, b in zip(ends, ends[1:])]))


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("kv_heads, dim", [(10, 80), (16, 128), (1, 16)])
def test_reads_of_every_length(pkg, kv_heads, dim, e4m3):
    """From one token to more than the chip's blocks hold at a time; what lies behind the last sequence stays as it was."""
    block, blocks = 24, 1600
    c = pkg.PagedKVCache(blocks, block, kv_heads, dim, E4M3 if e4m3 else torch.bfloat16)
    c.write(*rows_of(blocks * block, kv_heads, dim, seed=4), torch.arange(blocks * block, dtype=torch.int32, device="cuda"))
    pages = torch.randperm(blocks, generator=torch.Generator().manual_seed(5)).cuda()
    tables = torch.stack([pages[:800], pages[800:]]).to(torch.int32)
    for ends in ([0, 1, 1], [0, 700, 1000], [0, 5, 9001], [0, 19199, 30011], [0, 0, 7111]):
        rows = ends[-1] + 3
        out = [torch.full((rows, kv_heads, dim), 7.0, dtype=torch.bfloat16, device="cuda") for _ in "kv"]
        kernels().kv_cache_read(c.k, c.v, tables, torch.tensor(ends, dtype=torch.int32, device="cuda"), rows, c.k_scale, c.v_scale, *out)
        for cache, scale, got in ((c.k, c.k_scale, out[0]), (c.v, c.v_scale, out[1])):
            flat = (cache.float() * scale[..., None] if e4m3 else cache).to(torch.bfloat16)
            want = [flat[tables[b].long()].reshape(-1, kv_heads, dim)[:ends[b + 1] - ends[b]] for b in range(2)]
            assert torch.equal(got, torch.cat([*want, torch.full_like(got[:3], 7.0)]))


@pytest.mark.parametrize("rows", [0, 1, 37])
def test_results_of_a_read_are_tensors_of_their_own(pkg, rows):
    c = pkg.PagedKVCache(4, 16, 3, 48)
    k, v = rows_of(64, 3, 48, seed=6)
    c.write(k, v, torch.arange(64, dtype=torch.int32, device="cuda"))
    tables, cu = torch.arange(4, dtype=torch.int32, device="cuda")[None], torch.tensor([0, rows], dtype=torch.int32, device="cuda")
    mine = torch.empty(rows, 3, 48, dtype=torch.bfloat16, device="cuda")
    with torch.inference_mode():
        pairs = [c.read(tables, cu, rows), kernels().kv_cache_read(c.k, c.v, tables, cu, rows, v_out=mine), kernels().kv_cache_read(c.k, c.v, tables, cu, rows, k_out=mine)]
    pairs[1:1] = [c.read(tables, cu, rows)]
    for got in pairs[:2]:
        assert torch.equal(got[0], k[:rows]) and torch.equal(got[1], v[:rows])
        for x in got:
            assert x.shape == (rows, 3, 48) and x.is_contiguous() and not x.requires_grad and x._base is None
    assert torch.equal(pairs[2][0], k[:rows]) and torch.equal(pairs[3][1], v[:rows])
    a, b = pairs[1]
    a.zero_()                                             # (in place: one does not reach into the other)
    assert torch.equal(b, v[:rows]) and torch.equal(b.clone().float(), v[:rows].float())
    del a, pairs
    assert torch.equal(b, v[:rows])


@pytest.mark.parametrize("order", ["heads", "tokens", "wide"])
@pytest.mark.parametrize("e4m3", [False, True])
def test_read_of_a_batch(e4m3, order):
    c = Cache([5, 0, 700, 33, 0], 3, 80, 24, e4m3, order=order)
    cu = torch.tensor([0, 5, 5, 705, 738, 738], dtype=torch.int32, device="cuda")
    outs = [torch.full((750, 3, 96), 3.0, dtype=torch.bfloat16, device="cuda")[:, :, :80] for _ in range(2)]
    got = kernels().kv_cache_read(c.k, c.v, c.tables, cu, 750, c.ks, c.vs, outs[0], outs[1])
    for i, out in enumerate(got):
        assert out.data_ptr() == outs[i].data_ptr()
        want = torch.cat([r[i] for r in c.rows])
        torch.testing.assert_close(out[:738].double(), want, rtol=BF16_HALF + 2.0 ** -23, atol=0)
        assert (out[738:] == 3).all()                                   # rows behind the last sequence


def test_rows_that_are_not_finite(pkg):
    """An infinity or a NaN makes the row's scale one, and all that is read back of the row a NaN; its neighbours keep theirs."""
    k, v = rows_of(4, 2, 64)
    k[1, 0, 5], k[2, 1, 6], v[0, 0, 0] = math.inf, math.nan, -math.inf
    c = pkg.PagedKVCache(1, 16, 2, 64, E4M3)
    c.write(k, v, torch.arange(4, dtype=torch.int32, device="cuda"))
    for x, cache, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
        want, scales = plain_write(x, 16, 1, torch.arange(4), True, cache)
        np.testing.assert_array_equal(cache.float().cpu().numpy(), want.view(E4M3).float().cpu().numpy())
        np.testing.assert_array_equal(scale.cpu().numpy(), scales.cpu().numpy())
    rk, rv = c.read(torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([0, 4], dtype=torch.int32, device="cuda"), 4)
    bad = torch.zeros(4, 2, dtype=torch.bool, device="cuda")
    bad[1, 0] = bad[2, 1] = True
    assert torch.equal(torch.isnan(rk.float()).all(-1), bad) and torch.equal(torch.isnan(rk.float()).any(-1), bad)
    assert torch.isnan(rv[0, 0].float()).all() and torch.isfinite(rv[1:].float()).all()


def test_every_bf16_value_is_quantised_as_by_a_division(pkg):
    """All finite bf16 values, in rows of 64 with their neighbours: the codes and scales of the formula, bit for bit."""
    bits = torch.arange(0, 0x7f80, dtype=torch.int32)
    x = torch.cat([bits, bits | 0x8000]).to(torch.uint16).view(torch.bfloat16).cuda()
    x = torch.cat([x.view(-1, 1, 64), x[torch.randperm(x.numel(), generator=torch.Generator().manual_seed(1)).cuda()].view(-1, 1, 64)])
    c = pkg.PagedKVCache(x.shape[0], 1, 1, 64, E4M3)
    c.write(x, -x, torch.arange(x.shape[0], dtype=torch.int32, device="cuda"))
    codes, scale = quantised(x)
    assert torch.equal(c.k_scale[:, 0], scale) and torch.equal(c.v_scale[:, 0], scale)
    assert torch.equal(c.k[:, 0].view(torch.uint8), codes.view(torch.uint8))


# ---- refusals -----------------------------------------------------------------------------------------------------------------


def test_refusals_of_the_binding():
    Kn = kernels()
    c = Cache([5, 6], 2, 64, 16, True)
    q, k = queries(2, 14, 64), queries(2, 2, 64)
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    cu = torch.zeros(3, dtype=torch.int32, device="cuda")

    def refuses(fn, *a, **kw):
        with pytest.raises(ValueError):
            fn(*a, **kw)
    sc = c.scales()
    for bad in (dict(q=q.float()), dict(q=q[:, :13]), dict(q=q[:, :, :48]), dict(q=q[:1]), dict(q=q.cpu()), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(k_cache=c.k.float()), dict(k_cache=c.k[:, :, :1]), dict(v_cache=c.v.contiguous()), dict(k_cache=c.k.cpu()), dict(k_cache=c.k[0]),
                dict(block_tables=c.tables.long()), dict(block_tables=c.tables[0]), dict(block_tables=c.tables[:1]), dict(block_tables=c.tables.cpu()),
                dict(context_lens=c.lens.long()), dict(context_lens=c.lens[:1]), dict(k_scale=None), dict(k_scale=c.ks.half()), dict(v_scale=c.vs.contiguous()),
                dict(k_scale=c.ks[:1]), dict(out_scale=torch.ones(2, device="cuda")), dict(out_scale=torch.tensor(1.0)), dict(out=q.float()),
                dict(out=torch.empty(2, 13, 64, dtype=torch.bfloat16, device="cuda")), dict(out=torch.empty(2, 14, 64, dtype=torch.uint8, device="cuda"))):
        refuses(Kn.paged_attention, **{**dict(q=q, k_cache=c.k, v_cache=c.v, block_tables=c.tables, context_lens=c.lens, **sc), **bad})
    plain = Cache([5, 6], 2, 64, 16, False)
    refuses(Kn.paged_attention, q, *plain.args(), **sc)                  # scales beside a bf16 cache
    for bad in (dict(k=k.float()), dict(k=k[:1]), dict(v=k[:, :1]), dict(slot_mapping=i.long()), dict(slot_mapping=i[:1]), dict(k=k.cpu()), dict(slot_mapping=i.cpu()),
                dict(v_cache=c.k.view(torch.uint8))):
        refuses(Kn.kv_cache_write, **{**dict(k=k, v=k, slot_mapping=i, k_cache=c.k, v_cache=c.v, **sc), **bad})
    for bad in (dict(rows=-1), dict(cu_seqlens=cu[:2]), dict(cu_seqlens=cu.long()), dict(block_tables=c.tables.long()), dict(k_out=k.float()), dict(v_out=k[:1])):
        refuses(Kn.kv_cache_read, **{**dict(k_cache=c.k, v_cache=c.v, block_tables=c.tables, cu_seqlens=cu, rows=2, **sc), **bad})
    odd = torch.zeros(4 * 16 * 2 * 72 + 1, dtype=torch.bfloat16, device="cuda")
    refuses(Kn.paged_attention, q, odd[1:].view(4, 16, 2, 72)[..., :64], odd[1:].view(4, 16, 2, 72)[..., :64], c.tables, c.lens)      # not on 16 bytes
    torch.cuda.synchronize()
    assert Kn.read_status(torch.device("cuda", 0)) == 0


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_slot_or_page_outside_the_cache_is_reported(pkg, e4m3):
    """The kernels compare every page with the cache's before they go there; the next call on the stream raises."""
    Kn, dev = kernels(), torch.device("cuda", 0)
    c = Cache([40, 40], 2, 64, 16, e4m3)
    q = queries(2, 8, 64)
    want = check(c, q)

    def raises_once():
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="outside the key-value cache"):
            Kn.paged_attention(q, *c.args(), **c.scales())
        assert torch.equal(Kn.paged_attention(q, *c.args(), **c.scales()), want)     # the one after is clean
        assert Kn.read_status(dev) == 0
    blocks = c.k.shape[0]
    for page in (-1, blocks, 2 ** 31 - 1, -2 ** 31):
        tables = c.tables.clone()
        tables[0, 1] = page
        out = Kn.paged_attention(q, c.k, c.v, tables, c.lens, **c.scales())
        assert torch.equal(out[1], want[1])                                          # the other sequence
        raises_once()
    long = torch.tensor([40, 16 * c.tables.shape[1] + 1], dtype=torch.int32, device="cuda")
    Kn.paged_attention(q, c.k, c.v, c.tables[:, :3], long, **c.scales())             # longer than its table
    raises_once()
    k, v = rows_of(3, 2, 64)
    before = [t.clone() for t in (c.k.view(torch.uint8), c.v.view(torch.uint8))]
    Kn.kv_cache_write(k, v, torch.tensor([-1, blocks * 16, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), c.k, c.v, c.ks, c.vs)
    raises_once()
    assert all(torch.equal(x, y.view(torch.uint8)) for x, y in zip(before, (c.k, c.v)))
    tables = c.tables.clone()
    tables[1, 2] = blocks
    cu = torch.tensor([0, 40, 80], dtype=torch.int32, device="cuda")
    rows = Kn.kv_cache_read(c.k, c.v, tables, cu, 80, c.ks, c.vs)[0]
    torch.testing.assert_close(rows[:72].double(), torch.cat([c.rows[0][0], c.rows[1][0][:32]]), rtol=BF16_HALF + 2.0 ** -23, atol=0)
    raises_once()


# ---- streams, graphs, the layer -----------------------------------------------------------------------------------------------


def test_calls_on_several_streams():
    """Every stream has scratch of its own: calls that run beside one another give what they give alone."""
    Kn = kernels()
    caches = [Cache([20000 + 999 * i, 7], 2, 128, 64, bool(i % 2), seed=i) for i in range(4)]
    q = queries(2, 14, 128)
    want = [check(c, q) for c in caches]
    streams = [torch.cuda.Stream() for _ in caches]
    torch.cuda.synchronize()
    got = [[] for _ in caches]
    for _ in range(5):
        for c, s, g in zip(caches, streams, got):
            with torch.cuda.stream(s):
                g.append(Kn.paged_attention(q, *c.args(), **c.scales()))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_calls_of_several_threads():
    Kn = kernels()
    caches = [Cache([9000 + 555 * i, 40, 7], 4, 64, 32, bool(i % 2), seed=i) for i in range(3)]
    q = queries(3, 16, 64)
    want = [check(c, q) for c in caches]
    wrong = []

    def work(c, w):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    if not torch.equal(Kn.paged_attention(q, *c.args(), **c.scales()), w):
                        wrong.append("differs")
        except Exception as e:                            # noqa: BLE001  (shown by the assertion below)
            wrong.append(repr(e))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=x) for x in zip(caches, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("e4m3", [False, True])
def test_tables_and_lengths_of_any_layout(e4m3):
    """Slices of wider tables, tables of one page per sequence, of none."""
    Kn = kernels()
    c = Cache([40, 0, 700, 16], 2, 64, 16, e4m3, seed=8)
    q = queries(4, 14, 64)
    want = check(c, q)
    wide = torch.full((4, c.tables.shape[1] + 13), -9, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + c.tables.shape[1]] = c.tables
    lens = torch.stack([c.lens, c.lens + 1])[0]
    assert torch.equal(Kn.paged_attention(q, c.k, c.v, wide[:, 5:5 + c.tables.shape[1]], lens, **c.scales()), want)
    c = Cache([16, 3, 0, 9], 2, 64, 16, e4m3, seed=9)
    want = check(c, q)
    assert torch.equal(Kn.paged_attention(q, c.k, c.v, c.tables[:, :1], c.lens, **c.scales()), want)
    assert torch.equal(Kn.paged_attention(q, c.k, c.v, c.tables[:, 0].contiguous()[:, None], c.lens, **c.scales()), want)
    assert not Kn.paged_attention(q, c.k, c.v, c.tables[:, :0], torch.zeros_like(c.lens), **c.scales()).any()


def test_a_cache_of_all_layers(pkg):
    """The layout in which an engine allocates it: [2, layers, blocks, tokens, heads, channels] in one tensor."""
    Kn, layers, (blocks, block, heads, dim) = kernels(), 3, (9, 16, 2, 64)
    whole = torch.zeros(2, layers, blocks, block, heads, dim, dtype=torch.bfloat16, device="cuda")
    tables = torch.tensor([[3, 0, 8], [5, 2, 7]], dtype=torch.int32, device="cuda")
    lens = [40, 17]
    rows = [tuple(rows_of(57, heads, dim, seed=i)) for i in range(layers)]
    slots = torch.cat([tables[b].long().repeat_interleave(block)[:n] * block + torch.arange(n, device="cuda") % block for b, n in enumerate(lens)]).to(torch.int32)
    for (k, v), kc, vc in zip(rows, whole[0], whole[1]):
        Kn.kv_cache_write(k, v, slots, kc, vc)
    cu = torch.tensor([0, 40, 57], dtype=torch.int32, device="cuda")
    own = pkg.PagedKVCache(blocks, block, heads, dim)
    q = queries(2, 14, dim)
    for (k, v), kc, vc in zip(rows, whole[0], whole[1]):
        got = Kn.kv_cache_read(kc, vc, tables, cu, 57)
        assert torch.equal(got[0], k) and torch.equal(got[1], v)
        own.write(k, v, slots)
        n = torch.tensor(lens, dtype=torch.int32, device="cuda")
        assert torch.equal(Kn.paged_attention(q, kc, vc, tables, n), Kn.paged_attention(q, own.k, own.v, tables, n))


@pytest.mark.parametrize("e4m3", [False, True])
def test_a_captured_step_follows_lengths_pages_and_slots(pkg, e4m3):
    """One graph, replayed as the sequences grow over page ends and the batch's padding changes."""
    Kn = kernels()
    heads, kv_heads, dim, block, batch, steps = 14, 2, 64, 16, 4, 36
    layer = pkg.PagedAttention(heads, dim, num_kv_heads=kv_heads)
    layer.cache = pkg.PagedKVCache(16, block, kv_heads, dim, E4M3 if e4m3 else torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(0)
    data = torch.randn(steps, batch, (heads + 2 * kv_heads) * dim, generator=g, device="cuda").to(torch.bfloat16)
    qkv = torch.zeros(data.shape[1:], dtype=torch.bfloat16, device="cuda")
    slots, lens = torch.full((batch,), -1, dtype=torch.int32, device="cuda"), torch.zeros(batch, dtype=torch.int32, device="cuda")
    tables = torch.arange(16, dtype=torch.int32, device="cuda").view(4, 4).flip(1).contiguous()
    a, b = heads * dim, (heads + kv_heads) * dim
    run = lambda: layer(qkv[:, :a], qkv[:, a:b], qkv[:, b:], slots, tables, lens)           # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        Kn.reserve_workspace(torch.device("cuda", 0), Kn.paged_attention_workspace_bytes(heads, kv_heads, dim))
        run()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = run()
        kept = [[] for _ in range(batch)]
        for t in range(steps):
            live = [i for i in range(batch) if t >= 3 * i]                                  # sequences join one after the other
            at = torch.tensor([len(kept[i]) if i in live else 0 for i in range(batch)], device="cuda")
            slot = tables[torch.arange(batch, device="cuda"), at // block] * block + (at % block).to(torch.int32)
            alive = torch.tensor([i in live for i in range(batch)], device="cuda")
            slots.copy_(torch.where(alive, slot, -1))
            lens.copy_(torch.where(alive, at + 1, 0).to(torch.int32))
            qkv.copy_(data[t])
            graph.replay()
            got = out.clone()
            for i in live:
                kept[i].append(data[t, i])
            assert torch.equal(got, run())                                                  # (the same token written again)
            if t % 7 == 0 or t == steps - 1:
                for i in range(batch):
                    if i not in live:
                        assert not got[i].any()
                        continue
                    rows = torch.stack(kept[i])
                    c = Cache([len(rows)], kv_heads, dim, block, e4m3, k=lambda *_: rows[:, a:b].reshape(-1, kv_heads, dim),
                              v=lambda *_: rows[:, b:].reshape(-1, kv_heads, dim))
                    o, bound = definition(c, data[t, i:i + 1, :a].view(1, heads, dim), dim ** -0.5)
                    assert ((got[i].view(1, heads, dim).double() - o).abs() <= bound).all()
        assert Kn.read_status(torch.device("cuda", 0)) == 0


def test_two_graphs_share_a_streams_scratch(pkg):
    """Captured one after the other on one stream, replayed in turn on it."""
    Kn = kernels()
    caches = [Cache([9000, 5], 2, 128, 64, True, seed=1), Cache([33, 12345], 2, 128, 64, True, seed=2)]
    q = queries(2, 14, 128)
    want = [check(c, q) for c in caches]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        Kn.paged_attention(q, *caches[0].args(), **caches[0].scales())
        graphs, outs = [], []
        for c in caches:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                outs.append(Kn.paged_attention(q, *c.args(), **c.scales()))
            graphs.append(graph)
        for i in (0, 1, 1, 0, 1, 0):
            outs[i].zero_()
            graphs[i].replay()
            assert torch.equal(outs[i], want[i])


def test_growing_scratch_inside_a_capture_is_refused(pkg):
    Kn = kernels()
    c = Cache([100], 1, 128, 16, False)
    q = queries(1, 8, 128)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match="capture"):
            with torch.cuda.graph(graph, stream=side):
                Kn.paged_attention(q, *c.args())
    check(c, q)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("batch", [1, 5, 33])
def test_between_the_projections_of_a_decoder_layer(pkg, batch, e4m3):
    """norm -> codes -> qkv -> cache and attention -> codes -> o_proj: the codes give what the bf16 result gives, and both follow
    the definition."""
    Kn, ex = kernels(), importlib.import_module("nano-vllm-moe_b200.quantization.export")
    hidden, heads, kv_heads, dim, block = 512, 8, 2, 64, 16
    cfg = pkg.Fp8Config("fp8_w8a8_static")
    g = torch.Generator(device="cuda").manual_seed(batch)

    def fill(lay, scale):
        n, k = lay.weight_scale.numel(), lay.qweight.shape[0]
        codes, s = ex.quantize_weight(torch.randn(n, k, generator=g, device="cuda") * 0.05)
        lay.qweight.copy_(codes.t().cpu())
        lay.weight_scale.copy_(s.cpu())
        lay.input_scale.copy_(torch.tensor(scale))
        lay = lay.cuda()
        pkg.process_weights_after_loading(lay)
        return lay
    qkv_proj = fill(pkg.QKVParallelLinear(hidden, dim, heads, kv_heads, quant_method=cfg.get_quant_method(None, "qkv")), 5.0 / 448)
    o_proj = fill(pkg.RowParallelLinear(heads * dim, hidden, quant_method=cfg.get_quant_method(None, "o")), 2.0 / 448)
    norm = pkg.RMSNorm(hidden).cuda().bfloat16()
    attn = pkg.PagedAttention(heads, dim, num_kv_heads=kv_heads)
    lengths = [1 + (17 * b) % 50 for b in range(batch)]
    past = Cache([n - 1 for n in lengths], kv_heads, dim, block, e4m3, spare=batch + 1)
    owned = {p for pages in past.pages for p in pages}
    free = [p for p in range(past.k.shape[0]) if p not in owned]
    slots = []
    for b, n in enumerate(lengths):
        if (n - 1) % block == 0:
            past.pages[b].append(free.pop())
            past.tables[b, (n - 1) // block] = past.pages[b][-1]
        slots.append(past.pages[b][-1] * block + (n - 1) % block)
    slots = torch.tensor(slots, dtype=torch.int32, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    cache = pkg.PagedKVCache(1, block, kv_heads, dim, E4M3 if e4m3 else torch.bfloat16)
    cache.k, cache.v, cache.k_scale, cache.v_scale = past.k, past.v, past.ks, past.vs
    attn.cache = cache
    x = torch.randn(batch, hidden, generator=g, device="cuda").to(torch.bfloat16)
    codes, _ = norm.forward_quant(x, qkv_proj.input_scale)
    qkv = qkv_proj(codes)
    q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], -1)
    y = attn(q, k, v, slots, past.tables, lens)
    quant = attn.forward_quant(q, None, None, None, past.tables, lens, o_proj.input_scale)     # (the token is in the cache now)
    assert quant.codes.shape == (batch, heads * dim)
    assert torch.equal(o_proj(quant), o_proj(y) if batch > 16 else Kn.launch_w8a8_preq(Kn.quantize_activation(y, o_proj.input_scale), o_proj.qweight_packed,
                                                                                      o_proj.input_scale, o_proj.weight_scale))
    for i, t in enumerate((k, v)):
        for b in range(batch):
            r = t[b].view(1, kv_heads, dim)
            if e4m3:
                codes, s = quantised(r)
                r = codes.double() * s.double()[..., None]
            past.rows[b][i] = torch.cat([past.rows[b][i], r.double()])
    past.lengths = lengths
    o, bound = definition(past, q.view(batch, heads, dim), dim ** -0.5)
    assert ((y.view(batch, heads, dim).double() - o).abs() <= bound).all()
