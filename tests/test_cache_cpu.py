"""The paged cache and the decode attention without a GPU: what is refused, and how the cache lies in memory."""
import ctypes

import pytest
import torch

from helpers import kernels

E4M3 = torch.float8_e4m3fn


def cache_struct(L, p, **changed):
    # 3 pages of 4 tokens, 2 heads of 32 channels, [block][head][token][channel]
    fields = dict(k=p, v=p, k_scale=p, v_scale=p, num_blocks=3, stride_block=256, stride_token=32, stride_head=128,
                  scale_stride_block=8, scale_stride_token=1, scale_stride_head=4, block_size=4, num_kv_heads=2, head_dim=32,
                  dtype=L.CACHE_E4M3)
    return L.KvCache(**{**fields, **changed})


@pytest.fixture()
def memory():
    buf = ctypes.create_string_buffer(1 << 17)
    yield (ctypes.addressof(buf) + 255) & ~255


BAD_CACHES = [
    (dict(dtype=2), "ERR_ARG"), (dict(num_blocks=0), "ERR_SHAPE"), (dict(block_size=0), "ERR_SHAPE"), (dict(num_kv_heads=0), "ERR_SHAPE"),
    (dict(head_dim=8), "ERR_SHAPE"), (dict(head_dim=40), "ERR_SHAPE"), (dict(head_dim=272), "ERR_SHAPE"), (dict(k=None), "ERR_NULL"),
    (dict(v=None), "ERR_NULL"), (dict(k_scale=None), "ERR_NULL"), (dict(v_scale=None), "ERR_NULL"), (dict(k=1), "ERR_ALIGN"),
    (dict(stride_token=24), "ERR_ALIGN"), (dict(stride_block=0), "ERR_ALIGN"), (dict(stride_head=-128), "ERR_ALIGN"),
    (dict(scale_stride_head=0), "ERR_SHAPE"),
]


@pytest.mark.parametrize("changed, code", BAD_CACHES, ids=[f"{k}={v}" for c, _ in BAD_CACHES for k, v in c.items()])
def test_bad_caches_are_refused(pkg, memory, changed, code):
    L, lib, p = pkg._lib, pkg._lib.load(), memory
    c = ctypes.byref(cache_struct(L, p, **{k: (p + v if k == "k" and v else v) for k, v in changed.items()}))
    want = getattr(L, code)
    assert lib.fp8lin_kv_cache_write(c, p, 64, 32, p, 64, 32, p, 1, p, 65536, None) == want
    assert lib.fp8lin_kv_cache_read(c, p, 1, 1, p, 1, p, 64, 32, p, 64, 32, 1, p, 65536, None) == want
    assert lib.fp8lin_paged_attention(c, p, 64, 32, p, 1, 1, p, 1, 2, 1.0, None, p, 64, p, 65536, None) == want


def test_bad_arguments_are_refused(pkg, memory):
    L, lib, p = pkg._lib, pkg._lib.load(), memory
    c = ctypes.byref(cache_struct(L, p))
    assert lib.fp8lin_kv_cache_write(None, p, 64, 32, p, 64, 32, p, 1, p, 65536, None) == L.ERR_NULL

    def write(k=p, kt=64, kh=32, v=p, slots=p, tokens=2, ws=p, size=65536):
        return lib.fp8lin_kv_cache_write(c, k, kt, kh, v, 64, 32, slots, tokens, ws, size, None)
    assert write(tokens=0, k=None, slots=None) == L.OK
    assert write(tokens=-1) == L.ERR_SHAPE
    assert write(k=None) == write(v=None) == write(slots=None) == L.ERR_NULL
    assert write(k=p + 2) == write(kt=60) == write(kh=0) == L.ERR_ALIGN
    assert write(ws=None) == write(size=65535) == L.ERR_WORKSPACE

    def read(tables=p, ld=4, pages=4, cu=p, batch=2, k=p, rows=3, ws=p):
        return lib.fp8lin_kv_cache_read(c, tables, ld, pages, cu, batch, k, 64, 32, p, 64, 32, rows, ws, 65536, None)
    assert read(rows=0) == read(batch=0) == L.OK
    assert read(rows=-1) == read(batch=-1) == read(ld=3) == read(pages=-1) == L.ERR_SHAPE
    assert read(tables=None) == read(cu=None) == read(k=None) == L.ERR_NULL
    assert read(k=p + 8) == L.ERR_ALIGN
    assert read(ws=None) == L.ERR_WORKSPACE

    need = lib.fp8lin_paged_attention_workspace_bytes(4, 2, 32, L.CACHE_E4M3)
    assert need >= L.WS_HEADER_BYTES

    def attend(q=p, qr=128, qh=32, tables=p, ld=4, pages=4, lens=p, batch=2, heads=4, out_scale=None, out=p, ld_out=128, ws=p, size=need):
        return lib.fp8lin_paged_attention(c, q, qr, qh, tables, ld, pages, lens, batch, heads, 1.0, out_scale, out, ld_out, ws, size, None)
    assert attend(batch=0, q=None) == L.OK
    assert attend(batch=1 << 24, heads=256, qr=128 * 256) == L.ERR_SHAPE
    assert attend(heads=3) == attend(heads=0) == attend(batch=-1) == attend(ld=3) == L.ERR_SHAPE
    assert attend(q=None) == attend(tables=None) == attend(lens=None) == attend(out=None) == L.ERR_NULL
    assert attend(q=p + 2) == attend(qr=100) == attend(qh=12) == attend(out=p + 8) == attend(ld_out=120) == attend(ld_out=132) == L.ERR_ALIGN
    assert attend(out_scale=p, ld_out=136) == L.ERR_ALIGN
    assert attend(ws=None) == attend(size=need - 1) == L.ERR_WORKSPACE


def test_scratch_does_not_depend_on_the_batch(pkg):
    Kn = kernels()
    for heads, kv_heads, dim in [(28, 4, 128), (16, 16, 128), (20, 1, 128), (8, 1, 256), (14, 2, 64)]:
        for dtype in (torch.bfloat16, E4M3):
            need = Kn.paged_attention_workspace_bytes(heads, kv_heads, dim, dtype)
            assert pkg._lib.WS_HEADER_BYTES <= need < (32 << 20)


def test_cpu_tensors_are_refused(pkg):
    Kn = kernels()
    x = torch.zeros(2, 1, 16, dtype=torch.bfloat16)
    pages = torch.zeros(2, 4, 1, 16, dtype=torch.bfloat16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        Kn.kv_cache_write(x, x, i, pages, pages)
    with pytest.raises(ValueError, match="CUDA"):
        Kn.kv_cache_read(pages, pages, i[:1, None], i, 2)
    with pytest.raises(ValueError, match="CUDA"):
        Kn.paged_attention(x, pages, pages, i[:, None], i)
    layer = pkg.PagedAttention(1, 16)
    layer.cache = pkg.PagedKVCache(2, 4, 1, 16, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        layer(x.view(2, 16), x.view(2, 16), x.view(2, 16), i, i[:, None], i)


def test_layer_refusals(pkg):
    with pytest.raises(ValueError, match="multiple"):
        pkg.PagedAttention(6, 64, num_kv_heads=4)
    for bad in (dict(dtype=torch.float16), dict(head_dim=24), dict(head_dim=0), dict(num_blocks=0), dict(block_size=0)):
        with pytest.raises(ValueError):
            pkg.PagedKVCache(**{**dict(num_blocks=2, block_size=4, num_kv_heads=1, head_dim=16, device="cpu"), **bad})
    assert pkg.PagedAttention(4, 64).num_kv_heads == 4 and pkg.PagedAttention(4, 64).scale == 0.125


@pytest.mark.parametrize("dtype", [torch.bfloat16, E4M3])
def test_cache_layout(pkg, dtype):
    c = pkg.PagedKVCache(3, 8, 2, 32, dtype=dtype, device="cpu")
    for t in (c.k, c.v):
        assert t.shape == (3, 8, 2, 32) and t.dtype == dtype and t.stride() == (512, 32, 256, 1)
    assert not torch.any(c.k.float()) and c.k.data_ptr() != c.v.data_ptr()
    if dtype == E4M3:
        assert c.k_scale.shape == (3, 8, 2) and c.k_scale.stride() == (16, 1, 8)
    else:
        assert c.k_scale is None and c.v_scale is None


def test_row_parallel_sums_what_codes_give(pkg, monkeypatch):
    """Codes of a decode step through o_proj on several ranks: the local product, summed by the all-reduce."""
    from importlib import import_module
    linear = import_module("nano-vllm-moe_b200.layers.linear")
    seen = []

    class Method(pkg.QuantizeMethodBase):
        def create_weights(self, layer, **kw):
            pass

        def apply(self, layer, x, bias=None):
            seen.append((x, bias))
            return torch.ones(2, 8)

        def process_weights_after_loading(self, layer):
            pass
    lay = pkg.RowParallelLinear(32, 8, quant_method=Method())
    lay.tp_size, lay.tp_rank = 2, 1
    monkeypatch.setattr(linear.dist, "all_reduce", lambda y, group=None: y.mul_(2))
    codes = pkg.QuantizedActivation(torch.zeros(2, 16, dtype=torch.uint8), torch.tensor(1.0))
    assert torch.equal(lay(codes), torch.full((2, 8), 2.0)) and seen == [(codes, None)]
    lay.reduce_results = False
    assert torch.equal(lay(codes), torch.ones(2, 8))
    lay.reduce_results = "scatter"
    with pytest.raises(ValueError, match="codes"):
        lay(codes)
