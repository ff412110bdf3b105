"""Codes through a row-parallel layer on two gloo ranks: the ranks' products summed, whatever form bfloat16 activations would take."""
import importlib
import os
import socket
import sys
from pathlib import Path

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

ROOT = Path(__file__).resolve().parent.parent
K, N, ROWS = 32, 24, 700


def _worker(rank, world, port):
    sys.path.insert(0, str(ROOT))
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    pkg = importlib.import_module("nano-vllm-moe_b200")

    class Method(pkg.QuantizeMethodBase):               # a product of codes on the CPU; all sums are of whole numbers
        def create_weights(self, layer, **kw):
            layer.w = None

        def apply(self, layer, x, bias=None):
            y = x.codes.float() @ layer.w.t()
            return y if bias is None else y + bias

        def process_weights_after_loading(self, layer):
            pass
    g = torch.Generator().manual_seed(7)
    codes = torch.randint(0, 16, (ROWS, K), generator=g, dtype=torch.uint8)
    w = torch.randint(-8, 8, (N, K), generator=g).float()
    bias = torch.arange(N, dtype=torch.float32)
    part = slice(rank * K // world, (rank + 1) * K // world)
    for peer_reduce in ("auto", True, "rs", False):
        lay = pkg.RowParallelLinear(K, N, bias=True, quant_method=Method())
        lay.w, lay.peer_reduce, lay.peer_reduce_min_rows, lay.overlap_min_rows = w[:, part], peer_reduce, 1, 1
        lay.bias.data = bias
        x = pkg.QuantizedActivation(codes[:, part].contiguous(), torch.tensor(1.0))
        assert torch.equal(lay(x), codes.float() @ w.t() + bias), (rank, peer_reduce)
        lay.reduce_results = False
        assert torch.equal(lay(x), codes[:, part].float() @ w[:, part].t() + (bias if rank == 0 else 0)), (rank, peer_reduce)
        lay.reduce_results = "scatter"
        with pytest.raises(ValueError, match="codes"):
            lay(x)
    dist.destroy_process_group()


def test_codes_are_summed_over_the_ranks():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port), nprocs=2, join=True)
