"""ShardedIndex.search with an adapter, as two `gloo` ranks on the CPU: every rank maps
the same queries, and the result is the search of the mapped queries."""

import multiprocessing as mp
import os
import traceback
from datetime import timedelta

import numpy as np
import torch

from test_sharded_gloo import _corpus, _cpu_ops, _free_port


class Rotate(torch.nn.Module):
    """A stand-in for an adapter: any callable on a [b, d] tensor will do."""

    def __init__(self, d):
        super().__init__()
        g = torch.Generator().manual_seed(3)
        self.w = torch.nn.Parameter(torch.randn(d, d, generator=g) * d**-0.5)

    def forward(self, q):
        return q.float() @ self.w


def _worker(rank, world, port, out):
    try:
        import sys
        from pathlib import Path

        root = Path(__file__).resolve().parent.parent
        sys.path[:0] = [str(root), str(root / "cuda-vector-search_b200"), str(root / "tests")]
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        import torch.distributed as dist

        from cuda_vector_search import ShardedIndex

        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=timedelta(seconds=60))
        x, q = _corpus(n=500, d=48, b=5)
        n = len(x)
        index = ShardedIndex(ops=_cpu_ops(x[n * rank // world : n * (rank + 1) // world]))
        adapter = Rotate(48)
        v, i = index.search(torch.from_numpy(q), 7, adapter=adapter)
        v2, i2 = index.search(adapter(torch.from_numpy(q)).detach(), 7)
        v3, i3 = index.search(q[0], 7, adapter=adapter)  # one query, a numpy vector
        assert torch.equal(v, v2) and torch.equal(i, i2)
        assert torch.equal(i3, i[:1]) and not v.requires_grad
        out.put((rank, i.numpy(), None))
        dist.destroy_process_group()
    except Exception:
        out.put((rank, None, traceback.format_exc()))


def test_adapter_on_two_ranks():
    ctx = mp.get_context("spawn")
    out, port = ctx.Queue(), _free_port()
    ranks = [ctx.Process(target=_worker, args=(r, 2, port, out)) for r in range(2)]
    for p in ranks:
        p.start()
    got = [out.get(timeout=120) for _ in ranks]
    for p in ranks:
        p.join(60)
    assert all(err is None for _, _, err in got), [err for _, _, err in got]
    assert np.array_equal(got[0][1], got[1][1])
