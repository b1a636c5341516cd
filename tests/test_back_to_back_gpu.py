"""Searches issued back to back into one workspace, each with its own queries.

A search kernel may be scheduled while the search before it finishes; it must
still read the queries its own preparation wrote. The host runs ahead of the GPU
(a spinning kernel first), so that the launches really overlap.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 256, 384, 640, 1024])
@pytest.mark.parametrize("b", [1, 2, 3, 4, 5, 6, 7, 8, 9, 40, 200])
def test_alternating_queries_in_one_workspace(d, b):
    import cuda_vector_search as cvs
    from cuda_vector_search import _ext

    mod = _ext.load()
    g = torch.Generator().manual_seed(d + b)
    index = cvs.Index(torch.randn(3000, d, generator=g).half().cuda(), metric="cosine")
    queries = [torch.randn(b, d, generator=g).half().cuda() for _ in range(2)]
    ws = torch.zeros(mod.search_workspace_size(b, 3000, index._x.shape[1], 10), dtype=torch.uint8, device="cuda")
    want = []
    for q in queries:
        torch.cuda.synchronize()
        ws.zero_()
        torch.cuda.synchronize()
        want.append(index.search(q, 10))
    outs = [(torch.zeros(b, 10, device="cuda"), torch.zeros(b, 10, dtype=torch.int64, device="cuda")) for _ in range(8)]
    torch.cuda.synchronize()
    torch.cuda._sleep(3_000_000)
    for s, (v, i) in enumerate(outs):
        mod.search_into(queries[s % 2], index._x, 10, True, 0, v, i, ws)
    torch.cuda.synchronize()
    for s, (v, i) in enumerate(outs):
        rows = index.embeddings.double()[i]  # every returned score is its own query's score of that row
        q = index._prep_queries(queries[s % 2])[:, :d].double()
        assert ((rows * q[:, None]).sum(2) - v.double()).abs().max() < 1e-3, f"search {s}: another query's scores"
        assert torch.equal(i, want[s % 2][1])
