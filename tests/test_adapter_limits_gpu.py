"""The adapter's operators where a first set of sizes did not look."""

import pytest
import torch

import adapter_oracle as oracle
from test_adapter_gpu import DTYPES, E, check_norm, cvs, randn  # noqa: F401  (cvs: the fixture)

pytestmark = pytest.mark.gpu


# ---- layer norm -------------------------------------------------------------------
# One block of 256 threads takes a row wider than 4096 in four groups of 2048 columns.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [4104, 5120, 6136, 6144, 6152, 7000])
def test_layer_norm_widths_that_end_before_the_last_group(cvs, dtype, d):
    t = DTYPES[dtype]
    check_norm(cvs, randn(9, d, dtype=t, seed=1, shift=3.0), randn(d, dtype=t, seed=2, shift=1.0), randn(d, dtype=t, seed=3),
               randn(9, d, dtype=t, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(2048, 4104), (2500, 8191), (2500, 8192)])
def test_layer_norm_many_wide_rows(cvs, dtype, rows, d):
    t = DTYPES[dtype]
    check_norm(cvs, randn(rows, d, dtype=t, seed=1, shift=0.5), randn(d, dtype=t, seed=2, shift=1.0),
               randn(d, dtype=t, seed=3), randn(rows, d, dtype=t, seed=4))


# ---- few tiles: K shared by a cluster ---------------------------------------------------
@pytest.mark.parametrize("m,k", [(3, 384), (100, 384), (3, 576), (100, 576)])
def test_linear_clusters_with_ctas_without_a_slice(cvs, m, k):
    """6 and 9 slices of K among 8 CTAs: two or three of them have no product to wait for and
    send their zeros as soon as the cluster's CTAs are known to run. Call after call on a busy
    stream, the same bits, and the right ones."""
    t = torch.float16
    x, w = randn(m, k, dtype=t, seed=1), randn(1000, k, dtype=t, seed=2, scale=k**-0.5)
    want, _, _, scale = oracle.linear(x, w, None, "none", None)
    first = cvs.linear(x, w)
    oracle.close(first, want, (k / 8 + 16) * E * scale)
    assert all(torch.equal(cvs.linear(x, w), first) for _ in range(200))
