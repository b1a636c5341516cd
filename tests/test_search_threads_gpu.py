"""Searches of different widths and result counts from two host threads through the C ABI
(foreign calls release the interpreter lock): both run the same kernels with different
amounts of shared memory, and neither may lower the other's limit."""

import ctypes
import threading
from pathlib import Path

import pytest
import torch

from cases import make
from helpers import assert_topk_exact
from oracle import exact_topk

pytestmark = pytest.mark.gpu

LIB = Path(__file__).resolve().parent.parent / "cuda-vector-search_b200" / "cuda_vector_search" / "libcvs_b200.so"
vp, i64, i32, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    lib.cvs_fused_topk.argtypes = [vp, i64, vp, i64, i32, i32, i64, vp, vp, vp, size, i32, i32, vp, vp]
    lib.cvs_fused_topk_workspace_size.argtypes = [i64, i64, i32, i32, i32, i32, ctypes.POINTER(size)]
    lib.cvs_last_error.restype = ctypes.c_char_p
    return lib


# One-CTA and pair kernels with resident queries (widths up to 448); two merge sizes.
@pytest.mark.parametrize("b,first,second", [(16, (64, 10), (448, 10)), (256, (64, 10), (448, 10)), (16, (128, 10), (128, 1000))])
def test_two_searches_at_once(lib, b, first, second):
    n, work = 6000, []
    for d, k in (first, second):
        x, q = (t.cuda() for t in make(n, d, b, seed=d + k))
        need = size()
        assert lib.cvs_fused_topk_workspace_size(b, n, d, k, 0, 0, ctypes.byref(need)) == 0
        ws = torch.zeros(max(256, need.value), dtype=torch.uint8, device="cuda")
        v, i = torch.empty(b, k, device="cuda"), torch.empty(b, k, dtype=torch.int64, device="cuda")
        work.append((x, q, k, ws, v, i, torch.cuda.Stream()))
    torch.cuda.synchronize()
    errors, start = [None, None], threading.Barrier(2)

    def run(j):
        x, q, k, ws, v, i, s = work[j]
        start.wait()
        for _ in range(2000):
            st = lib.cvs_fused_topk(q.data_ptr(), b, x.data_ptr(), n, x.shape[1], k, 0, v.data_ptr(), i.data_ptr(), ws.data_ptr(),
                                    ws.numel(), 0, 0, None, s.cuda_stream)
            if st:
                errors[j] = (st, lib.cvs_last_error())
                return

    threads = [threading.Thread(target=run, args=(j,)) for j in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert errors == [None, None]
    for x, q, k, _, v, i, _ in work:
        x32, q32 = x.float().cpu().numpy(), q.float().cpu().numpy()
        ref_v, ref_i = exact_topk(q32, x32, k + 1)
        assert_topk_exact(v.cpu().numpy(), i.cpu().numpy(), q32, x32, ref_v, ref_i, k)
