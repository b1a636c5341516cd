"""What the query adapter refuses, without a GPU: the C ABI's contracts before any
device use, the binding's checks on CPU tensors, and the Python layer's."""

import ctypes
from pathlib import Path

import pytest
import torch

import cuda_vector_search as cvs
from cuda_vector_search import _C

LIB = Path(__file__).resolve().parent.parent / "cuda-vector-search_b200" / "cuda_vector_search" / "libcvs_b200.so"
vp, i64, i32, f32, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
P = vp(0x1000)  # aligned, never read: every call here is refused or has no rows


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    lib.cvs_last_error.restype = ctypes.c_char_p
    lib.cvs_layer_norm.argtypes = [vp, i32, i64, i32, i64, vp, vp, i32, f32, vp, i64, vp, vp, vp]
    lib.cvs_layer_norm_backward.argtypes = [vp, i64, vp, i32, i64, i32, i64, vp, i32, vp, vp, vp, i64, vp, vp, vp, size, vp]
    lib.cvs_linear.argtypes = [vp, i64, vp, i64, vp, vp, i64, i32, i32, i64, i32, i32, vp, i64, vp, i64, vp]
    lib.cvs_linear_backward.argtypes = [vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i64, i32, i32, vp, i64, vp, i64, vp, vp,
                                        size, vp]
    lib.cvs_preference_loss.argtypes = [vp, i32, i64, vp, i32, i64, i64, i32, i32, vp, i64, i32, vp, vp, i64, i32, f32, f32,
                                        i32, vp, vp, vp, vp, i64, vp, size, vp]
    lib.cvs_preference_grad.argtypes = [vp, i64, i64, i32, vp, vp, i32, vp, vp]
    return lib


def norm(lib, x=P, dtype=0, rows=4, d=64, stride=64, wt=0, y=P, ys=64):
    return lib.cvs_layer_norm(x, dtype, rows, d, stride, None, None, wt, 1e-5, y, ys, None, None, None)


@pytest.mark.parametrize("kw", [{"rows": -1}, {"d": 0}, {"d": 8193}, {"dtype": 3}, {"dtype": 1, "wt": 2}, {"x": None},
                                {"y": None}, {"ys": 63}, {"stride": -64}])
def test_layer_norm_contract(lib, kw):
    assert norm(lib, **kw) == 1 and lib.cvs_last_error()


def test_no_rows_is_nothing_to_do(lib):
    assert norm(lib, rows=0) == 0
    assert linear(lib, m=0) == 0
    n = size(7)
    assert lib.cvs_linear_backward_workspace_size(0, i64(0), 8, 8, ctypes.byref(n)) == 0 and n.value == 0


def linear(lib, x=P, xs=64, w=P, ws=64, res=None, rs=0, act=0, dtype=1, m=100, n=32, k=64, y=P, ys=32, z=None, zs=0):
    return lib.cvs_linear(x, xs, w, ws, None, res, rs, act, dtype, m, n, k, y, ys, z, zs, None)


@pytest.mark.parametrize("kw", [{"m": -1}, {"m": 2**31}, {"n": 0}, {"k": 0}, {"act": 4}, {"act": -1}, {"dtype": 0},
                                {"dtype": 3}, {"x": None}, {"w": None}, {"y": None}, {"ys": 31}, {"xs": 60}, {"xs": 56},
                                {"ws": 63}, {"x": vp(0x1002)}, {"w": vp(0x1008)}, {"z": vp(0x1004), "zs": 32},
                                {"z": P, "zs": 36}, {"z": P, "zs": 24}, {"res": P, "rs": -1}, {"n": 1 << 25},
                                {"m": 4, "ws": 63}])
def test_linear_contract(lib, kw):
    assert linear(lib, **kw) == 1 and lib.cvs_last_error()


def linear_backward(lib, dy=P, x=P, w=P, z=P, zs=32, act=2, dtype=1, m=100, dx=P, dxs=64, dw=P, dws=64, ws=P, nbytes=0):
    return lib.cvs_linear_backward(dy, 32, x, 64, w, 64, z, zs, act, dtype, m, 32, 64, dx, dxs, dw, dws, None, ws, nbytes,
                                   None)


@pytest.mark.parametrize("kw", [{"dy": None}, {"x": None}, {"w": None}, {"z": None}, {"zs": 33}, {"dxs": 60}, {"dws": 60},
                                {"act": 9}, {"dtype": 0}, {"x": vp(0x1002)}])
def test_linear_backward_contract(lib, kw):
    assert linear_backward(lib, **kw) == 1 and lib.cvs_last_error()


def test_linear_backward_with_nothing_wanted(lib):
    assert linear_backward(lib, dx=None, dw=None) == 0


def preference(lib, q=P, qt=0, b=4, d=100, x=P, n=50, dp=128, chosen=P, rejected=P, r=2, smooth=0.0, loss=P, margins=P,
               grad=None, gs=0):
    return lib.cvs_preference_loss(q, qt, d, None, 0, 0, b, d, 1, x, n, dp, chosen, rejected, r, r, 1.0, smooth, 1, loss, P,
                                   margins, grad, gs, P, 0, None)


@pytest.mark.parametrize("kw", [{"b": -1}, {"r": 0}, {"n": 0}, {"dp": 100}, {"dp": 2112}, {"d": 129}, {"d": 0}, {"qt": 3},
                                {"smooth": 1.5}, {"smooth": float("nan")}, {"x": None}, {"loss": None}, {"q": None},
                                {"chosen": None}, {"rejected": None}, {"margins": None}, {"grad": P, "gs": 100},
                                {"grad": vp(0x1004), "gs": 104}, {"grad": P, "gs": 96}])
def test_preference_contract(lib, kw):
    assert preference(lib, **kw) == 1 and lib.cvs_last_error()


def test_preference_grad_contract(lib):
    assert lib.cvs_preference_grad(P, 96, 4, 100, P, P, 0, P, None) == 1
    assert lib.cvs_preference_grad(None, 104, 4, 100, P, P, 0, P, None) == 1
    assert lib.cvs_preference_grad(P, 104, 4, 100, P, P, 3, P, None) == 1
    assert lib.cvs_preference_grad(P, 104, 0, 100, P, P, 0, P, None) == 0


def test_binding_refuses_host_tensors():
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        _C.layer_norm(x, None, None, 1e-5)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        _C.linear(x, torch.zeros(8, 64, dtype=torch.float16), None, 0, None)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        _C.preference_loss(x, None, torch.zeros(4, dtype=torch.int64), torch.zeros(4, 1, dtype=torch.int64), x, True, 1.0, 0.0,
                           True)


def test_python_layer():
    x = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="activation"):
        cvs.linear(x, x, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        cvs.Adapter(64, activation="tanh")
    with pytest.raises(ValueError, match="dtype"):
        cvs.Adapter(64, dtype=torch.float32)
    with pytest.raises(ValueError, match="positive"):
        cvs.Adapter(0)
    a = cvs.Adapter(64)
    assert a.weight1.shape == (128, 64) and a.weight2.shape == (64, 128) and (a.weight2 == 0).all()
    assert {p.dtype for p in a.parameters()} == {torch.float16}
    assert cvs.Adapter(64, hidden=100, dtype=torch.bfloat16).weight2.shape == (64, 100)
    again = cvs.Adapter(64)
    again.load_state_dict(a.state_dict())
    assert torch.equal(again.weight1, a.weight1)
