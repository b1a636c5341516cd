"""The adapter's operators where a first set of sizes did not look."""

import ctypes
import os
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

import adapter_oracle as oracle
from test_adapter_gpu import DTYPES, E, check_norm, cvs, ids, make_index, randn, strided  # noqa: F401  (cvs: the fixture)
from test_sharded_gloo import _free_port

pytestmark = pytest.mark.gpu

LIB = Path(__file__).resolve().parent.parent / "cuda-vector-search_b200" / "cuda_vector_search" / "libcvs_b200.so"
vp, i64, i32, f32, size = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    lib.cvs_last_error.restype = ctypes.c_char_p
    lib.cvs_layer_norm.argtypes = [vp, i32, i64, i32, i64, vp, vp, i32, f32, vp, i64, vp, vp, vp]
    lib.cvs_layer_norm_backward.argtypes = [vp, i64, vp, i32, i64, i32, i64, vp, i32, vp, vp, vp, i64, vp, vp, vp, size, vp]
    lib.cvs_linear.argtypes = [vp, i64, vp, i64, vp, vp, i64, i32, i32, i64, i32, i32, vp, i64, vp, i64, vp]
    lib.cvs_linear_backward_workspace_size.argtypes = [i32, i64, i32, i32, ctypes.POINTER(size)]
    lib.cvs_linear_backward.argtypes = [vp, i64, vp, i64, vp, i64, vp, i64, i32, i32, i64, i32, i32, vp, i64, vp, i64, vp, vp,
                                        size, vp]
    lib.cvs_preference_loss_workspace_size.argtypes = [i64, i32, ctypes.POINTER(size)]
    lib.cvs_preference_grad.argtypes = [vp, i64, i64, i32, vp, vp, i32, vp, vp]
    lib.cvs_align_rows.argtypes = [vp, i64, i32, i64, i32, vp, i64, vp]
    lib.cvs_debug_stall_next_norm.argtypes = [i64]
    lib.cvs_poll_device_error.argtypes = [i32, ctypes.POINTER(ctypes.c_int)]
    lib.cvs_preference_loss.argtypes = [vp, i32, i64, vp, i32, i64, i64, i32, i32, vp, i64, i32, vp, vp, i64, i32, f32, f32,
                                        i32, vp, vp, vp, vp, i64, vp, size, vp]
    return lib


def stream():
    return torch.cuda.current_stream().cuda_stream


# ---- layer norm -------------------------------------------------------------------
# One block of 256 threads takes a row wider than 4096 in four groups of 2048 columns.
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [4104, 5120, 6136, 6144, 6152, 7000])
def test_layer_norm_widths_that_end_before_the_last_group(cvs, dtype, d):
    t = DTYPES[dtype]
    check_norm(cvs, randn(9, d, dtype=t, seed=1, shift=3.0), randn(d, dtype=t, seed=2, shift=1.0), randn(d, dtype=t, seed=3),
               randn(9, d, dtype=t, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(2048, 4104), (2500, 8191), (2500, 8192), (4096, 4104), (4100, 8191), (8200, 4104)])
def test_layer_norm_many_wide_rows(cvs, dtype, rows, d):
    t = DTYPES[dtype]
    check_norm(cvs, randn(rows, d, dtype=t, seed=1, shift=0.5), randn(d, dtype=t, seed=2, shift=1.0),
               randn(d, dtype=t, seed=3), randn(rows, d, dtype=t, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1 << 20, 8), ((1 << 20) + 9, 8), (88000, 96), (140000, 60), (8200, 1024), (4200, 1001),
                                    (33000, 1024), (4100, 2048), (8200, 1032), (8200, 1031)])
def test_layer_norm_many_elements(cvs, dtype, rows, d):
    """Enough elements for the forward kernels that stage the weights and, aligned, the rows
    (types and widths differ in how many that is): the same bits as a few rows alone."""
    t = DTYPES[dtype]
    x, w, b = randn(rows, d, dtype=t, seed=1, scale=2.0, shift=0.5), randn(d, dtype=t, seed=2, shift=1.0), randn(d, dtype=t, seed=3)
    y = cvs.layer_norm(x, w, b)
    assert torch.equal(y[:3000], cvs.layer_norm(x[:3000], w, b)) and torch.equal(y[-999:], cvs.layer_norm(x[-999:], w, b))
    check_norm(cvs, x, w, b, randn(rows, d, dtype=t, seed=4))


def test_layer_norm_gradients_of_rows_far_from_zero(cvs):
    """Rows of 4099 plus whole numbers, whose fp32 mean is exact: the normalised values the
    backward pass computes again lose nothing to the offset. They are off by the variance's
    sum (64 terms of one row: half of 64 e at most) and four roundings."""
    g = torch.Generator(device="cuda").manual_seed(1)
    half = torch.randint(-8, 9, (500, 32), generator=g, device="cuda").float()
    x = (4099.0 + torch.cat([half, -half], 1)).requires_grad_()
    w = torch.ones(64, device="cuda", requires_grad=True)
    dy = x.detach() - 4099.0  # along the rows themselves: the term h mean(g h) is as large as g
    dx, dw = torch.autograd.grad(cvs.layer_norm(x, w), (x, w), dy)
    _, want_dx, want_dw, _, (h, rstd, gw) = oracle.layer_norm(x.detach(), w.detach(), None, 1e-5, dy)
    dh = 36 * E * h.abs()
    oracle.close(dw, want_dw, (80 + 500 / 64) * E * (dy.double() * h).abs().sum(0) + (dy.double().abs() * dh).sum(0))
    inner = (gw * h).mean(1, keepdim=True).abs()
    sums = 40 * E * (gw.abs().mean(1, keepdim=True) + h.abs() * (gw * h).abs().mean(1, keepdim=True))
    oracle.close(dx, want_dx, rstd * (sums + dh * inner + h.abs() * (gw.abs() * dh).mean(1, keepdim=True)
                                      + 4 * E * (gw.abs() + h.abs() * inner)) + 36 * E * want_dx.abs())


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


@pytest.mark.parametrize("k", [2048, 2056, 4096, 2050])
@pytest.mark.parametrize("m", [1, 2])
def test_linear_of_one_and_two_wide_rows(cvs, m, k):
    """Either side of the width where two rows leave the CUDA cores; 2050: unaligned rows stay."""
    t = torch.bfloat16
    x, w, b = randn(m, k, dtype=t, seed=1), randn(100, k, dtype=t, seed=2, scale=k**-0.5), randn(100, dtype=t, seed=3)
    want, z, _, scale = oracle.linear(x, w, b, "silu", None)
    oracle.close(cvs.linear(x, w, b, activation="silu"), want, 1.13 * (k / 8 + 16) * E * scale + 16 * E * z.abs())


# ---- two host threads ---------------------------------------------------------------
def in_threads(*calls, repeats=4000):
    """Each call over and over in a host thread of its own (foreign calls release the
    interpreter lock); the first error of each."""
    errors = [None] * len(calls)
    start = threading.Barrier(len(calls))

    def work(j):
        start.wait()
        for _ in range(repeats):
            try:
                why = calls[j]()
            except RuntimeError as e:
                why = str(e)
            if why:
                errors[j] = why
                return

    threads = [threading.Thread(target=work, args=(j,)) for j in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return errors


def test_layer_norm_of_two_widths_from_two_threads(lib):
    """Both widths run the same kernel with different amounts of shared memory."""
    rows, out, calls = 16384, [], []
    for j, d in enumerate((520, 768)):
        x = randn(rows, d, dtype=torch.float16, seed=j)
        y = torch.empty_like(x)
        s = torch.cuda.Stream()

        def call(x=x, y=y, d=d, s=s):
            st = lib.cvs_layer_norm(x.data_ptr(), 1, rows, d, d, None, None, 1, 1e-5, y.data_ptr(), d, None, None, s.cuda_stream)
            return lib.cvs_last_error() if st else None

        calls.append(call)
        out.append((x, y))
    torch.cuda.synchronize()
    assert in_threads(*calls) == [None, None]
    for x, y in out:
        want = oracle.layer_norm(x, None, None, 1e-5)
        oracle.close(y, want, 200 * E * (1 + want.abs()))


def test_preference_loss_of_two_widths_from_two_threads(lib):
    b, r, n, keep, calls = 64, 2, 200, [], []
    for j, d in enumerate((64, 256)):
        q = randn(b, d, dtype=torch.float32, seed=j)
        x = randn(n, d, dtype=torch.float16, seed=5 + j)
        chosen, rejected = ids(n, b, seed=7), ids(n, b, r, seed=8)
        loss, weight = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
        margins, ws = torch.empty(b, r, device="cuda"), torch.empty(1 << 16, dtype=torch.uint8, device="cuda")
        s = torch.cuda.Stream()

        def call(q=q, x=x, d=d, chosen=chosen, rejected=rejected, loss=loss, weight=weight, margins=margins, ws=ws, s=s):
            st = lib.cvs_preference_loss(q.data_ptr(), 0, d, None, 0, 0, b, d, 0, x.data_ptr(), n, d, chosen.data_ptr(),
                                         rejected.data_ptr(), r, r, 1.0, 0.0, 1, loss.data_ptr(), weight.data_ptr(),
                                         margins.data_ptr(), None, 0, ws.data_ptr(), ws.numel(), s.cuda_stream)
            return lib.cvs_last_error() if st else None

        calls.append(call)
        keep.append((q, x, chosen, rejected, margins))
    torch.cuda.synchronize()
    assert in_threads(*calls) == [None, None]
    for q, x, chosen, rejected, margins in keep:
        _, want, _ = oracle.preference(q, None, chosen, rejected, x, False, 1.0, 0.0, True)
        sizes = x.double().abs()[chosen][:, None] + x.double().abs()[rejected]
        oracle.close(margins, want, 150 * E * (sizes * q.double().abs()[:, None]).sum(2))


# ---- waits that run out ------------------------------------------------------------------
def norm_call(lib, x, y, dy=None, stats=None, ws=None):
    rows, d = x.shape
    s = stream()
    if dy is None:
        mean, rstd = stats if stats else (None, None)
        return lib.cvs_layer_norm(x.data_ptr(), 1, rows, d, d, None, None, 1, 1e-5, y.data_ptr(), d,
                                  mean.data_ptr() if stats else None, rstd.data_ptr() if stats else None, s)
    return lib.cvs_layer_norm_backward(dy.data_ptr(), d, x.data_ptr(), 1, rows, d, d, None, 1, stats[0].data_ptr(),
                                       stats[1].data_ptr(), y.data_ptr(), d, None, None, None, 0, s)


def poll(lib):
    code = ctypes.c_int(-1)
    torch.cuda.synchronize()
    return lib.cvs_poll_device_error(torch.cuda.current_device(), ctypes.byref(code)), code.value


@pytest.mark.parametrize("backward", [False, True])
def test_a_layer_norm_wait_that_runs_out_is_reported(lib, backward):
    """No row arrives, the waits end after 10^6 SM clocks: the device error word names the
    site, and the next call is an ordinary one."""
    x, dy = randn(16384, 768, dtype=torch.float16, seed=1), randn(16384, 768, dtype=torch.float16, seed=2)
    y, stats = torch.empty_like(x), (torch.empty(16384, device="cuda"), torch.empty(16384, device="cuda"))
    assert poll(lib) == (0, 0), "an earlier kernel left an error behind"
    assert norm_call(lib, x, y, stats=stats) == 0 and poll(lib) == (0, 0)
    args = (x, y, dy, stats) if backward else (x, y)
    assert lib.cvs_debug_stall_next_norm(1_000_000) == 0
    assert norm_call(lib, *args) == 0, lib.cvs_last_error()
    assert poll(lib) == (5, 0x100 | (41 if backward else 42))
    assert norm_call(lib, *args) == 0 and poll(lib) == (0, 0)
    want_y, want_dx, *_ = oracle.layer_norm(x, None, None, 1e-5, dy)
    oracle.close(y, want_dx if backward else want_y, 200 * E * (10 + want_y.abs()))


def test_the_layer_norm_hook_refuses_kernels_without_a_ring(lib):
    x = randn(100, 768, dtype=torch.float16, seed=1)
    y = torch.empty_like(x)
    assert lib.cvs_debug_stall_next_norm(1_000_000) == 0
    assert norm_call(lib, x, y) == 1 and b"hook" in lib.cvs_last_error()
    assert norm_call(lib, x, y) == 0 and poll(lib) == (0, 0)  # disarmed
    assert lib.cvs_debug_stall_next_norm(10) == 1


# ---- forward derivatives ------------------------------------------------------------
def test_forward_derivatives_are_refused(cvs):
    """A tangent would be lost: every differentiable input that carries one is refused."""
    import torch.autograd.forward_ad as fw

    x, w, b = randn(9, 64, dtype=torch.float16, seed=1), randn(64, 64, dtype=torch.float16, seed=2), randn(64, dtype=torch.float16, seed=3)
    index = make_index(cvs, 100, 64, "ip")
    c, rej = ids(100, 9, seed=4), ids(100, 9, seed=5)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: cvs.layer_norm(dual(x)), lambda: cvs.layer_norm(x, dual(b)), lambda: cvs.layer_norm(x, b, dual(b)),
                     lambda: cvs.linear(dual(x), w), lambda: cvs.linear(x, dual(w)), lambda: cvs.linear(x, w, dual(b)),
                     lambda: cvs.linear(x, w, residual=dual(x)), lambda: index.preference_loss(dual(x), c, rej),
                     lambda: cvs.layer_norm(dual(x).requires_grad_())):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        index.preference_loss(x, c, rej, reference=dual(x))  # a constant by definition
        a = cvs.Adapter(64, device="cuda")
        v, i = index.search(dual(x), 3, adapter=a)  # a search has no derivative
    v2, i2 = index.search(x, 3, adapter=a)
    assert torch.equal(v, v2) and torch.equal(i, i2)


# ---- values at absent rows -------------------------------------------------------------
@pytest.mark.parametrize("metric", ["cosine", "ip"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("b,r", [(6, 1), (6, 9), (3000, 2)])
def test_preference_absent_pairs_ignore_what_lies_there(cvs, metric, bad, b, r):
    """Padding holds anything: a query without a pair, a chosen row whose rejected rows are
    all absent. Its gradient is zero and nothing else changes."""
    x = randn(300, 96, dtype=torch.float16, seed=1, scale=0.3)
    x[299] = bad
    index = cvs.Index(torch.nn.functional.pad(x, (0, 32)), metric=metric, copy=False)  # as it is: not normalised again
    q, ref = randn(b, 96, dtype=torch.float32, seed=2), randn(b, 96, dtype=torch.float32, seed=3)
    q, ref = torch.nn.functional.pad(q, (0, 32)), torch.nn.functional.pad(ref, (0, 32))
    c, rej = ids(299, b, seed=4), ids(299, b, r, seed=5)
    q[1], ref[1], c[1] = bad, bad, -1           # a padded query
    q[2], rej[2] = bad, -1                      # a query whose rejected rows are all absent
    c[4], rej[4] = 299, -1                      # a bad chosen row in front of absent ones
    c[5], rej[5] = -1, 299                      # bad rejected rows behind an absent one
    want_q = q.clone()
    want_q[[1, 2]] = 0.5

    def run(q, ref, c, rej):
        q = q.detach().requires_grad_()
        loss, m = index.preference_loss(q, c, rej, reference=ref, scale=3.0, return_margins=True)
        return (loss.detach(), m, *torch.autograd.grad(loss, q))

    got = run(q, ref, c, rej)
    ref2, c2, rej2 = ref.clone(), c.clone(), rej.clone()
    ref2[1], c2[4], rej2[5] = 0.5, 0, 0
    want = run(want_q, ref2, c2, rej2)
    assert all(torch.isfinite(t).all() for t in got)
    assert (got[2][[1, 2, 4, 5]] == 0).all()
    for g, w in zip(got, want):
        assert torch.equal(g, w)


def test_preference_slopes_of_confident_pairs(cvs):
    """Margins that are exact (one column, one product): an fp32 gradient is then off by the
    slope's own roundings alone: exponential 4 e (2 ulp) and its argument's rest e, the sum
    1 + e^-|m| e, reciprocal 2 e (1 ulp), their product e; the other factors are one."""
    n = 80
    x = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    x[0, 0] = 1.0
    index = cvs.Index(x, metric="ip", copy=False)
    q = torch.zeros(n, 64, device="cuda")
    q[:, 0] = torch.linspace(-80.0, 80.0, n, device="cuda") + randn(n, dtype=torch.float32, seed=1)
    q.requires_grad_()
    loss = index.preference_loss(q, torch.zeros(n, dtype=torch.int64, device="cuda"), torch.ones(n, dtype=torch.int64, device="cuda"),
                                 reduction="sum")
    (dq,) = torch.autograd.grad(loss, q)
    oracle.close(dq[:, 0], -torch.sigmoid(-q.detach().double()[:, 0]), 9 * E * torch.sigmoid(-q.detach().double()[:, 0]))


def test_preference_infinite_margins(cvs):
    """A margin past fp32: the pair's slope is 0 or -scale, not NaN."""
    x = torch.zeros(2, 64, dtype=torch.float16, device="cuda")
    x[0, 0] = 60000.0
    index = cvs.Index(x, metric="ip", copy=False)
    q = torch.zeros(2, 64, device="cuda")
    q[0, 0], q[1, 0] = 1e38, -1e38
    q.requires_grad_()
    c, rej = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.ones(2, dtype=torch.int64, device="cuda")
    loss, m = index.preference_loss(q, c, rej, reduction="sum", label_smoothing=0.25, return_margins=True)
    (dq,) = torch.autograd.grad(loss, q)
    assert m[0, 0] == float("inf") and m[1, 0] == float("-inf") and torch.isinf(loss)
    assert dq[0, 0] == 0.25 * 60000.0 and dq[1, 0] == -0.75 * 60000.0


# ---- activations' tails ---------------------------------------------------------------
@pytest.mark.parametrize("m", [1, 2, 300])
def test_gelu_goes_to_zero(cvs, m):
    """Far below zero a bf16 GELU and its slope follow z Phi(z) down to fp32's smallest
    numbers instead of stopping at their value at -6: to 1e-3 above -9, 1e-2 above -11, and
    zero (or below 1e-27, where fp32 ends) beyond."""
    t = torch.bfloat16
    zs = torch.tensor([-5.0, -5.9375, -6.0, -6.0625, -6.5, -7.0, -8.0, -9.0, -10.0, -11.0, -12.0, -13.0, -14.0, -20.0, -50.0, -1e4])
    w = torch.zeros(16, 8, dtype=t, device="cuda")
    w[:, 0] = zs.to(t).cuda()
    x = torch.zeros(m, 8, dtype=t, device="cuda")
    x[:, 0] = 1.0
    y = cvs.linear(x, w, activation="gelu")
    z = w.double()[:, 0].expand(m, 16)
    want, slope = oracle.act(z, "gelu")
    rel = torch.where(z >= -9, 1e-3, torch.where(z >= -11, 1e-2, 1.0))
    oracle.close(y, want, rel * want.abs() + 1e-37)
    assert (y[:, z[0] <= -14] == 0).all()
    one = torch.zeros(1, 8, dtype=t, device="cuda")
    one[0, 0] = 1.0
    x = w.detach().clone().requires_grad_()  # rows with z in the first column: one output, its slope in dx's first column
    (dx,) = torch.autograd.grad(cvs.linear(x, one, activation="gelu"), x, torch.ones(16, 1, dtype=t, device="cuda"))
    oracle.close(dx[:, 0], slope[0], (rel[0] + 2.0**-8) * slope[0].abs() + 1e-37)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m", [2, 4000])
def test_gelu_error_is_a_share_of_z(cvs, dtype, m):
    """Products of two halves are exact pre-activations: over four million of them the GELU is
    off by its rounding and 16 e of |z| at most (its polynomial 12 e, the exponential's 2 ulp
    half of 4 e, product and sum e each)."""
    t = DTYPES[dtype]
    n = 4_000_000 // m
    x, w = randn(m, 1, dtype=t, seed=1), randn(n, 1, dtype=t, seed=2, scale=2.0)
    y = cvs.linear(x, w, activation="gelu")
    z = x.double() @ w.double().T
    oracle.close(y, oracle.act(z, "gelu")[0], 16 * E * z.abs())


# ---- counts past 32 bits ---------------------------------------------------------------
def test_counts_past_32_bits_are_refused(cvs):
    """A count of columns or rows is never cut to its low 32 bits."""
    x = randn(4, 1, dtype=torch.float16, seed=1)
    with pytest.raises(ValueError, match="at most"):
        cvs.linear(x, x[:1].expand((1 << 32) + 5, 1))
    with pytest.raises(ValueError, match="at most"):
        cvs.linear(x[:1].expand(4, (1 << 32) + 5), x[:1].expand(3, (1 << 32) + 5))
    index = make_index(cvs, 100, 64, "ip")
    with pytest.raises(ValueError, match="rejected"):
        index.preference_loss(randn(4, 64, dtype=torch.float32, seed=1), ids(100, 4, seed=2),
                              ids(100, 4, 1, seed=3).expand(4, (1 << 32) + 1))


# ---- training as documented ------------------------------------------------------------
def test_the_documented_training_loop(cvs):
    """The documented loop as it stands: the fp32 copies take every step, the parameters are their
    rounded values, and the gradient the loop ends on is the adapter's own."""
    text = (LIB.parent.parent.parent / "README.md").read_text()
    code = text[text.index("from cuda_vector_search import Adapter, Index") :]
    code = code[: code.index("```")]
    index = make_index(cvs, 2000, 768, "cosine")
    q = randn(100, 768, dtype=torch.bfloat16, seed=2)
    batch = (q, ids(2000, 100, seed=3), ids(2000, 100, 4, seed=4, gone=0.2))
    torch.manual_seed(0)
    names = {"torch": torch, "index": index, "batches": [batch] * 20, "q": q}
    exec(code, names)
    adapter, master, params = names["adapter"], names["master"], names["params"]
    torch.manual_seed(0)
    start = cvs.Adapter(768, dtype=torch.bfloat16, device="cuda")
    for m, p, p0 in zip(master, params, start.parameters()):
        assert m.dtype == torch.float32 and torch.isfinite(m).all() and torch.equal(p.detach(), m.to(p.dtype))
        # 20 AdamW steps move a value by at most 20 lr (1 + its decay) or so, and move it at all.
        moved = (m - p0.detach().float()).abs()
        assert (moved > 0).all() and moved.max() < 20 * 1e-4 * 2
    loss = index.preference_loss(adapter(q), *batch[1:], reference=q, scale=10.0)
    for g, p in zip(torch.autograd.grad(loss, params), params):
        assert torch.isfinite(g).all() and (g != 0).any() and g.shape == p.shape
    assert names["ids"].shape == (100, 10)


# ---- host threads that have made no CUDA call yet ----------------------------------------
def test_linear_from_a_new_thread(cvs):
    """Nothing has bound the device to the thread before its first call."""
    x, w = randn(700, 64, dtype=torch.float16, seed=1), randn(64, 64, dtype=torch.float16, seed=2)
    spare = cvs.linear(x, w)
    want = spare.clone()
    del spare  # the thread's result takes this block: no allocation binds the device either
    torch.cuda.synchronize()
    assert in_threads(lambda: None if torch.equal(cvs.linear(x, w), want) else "differs", repeats=1) == [None]


def test_backward_as_the_first_call_of_the_autograd_thread():
    """In a fresh process: a backward pass without activation starts with its product."""
    code = """
import torch, cuda_vector_search as cvs
x = torch.ones(700, 64, dtype=torch.float16, device="cuda", requires_grad=True)
w = torch.ones(64, 64, dtype=torch.float16, device="cuda")
y = cvs.linear(x, w)
dy = torch.ones_like(y)
spare = [torch.empty_like(y) for _ in range(4)]  # blocks for the backward pass to reuse
del spare
torch.cuda.synchronize()
(dx,) = torch.autograd.grad(y, x, dy)
assert (dx == 64).all()
"""
    root = LIB.parent.parent
    run = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=200)
    assert run.returncode == 0, run.stderr[-2000:]


# ---- the C ABI's own strides ----------------------------------------------------------
FILL = 77.0


def padded(rows, cols, stride, dtype, offset=0, values=None):
    """(buffer, view): rows `stride` apart in a buffer of FILL that goes on behind the last row."""
    buf = torch.full((offset + (rows + 2) * stride,), FILL, dtype=dtype, device="cuda")
    view = buf[offset : offset + rows * stride].view(rows, stride)[:, :cols]
    if values is not None:
        view.copy_(values)
    return buf, view


def untouched(buf, view, also=0):
    """Everything outside the view (and `also` columns behind it) is as it was."""
    kept = torch.ones_like(buf, dtype=torch.bool)
    rows, cols = view.shape
    kept.as_strided((rows, cols + also), (view.stride(0), 1), view.storage_offset()).fill_(False)
    return bool((buf[kept] == FILL).all())


@pytest.mark.parametrize("activation", ["none", "relu", "gelu"])
@pytest.mark.parametrize("more,offset", [(8, 0), (16, 8), (5, 1)])  # aligned and other strides, past the width
@pytest.mark.parametrize("m,k,n", [(1, 64, 72), (2, 72, 65), (40, 256, 72), (40, 256, 65), (700, 64, 72), (700, 64, 65), (700, 65, 200),
                                   (300, 391, 130)])
def test_c_abi_linear_strides(lib, m, k, n, more, offset, activation):
    t, act = torch.float16, ("none", "relu", "gelu").index(activation)
    up8 = lambda v: (v + 7) // 8 * 8  # noqa: E731
    _, x = padded(m, k, up8(k) + 8, t, 0, randn(m, k, dtype=t, seed=1))
    _, w = padded(n, k, up8(k) + 16, t, 0, randn(n, k, dtype=t, seed=2, scale=k**-0.5))
    b = randn(n, dtype=t, seed=3)
    aligned = more % 8 == 0
    s_out = (up8(n) if aligned else n) + more
    _, res = padded(m, n, s_out, t, offset, randn(m, n, dtype=t, seed=4))
    ybuf, y = padded(m, n, s_out, t, offset)
    zbuf, z = padded(m, n, up8(n) + 8, t)
    keep = activation != "none"
    st = lib.cvs_linear(x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), b.data_ptr(), res.data_ptr(), s_out, act, 1, m, n, k,
                        y.data_ptr(), s_out, z.data_ptr() if keep else None, z.stride(0) if keep else 0, stream())
    assert st == 0, lib.cvs_last_error()
    want, zd, slope, scale = oracle.linear(x, w, b, activation, res)
    dz_z = (k / 8 + 16) * E * scale
    oracle.close(y, want, 1.13 * dz_z + 16 * E * zd.abs() + 2 * E * want.abs())
    assert untouched(ybuf, y)
    if keep:
        oracle.close(z, zd, dz_z)
        assert untouched(zbuf, z, up8(n) - n)
    # Backward: all gradients, and each product alone.
    _, dy = padded(m, n, s_out, t, offset, randn(m, n, dtype=t, seed=5))
    nbytes = size()
    assert lib.cvs_linear_backward_workspace_size(act, m, n, k, ctypes.byref(nbytes)) == 0
    ws = torch.empty(max(nbytes.value, 256), dtype=torch.uint8, device="cuda")
    s_dx = k + more
    if keep:
        s_err = (zd.abs() <= dz_z).double() if activation == "relu" else 0.8 * (2.0**-11 * zd.abs() + 2.0**-25 + dz_z) + 16 * E
    else:
        s_err = torch.zeros_like(zd)
    dyd, wd, xd = dy.double(), w.double(), x.double()
    dz = dyd * slope
    dz_err = dyd.abs() * s_err + (2.0**-11 * dz.abs() + 2.0**-25 if keep else 0)
    for wanted in ("xwb", "x", "w", "b"):
        dxb, dx = padded(m, k, s_dx, t, offset)
        dwb, dw = padded(n, k, s_dx, t, offset)
        db = torch.full((n + 8,), FILL, dtype=t, device="cuda")
        p = lambda c, v: v.data_ptr() if c in wanted else None  # noqa: E731
        st = lib.cvs_linear_backward(dy.data_ptr(), s_out, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0),
                                     z.data_ptr() if keep else None, z.stride(0) if keep else 0, act, 1, m, n, k, p("x", dx), s_dx,
                                     p("w", dw), s_dx, p("b", db), ws.data_ptr(), ws.numel(), stream())
        assert st == 0, lib.cvs_last_error()
        if "x" in wanted:
            oracle.close(dx, dz @ wd, dz_err @ wd.abs() + (n / 8 + 16) * E * (dz.abs() @ wd.abs()))
            assert untouched(dxb, dx)
        if "w" in wanted:
            oracle.close(dw, dz.T @ xd, dz_err.T @ xd.abs() + (m / 8 + 32) * E * (dz.abs().T @ xd.abs()))
            assert untouched(dwb, dw)
        if "b" in wanted:
            oracle.close(db[:n], dz.sum(0), (dyd.abs() * s_err).sum(0) + (80 + m / 64) * E * dz.abs().sum(0))
            assert (db[n:] == FILL).all()


@pytest.mark.parametrize("rows,d", [(3, 64), (20, 391), (16390, 64), (5, 1032), (2100, 1031)])
@pytest.mark.parametrize("more,offset", [(8, 0), (8, 8), (5, 1)])
def test_c_abi_layer_norm_strides(lib, rows, d, more, offset):
    t = torch.float16
    _, x = padded(rows, d, d + more, t, offset, randn(rows, d, dtype=t, seed=1))
    _, dy = padded(rows, d, d + more, t, offset, randn(rows, d, dtype=t, seed=2))
    ybuf, y = padded(rows, d, d + more, t, offset)
    dxb, dx = padded(rows, d, d + more, t, offset)
    mean, rstd = torch.full((rows + 8,), FILL, device="cuda"), torch.full((rows + 8,), FILL, device="cuda")
    assert lib.cvs_layer_norm(x.data_ptr(), 1, rows, d, d + more, None, None, 1, 1e-5, y.data_ptr(), d + more, mean.data_ptr(),
                              rstd.data_ptr(), stream()) == 0
    assert lib.cvs_layer_norm_backward(dy.data_ptr(), d + more, x.data_ptr(), 1, rows, d, d + more, None, 1, mean.data_ptr(),
                                       rstd.data_ptr(), dx.data_ptr(), d + more, None, None, None, 0, stream()) == 0
    want, want_dx, *_ = oracle.layer_norm(x, None, None, 1e-5, dy)
    oracle.close(y, want, 200 * E * (1 + want.abs()))
    oracle.close(dx, want_dx, 2000 * E * (1 + want.abs()) * dy.double().abs().max())
    assert untouched(ybuf, y) and untouched(dxb, dx) and (mean[rows:] == FILL).all() and (rstd[rows:] == FILL).all()


# ---- workspace -------------------------------------------------------------------------
def test_linear_backward_without_activation_holds_no_copy_of_dy(cvs, lib):
    m, k, n = 32768, 64, 1536
    x, w = randn(m, k, dtype=torch.float16, seed=1).requires_grad_(), randn(n, k, dtype=torch.float16, seed=2)
    dy = randn(m, n, dtype=torch.float16, seed=3)
    y = cvs.linear(x, w)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    (dx,) = torch.autograd.grad(y, x, dy)
    held = torch.cuda.max_memory_allocated() - before
    assert held < dx.nbytes + dy.nbytes // 2  # dx itself, and no m x n halves
    # The C ABI: less is enough where dy can be read as it is, and refused where not.
    nbytes, less = size(), m * n * 2
    assert lib.cvs_linear_backward_workspace_size(0, m, n, k, ctypes.byref(nbytes)) == 0
    ws = torch.empty(max(nbytes.value - less, 256), dtype=torch.uint8, device="cuda")
    got = torch.empty_like(dx)

    def call(dy, act=0, z=None):
        return lib.cvs_linear_backward(dy.data_ptr(), dy.stride(0), x.data_ptr(), k, w.data_ptr(), k, z, n, act, 1, m, n, k,
                                       got.data_ptr(), k, None, k, None, ws.data_ptr(), nbytes.value - less, stream())

    assert call(dy) == 0 and torch.equal(got, dx)
    assert call(strided(dy, "odd")) == 3 and b"workspace" in lib.cvs_last_error()
    assert call(dy, act=2, z=dy.data_ptr()) == 3 and b"workspace" in lib.cvs_last_error()


# ---- graphs --------------------------------------------------------------------------------
def test_capture_after_a_warm_up_on_another_stream():
    """torch's own recipe in a process of its own: training steps on a side stream whose last
    loss stays alive, then the step captured on the capture's stream; the replay's gradients
    are the warm-up's."""
    code = """
import torch, cuda_vector_search as cvs
torch.manual_seed(0)
index = cvs.Index(torch.randn(2000, 128, device="cuda"))
adapter = cvs.Adapter(128, device="cuda")
q = torch.randn(64, 128, device="cuda", dtype=torch.float16)
c, r = torch.randint(2000, (64,), device="cuda"), torch.randint(2000, (64, 4), device="cuda")
def step():
    adapter.zero_grad(set_to_none=True)
    loss = index.preference_loss(adapter(q), c, r, reference=q)
    loss.backward()
    return loss
side = torch.cuda.Stream()
side.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(side):
    for _ in range(3):
        loss = step()
torch.cuda.current_stream().wait_stream(side)
want = [p.grad.clone() for p in adapter.parameters()]
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    captured = step()
for _ in range(3):
    for p in adapter.parameters():
        p.grad.fill_(7.0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(captured, loss) and all(torch.equal(p.grad, w) for p, w in zip(adapter.parameters(), want))
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=LIB.parent.parent, capture_output=True, text=True, timeout=200)
    assert run.returncode == 0, run.stderr[-2000:]


# ---- broadcast inputs ------------------------------------------------------------------
def test_preference_of_one_query_and_shared_rejected_rows(cvs):
    """One query expanded over several chosen rows, one list of rejected rows for all of them:
    the values of the copies, and the query's gradient summed over its uses."""
    index = make_index(cvs, 300, 96, "cosine")
    q = randn(1, 96, dtype=torch.float32, seed=1).requires_grad_()
    ref, c, rej = randn(1, 96, dtype=torch.float32, seed=2), ids(300, 20, seed=3, gone=0.1), ids(300, 1, 5, seed=4, gone=0.1)
    loss, m = index.preference_loss(q.expand(20, 96), c, rej.expand(20, 5), reference=ref.expand(20, 96), return_margins=True)
    (dq,) = torch.autograd.grad(loss, q)
    dense = q.detach().expand(20, 96).contiguous().requires_grad_()
    loss2, m2 = index.preference_loss(dense, c, rej.expand(20, 5).contiguous(), reference=ref.expand(20, 96).contiguous(),
                                      return_margins=True)
    (each,) = torch.autograd.grad(loss2, dense)
    assert torch.equal(loss, loss2) and torch.equal(m, m2)
    oracle.close(dq[0], each.double().sum(0), 20 * E * each.double().abs().sum(0))


def test_adapter_of_more_dimensions(cvs):
    """[2, 3, d] in, the same rows as [6, d], gradients included; a batch without rows."""
    torch.manual_seed(0)
    a = cvs.Adapter(64, activation="silu", device="cuda")
    with torch.no_grad():
        a.weight2.copy_(torch.randn(64, 128) * 0.1)
    x = randn(2, 3, 64, dtype=torch.float16, seed=1).requires_grad_()
    flat = x.detach().reshape(6, 64).requires_grad_()
    y, want = a(x), a(flat)
    assert y.shape == x.shape and torch.equal(y.reshape(6, 64), want)
    dy = randn(2, 3, 64, dtype=torch.float16, seed=2)
    got = torch.autograd.grad(y, (x, *a.parameters()), dy)
    exp = torch.autograd.grad(want, (flat, *a.parameters()), dy.reshape(6, 64))
    assert all(torch.equal(g.reshape(e.shape), e) for g, e in zip(got, exp))
    none = randn(0, 64, dtype=torch.float16, seed=1).requires_grad_()
    dx, *grads = torch.autograd.grad(a(none), (none, *a.parameters()), torch.empty(0, 64, dtype=torch.float16, device="cuda"))
    assert dx.shape == (0, 64) and all((g == 0).all() for g in grads)


def test_adapter_in_a_sharded_search():
    """The real adapter in front of a sharded index of one rank: the plain index's results."""
    code = """
import os, torch, torch.distributed as dist
from datetime import timedelta
import cuda_vector_search as cvs
dist.init_process_group("nccl", rank=0, world_size=1, timeout=timedelta(seconds=60), device_id=torch.device("cuda", 0))
torch.manual_seed(0)
x, q = torch.randn(3000, 96), torch.randn(20, 96)
a = cvs.Adapter(96, device="cuda")
with torch.no_grad():
    a.weight2.copy_(torch.randn(96, 192) * 0.1)
v, i = cvs.ShardedIndex(x.numpy()).search(q.numpy(), 5, adapter=a)
v2, i2 = cvs.Index(x).search(q.cuda(), 5, adapter=a)
assert torch.equal(v, v2) and torch.equal(i, i2) and not v.requires_grad
torch.cuda.synchronize()
dist.destroy_process_group()
"""
    env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=str(_free_port()), NCCL_SOCKET_IFNAME="lo")
    run = subprocess.run([sys.executable, "-c", code], cwd=LIB.parent.parent, capture_output=True, text=True, timeout=200, env=env)
    assert run.returncode == 0, run.stderr[-2000:]


@pytest.mark.parametrize("more,offset", [(8, 0), (5, 1)])
@pytest.mark.parametrize("b,r,d", [(3, 2, 64), (40, 9, 100), (3000, 1, 391)])
def test_c_abi_preference_strides(lib, b, r, d, more, offset):
    n, d_pad, up8 = 200, (d + 63) // 64 * 64, (d + 7) // 8 * 8
    x = torch.zeros(n, d_pad, dtype=torch.float16, device="cuda")
    x[:, :d] = randn(n, d, dtype=torch.float16, seed=1, scale=0.3)
    _, q = padded(b, d, d + more, torch.bfloat16, offset, randn(b, d, dtype=torch.bfloat16, seed=2))
    _, ref = padded(b, d, d + more, torch.float32, offset, randn(b, d, dtype=torch.float32, seed=3))
    chosen, rej = ids(n, b, seed=4, gone=0.1), ids(n, b, r, seed=5, gone=0.2)
    _, rejected = padded(b, r, r + 3, torch.int64, 0, rej)
    loss, weight = torch.full((4,), FILL, device="cuda"), torch.full((4,), FILL, device="cuda")
    mbuf = torch.full((b * r + 8,), FILL, device="cuda")
    gbuf = torch.full((b + 1, up8 + 16), FILL, device="cuda")
    need = size()
    assert lib.cvs_preference_loss_workspace_size(b, r, ctypes.byref(need)) == 0
    ws = torch.empty(max(need.value, 256), dtype=torch.uint8, device="cuda")
    st = lib.cvs_preference_loss(q.data_ptr(), 2, d + more, ref.data_ptr(), 0, d + more, b, d, 1, x.data_ptr(), n, d_pad,
                                 chosen.data_ptr(), rejected.data_ptr(), r + 3, r, 4.0, 0.1, 1, loss.data_ptr(),
                                 weight.data_ptr(), mbuf.data_ptr(), gbuf.data_ptr(), up8 + 16, ws.data_ptr(), ws.numel(), stream())
    assert st == 0, lib.cvs_last_error()
    want_loss, want_m, want_dq = oracle.preference(q, ref, chosen, rej, x[:, :d], True, 4.0, 0.1, True)
    unit = lambda v: (v.double() / v.double().norm(dim=1, keepdim=True)).abs()  # noqa: E731
    xa = x[:, :d].double().abs()
    sizes = xa[chosen.clamp_min(0)][:, None] + xa[rej.clamp_min(0)]
    m_err = 4.0 * 150 * E * (sizes * (unit(q) + unit(ref))[:, None]).sum(2)
    oracle.close(mbuf[: b * r].view(b, r), want_m, m_err + 4 * E * want_m.abs())
    oracle.close(loss[0], want_loss, m_err.mean() * 2 + 120 * E * want_loss.abs())
    assert (mbuf[b * r :] == FILL).all() and (loss[1:] == FILL).all() and (weight[1:] == FILL).all() and (gbuf[b] == FILL).all()
    upstream, dqb = torch.tensor([2.0], device="cuda"), torch.full((b * d + 8,), FILL, device="cuda")
    assert lib.cvs_preference_grad(gbuf.data_ptr(), up8 + 16, b, d, weight.data_ptr(), upstream.data_ptr(), 0, dqb.data_ptr(), stream()) == 0
    # Slopes of at most 0.9 x scale, each off by m_err / 4 and 16 e, over sums of r + 2 roundings, twice projected, over |q|.
    pairs = max(int(((chosen[:, None] >= 0) & (rej >= 0)).sum()), 1)
    per_row = (4.0 * (0.25 * m_err + 120 * E)[:, :, None] * sizes).sum(1)
    err = (per_row + unit(q) * (unit(q) * per_row).sum(1, keepdim=True) * 4) / q.double().norm(dim=1, keepdim=True) * 2.0 / pairs
    oracle.close(dqb[: b * d].view(b, d), 2.0 * want_dq, err)
    assert (dqb[b * d :] == FILL).all()


@pytest.mark.parametrize("rows,cols,more", [(1, 1, 0), (5, 64, 0), (700, 65, 8), (9, 300, 256), (3, 257, 512)])
def test_c_abi_align_rows(lib, rows, cols, more):
    _, src = padded(rows, cols, cols + 3, torch.bfloat16, 1, randn(rows, cols, dtype=torch.bfloat16, seed=1))
    stride = (cols + 7) // 8 * 8 + more
    buf, dst = padded(rows, cols, stride, torch.bfloat16)
    assert lib.cvs_align_rows(src.data_ptr(), cols + 3, 2, rows, cols, dst.data_ptr(), stride, stream()) == 0
    assert torch.equal(dst, src) and (buf[rows * stride :] == FILL).all()
    behind = buf[: rows * stride].view(rows, stride)[:, cols:]
    assert ((behind == 0) | (behind == FILL)).all()
