"""The query adapter's operators on the GPU against float64 forms of the same
formulas, at the sizes, types, strides and masks where each can go wrong.

Tolerances count roundings. u is half a step of a result's type (one rounding), e =
2^-24 one fp32 rounding. A sum of n fp32 terms taken in a tree or in lanes is off by at
most (n_seq + 16) e times the sum of the terms' magnitudes, n_seq the longest run of
sequential additions; n_seq <= 64 in every sum below over a row (32 elements a thread,
8 warps), and at most 64 + rows / 64 over rows. The tensor cores' accumulation over K
is taken as K / 8 e (at least one rounding or truncation per 16 products; 2 e each).
"""

import pytest
import torch

import adapter_oracle as oracle

pytestmark = pytest.mark.gpu

E = 2.0**-24
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def cvs():
    import cuda_vector_search
    from cuda_vector_search import _ext

    yield cuda_vector_search
    torch.cuda.synchronize()
    assert _ext.load().poll_device_error(0) == 0


def randn(*shape, dtype, seed, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale + shift).to(dtype)


def strided(t, kind):
    """The same values with other strides: rows further apart, an odd offset, or columns apart."""
    if kind == "dense":
        return t
    m, n = t.shape
    if kind == "rows":
        buf = torch.full((m, n + 24), float("nan"), dtype=t.dtype, device=t.device)
        view = buf[:, 8 : 8 + n]
    elif kind == "odd":
        buf = torch.full((m * (n + 3) + 1,), float("nan"), dtype=t.dtype, device=t.device)
        view = buf[1:].view(m, n + 3)[:, :n]
    else:  # columns apart
        buf = torch.full((n, m + 1), float("nan"), dtype=t.dtype, device=t.device)
        view = buf[:, :m].T
    view.copy_(t)
    return view


# ---- layer norm ---------------------------------------------------------------
def check_norm(cvs, x, w, b, dy, eps=1e-5):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b)]
    y = cvs.layer_norm(leaves[0], leaves[1], leaves[2], eps=eps)
    used = [t for t in leaves if t is not None]
    grads = dict(zip(("x", "w", "b"), (None, None, None)))
    got = torch.autograd.grad(y, used, dy)
    for (name, t), _ in zip([(n, t) for n, t in zip("xwb", leaves) if t is not None], got):
        grads[name] = got[[id(u) for u in used].index(id(t))]
    want_y, want_dx, want_dw, want_db, (h, rstd, g) = oracle.layer_norm(x, w, b, eps, dy)
    d, rows = x.shape[1], x.shape[0]
    xd = x.double()
    mean_abs = xd.abs().mean(1, keepdim=True)
    # h: the mean is off by 80 e mean|x|, the difference by that and a rounding, r by
    # 45 e (a sum of squares, a square root, a division) plus twice the mean's share.
    dh = 90 * E * (rstd * mean_abs) * (1 + h.abs()) + 50 * E * h.abs()
    wd = torch.ones(d, dtype=torch.float64, device="cuda") if w is None else w.double()
    oracle.close(y, want_y, dh * wd.abs() + 4 * E * (want_y.abs() + (h * wd).abs()))
    # dx: sums of g and g h over the row, each off by 90 e of its magnitudes and h's error.
    s1 = 90 * E * g.abs().mean(1, keepdim=True)
    s2 = (90 * E * (g * h).abs() + g.abs() * dh).mean(1, keepdim=True)
    inner = (g * h).mean(1, keepdim=True).abs()
    dx_err = rstd * (s1 + h.abs() * s2 + dh * inner + 4 * E * (g.abs() + h.abs() * inner)) + 50 * E * want_dx.abs()
    if grads["x"] is not None:
        oracle.close(grads["x"], want_dx, dx_err)
    run = (80 + rows / 64) * E
    dyd = dy.double()
    if grads["w"] is not None:
        oracle.close(grads["w"], want_dw, run * (dyd * h).abs().sum(0) + (dyd.abs() * dh).sum(0))
    if grads["b"] is not None:
        oracle.close(grads["b"], want_db, run * dyd.abs().sum(0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 2), (1, 768), (7, 8), (33, 100), (5, 255), (9, 256), (40, 391), (17, 1024),
                                    (11, 1025), (6, 2048), (5, 4096), (3, 8191), (4, 8192), (2500, 768), (5000, 64)])
def test_layer_norm(cvs, dtype, rows, d):
    t = DTYPES[dtype]
    check_norm(cvs, randn(rows, d, dtype=t, seed=1, scale=2.0, shift=0.5), randn(d, dtype=t, seed=2, shift=1.0),
               randn(d, dtype=t, seed=3), randn(rows, d, dtype=t, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,d", [(16384, 8), (16391, 96), (20000, 768), (18001, 1024), (17000, 65), (2500, 1032)])
def test_layer_norm_many_rows(cvs, dtype, rows, d):
    """Enough rows for the kernels that walk them through rings of row buffers."""
    t = DTYPES[dtype]
    check_norm(cvs, randn(rows, d, dtype=t, seed=1, scale=2.0, shift=0.5), randn(d, dtype=t, seed=2, shift=1.0),
               randn(d, dtype=t, seed=3), randn(rows, d, dtype=t, seed=4))


def test_layer_norm_many_strided_rows(cvs):
    x = strided(randn(17000, 320, dtype=torch.float16, seed=1), "rows")
    dy = strided(randn(17000, 320, dtype=torch.float16, seed=4), "rows")
    check_norm(cvs, x, randn(320, dtype=torch.float32, seed=2), None, dy)
    row = randn(1, 320, dtype=torch.float16, seed=5)
    y = cvs.layer_norm(row.expand(17000, 320))  # every row the same one in memory
    assert torch.equal(y, cvs.layer_norm(row).expand(17000, 320))


@pytest.mark.parametrize("kind", ["rows", "odd", "columns"])
@pytest.mark.parametrize("d", [64, 391])
def test_layer_norm_strides(cvs, kind, d):
    x = strided(randn(50, d, dtype=torch.bfloat16, seed=1), kind)
    dy = strided(randn(50, d, dtype=torch.bfloat16, seed=4), kind)
    check_norm(cvs, x, randn(d, dtype=torch.float32, seed=2), randn(d, dtype=torch.float32, seed=3), dy)


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
def test_layer_norm_without_weights(cvs, weight, bias):
    check_norm(cvs, randn(70, 320, dtype=torch.float16, seed=1), randn(320, dtype=torch.float16, seed=2) if weight else None,
               randn(320, dtype=torch.float16, seed=3) if bias else None, randn(70, 320, dtype=torch.float16, seed=4))


def test_layer_norm_constant_and_far_rows(cvs):
    """Rows without spread give the bias; a large common offset costs no more than
    the rows' own fp32 rounding."""
    x = randn(8, 512, dtype=torch.float32, seed=1)
    x[0] = 0.0
    x[1] = 3.0
    x[2] += 1000.0
    check_norm(cvs, x, randn(512, dtype=torch.float32, seed=2), randn(512, dtype=torch.float32, seed=3),
               randn(8, 512, dtype=torch.float32, seed=4), eps=1e-3)


def test_layer_norm_keeps_nan_to_its_row(cvs):
    x = randn(4, 384, dtype=torch.float16, seed=1)
    x[1, 7] = float("nan")
    x[2, 9] = float("inf")
    y = cvs.layer_norm(x)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64), (2, 3, 64), (64,)])
def test_layer_norm_shapes(cvs, shape):
    x = randn(*shape, dtype=torch.float16, seed=1).requires_grad_()
    w = randn(64, dtype=torch.float16, seed=2).requires_grad_()
    y = cvs.layer_norm(x, w)
    assert y.shape == x.shape and y.dtype == x.dtype
    dx, dw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape
    if x.numel() == 0:
        assert (dw == 0).all()


def test_layer_norm_gradient_against_differences(cvs):
    """The gradient along a direction against central differences in fp32: the
    difference's own error is e |f| / step + step^2 f''' / 6, below 2e-3 here."""
    x = randn(6, 96, dtype=torch.float32, seed=1).requires_grad_()
    w, b = randn(96, dtype=torch.float32, seed=2), randn(96, dtype=torch.float32, seed=3)
    dy, v = randn(6, 96, dtype=torch.float32, seed=4), randn(6, 96, dtype=torch.float32, seed=5)
    (dx,) = torch.autograd.grad(cvs.layer_norm(x, w, b), x, dy)
    s = 1e-2
    with torch.no_grad():
        up, down = cvs.layer_norm(x + s * v, w, b), cvs.layer_norm(x - s * v, w, b)
    num = (((up.double() - down.double()) / (2 * s)) * dy.double()).sum()
    assert abs(num - (dx.double() * v.double()).sum()) <= 2e-3 * (dx.double().abs() * v.double().abs()).sum()


# ---- linear -------------------------------------------------------------------
def check_linear(cvs, x, w, b, activation, residual, dy):
    leaves = [t.detach().requires_grad_() if t is not None else None for t in (x, w, b, residual)]
    y = cvs.linear(leaves[0], leaves[1], leaves[2], activation=activation, residual=leaves[3])
    used = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("x", "w", "b", "r"), leaves) if t is not None], torch.autograd.grad(y, used, dy)))
    want, z, slope, scale = oracle.linear(x, w, b, activation, residual)
    t, (m, k), n = x.dtype, x.shape, w.shape[0]
    u = oracle.HALF_STEP[t]
    # z: K products' accumulation and the bias; the activations' slopes are at most 1.13
    # and their own error at most 16 e of z; the residual's addition e.
    dz_z = (k / 8 + 16) * E * scale
    oracle.close(y, want, 1.13 * dz_z + 16 * E * z.abs() + 2 * E * want.abs())
    with torch.no_grad():
        y2 = cvs.linear(x, w, b, activation=activation, residual=residual)
    assert torch.equal(y2, y)  # keeping z for the backward pass changes nothing
    # slope: z is kept as fp16 (2^-11 relative, 2^-25 absolute), slopes change by at most
    # 0.8 per unit of z (relu: by 1 where z's sign is in doubt) and have 16 e of their own.
    dyd = dy.double()
    if activation == "none":
        s_err = torch.zeros_like(z)
    elif activation == "relu":
        s_err = (z.abs() <= dz_z).double()
    else:
        s_err = 0.8 * (2.0**-11 * z.abs() + 2.0**-25 + dz_z) + 16 * E
    dz = dyd * slope
    dz_err = dyd.abs() * s_err + (0 if activation == "none" else u * dz.abs() + oracle.TINY[t])
    if "r" in grads:
        assert torch.equal(grads["r"], dy)
    wd, xd = w.double(), x.double()
    oracle.close(grads["x"], dz @ wd, dz_err @ wd.abs() + (n / 8 + 16) * E * (dz.abs() @ wd.abs()))
    oracle.close(grads["w"], dz.T @ xd, dz_err.T @ xd.abs() + (m / 8 + 32) * E * (dz.abs().T @ xd.abs()))
    if "b" in grads:
        b_err = dyd.abs() * s_err
        oracle.close(grads["b"], dz.sum(0), b_err.sum(0) + (80 + m / 64) * E * dz.abs().sum(0))


SIZES = [(1, 64, 64), (1, 1, 1), (2, 96, 7), (5, 391, 130), (8, 768, 1536), (9, 64, 64), (16, 8, 8), (17, 391, 777),
         (64, 768, 256), (100, 64, 1000), (128, 128, 128), (129, 200, 129), (256, 768, 1536), (300, 1, 5), (1000, 72, 3),
         (513, 1536, 768), (2600, 384, 768), (4099, 100, 385)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(cvs, dtype, m, k, n):
    t = DTYPES[dtype]
    activation = ("none", "relu", "gelu", "silu")[(m + n) % 4]
    residual = randn(m, n, dtype=t, seed=5) if m % 2 else None
    check_linear(cvs, randn(m, k, dtype=t, seed=1), randn(n, k, dtype=t, seed=2, scale=k**-0.5),
                 randn(n, dtype=t, seed=3) if (m + k) % 3 else None, activation, residual,
                 randn(m, n, dtype=t, seed=4))


# Few tiles: a cluster of 2, 4 or 8 CTAs shares K; rings that go round; K that does not
# divide among them (CTAs without a slice); one tile and several rounds of tiles.
@pytest.mark.parametrize("m,k,n", [(3, 128, 64), (12, 320, 8), (40, 4096, 520), (200, 4104, 640), (9, 391, 65), (70, 448, 2000),
                                   (130, 2048, 3000), (500, 256, 64), (16, 64, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_linear_shared_k(cvs, m, k, n, residual):
    t = torch.bfloat16
    check_linear(cvs, randn(m, k, dtype=t, seed=1), randn(n, k, dtype=t, seed=2, scale=k**-0.5), randn(n, dtype=t, seed=3),
                 ("relu", "silu", "gelu", "none")[m % 4], randn(m, n, dtype=t, seed=5) if residual else None,
                 randn(m, n, dtype=t, seed=4))


@pytest.mark.parametrize("activation", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m", [3, 150, 700])
def test_linear_epilogues(cvs, activation, residual, m):
    t = torch.float16
    check_linear(cvs, randn(m, 192, dtype=t, seed=1), randn(320, 192, dtype=t, seed=2, scale=0.1), randn(320, dtype=t, seed=3),
                 activation, randn(m, 320, dtype=t, seed=5) if residual else None, randn(m, 320, dtype=t, seed=4))


@pytest.mark.parametrize("kind", ["rows", "odd", "columns"])
@pytest.mark.parametrize("m,k,n", [(4, 64, 72), (4, 65, 33), (200, 64, 72), (200, 65, 33)])
def test_linear_strides(cvs, kind, m, k, n):
    t = torch.bfloat16
    check_linear(cvs, strided(randn(m, k, dtype=t, seed=1), kind), strided(randn(n, k, dtype=t, seed=2, scale=0.2), kind),
                 randn(n, dtype=t, seed=3), "gelu", strided(randn(m, n, dtype=t, seed=5), kind),
                 strided(randn(m, n, dtype=t, seed=4), kind))


@pytest.mark.parametrize("n", [64, 320, 832])
@pytest.mark.parametrize("activation", ["none", "gelu"])
def test_linear_narrow_last_tiles(cvs, n, activation):
    """Tiles whose second half lies outside the matrix, many per CTA: every block of the
    result, and of the kept pre-activation, leaves before its buffer is written again."""
    t = torch.float16
    x, w = randn(60000, 64, dtype=t, seed=1), randn(n, 64, dtype=t, seed=2, scale=0.2)
    want, z, _, scale = oracle.linear(x, w, None, activation, None)
    with torch.no_grad():
        oracle.close(cvs.linear(x, w, activation=activation), want, 40 * E * scale + 16 * E * z.abs())
    wr = w.clone().requires_grad_()
    y = cvs.linear(x, wr, activation=activation)
    oracle.close(y, want, 40 * E * scale + 16 * E * z.abs())


def test_linear_broadcast_operands(cvs):
    """Rows that are one row in memory: an expanded input, residual and upstream
    gradient; the shared row's gradient is the sum over its uses."""
    t = torch.float16
    row = randn(1, 64, dtype=t, seed=1).requires_grad_()
    shared = randn(40, dtype=t, seed=2).requires_grad_()
    w = randn(40, 64, dtype=t, seed=3, scale=0.1).requires_grad_()
    for m in (4, 50):
        y = cvs.linear(row.expand(m, 64), w, residual=shared.expand(m, 40))
        want = row.double() @ w.double().T + shared.double()
        oracle.close(y, want.expand(m, 40), 64 * E * (row.double().abs() @ w.double().abs().T + shared.double().abs()).expand(m, 40))
        drow, dshared, dw = torch.autograd.grad(y.sum(), (row, shared, w))  # an expanded scalar of ones comes in
        assert torch.equal(dshared, torch.full_like(dshared, float(m)))
        oracle.close(drow, w.double().sum(0, keepdim=True) * m, 2.0**-11 * m * w.double().sum(0, keepdim=True).abs() + m * E * 64 + 2.0**-10)
        oracle.close(dw, (m * row.double()).expand(40, 64), m * E * row.double().abs().expand(40, 64))


def test_linear_nan_and_infinity_stay_in_their_row(cvs):
    for m in (4, 300):
        x = randn(m, 128, dtype=torch.float16, seed=1)
        x[1, 5] = float("nan")
        x[2, 6] = float("inf")
        y = cvs.linear(x, randn(96, 128, dtype=torch.float16, seed=2), activation="relu")
        assert torch.isnan(y[1]).all()
        assert not torch.isfinite(y[2].float()).all()
        keep = [i for i in range(m) if i not in (1, 2)]
        assert torch.isfinite(y[keep].float()).all()


def test_linear_kept_preactivation_beyond_fp16(cvs):
    """bf16 rows whose pre-activation overflows fp16: the slope there is 1 (or 0), not NaN."""
    x = torch.full((20, 64), 200.0, dtype=torch.bfloat16, device="cuda").requires_grad_()
    w = torch.full((8, 64), 100.0, dtype=torch.bfloat16, device="cuda")
    w[4:] = -100.0
    for activation in ("relu", "gelu", "silu"):
        y = cvs.linear(x, w, activation=activation)
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(dx, torch.full_like(dx, 400.0))


def test_linear_relu_sign_of_tiny_preactivations(cvs):
    """z > 0 far below fp16's smallest number still passes the gradient on."""
    for m in (4, 40):
        x = torch.full((m, 8), 2.0**-40, dtype=torch.bfloat16, device="cuda").requires_grad_()
        w = torch.ones(8, 8, dtype=torch.bfloat16, device="cuda")
        y = cvs.linear(x, w, activation="relu")
        (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
        assert torch.equal(dx, torch.full_like(dx, 8.0))


@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_linear_single_gradients(cvs, which):
    """One gradient at a time gives what all of them together give."""
    t = torch.float16
    ins = {"x": randn(70, 96, dtype=t, seed=1), "weight": randn(200, 96, dtype=t, seed=2, scale=0.1),
           "bias": randn(200, dtype=t, seed=3), "residual": randn(70, 200, dtype=t, seed=4)}
    dy = randn(70, 200, dtype=t, seed=5)

    def grads(names):
        args = {n: v.detach().requires_grad_(n in names) for n, v in ins.items()}
        y = cvs.linear(args["x"], args["weight"], args["bias"], activation="silu", residual=args["residual"])
        return dict(zip(names, torch.autograd.grad(y, [args[n] for n in names], dy)))

    assert torch.equal(grads([which])[which], grads(list(ins))[which])


@pytest.mark.parametrize("shape", [(0, 64), (2, 0, 64), (2, 30, 64), (64,)])
def test_linear_shapes(cvs, shape):
    x = randn(*shape, dtype=torch.float16, seed=1).requires_grad_()
    w = randn(24, 64, dtype=torch.float16, seed=2).requires_grad_()
    b = randn(24, dtype=torch.float16, seed=3).requires_grad_()
    y = cvs.linear(x, w, b, activation="gelu")
    assert y.shape == (*shape[:-1], 24)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
    assert dx.shape == x.shape and dw.shape == w.shape
    if x.numel() == 0:
        assert (dw == 0).all() and (db == 0).all()


def test_linear_is_the_same_every_run(cvs):
    t = torch.bfloat16
    x, w = randn(5000, 768, dtype=t, seed=1).requires_grad_(), randn(768, 768, dtype=t, seed=2).requires_grad_()
    b, dy = randn(768, dtype=t, seed=3).requires_grad_(), randn(5000, 768, dtype=t, seed=4)

    def once():
        y = cvs.linear(x, w, b, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))

    first = once()
    for _ in range(3):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


# ---- preference loss ------------------------------------------------------------
def check_preference(cvs, index, q, chosen, rejected, ref=None, scale=5.0, smoothing=0.0, reduction="mean", upstream=1.0):
    q = q.detach().requires_grad_()
    loss, margins = index.preference_loss(q, chosen, rejected, reference=ref, scale=scale, label_smoothing=smoothing,
                                          reduction=reduction, return_margins=True)
    (dq,) = torch.autograd.grad(loss, q, torch.tensor(upstream, device="cuda"))
    rej = rejected[:, None] if rejected.dim() == 1 else rejected
    cosine = index.metric == "cosine"
    x = index.embeddings
    want_loss, want_m, want_dq = oracle.preference(q.detach(), ref, chosen, rej, x, cosine, scale, smoothing, reduction == "mean")
    # Margins: scale (u.x_c - u.x_r), each of u and u_ref off by 60 e of itself (norm,
    # division, difference), each sum of d products off by 80 e of its magnitudes, which
    # are |u| (|x_c| + |x_r|) together.
    # Gradient: fl(S x_c - sum_j s_j x_j), S = fl(sum_j s_j) of r slopes: at most r + 2
    # roundings of partial sums no larger than sum_j |s_j| (|x_c| + |x_j|); r <= 64.
    qd = q.detach().double()
    mag = qd / qd.norm(dim=1, keepdim=True).clamp_min(1e-12) if cosine else qd
    mag = mag.abs()
    if ref is not None:
        rd = ref.double()
        mag = mag + (rd / rd.norm(dim=1, keepdim=True).clamp_min(1e-12) if cosine else rd).abs()
    there = (chosen[:, None] >= 0) & (rej >= 0)
    xc, xr = x.double()[chosen.clamp_min(0)][:, None], x.double()[rej.clamp_min(0)]
    apart, sizes = (xc - xr).abs(), xc.abs() + xr.abs()
    m_err = torch.where(there, scale * 150 * E * (sizes * mag[:, None]).sum(2), 0.0)
    oracle.close(margins, want_m, m_err + 4 * E * want_m.abs())
    pairs = max(int(there.sum()), 1)
    weight = 1.0 / pairs if reduction == "mean" else 1.0
    oracle.close(loss, want_loss, m_err.sum() * weight + 120 * E * want_loss.abs())
    # Gradient: slopes change by at most a quarter per unit of m.
    slope_err = torch.where(there, 0.25 * m_err + 16 * E, 0.0) * scale * weight
    slope = torch.where(there, torch.ones_like(m_err), 0.0) * scale * weight
    du_err = (slope_err[:, :, None] * apart).sum(1) + 100 * E * (slope[:, :, None] * sizes).sum(1)
    if cosine:
        n = qd.norm(dim=1, keepdim=True).clamp_min(1e-12)
        u = (qd / n).abs()
        du = (slope[:, :, None] * apart).sum(1)
        du_err = (du_err + u * (u * du_err).sum(1, keepdim=True) + 200 * E * u * (u * du).sum(1, keepdim=True)) / n + 8 * E * want_dq.abs()
    oracle.close(dq, want_dq * upstream, du_err * abs(upstream) + 8 * E * want_dq.abs() * abs(upstream))
    return loss, margins, dq


def make_index(cvs, n, d, metric, seed=11):
    return cvs.Index(randn(n, d, dtype=torch.float16, seed=seed, scale=0.3), metric=metric)


def ids(n, *shape, seed, gone=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = torch.randint(n, shape, generator=g, device="cuda")
    return torch.where(torch.rand(shape, generator=g, device="cuda") < gone, torch.full_like(t, -1), t)


@pytest.mark.parametrize("metric", ["cosine", "ip"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,r,d", [(1, 1, 1), (1, 1, 64), (1, 64, 384), (3, 5, 391), (32, 1, 384), (40, 2, 768), (7, 9, 1000),
                                   (20, 16, 1024), (5, 3, 1536), (2, 33, 2048), (3000, 4, 100)])
def test_preference(cvs, metric, dtype, b, r, d):
    index = make_index(cvs, 500, d, metric)
    t = DTYPES[dtype]
    q = randn(b, d, dtype=t, seed=1)
    ref = randn(b, d, dtype=t, seed=2) if (b + r) % 2 else None
    check_preference(cvs, index, q, ids(500, b, seed=3, gone=0.1), ids(500, b, r, seed=4, gone=0.2), ref=ref,
                     smoothing=0.1 if r > 4 else 0.0, reduction="sum" if d % 3 == 0 else "mean",
                     upstream=128.0 if dtype == "fp16" else 1.0)


def test_preference_one_rejected_as_a_vector(cvs):
    index = make_index(cvs, 300, 128, "cosine")
    check_preference(cvs, index, randn(10, 128, dtype=torch.float32, seed=1), ids(300, 10, seed=3), ids(300, 10, seed=4))


def test_preference_of_one_query_given_as_a_vector(cvs):
    index = make_index(cvs, 300, 128, "cosine")
    q, ref = randn(1, 128, dtype=torch.float32, seed=1), randn(1, 128, dtype=torch.float32, seed=2)
    a = index.preference_loss(q, [3], [4], reference=ref)
    b = index.preference_loss(q[0], torch.tensor([3]), [[4]], reference=ref[0])
    assert torch.equal(a, b)


def test_preference_absent_rows_only(cvs):
    """No pair at all: the loss and its gradient are zero, not NaN."""
    index = make_index(cvs, 300, 128, "cosine")
    q = randn(6, 128, dtype=torch.float32, seed=1)
    none = torch.full((6,), -1, device="cuda")
    loss, margins, dq = check_preference(cvs, index, q, none, ids(300, 6, 3, seed=4))
    assert loss == 0 and (margins == 0).all() and (dq == 0).all()
    check_preference(cvs, index, q, ids(300, 6, seed=4), torch.full((6, 3), -5, device="cuda"))
    q0 = torch.zeros(2, 128, device="cuda")  # padded queries: no direction, no pair
    check_preference(cvs, index, q0, none[:2], ids(300, 2, 3, seed=4))


def test_preference_same_row_twice(cvs):
    """A row chosen and rejected at once pulls nowhere; a row rejected twice counts twice."""
    index = make_index(cvs, 300, 192, "ip")
    c = ids(300, 8, seed=3)
    rej = torch.stack([c, (c + 1) % 300, (c + 1) % 300], dim=1)
    check_preference(cvs, index, randn(8, 192, dtype=torch.float32, seed=1), c, rej)


def test_preference_id_outside_the_index_is_nan(cvs):
    index = make_index(cvs, 300, 64, "ip")
    q = randn(4, 64, dtype=torch.float32, seed=1).requires_grad_()
    c, rej = ids(300, 4, seed=3), ids(300, 4, 2, seed=4)
    rej[1, 1] = 300
    loss, margins = index.preference_loss(q, c, rej, return_margins=True)
    (dq,) = torch.autograd.grad(loss, q)
    assert torch.isnan(loss) and torch.isnan(margins[1, 1]) and torch.isfinite(margins[1, 0])
    assert torch.isfinite(margins[[0, 2, 3]]).all()
    assert torch.isnan(dq[1]).all() and torch.isfinite(dq[[0, 2, 3]]).all()
    c[2] = 1 << 40
    _, margins = index.preference_loss(q, c, ids(300, 4, 2, seed=4), return_margins=True)
    assert torch.isnan(margins[2]).all() and torch.isfinite(margins[[0, 1, 3]]).all()


@pytest.mark.parametrize("scale", [1e-3, 200.0])
def test_preference_extreme_margins(cvs, scale):
    index = make_index(cvs, 300, 256, "ip")
    check_preference(cvs, index, randn(9, 256, dtype=torch.float32, seed=1), ids(300, 9, seed=3), ids(300, 9, 4, seed=4),
                     scale=scale, smoothing=0.2)


def test_preference_strides_and_empty_batches(cvs):
    index = make_index(cvs, 300, 100, "cosine")
    for kind in ("rows", "odd", "columns"):
        check_preference(cvs, index, strided(randn(12, 100, dtype=torch.bfloat16, seed=1), kind), ids(300, 24, seed=3)[::2],
                         ids(300, 5, 12, seed=4).T, ref=strided(randn(12, 100, dtype=torch.float32, seed=2), kind))
    q = torch.zeros(0, 100, device="cuda", requires_grad=True)
    loss = index.preference_loss(q, ids(300, 0, seed=3), ids(300, 0, 2, seed=4))
    (dq,) = torch.autograd.grad(loss, q)
    assert loss == 0 and dq.shape == (0, 100)


def test_preference_gradient_against_differences(cvs):
    """Along a direction: central differences of an fp32 loss, step 1e-2, error below 5e-3."""
    index = make_index(cvs, 300, 64, "cosine")
    q = randn(5, 64, dtype=torch.float32, seed=1).requires_grad_()
    c, rej, v = ids(300, 5, seed=3), ids(300, 5, 3, seed=4), randn(5, 64, dtype=torch.float32, seed=5)
    (dq,) = torch.autograd.grad(index.preference_loss(q, c, rej, scale=4.0), q)
    with torch.no_grad():
        up, down = (index.preference_loss(q + s * v, c, rej, scale=4.0).double() for s in (1e-2, -1e-2))
    assert abs((up - down) / 2e-2 - (dq.double() * v.double()).sum()) <= 5e-3 * (dq.double().abs() * v.double().abs()).sum()


def test_preference_half_gradients_are_rounded_after_their_scaling(cvs):
    """fp16 gradients of a mean over many pairs would be lost without the upstream scale."""
    index = make_index(cvs, 300, 64, "cosine")
    b = 4000
    check_preference(cvs, index, randn(b, 64, dtype=torch.float16, seed=1), ids(300, b, seed=3), ids(300, b, 2, seed=4),
                     upstream=65536.0)


# ---- together --------------------------------------------------------------------
def plain_adapter(a, x):
    """The adapter's forward pass in float64 from its parameters."""
    p = {n: t.double() for n, t in a.named_parameters()}
    x = x.double()
    h = oracle.layer_norm(x, p["norm_weight"], p["norm_bias"], a.eps)
    z = h @ p["weight1"].T + p["bias1"]
    return oracle.act(z, a.activation)[0] @ p["weight2"].T + p["bias2"] + x


def trained(cvs, dim, dtype, seed=0):
    torch.manual_seed(seed)
    a = cvs.Adapter(dim, dtype=dtype, device="cuda")
    with torch.no_grad():
        a.weight2.copy_(torch.randn(dim, 2 * dim, device="cuda") * 0.05)
        a.bias2.copy_(torch.randn(dim, device="cuda") * 0.05)
    return a


@pytest.mark.parametrize("b", [1, 8, 33, 256])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_adapter_in_a_search(cvs, b, dtype):
    """Index.search with an adapter is the search of the adapted queries, and the
    adapted queries are the float64 form's to a few half-precision roundings."""
    index = make_index(cvs, 3000, 384, "cosine")
    a = trained(cvs, 384, dtype)
    q = randn(b, 384, dtype=torch.float32, seed=2)
    v, i = index.search(q, 10, adapter=a)
    with torch.no_grad():
        moved = a(q)
        v2, i2 = index.search(moved, 10)
    assert torch.equal(v, v2) and torch.equal(i, i2)
    v3, i3 = index.search(q.cpu().numpy(), 10, adapter=a)
    assert torch.equal(v, v3) and torch.equal(i, i3)
    want = plain_adapter(a, q.to(dtype))
    u = oracle.HALF_STEP[dtype]
    # Three rounded vectors (norm, hidden, result): each hidden unit is off by 2 u of its
    # inputs' magnitudes, carried through W2; sums of 768 terms of 0.05 x 1.
    p = {n: t.double().abs() for n, t in a.named_parameters()}
    h = oracle.layer_norm(q.to(dtype), a.norm_weight, a.norm_bias, a.eps).abs()
    hid = 1.13 * (u * (h @ p["weight1"].T)) + u * (h @ p["weight1"].T)
    oracle.close(moved, want, hid @ p["weight2"].T + 200 * E * (h @ p["weight1"].T) @ p["weight2"].T)
    fresh = cvs.Adapter(384, dtype=dtype, device="cuda")
    v4, i4 = index.search(q.to(dtype), 10, adapter=fresh)  # an untrained adapter changes nothing
    v5, i5 = index.search(q.to(dtype), 10)
    assert torch.equal(v4, v5) and torch.equal(i4, i5)


def test_adapter_training_step(cvs):
    """Layer norm, two linear layers and the loss in one autograd graph: every
    parameter's gradient against the float64 graph, to 3% of its norm (five chained
    bf16 roundings of 2^-9 typical size each, amplified at most by the layers' gains)."""
    index = make_index(cvs, 2000, 192, "cosine")
    a = trained(cvs, 192, torch.bfloat16)
    q = randn(300, 192, dtype=torch.bfloat16, seed=2)
    c, rej = ids(2000, 300, seed=3), ids(2000, 300, 4, seed=4, gone=0.2)
    loss = index.preference_loss(a(q), c, rej, reference=q, scale=8.0)
    loss.backward()
    double = {n: t.detach().double().requires_grad_() for n, t in a.named_parameters()}
    x = q.double()
    norm = torch.nn.functional.layer_norm(x, (192,), double["norm_weight"], double["norm_bias"], a.eps)
    hidden = torch.nn.functional.gelu(norm @ double["weight1"].T + double["bias1"])
    out = hidden @ double["weight2"].T + double["bias2"] + x
    unit = torch.nn.functional.normalize
    moved = unit(out, dim=1) - unit(x, dim=1)
    rows = index.embeddings.double()
    there = (rej >= 0).double()
    m = 8.0 * ((rows[c][:, None] - rows[rej.clamp_min(0)]) * moved[:, None]).sum(2)
    want = (torch.nn.functional.softplus(-m) * there).sum() / there.sum()
    want.backward()
    assert abs(loss.item() - want.item()) < 1e-2 * abs(want.item())
    for n, t in a.named_parameters():
        g, e = t.grad.double(), double[n].grad
        assert (g - e).norm() <= 0.03 * e.norm(), n


def test_optimizer_step_lowers_the_loss_direction(cvs):
    """The gradient of the whole step along itself: a small step against it moves the
    loss by -step |g|^2 to first order (checked for sign only)."""
    index = make_index(cvs, 2000, 128, "cosine")
    a = trained(cvs, 128, torch.float16)
    q = randn(200, 128, dtype=torch.float16, seed=2)
    c, rej = ids(2000, 200, seed=3), ids(2000, 200, 4, seed=4)

    def value():
        with torch.no_grad():
            return index.preference_loss(a(q), c, rej, scale=8.0).item()

    before = value()
    (index.preference_loss(a(q), c, rej, scale=8.0) * 256).backward()
    with torch.no_grad():
        for p in a.parameters():
            p -= (p.grad.float() / 256 * 0.5).to(p.dtype)
    assert value() < before


# ---- streams and graphs -----------------------------------------------------------
def test_on_a_side_stream(cvs):
    index = make_index(cvs, 1000, 256, "cosine")
    a = trained(cvs, 256, torch.float16)
    q = randn(100, 256, dtype=torch.float16, seed=2)
    c, rej = ids(1000, 100, seed=3), ids(1000, 100, 3, seed=4)

    def step():
        x = q.detach().requires_grad_()
        loss = index.preference_loss(a(x), c, rej)
        return (loss.detach(), *torch.autograd.grad(loss, (x, *a.parameters())))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda._sleep(2_000_000)
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000)
        got = step()
    side.synchronize()
    assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_captured_inference_and_training_replay(cvs):
    index = make_index(cvs, 1000, 256, "cosine")
    a = trained(cvs, 256, torch.float16)
    q = randn(64, 256, dtype=torch.float16, seed=2).requires_grad_()
    c, rej = ids(1000, 64, seed=3), ids(1000, 64, 3, seed=4)
    params = (q, *a.parameters())

    def step():
        loss = index.preference_loss(a(q), c, rej, scale=4.0)
        return (loss.detach(), *torch.autograd.grad(loss, params))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    with torch.cuda.graph(other, stream=side), torch.no_grad():
        v, i = index.search(q, 5, adapter=a)
    for seed in (21, 22):
        with torch.no_grad():
            q.copy_(randn(64, 256, dtype=torch.float16, seed=seed))
        graph.replay()
        other.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(out, step()))
        with torch.no_grad():
            v2, i2 = index.search(q, 5, adapter=a)
        assert torch.equal(v, v2) and torch.equal(i, i2)


def test_capture_with_an_eager_graph_alive_is_refused(cvs):
    """An autograd graph of the same leaf made on another stream and still alive:
    the captured call raises instead of ending the process in the backward pass."""
    w = randn(64, 64, dtype=torch.float16, seed=2).requires_grad_()
    x = randn(16, 64, dtype=torch.float16, seed=1)
    alive = cvs.linear(x, w)  # keeps w's gradient accumulator on this stream
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="another stream"):
        with torch.cuda.graph(graph, stream=side):
            cvs.linear(x, w)
    del alive
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):  # released: the same capture goes through
        y = cvs.linear(x, w)
        (dw,) = torch.autograd.grad(y, w, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    oracle.close(dw, x.double().sum(0).expand(64, 64), 40 * E * x.double().abs().sum(0).expand(64, 64))


def test_second_derivatives_are_refused(cvs):
    x = randn(4, 64, dtype=torch.float32, seed=1).requires_grad_()
    y = cvs.layer_norm(x)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


# ---- sizes past 32 bits -----------------------------------------------------------
def test_more_than_two_to_the_31_elements(cvs):
    """Inputs, results and gradients of more than 2^31 elements: their last rows (and
    first) agree with the same rows computed alone."""
    t = torch.float16
    d = 1024
    rows = (1 << 31) // d + 777
    x = torch.zeros(rows, d, dtype=t, device="cuda")
    x[:100] = randn(100, d, dtype=t, seed=1)
    x[-100:] = randn(100, d, dtype=t, seed=2)
    w = randn(d, dtype=t, seed=3)
    y = cvs.layer_norm(x, w)
    assert torch.equal(y[-100:], cvs.layer_norm(x[-100:], w)) and torch.equal(y[:100], cvs.layer_norm(x[:100], w))
    assert (y[100:-100][:: 1 << 12] == 0).all()
    del y
    w2 = randn(24, d, dtype=t, seed=4, scale=0.03)
    y = cvs.linear(x, w2)  # the largest input
    oracle.close(y[-100:], x[-100:].double() @ w2.double().T, 200 * E * (x[-100:].double().abs() @ w2.double().abs().T))
    del y
    xr = x.requires_grad_()
    yn = cvs.layer_norm(xr, w)
    dy = torch.zeros_like(x)
    dy[-100:] = randn(100, d, dtype=t, seed=5)
    (dx,) = torch.autograd.grad(yn, xr, dy)
    _, want, _, _, _ = oracle.layer_norm(x[-100:].detach(), w, None, 1e-5, dy[-100:])
    oracle.close(dx[-100:], want, 2.0**-16 * want.abs() + 2.0**-18)
    assert (dx[:-100][:: 1 << 12] == 0).all()


def test_linear_result_past_32_bits(cvs):
    t = torch.bfloat16
    n = 520
    m = (1 << 31) // n + 300
    x, w, b = randn(m, 64, dtype=t, seed=1), randn(n, 64, dtype=t, seed=2, scale=0.1), randn(n, dtype=t, seed=3)
    y = cvs.linear(x, w, b, activation="gelu")
    for part in (slice(0, 300), slice(m - 300, m)):
        want, z, _, scale = oracle.linear(x[part], w, b, "gelu", None)
        oracle.close(y[part], want, 40 * E * scale + 16 * E * z.abs())


def test_preference_over_a_corpus_past_32_bits(cvs):
    rows = (1 << 31) // 1024 + 500
    x = torch.zeros(rows, 1024, dtype=torch.float16, device="cuda")
    x[:300] = randn(300, 1024, dtype=torch.float16, seed=1, scale=0.05)
    x[-300:] = randn(300, 1024, dtype=torch.float16, seed=2, scale=0.05)
    index = cvs.Index(x, metric="ip", copy=False)
    q = randn(20, 1024, dtype=torch.float32, seed=3).requires_grad_()
    c, rej = rows - 1 - ids(300, 20, seed=4), torch.cat([rows - 1 - ids(300, 20, 2, seed=5), ids(300, 20, 2, seed=6)], 1)
    loss, m = index.preference_loss(q, c, rej, return_margins=True)
    (dq,) = torch.autograd.grad(loss, q)
    small = torch.cat([x[:300], x[-300:]])
    there = cvs.Index(small, metric="ip")
    near = lambda i: torch.where(i < 300, i, i - (rows - 600))  # noqa: E731
    q2 = q.detach().requires_grad_()
    loss2, m2 = there.preference_loss(q2, near(c), near(rej), return_margins=True)
    (dq2,) = torch.autograd.grad(loss2, q2)
    assert torch.equal(loss, loss2) and torch.equal(m, m2) and torch.equal(dq, dq2)


# ---- several at once ----------------------------------------------------------------
def test_threads_on_streams_of_their_own(cvs):
    """Two host threads train and search at the same time, each on its own stream: both
    get what they get alone."""
    import threading

    index = make_index(cvs, 3000, 384, "cosine")
    adapters = [trained(cvs, 384, torch.bfloat16, seed=s) for s in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def work(s, out):
        a = adapters[s]
        with torch.cuda.stream(streams[s]):
            got = []
            for i in range(8):
                q = randn(60 + 97 * s, 384, dtype=torch.bfloat16, seed=100 * s + i).requires_grad_()
                b = q.shape[0]
                loss, m = index.preference_loss(a(q), ids(3000, b, seed=i), ids(3000, b, 3, seed=i + 50), reference=q,
                                                return_margins=True)
                got.append((loss.detach(), m, *torch.autograd.grad(loss, (q, *a.parameters())),
                            *index.search(q.detach(), 5, adapter=a)))
            streams[s].synchronize()
            out[s] = got

    alone, together = {}, {}
    for s in range(2):
        work(s, alone)
    threads = [threading.Thread(target=work, args=(s, together)) for s in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(together) == [0, 1]
    for s in range(2):
        for w, g in zip(alone[s], together[s]):
            assert all(torch.equal(x, y) for x, y in zip(w, g))
