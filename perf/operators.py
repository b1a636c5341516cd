"""The operators of a query adapter, as they are measured: layer norm, linear
(matrix product with bias, activation and residual) and the preference loss.

An adapter is the small residual network that retrieval systems train on top of a
frozen embedding model: it moves the queries (or re-embeds the corpus) so that the
preferred documents score higher, and the corpus index stays as it is. ``run``
computes one pass of one operator, either in its plain form (elementary torch
operations in 32 bits) or, with ``own`` set, through this package's calls.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
_EPS = 1e-5


def _package():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cuda-vector-search_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import cuda_vector_search

    return cuda_vector_search


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _layer_norm(rows, dim, dtype, train):
    return {"op": "layer_norm", "rows": rows, "dim": dim, "type": dtype, "train": train}


def _linear(rows, inputs, outputs, dtype, activation, residual, train):
    return {"op": "linear", "rows": rows, "inputs": inputs, "outputs": outputs, "type": dtype,
            "activation": activation, "residual": residual, "train": train}


def _preference(queries, rejected, dim, corpus, dtype, metric, reference, smoothing, missing):
    return {"op": "preference", "queries": queries, "rejected": rejected, "dim": dim, "corpus": corpus, "type": dtype,
            "metric": metric, "reference": reference, "smoothing": smoothing, "missing": missing}


def listed():
    cases = {
        # One query on its way to a search: a single row, latency only.
        "norm_one_query": _layer_norm(1, 768, "float16", False),
        # A training batch through the adapter's norm, with the weights' gradients.
        "norm_train": _layer_norm(16384, 768, "bfloat16", True),
        # A corpus chunk of the ingest's size normalised before it is re-embedded.
        "norm_corpus": _layer_norm(262144, 768, "float16", False),
        # Single precision, a ragged width and row count (an embedding with appended features).
        "norm_train_odd": _layer_norm(20011, 391, "float32", True),
        # The first layer for a single query, and for the 256-query batch of the main search workload.
        "linear_one_query": _linear(1, 768, 1536, "float16", "gelu", False, False),
        "linear_batch": _linear(256, 768, 1536, "float16", "gelu", False, False),
        # The second layer over half an ingest chunk: a corpus being re-embedded.
        "linear_corpus": _linear(131072, 1536, 768, "bfloat16", "none", True, False),
        # Training: the first layer with its activation, and a ragged one with everything on.
        "linear_train": _linear(16384, 768, 1536, "bfloat16", "gelu", False, True),
        "linear_train_odd": _linear(3001, 391, 777, "float16", "silu", True, True),
        # The loss: a small batch of single pairs against the smallest corpus of the benchmark,
        # a large one with several rejected rows each, and one without a reference and with gaps.
        "preference_small": _preference(32, 1, 384, 100000, "float32", "cosine", True, 0.0, 0.0),
        "preference_train": _preference(16384, 4, 768, 1000000, "bfloat16", "cosine", True, 0.1, 0.0),
        "preference_many": _preference(2047, 31, 391, 400000, "float16", "ip", False, 0.0, 0.2),
    }
    return [dict(c, name=n) for n, c in cases.items()]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _width(rng, low, high):
    w = _log_int(rng, low, high)
    return max(low, w // 64 * 64) if rng.random() < 0.6 else w


def draw(rng):
    op = rng.choice(["layer_norm", "linear", "linear", "preference"])
    if op == "layer_norm":
        dim = _width(rng, 64, 2048)
        dtype = rng.choice(["float16", "bfloat16", "float32"])
        train = rng.random() < 0.5
        cell = (4 if dtype == "float32" else 2) * (4 if train else 2)  # bytes that a component costs
        return _layer_norm(_log_int(rng, 1, min(262144, 800_000_000 // (cell * dim))), dim, dtype, train)
    if op == "linear":
        inputs, outputs = _width(rng, 64, 2048), _width(rng, 64, 2048)
        train = rng.random() < 0.5
        rows = _log_int(rng, 1, min(131072, 150_000_000_000 // (inputs * outputs * (3 if train else 1)) + 1))
        return _linear(rows, inputs, outputs, rng.choice(["float16", "bfloat16"]),
                       rng.choice(["none", "relu", "gelu", "silu"]), rng.random() < 0.5, train)
    dim = _width(rng, 64, 1024)
    rejected = _log_int(rng, 1, 64)
    queries = _log_int(rng, 1, min(16384, 48_000_000 // (dim * rejected)))
    corpus = _log_int(rng, 1000, 500_000_000 // dim)
    return _preference(queries, rejected, dim, corpus, rng.choice(["float16", "bfloat16", "float32"]),
                       rng.choice(["cosine", "ip"]), rng.random() < 0.7, rng.choice([0.0, 0.1]),
                       rng.choice([0.0, 0.2]))


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPES[case["type"]]

    def randn(*shape, dtype=t, scale=1.0, shift=0.0):
        x = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(shift, scale, generator=g)
        return x.to(dtype)

    state = {"case": case}
    if case["op"] == "layer_norm":
        rows, dim = case["rows"], case["dim"]
        # Raw embeddings: each component has its own offset and spread.
        spread = torch.empty(dim, device="cuda").uniform_(0.2, 2.0, generator=g)
        x = randn(rows, dim, dtype=torch.float32)
        state["x"] = (x * spread + randn(dim, dtype=torch.float32, scale=0.5)).to(t)
        state["weight"] = randn(dim, scale=0.1, shift=1.0)
        state["bias"] = randn(dim, scale=0.1)
        if case["train"]:
            state["dy"] = randn(rows, dim, scale=0.05)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
    elif case["op"] == "linear":
        rows, k, n = case["rows"], case["inputs"], case["outputs"]
        # Normalised activations against weights at their usual scale.
        state["x"] = randn(rows, k)
        state["weight"] = randn(n, k, scale=1 / math.sqrt(k))
        state["bias"] = randn(n, scale=0.1)
        state["residual"] = randn(rows, n) if case["residual"] else None
        if case["train"]:
            state["dy"] = randn(rows, n, scale=0.05)
            for name in ("x", "weight", "bias", "residual"):
                if state[name] is not None:
                    state[name].requires_grad_()
    else:
        b, r, d, n = case["queries"], case["rejected"], case["dim"], case["corpus"]
        # Unit rows as the index stores them; queries near a corpus row, their
        # adapted form a little away from the reference, as during training.
        corpus = randn(n, d, dtype=torch.float16)
        for part in corpus.split(1 << 18):
            part.copy_(part.float() / part.float().norm(dim=1, keepdim=True).clamp_min(1e-12))
        chosen = torch.randint(n, (b,), device="cuda", generator=g)
        rejected = torch.randint(n, (b, r), device="cuda", generator=g)
        if case["missing"]:
            gone = torch.empty(b, r, device="cuda").uniform_(generator=g) < case["missing"]
            rejected = torch.where(gone, torch.full_like(rejected, -1), rejected)
            alone = torch.empty(b, device="cuda").uniform_(generator=g) < case["missing"] / 4
            chosen = torch.where(alone, torch.full_like(chosen, -1), chosen)
        base = 0.4 * corpus[chosen.clamp_min(0)].float() + randn(b, d, dtype=torch.float32, scale=1 / math.sqrt(d))
        state["reference"] = base.to(t) if case["reference"] else None
        state["queries"] = (base + randn(b, d, dtype=torch.float32, scale=0.2 / math.sqrt(d))).to(t).requires_grad_()
        state["chosen"], state["rejected"], state["corpus"] = chosen, rejected, corpus
        # The loss's gradient is scaled so that half-precision gradients keep their digits.
        state["loss_scale"] = torch.tensor(1024.0 if case["type"] == "float16" else 1.0, device="cuda")
        if own:
            # The rows are normalised already and the index takes them as they are
            # where the width allows it.
            state["index"] = _package().Index(corpus, metric=case["metric"], copy=False)
    return state


_SCALE = 10.0  # the loss's inverse temperature


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _own(state, case)
    with torch.no_grad():
        if case["op"] == "layer_norm":
            return _plain_layer_norm(state, case)
        if case["op"] == "linear":
            return _plain_linear(state, case)
        return _plain_preference(state, case)


def _own(state, case):
    cvs = _package()
    if case["op"] == "layer_norm":
        y = cvs.layer_norm(state["x"], state["weight"], state["bias"], eps=_EPS)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    if case["op"] == "linear":
        y = cvs.linear(state["x"], state["weight"], state["bias"], activation=case["activation"],
                       residual=state["residual"])
        if not case["train"]:
            return {"y": y}
        leaves = [state[name] for name in ("x", "weight", "bias", "residual") if state[name] is not None]
        grads = torch.autograd.grad(y, leaves, state["dy"])
        return dict(zip(("y", "dx", "dweight", "dbias", "dresidual"), (y.detach(), *grads)))
    loss, margins = state["index"].preference_loss(
        state["queries"], state["chosen"], state["rejected"], reference=state["reference"], scale=_SCALE,
        label_smoothing=case["smoothing"], return_margins=True)
    (dq,) = torch.autograd.grad(loss, (state["queries"],), state["loss_scale"])
    return {"loss": loss.detach(), "margins": margins, "dqueries": dq}


def _plain_layer_norm(state, case):
    x, w, b = state["x"].float(), state["weight"].float(), state["bias"].float()
    centred = x - x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(1, keepdim=True) + _EPS)
    xhat = centred * rstd
    t = state["x"].dtype
    out = {"y": (xhat * w + b).to(t)}
    if case["train"]:
        dy = state["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        out.update(dx=dx.to(t), dweight=(dy * xhat).sum(0).to(t), dbias=dy.sum(0).to(t))
    return out


def _plain_linear(state, case):
    x, w, t = state["x"].float(), state["weight"].float(), state["x"].dtype
    z = x @ w.T + state["bias"].float()
    act = case["activation"]
    if act == "none":
        y, slope = z, None
    elif act == "relu":
        y, slope = z.clamp_min(0), (z > 0).float()
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    else:
        s = 1 / (1 + torch.exp(-z))
        y, slope = z * s, s * (1 + z * (1 - s))
    if state["residual"] is not None:
        y = y + state["residual"].float()
    out = {"y": y.to(t)}
    if case["train"]:
        dy = state["dy"].float()
        dz = dy if slope is None else dy * slope
        out.update(dx=(dz @ w).to(t), dweight=(dz.T @ x).to(t), dbias=dz.sum(0).to(t))
        if state["residual"] is not None:
            out["dresidual"] = dy.to(t)
    return out


def _plain_preference(state, case):
    q = state["queries"].float()
    cosine = case["metric"] == "cosine"
    norm = torch.sqrt((q * q).sum(1, keepdim=True)).clamp_min(1e-12) if cosine else torch.ones_like(q[:, :1])
    u = q / norm
    moved = u
    if state["reference"] is not None:
        ref = state["reference"].float()
        if cosine:
            ref = ref / torch.sqrt((ref * ref).sum(1, keepdim=True)).clamp_min(1e-12)
        moved = u - ref
    there = (state["chosen"][:, None] >= 0) & (state["rejected"] >= 0)
    better = state["corpus"][state["chosen"].clamp_min(0)].float()
    apart = better[:, None, :] - state["corpus"][state["rejected"].clamp_min(0)].float()
    m = _SCALE * (apart * moved[:, None, :]).sum(2)
    m = torch.where(there, m, torch.zeros_like(m))
    eps = case["smoothing"]
    tail = torch.log1p(torch.exp(-m.abs()))
    each = (1 - eps) * ((-m).clamp_min(0) + tail) + eps * (m.clamp_min(0) + tail)
    count = there.sum().clamp_min(1).float()
    loss = torch.where(there, each, torch.zeros_like(each)).sum() / count
    slope = eps - 1 / (1 + torch.exp(m))
    slope = torch.where(there, slope, torch.zeros_like(slope)) * (state["loss_scale"] * _SCALE / count)
    du = (slope[:, :, None] * apart).sum(1)
    dq = (du - u * (u * du).sum(1, keepdim=True)) / norm if cosine else du
    return {"loss": loss, "margins": m, "dqueries": dq.to(state["queries"].dtype)}


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    d = {k: v.detach().double() for k, v in state.items() if torch.is_tensor(v) and v.is_floating_point() and k != "corpus"}
    if case["op"] == "layer_norm":
        x = d["x"]
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        xhat = (x - mean) * (var + _EPS).rsqrt()
        out = {"y": torch.addcmul(d["bias"], xhat, d["weight"])}
        if case["train"]:
            dxhat = d["dy"] * d["weight"]
            n = x.shape[1]
            # The Jacobian of the normalisation: (I - 1 1^T / n - xhat xhat^T / n) / std.
            inner = torch.einsum("rc,rc->r", dxhat, xhat)[:, None] / n
            out["dx"] = (dxhat - dxhat.sum(1, keepdim=True) / n - xhat * inner) * (var + _EPS).rsqrt()
            out["dweight"] = torch.einsum("rc,rc->c", d["dy"], xhat)
            out["dbias"] = d["dy"].sum(0)
        return out
    if case["op"] == "linear":
        z = torch.addmm(d["bias"], d["x"], d["weight"].t())
        z.requires_grad_(case["train"])
        with torch.enable_grad():
            if case["activation"] == "relu":
                a = torch.where(z > 0, z, 0.0)
            elif case["activation"] == "gelu":
                a = 0.5 * z * torch.erfc(-z / math.sqrt(2.0))
            elif case["activation"] == "silu":
                a = z * torch.sigmoid(z)
            else:
                a = z * 1.0
        y = a.detach()
        out = {"y": y + d["residual"] if "residual" in d else y}
        if case["train"]:
            (dz,) = torch.autograd.grad(a, z, d["dy"])
            out["dx"] = torch.mm(dz, d["weight"])
            out["dweight"] = torch.mm(dz.t(), d["x"])
            out["dbias"] = torch.sum(dz, 0)
            if "residual" in d:
                out["dresidual"] = d["dy"]
        return out
    q = d["queries"].requires_grad_()
    unit = (lambda v: torch.nn.functional.normalize(v, dim=1, eps=1e-12)) if case["metric"] == "cosine" else (lambda v: v)
    chosen, rejected = state["chosen"], state["rejected"]
    there = ((chosen >= 0).unsqueeze(1) & (rejected >= 0)).double()

    def scores(v):
        s = torch.empty(rejected.shape, dtype=torch.float64, device=v.device)
        parts = []
        for i in range(0, len(v), 1024):
            up = torch.einsum("bd,bd->b", v[i:i + 1024], state["corpus"][chosen[i:i + 1024].clamp_min(0)].double())
            down = torch.einsum("bd,brd->br", v[i:i + 1024], state["corpus"][rejected[i:i + 1024].clamp_min(0)].double())
            parts.append(up.unsqueeze(1) - down)
        return torch.cat(parts) if parts else s

    with torch.enable_grad():
        m = scores(unit(q))
        if "reference" in d:
            m = m - scores(unit(d["reference"]))
        m = m * _SCALE * there
        eps = case["smoothing"]
        each = -(1 - eps) * torch.nn.functional.logsigmoid(m) - eps * torch.nn.functional.logsigmoid(-m)
        loss = (each * there).sum() / there.sum().clamp_min(1)
    (dq,) = torch.autograd.grad(loss, q, d["loss_scale"])
    return {"loss": loss.detach(), "margins": m.detach(), "dqueries": dq}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "float32" else 2
    if case["op"] == "layer_norm":
        cells, dim = case["rows"] * case["dim"], case["dim"]
        if case["train"]:  # x, dy in; y, dx out; weight, bias in; their gradients out
            return {"bytes": e * (4 * cells + 4 * dim), "flops": 22 * cells}
        return {"bytes": e * (2 * cells + 2 * dim), "flops": 8 * cells}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["inputs"], case["outputs"]
        moved = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if case["train"]:  # dy in; dx, dweight, dbias out (the residual's gradient is dy itself)
            moved += m * n + m * k + n * k + n
        return {"bytes": e * moved, "flops": 2 * m * k * n * (3 if case["train"] else 1)}
    b, r, d = case["queries"], case["rejected"], case["dim"]
    kept = 1 - case["missing"]
    rows = int(b * (1 + r * kept))
    moved = 2 * d * rows + e * b * d * (3 if case["reference"] else 2) + 8 * b * (1 + r) + 4 * b * r + 4
    return {"bytes": moved, "flops": 5 * d * b * r + 12 * b * d}
