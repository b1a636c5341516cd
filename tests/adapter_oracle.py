"""Plain float64 forms of the query adapter's operators (test infrastructure).

Inputs are the operators' own (rounded) inputs, widened exactly; results and
gradients are float64. ``close`` compares with a tolerance counted in roundings.
"""

from __future__ import annotations

import math

import numpy as np
import torch

# Half a step of each type: one rounding's largest relative error.
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}  # half of the smallest step


def close(got, want, extra=0.0, roundings=1):
    """|got - want| <= roundings x half a step of got's type x |want|, plus ``extra``
    (a float64 array or number: the error of everything before the last rounding)."""
    g = got.detach().double().cpu().numpy()
    w = want.detach().double().cpu().numpy()
    assert g.shape == w.shape, (g.shape, w.shape)
    e = extra.detach().double().cpu().numpy() if torch.is_tensor(extra) else np.asarray(extra, dtype=np.float64)
    u = HALF_STEP[got.dtype]
    tol = roundings * u * np.abs(w) + (1 + u) * e + TINY[got.dtype]
    nan = np.isnan(w)
    assert (np.isnan(g) == nan).all(), "NaN in other places"
    bad = ~(np.abs(g - w) <= tol) & ~nan & ~(np.isinf(w) & (g == w))
    assert not bad.any(), f"{bad.sum()} of {bad.size} off; worst {np.nanmax(np.abs(g - w) - tol)} over its tolerance"


def layer_norm(x, w, b, eps, dy=None):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    h = (x - mean) * rstd
    w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if w is None else w.double()
    b = torch.zeros_like(w) if b is None else b.double()
    y = h * w + b
    if dy is None:
        return y
    dy = dy.double()
    g = dy * w
    dx = rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
    return y, dx, (dy * h).sum(0), dy.sum(0), (h, rstd, g)


def act(z, name):
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def linear(x, w, b, activation, residual):
    """(y, z, slope, scale): scale bounds the sum of the products' magnitudes."""
    z = x.double() @ w.double().T
    scale = x.double().abs() @ w.double().abs().T
    if b is not None:
        z = z + b.double()
        scale = scale + b.double().abs()
    a, slope = act(z, activation)
    y = a if residual is None else a + residual.double()
    return y, z, slope, scale


def preference(q, ref, chosen, rejected, corpus, cosine, scale, smoothing, mean):
    """(loss, margins, dq) with dq the gradient of the loss."""
    q = q.double()

    def unit(v):
        return v / v.norm(dim=1, keepdim=True).clamp_min(1e-12) if cosine else v

    u = unit(q)
    moved = u if ref is None else u - unit(ref.double())
    there = (chosen[:, None] >= 0) & (rejected >= 0)
    x = corpus.double()
    apart = x[chosen.clamp_min(0)][:, None] - x[rejected.clamp_min(0)]
    m = torch.where(there, scale * (apart * moved[:, None]).sum(2), 0.0)
    soft = torch.nn.functional.softplus
    each = (1 - smoothing) * soft(-m) + smoothing * soft(m)
    weight = 1.0 / max(int(there.sum()), 1) if mean else 1.0
    loss = torch.where(there, each, 0.0).sum() * weight
    slope = torch.where(there, smoothing - torch.sigmoid(-m), 0.0) * scale * weight
    du = (slope[:, :, None] * apart).sum(1)
    if cosine:
        norm = q.norm(dim=1, keepdim=True)
        along = torch.where(norm > 1e-12, (u * du).sum(1, keepdim=True), 0.0)
        du = (du - u * along) / norm.clamp_min(1e-12)
    return loss, m, du
