"""A query adapter: a small residual network between an embedding model and a
fixed index, the operators it is made of, and its use in a search.

``Adapter`` maps embeddings ``x`` to ``x + W2 act(W1 layer_norm(x) + b1) + b2``. It is
trained with ``Index.preference_loss`` (queries, the rows users preferred, the rows they
passed over) while the corpus stays as it is, and used with
``Index.search(queries, k, adapter=adapter)``. All operators run on this package's own
kernels, on the current stream of their inputs' device; they are differentiable once (in
reverse mode: tangents of ``torch.autograd.forward_ad`` are refused), allocate through
torch's caching allocator only, and can be captured into CUDA graphs.
"""

from __future__ import annotations

import torch

from . import _ext

ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


def layer_norm(x, weight=None, bias=None, eps: float = 1e-5):
    """Layer norm over the last dimension (up to 8192 wide), in x's dtype.

    x: float32, float16 or bfloat16. weight, bias: one value per column, float32 or
    x's dtype, or None (ones / zeros). Statistics and sums are float32.
    """
    return _ext.load().layer_norm(x, weight, bias, float(eps))


def linear(x, weight, bias=None, activation: str = "none", residual=None):
    """``activation(x @ weight.T + bias) + residual``, rounded once to x's dtype.

    x: [..., k], float16 or bfloat16, and every other operand of the same dtype;
    weight: [n, k]; bias: [n]; residual: [..., n], of the result's shape.
    activation: "none", "relu", "gelu" (the exact one) or "silu". Rows whose address
    or stride is not a multiple of 16 bytes are copied first when there are more than
    8 of them.
    """
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
    return _ext.load().linear(x, weight, bias, ACTIVATIONS[activation], residual)


class Adapter(torch.nn.Module):
    """Residual network over embeddings: ``x + W2 act(W1 layer_norm(x) + b1) + b2``.

    W2 and b2 start at zero, so an untrained adapter leaves embeddings as they are.

    Args:
        dim: embedding width.
        hidden: width of the hidden layer (default: twice the embedding's).
        activation: "gelu", "relu", "silu" or "none".
        dtype: float16 or bfloat16, of the parameters and of the computation. An
            optimizer's small steps are lost in either: let it work on float32 copies of
            the parameters and copy them back after each step.
    """

    def __init__(self, dim: int, hidden: int | None = None, activation: str = "gelu", eps: float = 1e-5,
                 dtype=torch.float16, device=None):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation must be one of {tuple(ACTIVATIONS)}")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("an adapter's dtype must be float16 or bfloat16")
        hidden = 2 * dim if hidden is None else hidden
        if dim < 1 or hidden < 1:
            raise ValueError("dim and hidden must be positive")
        self.dim, self.hidden, self.activation, self.eps = dim, hidden, activation, eps
        kw = {"dtype": dtype, "device": device}
        self.norm_weight = torch.nn.Parameter(torch.ones(dim, **kw))
        self.norm_bias = torch.nn.Parameter(torch.zeros(dim, **kw))
        self.weight1 = torch.nn.Parameter((torch.randn(hidden, dim, device=device) * dim**-0.5).to(dtype))
        self.bias1 = torch.nn.Parameter(torch.zeros(hidden, **kw))
        self.weight2 = torch.nn.Parameter(torch.zeros(dim, hidden, **kw))
        self.bias2 = torch.nn.Parameter(torch.zeros(dim, **kw))

    def forward(self, x):
        """Adapted embeddings of x [..., dim], in the adapter's dtype."""
        x = x.to(self.weight1.dtype)
        h = layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        h = linear(h, self.weight1, self.bias1, activation=self.activation)
        return linear(h, self.weight2, self.bias2, residual=x)

    def extra_repr(self) -> str:
        return f"dim={self.dim}, hidden={self.hidden}, activation={self.activation!r}"
