"""Exact top-k vector search on NVIDIA B200 (sm_100a) with hand-written kernels.

Drop-in for the reference package's public API (cuda_vector_search/__init__.py:3-7):
``Index``, ``exact_topk_fp32``, ``torch_topk``. ``ShardedIndex`` adds row-sharded
search over a torch.distributed process group (one rank per GPU). ``Adapter``, with
its operators ``layer_norm`` and ``linear`` and the training loss
``Index.preference_loss``, adapts the queries to a fixed index.
"""

from .adapter import Adapter, layer_norm, linear
from .index import Index
from .reference import exact_topk_fp32, torch_topk
from .sharded import ShardedIndex

__all__ = ["Adapter", "Index", "ShardedIndex", "exact_topk_fp32", "layer_norm", "linear", "torch_topk"]
__version__ = "0.1.0"
