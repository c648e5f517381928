"""Output postprocessors — drop-in for reference ``models/postprocessors/postprocessors.py``
(Hydra ``_target_: ...postprocessors.postprocessors.L2NormEmbeddingPostprocessor``).

``L2NormEmbeddingPostprocessor`` (postprocessors.py:34-56) runs the
``gr_l2_normalize`` kernel forward and backward; ``LayerNormEmbeddingPostprocessor``
(postprocessors.py:59-80) the ``gr_layer_norm`` kernels where they apply.
"""
from __future__ import annotations

import abc

import torch
import torch.nn.functional as F
from torch.autograd.forward_ad import unpack_dual

from . import ops


class OutputPostprocessorModule(torch.nn.Module):
    """postprocessors.py:21-31."""

    @abc.abstractmethod
    def debug_str(self) -> str:
        pass

    @abc.abstractmethod
    def forward(self, output_embeddings: torch.Tensor) -> torch.Tensor:
        pass


class L2NormEmbeddingPostprocessor(OutputPostprocessorModule):
    def __init__(self, embedding_dim: int, eps: float = 1e-6) -> None:
        super().__init__()
        self._embedding_dim: int = embedding_dim
        self._eps: float = eps

    def debug_str(self) -> str:
        return "l2"

    def forward(self, output_embeddings: torch.Tensor) -> torch.Tensor:
        return ops.l2_normalize(output_embeddings[..., : self._embedding_dim], self._eps)


class LayerNormEmbeddingPostprocessor(OutputPostprocessorModule):
    """postprocessors.py:59-80.  float32 and bfloat16 rows on the GPU run ``ops.layer_norm``;
    everything else (CPU tensors, other types, autocast, forward-mode derivatives, traced or transformed
    calls) is torch's ``F.layer_norm``."""

    def __init__(self, embedding_dim: int, eps: float = 1e-6) -> None:
        super().__init__()
        self._embedding_dim: int = embedding_dim
        self._eps: float = eps

    def debug_str(self) -> str:
        return "ln"

    def forward(self, output_embeddings: torch.Tensor) -> torch.Tensor:
        output_embeddings = output_embeddings[..., : self._embedding_dim]
        if not torch.jit.is_scripting():
            if _kernel_takes(output_embeddings, self._embedding_dim):
                return ops.layer_norm(output_embeddings, eps=self._eps)
        return F.layer_norm(output_embeddings, normalized_shape=(self._embedding_dim,),
                            eps=self._eps)


def _kernel_takes(x, dim: int) -> bool:
    """Whether ``ops.layer_norm`` runs x, a plain tensor that no tracer or transform watches."""
    return (not torch.jit.is_tracing() and not torch.compiler.is_compiling()
            and type(x) is torch.Tensor and x.is_cuda and x.dtype in (torch.float32, torch.bfloat16)
            and 0 < dim == x.shape[-1] < ops.LN_COLUMNS and unpack_dual(x).tangent is None
            and not torch.is_autocast_enabled() and not torch._C._are_functorch_transforms_active()
            and not torch._C._len_torch_dispatch_stack()
            and not torch._C._dispatch_tls_is_dispatch_key_included(torch._C.DispatchKey.PreDispatch))
