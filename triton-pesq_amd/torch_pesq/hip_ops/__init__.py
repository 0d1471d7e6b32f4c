"""HIP operators of the PESQ pipeline, one module per stage.

Mirrors the operator set of the reference's ``torch_pesq/triton_ops``:
``HipIIR`` (``TritonIIR``), ``HipResample`` (``TritonResample``),
``HipStftBark`` (``TritonStftBark``), ``HipPesqChain`` (``TritonPesqChain``),
the element-wise functions and ``PesqLossHip`` (``PesqLossTriton``).

Additions for the networks that the loss trains: ``recurrence`` (the gated
linear recurrence), ``norm`` (norms around a residual block) and ``adamw`` (the
optimizer's step over all tensors).
"""

import torch

HAS_HIP = torch.cuda.is_available()

__all__ = ["HAS_HIP"]
