"""Low-rank adapters of many requests beside one shared projection (no reference counterpart).

Row m of a batch uses adapter g = ids[m], or none; with s_g = scale (a number, or scale[g])::

    low[m] = s_g * A[m] @ down[g].T                 [M, R]
    C[m]   = A[m] @ B.T + low[m] @ up[g].T          [M, N]

`LoraPlan` is made once per batch and serves every projection of the model; `gemm_lora` is the
forward pass from one token to long prompts, `gemm_lora_backward` the gradients of A, down and up
(B is frozen; its gradient, where one is wanted, is ``gemm(dC, A, a_is_km=True)``).
"""
from __future__ import annotations

import torch

from . import _C

MAX_RANK = 128        # GEMM_SM100_LORA_MAX_RANK
MAX_ADAPTERS = 4096   # GEMM_SM100_LORA_MAX_ADAPTERS


class LoraPlan:
    """Which adapter each row of a batch uses, prepared on the device without waiting for it.

    ``ids`` holds one int32 or int64 index per row; a value outside ``[0, num_adapters)`` means that
    the row has no adapter.  ``update(ids)`` refills the plan for another batch of as many rows in
    stream order (also inside a captured CUDA graph): use and refill it on one stream, or order the
    streams yourself.
    """

    def __init__(self, ids: torch.Tensor, num_adapters: int):
        if ids.dim() != 1:
            raise ValueError("ids must be a 1D tensor with one adapter index per row")
        if not 1 <= num_adapters <= MAX_ADAPTERS:
            raise ValueError(f"num_adapters must be between 1 and {MAX_ADAPTERS}, got {num_adapters}")
        if not ids.is_cuda:
            raise ValueError("ids must be a CUDA tensor")
        self.rows = ids.shape[0]
        self.num_adapters = num_adapters
        self.buffer = torch.empty(_C.lora_plan_bytes(self.rows, num_adapters), dtype=torch.uint8, device=ids.device)
        self.stream = torch.cuda.current_stream(ids.device).cuda_stream   # the memory's own stream
        _C.lora_plan(ids, num_adapters, self.buffer)

    def update(self, ids: torch.Tensor) -> "LoraPlan":
        if ids.dim() != 1 or ids.shape[0] != self.rows:
            raise ValueError(f"the plan is for {self.rows} rows, ids has shape {tuple(ids.shape)}")
        stream = torch.cuda.current_stream(self.buffer.device)
        if stream.cuda_stream != self.stream:
            self.buffer.record_stream(stream)
        _C.lora_plan(ids, self.num_adapters, self.buffer)
        return self


def _scales(scale) -> tuple[torch.Tensor | None, float]:
    return (scale, 1.0) if isinstance(scale, torch.Tensor) else (None, float(scale))


def gemm_lora(A: torch.Tensor, B: torch.Tensor, down: torch.Tensor, up: torch.Tensor, plan: LoraPlan,
              scale: float | torch.Tensor = 1.0, out: torch.Tensor | None = None,
              low: torch.Tensor | None = None) -> torch.Tensor:
    """``A @ B.T`` plus, for every row, the product through its own adapter; returns ``out``.

    A ``[M,K]``, B ``[N,K]``, down ``[adapters,R,K]``, up ``[adapters,N,R]``, all bf16 or all fp16; R is a
    multiple of 8 up to 128, K a multiple of 8.  ``scale`` is a number or a float32 tensor with one
    value per adapter.  ``low`` (``[M,R]``) receives the scaled low-rank rows, which the backward pass
    can use again.  ``out`` may have a row pitch; with more than one row it has to be a multiple of 8
    elements.  Without ``out`` and with N no multiple of 8 the result is the first N columns of such rows.
    """
    scales, factor = _scales(scale)
    return _C.gemm_lora(A, B, down, up, plan.buffer, plan.rows, plan.num_adapters, plan.stream, scales, factor, out, low)


def gemm_lora_backward(dC: torch.Tensor, A: torch.Tensor, B: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                       plan: LoraPlan, scale: float | torch.Tensor = 1.0, low: torch.Tensor | None = None,
                       needs: tuple[bool, bool, bool] = (True, True, True)):
    """``(dA, d_down, d_up)`` for the gradient ``dC`` ``[M,N]`` of `gemm_lora`'s result; N a multiple of 8.

    ``low`` is what `gemm_lora` was given (computed again when None).  Entries of ``needs`` that are
    False come back as None and are not computed.  Adapters without rows get zeros.
    """
    scales, factor = _scales(scale)
    return tuple(_C.gemm_lora_backward(dC, A, B, down, up, plan.buffer, plan.rows, plan.num_adapters, plan.stream, scales,
                                       factor, low, *needs))
