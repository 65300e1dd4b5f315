"""A shared projection with the low-rank adapters of many requests (csrc/kernels/lora.cu)."""
from __future__ import annotations

from typing import Optional

import torch

from .. import native
from .ffn import _writable


def lora_linear(x: torch.Tensor, w: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, adapter: torch.Tensor,
                scale: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None, tile: int = 0) -> torch.Tensor:
    """``y[t] = w x[t] + scale[a] * lora_b[a] (lora_a[a] x[t])`` with ``a = adapter[t]``.

    x [T, K], w [N, K], lora_a [L, r, K], lora_b [L, N, r], all bf16 or all fp16; adapter int32
    [T], -1 for a row without one; scale f32 [L] (default 1).  Rows may use any adapters in any
    order; only the adapters in use are read.  K and r multiples of 8, r <= 128, L <= 8192,
    16-byte aligned rows of x and w; T and N are free.  Sums are f32; scale times
    lora_a x is rounded to the inputs' type before lora_b (so in fp16 it has to stay within 65504).

    The indexes stay on the device: one outside [-1, L) gives its row no adapter and raises at
    the next ``ops.gemm.check_errors()``.  Inference only: an input that requires a gradient is
    refused while gradients are enabled, one with a forward-mode tangent always.  Runs on the
    current stream of x's device and can be captured in a CUDA graph.  ``tile``: 0 by shape, 1
    split-K clusters (few rows), 2 and 3 CTA pairs with 256 x 512 and 256 x 256 tiles."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in (x, w, lora_a, lora_b) + (() if scale is None else (scale,))):
        raise RuntimeError("lora_linear has no backward pass: call it under torch.no_grad()")
    return native().lora_linear(x, w, lora_a, lora_b, adapter, scale, _writable(out), int(tile))
