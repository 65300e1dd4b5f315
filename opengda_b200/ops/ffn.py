"""The gated half of a feed-forward block: ``h = act(x @ w_gate^T) * (x @ w_up^T)``.

Both projections, the activation and the product run in one tcgen05 kernel
(csrc/kernels/ffn.cu); the backward pass in two.  The dense counterpart of the expert layer's
first grouped GEMM (``models.moe``); the down projection is ``ops.gemm.gemm`` or, with
adapters, ``ops.lora.lora_linear``.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import native

ACTS = {"silu": 0, "gelu": 1, "gelu_tanh": 2}


def _writable(out: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """``out`` as a target of a kernel: not part of an autograd graph, and its version advanced
    so that a graph that saved it notices the overwrite."""
    if out is not None:
        if out.requires_grad:
            raise ValueError("out must not require a gradient")
        if not out.is_inference():
            torch.autograd.graph.increment_version(out)
    return out


def _act(act: str) -> int:
    if act not in ACTS:
        raise ValueError(f"act must be one of {sorted(ACTS)}, not {act!r}")
    return ACTS[act]


def gated_linear_forward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, act: str = "silu",
                         save: bool = True, out: Optional[torch.Tensor] = None,
                         tile: int = 0) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """``gated_linear`` without autograd: returns ``(h, saved)``; ``saved`` is what
    ``gated_linear_backward`` needs (g and u in f32, 8 bytes per element of h, in a private
    layout), or None with ``save=False``."""
    h, saved = native().gated_linear(x, w_gate, w_up, _act(act), bool(save), _writable(out), int(tile))
    return h, saved


def gated_linear_backward(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                          saved: torch.Tensor, act: str = "silu", need_dx: bool = True,
                          need_dw: bool = True, tile: int = 0) -> Tuple[Optional[torch.Tensor], ...]:
    """Gradients ``(dx, dw_gate, dw_up)`` of ``gated_linear`` from ``dh`` (row-major) and the
    forward's ``saved``; None for those not wanted.  The gradients of g and u are rounded to the
    inputs' type once, between the activation's derivative and the products (in fp16, scale the loss so
    that they stay above 6e-5); sums are f32."""
    return native().gated_linear_backward(dh, x, w_gate, w_up, saved, _act(act), bool(need_dx), bool(need_dw),
                                          int(tile))


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, act: str = "silu",
                 out: Optional[torch.Tensor] = None, tile: int = 0) -> torch.Tensor:
    """``h[T, I] = act(x[T, H] @ w_gate[I, H]^T) * (x @ w_up[I, H]^T)``, differentiable
    once, in reverse mode (an argument with a forward-mode tangent is refused).

    bf16 or fp16 (all alike), f32 accumulation and activation, one rounding.  ``act``: "silu",
    "gelu" (erf) or "gelu_tanh".  H a multiple of 8 and 16-byte aligned rows (as ``ops.gemm``);
    T and I are free.  ``out`` and ``tile`` (0 by shape, 1 split-K clusters for few rows, 2 and 3
    CTA pairs with 256 x 512 and 256 x 256 tiles) are for calls without gradients.

    Runs on the current stream of x's device and can be captured in a CUDA graph.  To capture a
    training step, call ``gated_linear_forward`` and ``gated_linear_backward``, or make sure that
    no autograd graph made on the default stream of the same parameters (or of what the weights are
    computed from) is alive: such a call is refused."""
    if torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad):
        if out is not None or tile:
            raise ValueError("gated_linear: out and tile are for calls without gradients")
        return native().gated_linear_autograd(x, w_gate, w_up, _act(act))
    return gated_linear_forward(x, w_gate, w_up, act, save=False, out=out, tile=tile)[0]
