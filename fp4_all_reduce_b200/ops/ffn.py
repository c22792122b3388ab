"""Gated projections of the feed-forward block, the column-parallel half in front of the row-parallel linear
(tcgen05 / TMEM kernels, csrc/kernels/gated.cu).

    h = gated_linear(x, wt)                          # act(x @ wt[:F].T) * (x @ wt[F:].T), [M, F]; differentiable
    h, pre = gated_linear_forward(x, wt)             # the same, keeping the two projections [M, 2 F] for
    dx, dwt = gated_linear_backward(dh, pre, x, wt)  # their gradients

`wt` is [2 F, K] in nn.Linear layout, this rank's F gate rows followed by its F up rows; x is what the AllReduce block before it
returns, h is the input of the row-parallel linear behind it.  Under tensor parallelism dx is this rank's partial of the
gradient, to be summed by `ctx.all_reduce`.

BF16 tensors, contiguous, starting on 16-byte boundaries; K and F are multiples of 8, M is any row count.  Sums, the activation and
the product are FP32, h is rounded once.  The backward pass hands the gradients of
the projections to its matrix products in BF16.  Everything runs on the current stream.

Second derivatives and forward mode are refused, by `torch.ops.fp4ar.gated_linear` as well.  A given `out` gets a new version, as
after any in-place operation; where autograd records it must not require a gradient.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native as N

ACTIVATIONS = {"silu": N.ACT_SILU, "gelu": N.ACT_GELU, "gelu_tanh": N.ACT_GELU_TANH}


def gated_linear(x: torch.Tensor, wt: torch.Tensor, activation: int = N.ACT_SILU, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x @ wt[:F].T) * (x @ wt[F:].T).  Where autograd records, the projections are kept for the backward pass and `out`
    cannot be given."""
    return N.front().gated_linear(x, wt, activation, out)


def gated_linear_forward(x: torch.Tensor, wt: torch.Tensor, activation: int = N.ACT_SILU, *,
                         out: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(h, pre): pre [M, 2 F] holds the gate and the up projections in FP32; h is the same as without it.  Records no gradient."""
    return N.front().gated_linear_pre(x, wt, activation, out)


def gated_linear_backward(dh: torch.Tensor, pre: torch.Tensor, x: torch.Tensor, wt: torch.Tensor, activation: int = N.ACT_SILU, *,
                          need_dx: bool = True, need_dwt: bool = True) -> tuple[Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dwt) for the gradient dh of h, each None where it is not needed.  dh may have any strides and any place in
    its storage.  Records no gradient."""
    return N.front().gated_backward(dh, pre, x, wt, activation, need_dx, need_dwt)
