"""Row-parallel linear with low-rank adapters of many requests at once (tcgen05 / TMEM kernels, csrc/kernels/adapters.cu).

    y = linear_adapters(x, wt, ids, a, b, scales)    # y[i] = x[i] @ wt.T + scales[j] * (x[i] @ a[j].T) @ b[j].T,  j = ids[i]

`wt` [N, K] in nn.Linear layout is shared by all rows; `a` [adapters, R, K] and `b` [adapters, N, R] hold the adapters, smaller ranks
padded with zeros; `ids` [M] int32 names the adapter of every row, any value outside 0 .. adapters-1 (-1 by convention) none.
Rows of one request need not be neighbours, and a row depends on its own adapter only, whatever the others hold.  Under tensor
parallelism every rank has its K columns of `wt` and `a` and all of `b`; y is its partial, the BF16 input of
`ctx.all_reduce_add_rms_norm` (N = 6144 there, any multiple of 8 here).

BF16 tensors, contiguous, starting on 16-byte boundaries; K, N and R are multiples of 8, R is at most 128.  All sums are FP32; x a.T is
not rounded below 16 bits of mantissa before it meets b, and y is rounded once.  Runs on the current stream; forward only: a call that
autograd would record and tangents of forward mode are refused, by `torch.ops.fp4ar.linear_adapters` as well.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _native as N


def linear_adapters(x: torch.Tensor, wt: torch.Tensor, ids: torch.Tensor, a: torch.Tensor, b: torch.Tensor,
                    scales: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x @ wt.T plus every row's own adapter, BF16 [M, N] (into `out` when given)."""
    return N.front().linear_adapters(x, wt, ids, a, b, scales, out)
