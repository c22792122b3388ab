"""The feed-forward half of one transformer layer under tensor parallelism, inference:

    h = act(x Wg^T) * (x Wu^T)                        gated projections, this rank's F columns
    partial = h Wd^T  (+ the adapters of the rows)    row-parallel down projection
    AllReduce -> residual add -> Gemma RMSNorm        the fused block of `ctx`

This is the MLP end of a block of `models/m3_block.py`, with its matrix products in place of the pre-computed partials.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from .. import _native as N
from ..ops import adapters as _adapters
from ..ops import ffn
from ..ops import gemm as _gemm


class FeedForward:
    """`gate_up` [2 F, 6144] (gate rows, then up rows), `down` [6144, F], `norm_weight` [6144], all BF16, of this rank.

    Rows without adapters go through the NVFP4 GEMM, which needs `gs`, every rank's static scale of its partial
    (`calibrate` measures this rank's), and F a multiple of 64.  `a` [adapters, R, F], `b` [adapters, 6144, R] and `scales`
    are the down projection's adapters; a call that names `ids` adds them, and hands the AllReduce a BF16 partial."""

    def __init__(self, ctx, gate_up: torch.Tensor, down: torch.Tensor, norm_weight: torch.Tensor, *, activation: int = N.ACT_SILU,
                 gs: Optional[Sequence[float]] = None, a: Optional[torch.Tensor] = None, b: Optional[torch.Tensor] = None,
                 scales: Optional[torch.Tensor] = None, eps: float = 1e-6, weight_bias: float = 1.0):
        if gate_up.dim() != 2 or gate_up.shape[1] != N.HIDDEN or gate_up.shape[0] % 2:
            raise ValueError(f"gate_up must have shape [2 F, {N.HIDDEN}], got {tuple(gate_up.shape)}")
        if tuple(down.shape) != (N.HIDDEN, gate_up.shape[0] // 2):
            raise ValueError(f"down must have shape [{N.HIDDEN}, {gate_up.shape[0] // 2}], got {tuple(down.shape)}")
        if (a is None) != (b is None):
            raise ValueError("a and b come together")
        self.ctx, self.gate_up, self.down, self.norm_weight, self.activation = ctx, gate_up, down, norm_weight, activation
        self.gs, self.a, self.b, self.scales, self.eps, self.weight_bias = gs, a, b, scales, eps, weight_bias

    def calibrate(self, x: torch.Tensor) -> float:
        """This rank's static scale from a batch of inputs; gather every rank's into `gs`."""
        with torch.no_grad():
            return _gemm.calibrate_gs(ffn.gated_linear(x, self.gate_up, self.activation), self.down)

    @torch.no_grad()
    def __call__(self, x: torch.Tensor, residual: torch.Tensor, ids: Optional[torch.Tensor] = None, *, epilogue: int = N.EPI_NORM_BF16,
                 qscale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
        """(normed output, residual updated in place) of x [M, 6144]."""
        if ids is not None and self.a is None:
            raise ValueError("ids name adapters, but the block has none")
        if ids is None and self.gs is None:
            raise ValueError("without ids the NVFP4 GEMM runs, which needs gs (see calibrate)")
        h = ffn.gated_linear(x, self.gate_up, self.activation)
        if ids is None and self.ctx.nranks == 1:          # nobody to push to
            q = _gemm.gemm_nvfp4(h, self.down, self.gs[0])
            return self.ctx.all_reduce_add_rms_norm(q, residual, self.norm_weight, eps=self.eps, weight_bias=self.weight_bias,
                                                    epilogue=epilogue, qscale=qscale, gs=self.gs)
        if ids is None:
            return _gemm.gemm_all_reduce_add_rms_norm(self.ctx, h, self.down, self.gs, residual, self.norm_weight, eps=self.eps,
                                                      weight_bias=self.weight_bias, epilogue=epilogue, qscale=qscale)
        y = _adapters.linear_adapters(h, self.down, ids, self.a, self.b, self.scales)
        return self.ctx.all_reduce_add_rms_norm(y, residual, self.norm_weight, eps=self.eps, weight_bias=self.weight_bias, epilogue=epilogue,
                                                qscale=qscale)
