"""Gated projections and their gradients against 64-bit references, at the sizes where tiles, K blocks and rows end inside one."""
import pytest
import torch

import layer_ref as R
from fp4_all_reduce_b200 import _native as N
from fp4_all_reduce_b200.ops import allreduce as A  # noqa: F401  (registers torch.ops.fp4ar)
from fp4_all_reduce_b200.ops import ffn
from fp4_all_reduce_b200.ops import gemm as G

pytestmark = pytest.mark.gpu


def _data(M, K, F, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wt = (torch.randn(2 * F, K, generator=g, device="cuda") / K ** 0.5).to(torch.bfloat16)
    dh = torch.randn(M, F, generator=g, device="cuda").to(torch.bfloat16)
    return x, wt, dh


def _within(got, want, bound, dtype=torch.bfloat16):
    assert got.shape == want.shape and got.dtype == dtype
    d = (got.double() - want).abs()
    assert bool((d <= bound).all()), float((d / bound).max())


SHAPES = [(1, 8, 8), (1, 64, 64), (2, 520, 72), (7, 1024, 136), (16, 2048, 256), (17, 72, 1000), (33, 200, 128), (63, 1000, 520),
          (64, 256, 264), (65, 6144, 64), (127, 128, 8), (128, 192, 128), (129, 4104, 200), (255, 136, 1368), (256, 64, 320), (257, 320, 136),
          (385, 2048, 512), (1031, 264, 648), (2050, 128, 1160)]


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_forward(M, K, F, act):
    x, wt, _ = _data(M, K, F)
    h = ffn.gated_linear(x, wt, act)
    want, gate, up, bound, eg, eu = R.gated(x, wt, act)
    _within(h, want, bound)
    h2, pre = ffn.gated_linear_forward(x, wt, act)
    assert torch.equal(h, h2)
    _within(pre, torch.cat([gate, up], 1), torch.cat([eg, eu], 1) + 1e-30, torch.float32)
    assert G.gemm_status().code == 0


@pytest.mark.parametrize("act", [0, 1, 2])
@pytest.mark.parametrize("M,K,F", SHAPES)
def test_gradients(M, K, F, act):
    x, wt, dh = _data(M, K, F, 1)
    x.requires_grad_(), wt.requires_grad_()
    h = ffn.gated_linear(x, wt, act)
    dx, dw = torch.autograd.grad(h, (x, wt), dh)
    wx, ww, bx, bw = R.gated_grads(dh, x, wt, act)
    _within(dx, wx, bx)
    _within(dw, ww, bw)
    # two roundings (dpre, result) of at most 2^-8 each, of independent sizes: their rms is below 2^-8 sqrt(2 / 3)
    for got, want in ((dx, wx), (dw, ww)):
        assert (got.double() - want).norm() <= R.BF16 * want.norm()
    assert G.gemm_status().code == 0
