"""Tensors that a call writes into (`out`, an updated residual) get a new version: autograd notices that one of them was saved for a
backward pass."""
import pytest
import torch

from fp4_all_reduce_b200 import _native as N
from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import allreduce as A  # noqa: F401  (registers torch.ops.fp4ar)
from fp4_all_reduce_b200.ops import codec
from fp4_all_reduce_b200.ops import ffn
from fp4_all_reduce_b200.ops import gemm as G
from fp4_all_reduce_b200.parallel.context import SoloRankContext

pytestmark = pytest.mark.gpu


def _bf16(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


def _noticed(call, *written):
    """`call` writes every tensor of `written`: one new version each, shared with the storage's other views, and a backward pass that
    has saved it raises."""
    w = torch.ones((), device="cuda", requires_grad=True)
    losses = [(t.float() * w).sum() if t.dtype == torch.uint8 else (t * w.to(t.dtype)).sum() for t in written]
    views, versions = [t[:1] for t in written], [t._version for t in written]
    call()
    for t, v, n, loss in zip(written, views, versions, losses):
        assert t._version == n + 1 and v._version == n + 1
        if t.dtype != torch.uint8:                                   # (the product saved a copy of those)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()


@pytest.mark.parametrize("rows", [4, 600])
def test_outputs_of_the_feed_forward_ops(rows):
    x, wt, a, b = _bf16(rows, 64), _bf16(48, 64, seed=1), _bf16(2, 8, 64, seed=2), _bf16(2, 48, 8, seed=3)
    ids = (torch.arange(rows, device="cuda") % 3).to(torch.int32)
    h, y = torch.zeros(rows + 1, 24, device="cuda", dtype=torch.bfloat16)[:rows], torch.zeros(rows, 48, device="cuda", dtype=torch.bfloat16)
    before = [t._version for t in (x, wt, ids, a, b)]
    _noticed(lambda: ffn.gated_linear(x, wt, out=h), h)
    _noticed(lambda: ffn.gated_linear_forward(x, wt, out=h), h)
    _noticed(lambda: AD.linear_adapters(x, wt, ids, a, b, out=y), y)
    assert [t._version for t in (x, wt, ids, a, b)] == before


def test_outputs_made_under_inference_mode_may_be_written_anywhere():
    """Such a tensor has no version, and autograd cannot have saved it."""
    x, wt = _bf16(4, 64), _bf16(48, 64, seed=1)
    want = ffn.gated_linear(x, wt)
    with torch.inference_mode():
        h = torch.empty(4, 24, device="cuda", dtype=torch.bfloat16)
        assert torch.equal(ffn.gated_linear(x, wt, out=h), want)
    assert torch.equal(ffn.gated_linear(x, wt, out=h), want)


ROWS = 8


def test_outputs_of_the_codec_norm_and_gemm_ops():
    x, w = _bf16(ROWS, N.HIDDEN), _bf16(N.HIDDEN, seed=1)
    res, out = _bf16(ROWS, N.HIDDEN, seed=2), _bf16(ROWS, N.HIDDEN, seed=3)
    _noticed(lambda: codec.add_rmsnorm(x, res, w, out=out), out)
    _noticed(lambda: codec.add_rmsnorm(x, res, w, inplace_residual=True), res)
    _noticed(lambda: codec.add_rmsnorm(x, res, w, inplace_residual=True, out=out), res, out)
    _noticed(lambda: torch.ops.fp4ar.add_rms_norm(x, res, w, 1e-6, 1.0), res)
    q = torch.zeros(ROWS, N.QROW_BYTES, device="cuda", dtype=torch.uint8)
    _noticed(lambda: G.gemm_nvfp4(_bf16(ROWS, 64), _bf16(N.HIDDEN, 64), 1.0, out=q), q)
    before = [t._version for t in (x, w, res)]
    codec.add_rmsnorm(x, res, w)
    assert [t._version for t in (x, w, res)] == before


@pytest.mark.parametrize("native", [True, False])
def test_outputs_of_a_context(native):
    """By the native front end and by the Python wrappers behind it (a NumPy scale is theirs)."""
    import numpy as np

    ctx, kw = SoloRankContext(2, ROWS), dict(mode=N.MODE_COMPUTE)
    if not native:
        ctx._front = None
    x, w = _bf16(ROWS, N.HIDDEN), _bf16(N.HIDDEN, seed=1)
    res, out, other = _bf16(ROWS, N.HIDDEN, seed=2), _bf16(ROWS, N.HIDDEN, seed=3), _bf16(ROWS, N.HIDDEN, seed=4)
    q = torch.zeros(ROWS, N.QROW_BYTES, device="cuda", dtype=torch.uint8)
    _noticed(lambda: ctx.all_reduce(x, out, **kw), out)
    _noticed(lambda: ctx.all_reduce_add_rms_norm(x, res, w, **kw), res)
    _noticed(lambda: ctx.all_reduce_add_rms_norm(x, res, w, out=out, residual_out=other, **kw), out, other)
    _noticed(lambda: ctx.all_reduce_add_rms_norm(x, res, w, epilogue=N.EPI_NORM_NVFP4, out=q, **kw), res, q)
    _noticed(lambda: ctx.all_reduce_add_rms_norm(x, res, w, eps=np.float32(1e-6), **kw), res)
    n = x._version
    with torch.inference_mode():
        made = torch.zeros_like(x)
    ctx.all_reduce(x, made, **kw)
    assert x._version == n and torch.equal(made, ctx.all_reduce(x, **kw))
    ctx.close()


class _PushOnly(SoloRankContext):
    """A rank whose pushes go into its own window and whose AllReduce is left out (its peers do not exist)."""

    def launch(self, args, stream=None):
        pass


def test_tensors_of_the_fused_linear():
    ctx = _PushOnly(2, ROWS)
    x, wt, w = _bf16(ROWS, 64), _bf16(N.HIDDEN, 64, seed=1), _bf16(N.HIDDEN, seed=2)
    res, out = _bf16(ROWS, N.HIDDEN, seed=3), _bf16(ROWS, N.HIDDEN, seed=4)
    q = torch.zeros(ROWS, N.QROW_BYTES, device="cuda", dtype=torch.uint8)
    _noticed(lambda: G.gemm_all_reduce_add_rms_norm(ctx, x, wt, [1.0, 1.0], res, w), res)
    _noticed(lambda: G.gemm_all_reduce_add_rms_norm(ctx, x, wt, [1.0, 1.0], res, w, out=out), res, out)
    _noticed(lambda: G.gemm_push(ctx, x, wt, 1.0, local_q=q), q)
    ctx.close()
