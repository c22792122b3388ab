"""Tensors that a call writes into (`out`, an updated residual) get a new version: autograd notices that one of them was saved for a
backward pass."""
import pytest
import torch

from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import allreduce as A  # noqa: F401  (registers torch.ops.fp4ar)
from fp4_all_reduce_b200.ops import ffn

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
