"""Derivatives that the feed-forward ops do not have are refused on the GPU as on the host, those they have stay as they were."""
import pytest
import torch

from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import allreduce as A  # noqa: F401  (registers torch.ops.fp4ar)
from fp4_all_reduce_b200.ops import ffn

pytestmark = pytest.mark.gpu


def _bf16(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("gated", [ffn.gated_linear, lambda x, wt: torch.ops.fp4ar.gated_linear(x, wt, 0)], ids=["ffn", "op"])
@pytest.mark.parametrize("rows", [4, 300])
def test_a_gradient_penalty_raises(gated, rows):
    """First gradients taken with create_graph=True are those taken without; differentiating them raises."""
    x, wt = _bf16(rows, 16).requires_grad_(), _bf16(48, 16, seed=1).requires_grad_()
    want = torch.autograd.grad(gated(x, wt).sum(), (x, wt))
    h = gated(x, wt)
    grads = torch.autograd.grad(h.sum(), (x, wt), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        (h.sum() + grads[0].square().sum()).backward()
    assert x.grad is None and wt.grad is None


@pytest.mark.parametrize("rows", [4, 600])
def test_adapters_refuse_a_recording_by_both_entries(rows):
    x, wt, a, b = _bf16(rows, 64), _bf16(48, 64, seed=1), _bf16(2, 8, 64, seed=2), _bf16(2, 48, 8, seed=3)
    ids = (torch.arange(rows, device="cuda") % 3).to(torch.int32)
    scales = torch.full((2,), 0.5, device="cuda")
    want = AD.linear_adapters(x, wt, ids, a, b, scales)
    assert torch.equal(torch.ops.fp4ar.linear_adapters(x, wt, ids, a, b, scales), want)
    for call in (AD.linear_adapters, torch.ops.fp4ar.linear_adapters):
        for i in (0, 1, 3, 4, 5):
            args = [x, wt, ids, a, b, scales]
            args[i] = args[i].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="linear_adapters has no backward pass"):
                call(*args)
            with torch.no_grad():
                y = call(*args)
            assert torch.equal(y, want) and not y.requires_grad


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    x, wt, a, b = _bf16(4, 64), _bf16(48, 64, seed=1), _bf16(2, 8, 64, seed=2), _bf16(2, 48, 8, seed=3)
    ids = torch.zeros(4, device="cuda", dtype=torch.int32)
    h, pre = ffn.gated_linear_forward(x, wt)
    for fn, args in ((ffn.gated_linear, (x, wt)), (ffn.gated_linear_forward, (x, wt)), (ffn.gated_linear_backward, (h, pre, x, wt)),
                     (lambda *t: torch.ops.fp4ar.gated_linear(*t, 0), (x, wt)), (lambda *t: torch.ops.fp4ar.gated_linear_pre(*t, 0), (x, wt)),
                     (lambda *t: torch.ops.fp4ar.gated_linear_backward(*t, 0, True, True), (h, pre, x, wt)),
                     (lambda *t: AD.linear_adapters(t[0], t[1], ids, t[2], t[3]), (x, wt, a, b)),
                     (lambda *t: torch.ops.fp4ar.linear_adapters(t[0], t[1], ids, t[2], t[3], None), (x, wt, a, b))):
        fn(*args)
        for i in range(len(args)):
            with forward_ad.dual_level():
                dual = list(args)
                dual[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(RuntimeError, match="has no forward-mode derivative"):
                    fn(*dual)
    g = x.clone().requires_grad_()
    for gated in (ffn.gated_linear, lambda p, q: torch.ops.fp4ar.gated_linear(p, q, 0)):      # forward over reverse
        with forward_ad.dual_level(), pytest.raises(RuntimeError):
            torch.autograd.grad(gated(g, wt), g, forward_ad.make_dual(h, h))


@pytest.mark.parametrize("gated", [ffn.gated_linear, lambda x, wt: torch.ops.fp4ar.gated_linear(x, wt, 0)], ids=["ffn", "op"])
def test_a_gradient_penalty_raises_where_only_some_gradients_are_asked_for(gated):
    """autograd.grad and backward(inputs=...) run only what leads to the tensors they are given: the refusal stands on the way to every
    input of the first backward pass."""
    x, wt, dh = (t.requires_grad_() for t in (_bf16(4, 16), _bf16(48, 16, seed=1), _bf16(4, 24, seed=2)))
    for wanted in ((x, wt), (x,), (wt,), (dh,)):
        for first in (x, wt):
            h = gated(x, wt)
            (g,) = torch.autograd.grad(h, first, dh, create_graph=True)
            with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
                torch.autograd.grad(h.sum() + g.square().sum(), wanted, allow_unused=True)
            h = gated(x, wt)
            (g,) = torch.autograd.grad(h, first, dh, create_graph=True)
            with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
                (h.sum() + g.square().sum()).backward(inputs=list(wanted))
