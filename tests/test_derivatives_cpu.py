"""Derivatives that the feed-forward ops do not have are refused, on meta tensors and, where the refusal comes before the checks of the
device, on CPU tensors: nothing is dropped in silence."""
import pytest
import torch


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from fp4_all_reduce_b200 import _native as N
    from fp4_all_reduce_b200.ops import allreduce  # noqa: F401  (registers torch.ops.fp4ar)

    try:
        N.front()
    except RuntimeError as e:
        pytest.skip(str(e))
    return torch.ops.fp4ar


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("needs", ["x", "wt", "both"])
def test_the_custom_op_has_no_second_derivative(ops, needs):
    """A loss with a gradient penalty: its backward pass raises, whichever input the gradient is taken of."""
    x, wt = _meta(5, 16), _meta(48, 16)
    wanted = {"x": [x], "wt": [wt], "both": [x, wt]}[needs]
    for t in wanted:
        t.requires_grad_()
    h = ops.gated_linear(x, wt, 0)
    grads = torch.autograd.grad(h.sum(), wanted, create_graph=True)
    assert [g.shape for g in grads] == [t.shape for t in wanted]
    loss = h.sum() + sum(g.square().sum() for g in grads)
    with pytest.raises(RuntimeError, match="gated_linear cannot be differentiated twice"):
        loss.backward()
    assert x.grad is None and wt.grad is None


def test_a_gradient_of_the_gradient_of_h_is_refused_too(ops):
    x, wt, dh = _meta(5, 16).requires_grad_(), _meta(48, 16), _meta(5, 24).requires_grad_()
    (dx,) = torch.autograd.grad(ops.gated_linear(x, wt, 0), x, dh, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        torch.autograd.grad(dx.sum(), dh)


def test_the_parts_of_the_backward_pass_have_no_gradient_of_their_own(ops):
    x, wt = _meta(5, 16).requires_grad_(), _meta(48, 16)
    h, pre = ops.gated_linear_pre(x, wt, 0)
    for out in (h, pre):
        with pytest.raises(RuntimeError, match="gated_linear_pre records no gradient"):
            torch.autograd.grad(out.sum(), x, retain_graph=True)
    dx, dw = ops.gated_linear_backward(_meta(5, 24), pre.detach(), x, wt, 0, True, True)
    with pytest.raises(RuntimeError, match="cannot be differentiated twice"):
        (dx.sum() + dw.sum()).backward()


def test_first_gradients_of_the_custom_op_stay(ops):
    x, wt = _meta(5, 16).requires_grad_(), _meta(48, 16).requires_grad_()
    ops.gated_linear(x, wt, 0).sum().backward()
    assert x.grad.shape == x.shape and wt.grad.shape == wt.shape
    assert not x.grad.requires_grad and not wt.grad.requires_grad


def test_a_compiled_step_still_traces(ops):
    x, wt = _meta(5, 16).requires_grad_(), _meta(48, 16).requires_grad_()
    h = torch.compile(lambda a, b: ops.gated_linear(a, b, 1), fullgraph=True, backend="aot_eager")(x, wt)
    dx, dw = torch.autograd.grad(h.sum(), (x, wt))
    assert dx.shape == x.shape and dw.shape == wt.shape


def _adapter_tensors(make):
    return dict(x=make(5, 16), wt=make(48, 16), ids=torch.zeros(5, dtype=torch.int32, device=make(1).device), a=make(2, 8, 16), b=make(2, 48, 8),
                scales=make(2, dtype=torch.float32))


@pytest.mark.parametrize("name", ["x", "wt", "a", "b", "scales"])
def test_the_op_with_adapters_has_no_backward_pass(ops, name):
    """As the function in ops/adapters.py, the op refuses the call; without a recording it takes the same tensors."""
    t = _adapter_tensors(_meta)
    t[name].requires_grad_()
    with pytest.raises(RuntimeError, match="linear_adapters has no backward pass"):
        ops.linear_adapters(**t)
    with torch.no_grad():
        y = ops.linear_adapters(**t)
    assert y.shape == (5, 48) and not y.requires_grad
    t[name] = t[name].detach()
    assert not ops.linear_adapters(**t).requires_grad


def test_a_compiled_call_with_adapters(ops):
    t = _adapter_tensors(_meta)
    fn = torch.compile(lambda *a: ops.linear_adapters(*a), fullgraph=True, backend="aot_eager")
    assert fn(*t.values()).shape == (5, 48)
    with pytest.raises(RuntimeError, match="linear_adapters has no backward pass"):
        fn(t["x"].clone().requires_grad_(), *list(t.values())[1:])


def _forward_mode(fn, args, i):
    """fn(*args) with a tangent on argument i."""
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        args = list(args)
        args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
        return fn(*args)


def test_the_functions_have_no_forward_mode(ops):
    """A dual tensor that requires no gradient would pass every other check; the result would have no tangent, which torch takes as zero."""
    from fp4_all_reduce_b200.ops import adapters, ffn

    def make(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype)

    x, wt, h, pre = make(5, 16), make(48, 16), make(5, 24), make(5, 48, dtype=torch.float32)
    t = list(_adapter_tensors(make).values())
    for name, fn, args, which in (("gated_linear", ffn.gated_linear, (x, wt), (0, 1)), ("gated_linear", ffn.gated_linear_forward, (x, wt), (0, 1)),
                                  ("gated_linear", ffn.gated_linear_backward, (h, pre, x, wt), (0, 1, 2, 3)),
                                  ("linear_adapters", adapters.linear_adapters, t, (0, 1, 3, 4, 5))):
        for i in which:
            with pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                _forward_mode(fn, args, i)
        with pytest.raises(ValueError, match="CUDA"):                # as before without a tangent
            fn(*args)
    with pytest.raises(RuntimeError, match="gated_linear has no forward-mode derivative"):
        _forward_mode(lambda a, b: ffn.gated_linear(a, b.requires_grad_()), (x, wt), 0)
    with pytest.raises(RuntimeError, match="gated_linear has no forward-mode derivative"):
        torch.func.jvp(lambda a: ffn.gated_linear(a, wt.detach()), (x,), (x,))


def test_the_custom_ops_have_no_forward_mode(ops):
    x, wt, h, pre = _meta(5, 16), _meta(48, 16), _meta(5, 24), _meta(5, 48, dtype=torch.float32)
    t = list(_adapter_tensors(_meta).values())
    for name, fn, args, which in (("gated_linear", lambda *a: ops.gated_linear(*a, 0), (x, wt), (0, 1)),
                                  ("gated_linear_pre", lambda *a: ops.gated_linear_pre(*a, 0), (x, wt), (0, 1)),
                                  ("gated_linear_backward", lambda *a: ops.gated_linear_backward(*a, 0, True, True), (h, pre, x, wt), (0, 1, 2, 3)),
                                  ("linear_adapters", ops.linear_adapters, t, (0, 1, 3, 4, 5))):
        for i in which:
            for recording in (True, False):
                with torch.set_grad_enabled(recording), pytest.raises(RuntimeError, match=f"{name} has no forward-mode derivative"):
                    _forward_mode(fn, args, i)
        fn(*args)
    with pytest.raises(RuntimeError):                                # recorded too: torch's own refusal
        _forward_mode(lambda a, b: ops.gated_linear(a, b.clone().requires_grad_(), 0), (x, wt), 0)
    # forward over reverse: the tangent of h's gradient does not get lost
    g = x.clone().requires_grad_()
    with pytest.raises(RuntimeError):
        _forward_mode(lambda d: torch.autograd.grad(ops.gated_linear(g, wt, 0), g, d), (h,), 0)


def test_an_out_with_a_history_is_refused(ops):
    """Its gradient would go on to whoever made the values that the call writes over."""
    from fp4_all_reduce_b200.ops import adapters, ffn

    x, wt = torch.zeros(5, 16, dtype=torch.bfloat16), torch.zeros(48, 16, dtype=torch.bfloat16)
    t = list(_adapter_tensors(lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)).values())
    for fn, args, out in ((ffn.gated_linear, (x, wt), torch.zeros(5, 24, dtype=torch.bfloat16)),
                          (ffn.gated_linear_forward, (x, wt), torch.zeros(5, 24, dtype=torch.bfloat16)),
                          (adapters.linear_adapters, t, torch.zeros(5, 48, dtype=torch.bfloat16))):
        leaf = out.requires_grad_()
        for bad in (leaf, leaf * 2):
            with pytest.raises(ValueError, match="out must not require a gradient"):
                fn(*args, out=bad)
            with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):       # nothing is recorded: taken as any other
                fn(*args, out=bad)
