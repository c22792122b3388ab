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
          (385, 2048, 512), (1031, 264, 648), (2050, 128, 1160), (500, 512, 264), (900, 136, 72),
          (1024, 256, 136), (400, 128, 4104), (200000, 8, 8), (1, 64, 100000), (3, 32768, 16)]


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


def test_gradients_against_differences():
    """d/de sum(c h(x + e dx, W + e dW)) at e = 0 by central differences of the 64-bit formula, against <dx, grad x> + <dW, grad W>.
    The third derivative of the loss along the direction is of the order of the loss itself, so the step 2^-8 leaves 2^-16 of it;
    the gradients are off by 2^-8 of their norm at most (see above), and so is a product with a direction, relative to the norms."""
    M, K, F = 40, 136, 88
    x, wt, c = _data(M, K, F, 4)
    g = torch.Generator(device="cuda").manual_seed(5)
    vx = torch.randn(M, K, generator=g, device="cuda", dtype=torch.float64)
    vw = torch.randn(2 * F, K, generator=g, device="cuda", dtype=torch.float64) / K ** 0.5
    for act in range(3):
        _, pre = ffn.gated_linear_forward(x, wt, act)
        dx, dw = ffn.gated_linear_backward(c, pre, x, wt, act)
        step = 2.0 ** -8

        def loss(e):
            p = (x.double() + e * vx) @ (wt.double() + e * vw).t()
            return (c.double() * R.act(p[:, :F], act) * p[:, F:]).sum()

        want = (loss(step) - loss(-step)) / (2 * step)
        got = (dx.double() * vx).sum() + (dw.double() * vw).sum()
        size = dx.double().norm() * vx.norm() + dw.double().norm() * vw.norm()
        assert abs(got - want) <= (R.BF16 + 2.0 ** -14) * size, (act, float(got), float(want))


def test_the_op_alone_recomputes_and_gives_the_same_gradients():
    x, wt, dh = _data(150, 264, 136, 6)
    x.requires_grad_(), wt.requires_grad_()
    h = ffn.gated_linear(x, wt, 1)
    want = torch.autograd.grad(h, (x, wt), dh)
    h2 = torch.ops.fp4ar.gated_linear(x, wt, 1)
    got = torch.autograd.grad(h2, (x, wt), dh)
    assert torch.equal(h, h2) and all(torch.equal(a, b) for a, b in zip(got, want))
    fn = torch.compile(lambda a, b: torch.ops.fp4ar.gated_linear(a, b, 1), fullgraph=True, backend="aot_eager")
    h3 = fn(x, wt)
    got = torch.autograd.grad(h3, (x, wt), dh)
    assert torch.equal(h, h3) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("M", [5, 300])
def test_one_input_needs_a_gradient_and_any_layout_of_dh(M):
    x, wt, _ = _data(M, 72, 40, 7)
    wx, ww, bx, bw = R.gated_grads(torch.ones(M, 40, device="cuda").to(torch.bfloat16), x, wt, 0)
    xg = x.clone().requires_grad_()
    ffn.gated_linear(xg, wt).sum().backward()                       # an expanded gradient, strides 0
    _within(xg.grad, wx, bx)
    wg = wt.clone().requires_grad_()
    ffn.gated_linear(x, wg).sum().backward()
    _within(wg.grad, ww, bw)
    _, pre = ffn.gated_linear_forward(x, wt)
    dh = torch.randn(40, M, device="cuda").to(torch.bfloat16).t()
    a = ffn.gated_linear_backward(dh, pre, x, wt, need_dwt=False)
    b = ffn.gated_linear_backward(dh.contiguous(), pre, x, wt, need_dx=False)
    assert a[1] is None and b[0] is None
    wx, ww, bx, bw = R.gated_grads(dh, x, wt, 0)
    _within(a[0], wx, bx), _within(b[1], ww, bw)


def test_a_gradient_that_starts_anywhere():
    x, wt, _ = _data(6, 72, 40, 7)
    _, pre = ffn.gated_linear_forward(x, wt)
    room = torch.randn(6 * 40 + 3, device="cuda").to(torch.bfloat16)
    dh = room[3:].view(6, 40)                                        # contiguous, six bytes behind a boundary
    a, b = ffn.gated_linear_backward(dh, pre, x, wt), ffn.gated_linear_backward(dh.clone(), pre, x, wt)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_no_second_derivative():
    x, wt, _ = _data(4, 16, 8, 8)
    x.requires_grad_()
    (dx,) = torch.autograd.grad(ffn.gated_linear(x, wt).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="differentiated twice"):
        dx.sum().backward()


def test_a_changed_input_is_noticed():
    x, wt, _ = _data(4, 16, 8, 8)
    wt.requires_grad_()
    x = x.clone()
    h = ffn.gated_linear(x, wt)
    x.zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_no_rows():
    x, wt, dh = _data(0, 64, 32)
    x.requires_grad_(), wt.requires_grad_()
    h = ffn.gated_linear(x, wt)
    dx, dw = torch.autograd.grad(h, (x, wt), dh)
    assert h.shape == (0, 32) and dx.shape == (0, 64) and bool((dw == 0).all()) and dw.shape == (64, 64)


@pytest.mark.parametrize("M", [3, 129, 600])
def test_out_is_written_and_nothing_behind_it(M):
    x, wt, _ = _data(M, 72, 40, 9)
    room = torch.full((M + 2, 40), 7.0, device="cuda", dtype=torch.bfloat16)
    h = ffn.gated_linear(x, wt, out=room[:M])
    assert h.data_ptr() == room.data_ptr() and torch.equal(h, ffn.gated_linear(x, wt)) and bool((room[M:] == 7).all())


@pytest.mark.parametrize("M", [9, 200, 700])
def test_a_bad_row_stays_in_its_row(M):
    """Infinities and NaN in one row of x, or in the weights of one column of h, reach nothing else."""
    x, wt, dh = _data(M, 136, 72, 10)
    h, pre = ffn.gated_linear_forward(x, wt)
    dx, _ = ffn.gated_linear_backward(dh, pre, x, wt)
    x2, wt2 = x.clone(), wt.clone()
    x2[4, 3], x2[5, 0] = float("nan"), float("inf")
    wt2[7, 1] = float("nan")                                         # gate row of column 7
    h2, pre2 = ffn.gated_linear_forward(x2, wt2)
    rows = [i for i in range(M) if i not in (4, 5)]
    cols = [i for i in range(72) if i != 7]
    assert torch.equal(h2[rows][:, cols], h[rows][:, cols])
    assert bool(torch.isnan(h2[:, 7]).all() and torch.isnan(h2[4]).all())
    _, pre3 = ffn.gated_linear_forward(x2, wt)
    dx3, _ = ffn.gated_linear_backward(dh, pre3, x2, wt)
    assert torch.equal(dx3[rows], dx[rows])


@pytest.mark.parametrize("act", [0, 1, 2])
def test_gates_far_from_zero(act):
    """Gates from -3e38 to 3e38: the values and slopes go to their limits without NaN, in both kernels."""
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, -1.5, 3.0, -9.0, 12.0, -40.0, 88.0, -88.0, -100.0, 1e4, -1e4, 1e19, -1e19, 1e20, -1e20, 3e38, -3e38],
                     device="cuda").to(torch.bfloat16)
    for M in (g.numel(), 26 * g.numel()):
        x = torch.zeros(M, 8, device="cuda", dtype=torch.bfloat16)
        x[:, 0] = g.repeat(M // g.numel())
        x[:, 1] = 1.0
        wt = torch.zeros(16, 8, device="cuda", dtype=torch.bfloat16)
        wt[:8, 0], wt[8:, 1] = 1.0, 1.0                              # gate = g, up = 1
        h, pre = ffn.gated_linear_forward(x, wt, act)
        dx, _ = ffn.gated_linear_backward(torch.ones_like(h), pre, x, wt, act)
        want, slope = R.act(x[:, 0].double(), act), R.act_grad(x[:, 0].double(), act)
        want, slope = torch.nan_to_num(want), torch.nan_to_num(slope, nan=float((act >= 0)))
        far = x[:, 0].double().abs() > 1e5                           # there the 64-bit formula may overflow: limits 0, g; slopes 0, 1
        want = torch.where(far, x[:, 0].double().clamp(min=0), want)
        slope = torch.where(far, (x[:, 0] > 0).double(), slope)
        # the FP32 exponential of an argument t is off by t 2^-23: of -g^2 / 2 at -9 5e-6, of 88 1e-5; tiny values vanish
        assert bool(((h[:, 0].double() - want).abs() <= (R.BF16 + 2.0 ** -16) * want.abs() + 1e-35).all())
        # eight equal terms summed, each with its own rounding
        assert bool(((dx[:, 0].double() - 8 * slope).abs() <= 8 * (2.1 * R.BF16 * slope.abs() + 2.0 ** -20)).all())


def test_offsets_beyond_32_bits():
    """pre has more than 2^32 bytes and 2^31 elements; rows at its end are looked at."""
    M, K, F = 70000, 8, 16384
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wt = torch.randn(2 * F, K, generator=g, device="cuda").to(torch.bfloat16)
    h, pre = ffn.gated_linear_forward(x, wt)
    rows = torch.tensor([0, 1, 32767, 32768, 65535, 65536, 69998, 69999], device="cuda")
    want, gate, up, bound, eg, eu = R.gated(x[rows], wt, 0)
    _within(h[rows], want, bound)
    _within(pre[rows], torch.cat([gate, up], 1), torch.cat([eg, eu], 1) + 1e-30, torch.float32)
    dh = torch.ones(M, F, device="cuda", dtype=torch.bfloat16)
    dx, _ = ffn.gated_linear_backward(dh, pre, x, wt, need_dwt=False)
    wx, _, bx, _ = R.gated_grads(dh[rows], x[rows], wt, 0)
    _within(dx[rows], wx, bx)


@pytest.mark.parametrize("M,K,F", [(6, 2048, 512), (200, 512, 264), (1100, 6144, 2048)])
def test_captured_and_replayed(M, K, F):
    """Forward and backward in one CUDA graph (the last shape cuts K loops), replayed on new data beside eager calls on another
    stream: the same bits as eagerly."""
    x, wt, dh = _data(M, K, F, 11)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        xg, wg = x.clone().requires_grad_(), wt.clone().requires_grad_()
        torch.autograd.grad(ffn.gated_linear(xg, wg), (xg, wg), dh)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        h = ffn.gated_linear(xg, wg)
        dx, dw = torch.autograd.grad(h, (xg, wg), dh)
    torch.cuda.synchronize()
    for seed in (12, 13):
        x2, wt2, dh2 = _data(M, K, F, seed)
        with torch.no_grad():
            xg.copy_(x2), wg.copy_(wt2), dh.copy_(dh2)
        torch.cuda.synchronize()
        graph.replay()
        h2, pre2 = ffn.gated_linear_forward(x2, wt2)                 # on the current stream, at the same time
        dx2, dw2 = ffn.gated_linear_backward(dh2, pre2, x2, wt2)
        torch.cuda.synchronize()
        assert torch.equal(h, h2) and torch.equal(dx, dx2) and torch.equal(dw, dw2)
    assert G.gemm_status().code == 0


_FIRST = """
import torch
from fp4_all_reduce_b200.ops import adapters, ffn, gemm
for rows in (4, 300, 1100):
    x = torch.ones(rows, 4096, device="cuda", dtype=torch.bfloat16)
    wt = torch.full((4096, 4096), 2.0 ** -12, device="cuda", dtype=torch.bfloat16)
    a, b = torch.zeros(3, 8, 4096, device="cuda", dtype=torch.bfloat16), torch.ones(3, 4096, 8, device="cuda", dtype=torch.bfloat16)
    ids = torch.zeros(rows, device="cuda", dtype=torch.int32)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h, pre = ffn.gated_linear_forward(x, wt)
        dx, dw = ffn.gated_linear_backward(torch.ones_like(h), pre, x, wt)
        y = adapters.linear_adapters(x, wt, ids, a, b)
    g.replay()
    torch.cuda.synchronize()
    want = torch.sigmoid(torch.ones(()).double()).item()             # gate = up = 1
    assert abs(h.double() - want).max().item() <= want * 2 ** -8 and (pre == 1).all() and (y == 1).all()
    assert gemm.gemm_status().code == 0
print("captured first")
"""


def test_the_first_call_of_a_process_may_be_captured():
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    p = subprocess.run([sys.executable, "-c", _FIRST], cwd=root, capture_output=True, text=True, timeout=300)
    assert p.returncode == 0 and "captured first" in p.stdout, p.stderr[-2000:]


def test_calls_on_several_streams_at_once():
    shapes = [(1100, 6144, 2048), (30, 2048, 512), (4000, 4096, 1024)]
    data = [_data(*s, seed=20 + i) for i, s in enumerate(shapes)]
    want = []
    for x, wt, dh in data:
        h, pre = ffn.gated_linear_forward(x, wt)
        want.append((h, *ffn.gated_linear_backward(dh, pre, x, wt)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(11)]           # more than have a workspace of their own
    got = []
    for r in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, wt, dh = data[i % 3]
                h, pre = ffn.gated_linear_forward(x, wt)
                got.append((i % 3, (h, *ffn.gated_linear_backward(dh, pre, x, wt))))
    torch.cuda.synchronize()
    for i, outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
    assert G.gemm_status().code == 0


def test_refusals():
    x, wt, dh = _data(4, 16, 8)
    h, pre = ffn.gated_linear_forward(x, wt)
    shifted = torch.zeros(4 * 16 + 4, device="cuda", dtype=torch.bfloat16)[4:].view(4, 16)
    for bad, why in ((x.float(), "x must be torch.bfloat16"), (x[:, :12], "wt must have shape"), (x.t().contiguous().t(), "x must be contiguous"),
                     (shifted, "16-byte boundary"), (x[0], "x must have shape")):
        with pytest.raises(ValueError, match=why):
            ffn.gated_linear(bad, wt)
    for bad, why in ((wt.half(), "wt must be torch.bfloat16"), (wt[:12], "multiple of 8"), (wt.cpu(), "CUDA"), (wt[::2][:0], "multiple of 8")):
        with pytest.raises(ValueError, match=why):
            ffn.gated_linear(x, bad)
    with pytest.raises(ValueError, match="K must be"):
        ffn.gated_linear(x[:, :4].contiguous(), wt[:, :4].contiguous())
    with pytest.raises(ValueError, match="activation"):
        ffn.gated_linear(x, wt, 3)
    for out, why in ((torch.empty(4, 16, device="cuda", dtype=torch.bfloat16), "out must have shape"), (h.float(), "out must be"),
                     (x.view(-1)[:32].view(4, 8), "overlap x"), (wt.view(-1)[:32].view(4, 8), "overlap wt")):
        with pytest.raises(ValueError, match=why):
            ffn.gated_linear(x, wt, out=out)
    with pytest.raises(ValueError, match="gradient is recorded"):
        ffn.gated_linear(x.clone().requires_grad_(), wt, out=h)
    for args, why in (((dh[:3], pre, x, wt), "dh must have shape"), ((dh, pre.to(torch.bfloat16), x, wt), "pre must be torch.float32"),
                      ((dh.float(), pre, x, wt), "dh must be"), ((dh, pre[:, :8], x, wt), "pre must have shape")):
        with pytest.raises(ValueError, match=why):
            ffn.gated_linear_backward(*args)
    with pytest.raises(TypeError, match="x must be a tensor"):
        ffn.gated_linear([1.0], wt)


@pytest.mark.multigpu
def test_tensors_of_another_device():
    x, wt, dh = _data(40, 64, 32)
    there = "cuda:1"
    with pytest.raises(ValueError, match="is on cuda:1"):
        ffn.gated_linear(x, wt.to(there))
    h, pre = ffn.gated_linear_forward(x.to(there), wt.to(there))     # the current device is another one
    dx, dw = ffn.gated_linear_backward(dh.to(there), pre, x.to(there), wt.to(there))
    h0, pre0 = ffn.gated_linear_forward(x, wt)
    dx0, dw0 = ffn.gated_linear_backward(dh, pre0, x, wt)
    assert torch.equal(h.cpu(), h0.cpu()) and torch.equal(dx.cpu(), dx0.cpu()) and torch.equal(dw.cpu(), dw0.cpu())
