"""The feed-forward half of a layer as it is used: gated projections, down projection with or without adapters, AllReduce + norm of a
one-rank group, and the gradient of its input summed by the AllReduce; step by step against 64 bits and the host model."""
import pytest
import torch

import layer_ref as R
from fp4_all_reduce_b200 import _native as N
from fp4_all_reduce_b200 import oracle as O
from fp4_all_reduce_b200.models.feed_forward import FeedForward
from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import codec
from fp4_all_reduce_b200.ops import ffn
from fp4_all_reduce_b200.ops import gemm as G
from fp4_all_reduce_b200.utils import data as D

pytestmark = pytest.mark.gpu
F, POOL, RANK = 320, 5, 16


@pytest.fixture(scope="module")
def ctx():
    from fp4_all_reduce_b200.parallel.context import Fp4ArContext

    c = Fp4ArContext(640, device=torch.device("cuda", 0))
    yield c
    c.close()


def _block(ctx, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, std):
        return (torch.randn(*s, generator=g, device="cuda") * std).to(torch.bfloat16)

    return FeedForward(ctx, rnd(2 * F, N.HIDDEN, std=N.HIDDEN ** -0.5), rnd(N.HIDDEN, F, std=F ** -0.5), D.norm_weight().cuda(),
                       a=rnd(POOL, RANK, F, std=F ** -0.5), b=rnd(POOL, N.HIDDEN, RANK, std=0.3), scales=torch.rand(POOL, generator=g, device="cuda") + 0.5)


def _x(rows, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, N.HIDDEN, generator=g, device="cuda").to(torch.bfloat16)


@pytest.mark.parametrize("rows", [1, 40, 130, 600])
def test_with_adapters(ctx, rows):
    blk, x = _block(ctx), _x(rows)
    ids = (torch.arange(rows, device="cuda") % (POOL + 1) - 1).to(torch.int32)
    residual = D.residual(rows).cuda()
    res0 = residual.clone()
    out, res = blk(x, residual, ids)
    assert res.data_ptr() == residual.data_ptr()
    h = ffn.gated_linear(x, blk.gate_up)
    want, _, _, bound, _, _ = R.gated(x, blk.gate_up, 0)
    assert bool(((h.double() - want).abs() <= bound).all())
    y = AD.linear_adapters(h, blk.down, ids, blk.a, blk.b, blk.scales)
    want, bound = R.adapters(h, blk.down, ids, blk.a, blk.b, blk.scales)
    assert bool(((y.double() - want).abs() <= bound).all())
    exp = O.allreduce([O.bf16_bits(y)], epi=1, res_in=O.bf16_bits(res0), weight=O.bf16_bits(blk.norm_weight), eps=1e-6, wbias=1.0)
    assert (O.bf16_bits(out) == exp["out"]).all() and (O.bf16_bits(res) == exp["res_out"]).all()
    assert ctx.status().ok and G.gemm_status().code == 0


def test_without_adapters(ctx):
    blk, x = _block(ctx, 3), _x(70, 4)
    with pytest.raises(ValueError, match="needs gs"):
        blk(x, D.residual(70).cuda())
    blk.gs = [blk.calibrate(x)]
    residual = D.residual(70).cuda()
    res0 = residual.clone()
    out, res = blk(x, residual, epilogue=N.EPI_NORM_NVFP4, qscale=168.0)
    q = G.gemm_nvfp4(ffn.gated_linear(x, blk.gate_up), blk.down, blk.gs[0])
    exp = O.allreduce([q.cpu().numpy()], input_kind=1, gs=blk.gs, epi=2, res_in=O.bf16_bits(res0), weight=O.bf16_bits(blk.norm_weight), eps=1e-6,
                      wbias=1.0, qscale=168.0)
    assert (out.cpu().numpy() == exp["outq"]).all() and (O.bf16_bits(res) == exp["res_out"]).all()


def test_gradient_of_the_input_goes_through_the_all_reduce(ctx):
    """Training: dx of the column-parallel projections is a partial; its sum over the ranks is one AllReduce."""
    blk, x = _block(ctx, 5), _x(200, 6)
    dh = torch.randn(200, F, device="cuda").to(torch.bfloat16)
    xg, wg = x.clone().requires_grad_(), blk.gate_up.clone().requires_grad_()
    dx, dw = torch.autograd.grad(ffn.gated_linear(xg, wg), (xg, wg), dh)
    wx, ww, bx, bw = R.gated_grads(dh, x, blk.gate_up, 0)
    assert bool(((dx.double() - wx).abs() <= bx).all() and ((dw.double() - ww).abs() <= bw).all())
    total = ctx.all_reduce(dx)
    assert (O.bf16_bits(total) == O.allreduce([O.bf16_bits(dx)])["out"]).all()


def test_a_step_in_a_cuda_graph(ctx):
    blk, x = _block(ctx, 7), _x(48, 8)
    ids = (torch.arange(48, device="cuda") % POOL).to(torch.int32)
    residual = D.residual(48).cuda()
    res0 = residual.clone()
    want, res_want = blk(x, residual, ids)
    want, res_want = want.clone(), res_want.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, _ = blk(x, residual, ids)
    for _ in range(3):
        residual.copy_(res0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(residual, res_want)


def test_the_block_refuses_what_does_not_fit(ctx):
    blk = _block(ctx)
    with pytest.raises(ValueError, match="gate_up must have shape"):
        FeedForward(ctx, blk.gate_up[:, :64], blk.down, blk.norm_weight)
    with pytest.raises(ValueError, match="down must have shape"):
        FeedForward(ctx, blk.gate_up, blk.down[:, :64], blk.norm_weight)
    with pytest.raises(ValueError, match="come together"):
        FeedForward(ctx, blk.gate_up, blk.down, blk.norm_weight, a=blk.a)
    with pytest.raises(ValueError, match="has none"):
        FeedForward(ctx, blk.gate_up, blk.down, blk.norm_weight)(_x(2), D.residual(2).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"))
    for x, why in ((codec.encode_static(_x(2), 1.0), "wt must have shape"), (_x(2).float(), "x must be torch.bfloat16")):
        with pytest.raises(ValueError, match=why):
            blk(x, D.residual(2).cuda(), torch.zeros(2, dtype=torch.int32, device="cuda"))
