"""The linear with adapters where tiles of 256 rows take it: offsets beyond 32 bits."""
import pytest
import torch

import layer_ref as R
from fp4_all_reduce_b200 import _native as N
from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import gemm as G

pytestmark = pytest.mark.gpu


def _tiled(M, adapters):
    assert N.cuda().fp4ar_adapters_few_rows(M, adapters) == 0


@pytest.mark.parametrize("M", [513, 600])
def test_offsets_beyond_32_bits(M):
    """b has 2.6e9 elements; the last adapters and the last columns are looked at, one of the adapters not finite in one of them."""
    n, Nn, r, K = 160, 131072, 128, 8
    _tiled(M, n)
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wt = torch.randn(Nn, K, generator=g, device="cuda").to(torch.bfloat16)
    a = torch.randn(n, r, K, generator=g, device="cuda").to(torch.bfloat16)
    b = torch.empty(n, Nn, r, device="cuda", dtype=torch.bfloat16)
    b[n - 2:].normal_(generator=g)
    b[:n - 2] = float("nan")                                         # nobody's
    ids = (n - 1 - torch.arange(M, device="cuda") % 2).to(torch.int32)
    cols = torch.tensor([0, 1, 255, 256, 65535, 65536, Nn - 257, Nn - 1], device="cuda")
    want, bound = R.adapters(x, wt[cols], ids - (n - 2), a[n - 2:], b[n - 2:][:, cols], None)
    y = AD.linear_adapters(x, wt, ids, a, b)
    assert bool(((y[:, cols].double() - want).abs() <= bound).all())
    b[n - 1, Nn - 2, 77] = float("nan")                              # in the last tile, beside the last column
    y2 = AD.linear_adapters(x, wt, ids, a, b)
    other = ids == n - 2
    assert torch.equal(y2[other], y[other]) and bool(torch.isnan(y2[~other, Nn - 2]).all())
    assert torch.equal(y2[:, :Nn - 256], y[:, :Nn - 256])            # tiles without it are as before
    # the last tile of the adapter that is not finite there: r products are added one by one to the finished sum
    v, va = x.double() @ a[n - 1].double().t(), b[n - 1][cols].double().abs()
    extra = r * 2.0 ** -24 * (v.abs() @ va.t()) + 2.0 ** -24 * want.abs()
    assert bool(((y2[:, cols].double() - want).abs() <= bound + extra)[~other].all())
    assert G.gemm_status().code == 0
