"""The row-parallel linear with adapters of many requests against 64-bit references."""
import pytest
import torch

import layer_ref as R
from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import gemm as G

pytestmark = pytest.mark.gpu


def _data(M, K, Nn, n, r, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rnd(*s, std=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * std).to(torch.bfloat16)

    return (rnd(M, K), rnd(Nn, K, std=K ** -0.5), torch.randint(-1, n, (M,), generator=g, device="cuda", dtype=torch.int32),
            rnd(n, r, K, std=K ** -0.5), rnd(n, Nn, r, std=0.3), 0.5 + torch.rand(n, generator=g, device="cuda"))


def _check(args):
    y = AD.linear_adapters(*args)
    want, bound = R.adapters(*args)
    d = (y.double() - want).abs()
    assert y.shape == want.shape and bool((d <= bound).all()), float((d / bound).max())
    assert G.gemm_status().code == 0
    return y


@pytest.mark.parametrize("M,K,Nn,n,r", [(1, 8, 8, 1, 8), (1, 2048, 6144, 8, 16), (2, 72, 264, 3, 24), (5, 520, 1000, 5, 64), (16, 128, 128, 4, 8),
                                        (33, 1992, 328, 40, 16), (64, 2048, 512, 48, 16), (65, 64, 64, 70, 32), (100, 256, 200, 7, 128),
                                        (128, 320, 256, 1, 40), (129, 136, 520, 9, 48), (255, 1000, 136, 300, 16), (257, 264, 264, 12, 72),
                                        (700, 512, 1032, 6, 104), (1031, 200, 648, 16, 32), (2050, 128, 1160, 3, 64)])
def test_mixed_rows(M, K, Nn, n, r):
    _check(_data(M, K, Nn, n, r))


@pytest.mark.parametrize("M", [1, 20, 64, 130, 513])
def test_requests_in_any_order(M):
    """All rows without an adapter, all with one, contiguous requests, ids far outside the range, no scales."""
    x, wt, _, a, b, sc = _data(M, 264, 392, 6, 16, 2)
    for ids in (torch.full((M,), -1), torch.full((M,), 5), torch.arange(M) * 6 // M, 5 - torch.arange(M) % 6,
                torch.tensor([6, 2 ** 31 - 1, -2 ** 31, -7, 3])[torch.arange(M) % 5]):
        ids = ids.to(torch.int32).cuda()
        y = _check((x, wt, ids, a, b, sc))
        plain = AD.linear_adapters(x, wt, torch.full_like(ids, -1), a, b, sc)
        bare = (ids < 0) | (ids >= 6)
        assert torch.equal(y[bare], plain[bare])
    _check((x, wt, ids, a, b, None))


@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("where", ["a", "b"])
def test_a_broken_adapter_stays_with_its_rows(M, where):
    """Infinities and NaN in one request's adapter or input row reach no other row; its own rows get what the formula gives."""
    x, wt, _, a, b, sc = _data(M, 128, 264, 3, 16, 3)
    ids = (torch.arange(M, device="cuda") % 3).to(torch.int32)
    clean = AD.linear_adapters(x, wt, ids, a, b, sc)
    t = (a if where == "a" else b).clone()
    t[1, 5, 7], t[1, 6, 3] = float("inf"), float("nan")
    x2 = x.clone()
    x2[2] = float("nan")
    y = AD.linear_adapters(x2, wt, ids, t if where == "a" else a, t if where == "b" else b, sc)
    others = ids != 1
    others[2] = False
    assert torch.equal(y[others], clean[others])
    assert torch.isnan(y[2]).all()
    mine = ids == 1
    if where == "a":
        assert torch.isnan(y[mine]).all()
    else:
        assert torch.isnan(y[mine][:, 6]).all() and torch.isinf(y[mine][:, 5]).all()
        keep = [c for c in range(264) if c not in (5, 6)]
        want, bound = R.adapters(x, wt, ids, a, b, sc)
        assert bool(((y.double() - want).abs() <= bound)[mine][:, keep].all())
