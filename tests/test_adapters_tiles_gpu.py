"""The linear with adapters where tiles of 256 rows take it: offsets beyond 32 bits, and adapters that are not finite in every state that
the tiled kernel can be in (several tiles per CTA pair, several blocks per adapter, cut K loops)."""
import ctypes as C

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


def _plan(M, Nn, K):
    """(tiles of the busiest unit, whether K loops are cut) on 74 CTA pairs"""
    used, segs = C.c_int(), (C.c_int * (5 * 64))()
    tiles, kblocks, most, cut = -(-M // 256) * -(-Nn // 256), -(-K // 64), 0, False
    assert N.cuda().fp4ar_layer_plan(tiles, kblocks, 74, 0, C.byref(used), None, 0) == 0
    for u in range(used.value):
        n = N.cuda().fp4ar_layer_plan(tiles, kblocks, 74, u, C.byref(used), segs, 64)
        most, cut = max(most, n), cut or any(segs[5 * i + 3] for i in range(n))
    return most, cut


# (rows, K, N, adapters, rank), tiles of a unit at least, K loops cut
STATES = [((600, 264, 6144, 3, 16), 1, False), ((1100, 264, 6144, 5, 72), 2, False), ((600, 64, 107600, 3, 16), 17, False),
          ((1500, 128, 5000, 4, 128), 2, False), ((513, 200, 264, 30, 40), 1, False), ((600, 8192, 2048, 3, 72), 1, True),
          ((1100, 6144, 4096, 5, 16), 2, True), ((700, 8192, 520, 4, 128), 1, True)]


@pytest.mark.parametrize("shape,tiles,cut", STATES)
@pytest.mark.parametrize("where", ["a", "b"])
def test_a_broken_adapter_stays_with_its_rows(shape, tiles, cut, where):
    """Infinities and NaN of one request in the first, a middle and the last tile of columns reach no other row; its own rows get what
    the formula gives, in the broken columns too."""
    M, K, Nn, n, r = shape
    _tiled(M, n)
    most, cuts = _plan(M, Nn, K)
    assert most >= tiles and cuts == cut
    g = torch.Generator(device="cuda").manual_seed(11)

    def rnd(*s, std=1.0):
        return (torch.randn(*s, generator=g, device="cuda") * std).to(torch.bfloat16)

    x, wt, a, b = rnd(M, K), rnd(Nn, K, std=K ** -0.5), rnd(n, r, K, std=K ** -0.5), rnd(n, Nn, r, std=0.3)
    sc = 0.5 + torch.rand(n, generator=g, device="cuda")
    ids = (torch.arange(M, device="cuda") % (n + 1) - 1).to(torch.int32)
    clean = AD.linear_adapters(x, wt, ids, a, b, sc)
    want, bound = R.adapters(x, wt, ids, a, b, sc)
    assert bool(((clean.double() - want).abs() <= bound).all())
    broken, bad = n - 1, (5, 6, (Nn // 2) | 1, Nn - 3)
    t = (a if where == "a" else b).clone()
    if where == "a":
        t[broken, r - 1, K - 1] = float("nan")
    else:
        t[broken, bad[0], r - 1], t[broken, bad[1], 0], t[broken, bad[2], r // 2], t[broken, bad[3], 3] = (float(f) for f in ("inf", "nan", "-inf", "nan"))
    x2 = x.clone()
    x2[2] = float("nan")                                             # ids[2] is 1: not the broken one
    for _ in range(2):
        y = AD.linear_adapters(x2, wt, ids, t if where == "a" else a, t if where == "b" else b, sc)
        mine, others = ids == broken, ids != broken
        others[2] = mine[2] = False
        assert torch.equal(y[others], clean[others])
        assert bool(torch.isnan(y[2]).all())
        if where == "a":
            assert bool(torch.isnan(y[mine]).all())
            continue
        good = torch.ones(Nn, dtype=torch.bool, device="cuda")
        good[list(bad)] = False
        v = sc[broken].double() * (x[mine].double() @ a[broken].double().t())
        # the broken tiles add r products one by one to the finished sum
        extra = r * 2.0 ** -24 * (v.abs() @ b[broken].double().abs().t()) + 2.0 ** -24 * want[mine].abs()
        assert bool(((y[mine].double() - want[mine]).abs() <= bound[mine] + extra)[:, good].all())
        assert bool(torch.isnan(y[mine][:, [bad[1], bad[3]]]).all())
        assert torch.equal(y[mine][:, bad[0]].double(), torch.sign(v[:, r - 1]) * float("inf"))
        assert torch.equal(y[mine][:, bad[2]].double(), torch.sign(v[:, r // 2]) * -float("inf"))
    assert G.gemm_status().code == 0


def test_every_adapter_broken_but_one():
    """All blocks of a tile but one adapter's are zeros, in all orders of the list."""
    M, K, Nn, n, r = 700, 264, 1032, 12, 72
    _tiled(M, n)
    g = torch.Generator(device="cuda").manual_seed(12)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wt = (torch.randn(Nn, K, generator=g, device="cuda") * K ** -0.5).to(torch.bfloat16)
    a = (torch.randn(n, r, K, generator=g, device="cuda") * K ** -0.5).to(torch.bfloat16)
    b = (torch.randn(n, Nn, r, generator=g, device="cuda") * 0.3).to(torch.bfloat16)
    for keep in (0, 5, n - 1):
        ids = ((torch.arange(M, device="cuda") * 7 + keep) % n).to(torch.int32)
        clean = AD.linear_adapters(x, wt, ids, a, b)
        t = b.clone()
        t[torch.arange(n, device="cuda") != keep, ::256, 9] = float("nan")       # a column of every tile
        y = AD.linear_adapters(x, wt, ids, a, t)
        assert torch.equal(y[ids == keep], clean[ids == keep])
        assert bool(torch.isnan(y[ids != keep][:, ::256]).all())
        want, bound = R.adapters(x, wt, ids, a, b, None)
        v = torch.stack([x.double() @ a[j].double().t() for j in range(n)])[ids.long(), torch.arange(M, device="cuda")]
        size = torch.stack([v.abs() @ b[j].double().abs().t() for j in range(n)])[ids.long(), torch.arange(M, device="cuda")]
        fine = torch.ones(Nn, dtype=torch.bool, device="cuda")
        fine[::256] = False
        assert bool(((y.double() - want).abs() <= bound + r * 2.0 ** -24 * size + 2.0 ** -24 * want.abs())[:, fine].all())
    assert G.gemm_status().code == 0
