"""The row-parallel linear with adapters of many requests against 64-bit references."""
import pytest
import torch

import layer_ref as R
from fp4_all_reduce_b200.ops import adapters as AD
from fp4_all_reduce_b200.ops import allreduce as A  # noqa: F401  (registers torch.ops.fp4ar)
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
                                        (700, 512, 1032, 6, 104), (1031, 200, 648, 16, 32), (2050, 128, 1160, 3, 64),
                                        (1500, 72, 136, 900, 8), (600, 256, 264, 700, 128), (513, 320, 520, 513, 40), (300, 6144, 264, 4, 16), (100000, 16, 8, 5, 8), (7, 32768, 16, 3, 32), (2, 64, 100000, 4, 16)])
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


@pytest.mark.parametrize("M,K,Nn", [(128, 64, 264), (112, 72, 520), (128, 256, 40000), (256, 64, 136), (250, 2048, 6144), (225, 128, 1000), (500, 136, 264)])
def test_many_rows_of_one_tile(M, K, Nn):
    """Short K loops and wide outputs leave K whole: a CTA then holds the sums and the low-rank parts of all its rows."""
    _check(_data(M, K, Nn, 40, 16, 6))


def test_no_rows_out_and_the_custom_op():
    x, wt, ids, a, b, sc = _data(20, 72, 40, 3, 8, 4)
    assert AD.linear_adapters(x[:0], wt, ids[:0], a, b, sc).shape == (0, 40)
    y = _check((x, wt, ids, a, b, sc))
    room = torch.full((22, 40), 7.0, device="cuda", dtype=torch.bfloat16)
    out = AD.linear_adapters(x, wt, ids, a, b, sc, out=room[:20])
    assert out.data_ptr() == room.data_ptr() and torch.equal(out, y) and bool((room[20:] == 7).all())
    assert torch.equal(torch.ops.fp4ar.linear_adapters(x, wt, ids, a, b, sc), y)
    fn = torch.compile(lambda *t: torch.ops.fp4ar.linear_adapters(*t), fullgraph=True, backend="eager")
    assert torch.equal(fn(x, wt, ids, a, b, sc), y)


@pytest.mark.parametrize("M", [4, 300])
def test_every_rank_and_every_adapter_counts(M):
    """One nonzero rank at a time, in the last adapter too: nothing of B or A is skipped or taken twice."""
    K, Nn, n = 64, 264, 5
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wt = torch.zeros(Nn, K, device="cuda", dtype=torch.bfloat16)
    ids = (torch.arange(M, device="cuda") % n).to(torch.int32)
    for r in (8, 40, 128):
        for at in range(0, r, 7):
            a = torch.zeros(n, r, K, device="cuda", dtype=torch.bfloat16)
            b = torch.zeros(n, Nn, r, device="cuda", dtype=torch.bfloat16)
            a[:, at, 0] = torch.arange(1, n + 1, device="cuda").to(torch.bfloat16)
            b[:, :, at] = 1.0
            y = AD.linear_adapters(x, wt, ids, a, b)
            want = (x[:, 0].double() * (ids + 1)).unsqueeze(1).expand(M, Nn)
            assert bool(((y.double() - want).abs() <= (R.BF16 + 2.0 ** -16) * want.abs()).all()), (r, at)


@pytest.mark.parametrize("M", [5, 300])
def test_offsets_beyond_32_bits(M):
    """b has 2.6e9 elements; the last adapters and the last columns are looked at."""
    n, Nn, r, K = 160, 131072, 128, 8
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    wt = torch.randn(Nn, K, generator=g, device="cuda").to(torch.bfloat16)
    a = torch.randn(n, r, K, generator=g, device="cuda").to(torch.bfloat16)
    b = torch.empty(n, Nn, r, device="cuda", dtype=torch.bfloat16)
    b[n - 2:].normal_(generator=g)
    b[:n - 2] = float("nan")                                         # nobody's
    ids = (n - 1 - torch.arange(M, device="cuda") % 2).to(torch.int32)
    y = AD.linear_adapters(x, wt, ids, a, b)
    cols = torch.tensor([0, 1, 255, 256, 65535, 65536, Nn - 257, Nn - 1], device="cuda")
    want, bound = R.adapters(x, wt[cols], ids - (n - 2), a[n - 2:], b[n - 2:][:, cols], None)
    assert bool(((y[:, cols].double() - want).abs() <= bound).all())


@pytest.mark.parametrize("M", [6, 500, 3000])
def test_captured_and_replayed_beside_eager_calls(M):
    x, wt, ids, a, b, sc = _data(M, 1024, 2048, 9, 24, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        AD.linear_adapters(x, wt, ids, a, b, sc)
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        y = AD.linear_adapters(x, wt, ids, a, b, sc)
    torch.cuda.synchronize()
    for seed in (6, 7, 8):
        x2, _, ids2, a2, b2, sc2 = _data(M, 1024, 2048, 9, 24, seed)
        x.copy_(x2), ids.copy_(ids2), a.copy_(a2), b.copy_(b2), sc.copy_(sc2)
        torch.cuda.synchronize()
        graph.replay()
        y2 = AD.linear_adapters(x2, wt, ids2, a2, b2, sc2)
        torch.cuda.synchronize()
        assert torch.equal(y, y2)
    assert G.gemm_status().code == 0


def test_many_calls_in_a_row_give_the_same_bits():
    """Back-to-back launches overlap at their ends; every one sees its own V, lists and flags."""
    sets = [_data(m, 520, 1032, 20, 16, 30 + i) for i, m in enumerate((1, 64, 128, 129, 600, 1500))]
    want = [AD.linear_adapters(*s) for s in sets]
    torch.cuda.synchronize()
    got = [(i % 6, AD.linear_adapters(*sets[i % 6])) for i in range(60)]
    assert all(torch.equal(y, want[i]) for i, y in got)
    assert G.gemm_status().code == 0


@pytest.mark.parametrize("which", ["few rows", "tiles", "gated", "NVFP4"])
def test_the_first_cuda_call_of_a_thread(which):
    """A new thread has no context of its own yet when the tensor maps are made."""
    import threading

    from fp4_all_reduce_b200.ops import ffn

    s = _data(40 if which == "few rows" else 700, 256, 512, 3, 16, 8)
    call = {"gated": lambda: ffn.gated_linear(s[0], s[1]), "NVFP4": lambda: G.gemm_nvfp4(s[0], s[1], 1.0)}.get(which, lambda: AD.linear_adapters(*s))
    want = call()
    del want                                        # (its memory serves the thread's call: nothing there but the launch needs CUDA)
    want, got = call(), []
    spare = call()
    del spare

    def work():
        try:
            got.append(call())
        except Exception as e:
            got.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert torch.is_tensor(got[0]) and torch.equal(got[0], want), got


def test_two_threads_on_one_stream():
    """Launches of two threads interleave on their common stream; the last two shapes cut K loops, whose slots they share."""
    import threading

    from fp4_all_reduce_b200.ops import ffn

    sets = [_data(m, k, nn, n, 16, 40 + i) for i, (m, k, nn, n) in enumerate(((64, 512, 1032, 9), (600, 512, 1032, 9), (600, 8192, 2048, 3), (1100, 6144, 4096, 5)))]
    gate = [s[1].repeat(2, 1) for s in sets]
    want = [AD.linear_adapters(*s) for s in sets]
    want_h = [ffn.gated_linear(s[0], g) for s, g in zip(sets, gate)]
    torch.cuda.synchronize()
    bad = []

    def work(seed):
        try:
            for i in range(40):
                j = (i * 7 + seed) % 4
                y, h = AD.linear_adapters(*sets[j]), ffn.gated_linear(sets[j][0], gate[j])
                if not (torch.equal(y, want[j]) and torch.equal(h, want_h[j])):
                    bad.append((seed, i, j))
        except Exception as e:
            bad.append((seed, e))

    threads = [threading.Thread(target=work, args=(s,)) for s in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad and G.gemm_status().code == 0, bad


def test_refusals():
    x, wt, ids, a, b, sc = _data(4, 16, 24, 3, 8)
    ok = dict(x=x, wt=wt, ids=ids, a=a, b=b, scales=sc)
    for name, bad, why in (("x", x.half(), "x must be torch.bfloat16"), ("x", x[:, :8], "wt must have shape"), ("x", x.t().contiguous().t(), "contiguous"),
                           ("wt", wt[:20], "multiples of 8"), ("wt", wt.cpu(), "CUDA"), ("ids", ids.long(), "ids must be torch.int32"),
                           ("ids", ids[:3], "ids must have shape"), ("ids", ids.cpu(), "CUDA"), ("ids", ids.repeat(2)[::2], "contiguous"),
                           ("a", a[:, :, :8], "a must have shape"), ("a", a[:, :4], "multiple of 8"), ("a", a[:0], "at least one"),
                           ("a", a.float(), "a must be"), ("b", b[:2], "b must have shape"), ("b", b[:, :, :4], "b must have shape"),
                           ("b", b.transpose(1, 2).contiguous().transpose(1, 2), "b must be contiguous"), ("scales", sc.half(), "scales must be torch.float32"),
                           ("scales", sc[:2], "scales must have shape"), ("scales", sc.cpu(), "CUDA")):
        with pytest.raises(ValueError, match=why):
            AD.linear_adapters(**{**ok, name: bad})
    with pytest.raises(ValueError, match="up to 128"):
        AD.linear_adapters(x, wt, ids, torch.zeros(3, 136, 16, device="cuda", dtype=torch.bfloat16),
                           torch.zeros(3, 24, 136, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="out must have shape"):
        AD.linear_adapters(**ok, out=x)
    with pytest.raises(ValueError, match="overlap b"):
        AD.linear_adapters(**ok, out=b.view(-1)[:96].view(4, 24))
    with pytest.raises(RuntimeError, match="no backward pass"):
        AD.linear_adapters(**{**ok, "a": a.clone().requires_grad_()})
    with torch.no_grad():
        AD.linear_adapters(**{**ok, "a": a.clone().requires_grad_()})
