"""Host side of the feed-forward ops without a GPU: refusals of the front end and of the C interface, shapes of the fake kernels."""
import ctypes as C

import pytest
import torch

from fp4_all_reduce_b200 import _native as N


@pytest.fixture(scope="module")
def ops(cuda_lib):
    from fp4_all_reduce_b200.ops import adapters, allreduce, ffn

    try:
        N.front()
    except RuntimeError as e:
        pytest.skip(str(e))
    return ffn, adapters, allreduce


def _bf16(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def test_cpu_tensors_and_shapes_are_refused_by_name(ops):
    ffn, adapters, _ = ops
    x, wt = _bf16(4, 16), _bf16(16, 16)
    for args, why in (((x, wt), "x must be a CUDA tensor"), ((x.float(), wt), "x must be torch.bfloat16, got torch.float32"),
                      ((_bf16(4, 12), _bf16(16, 12)), "K must be a positive multiple of 8, got 12"), ((x, _bf16(16, 8)), r"wt must have shape \[2 F, 16\]"),
                      ((x, _bf16(24, 16)), "F a positive multiple of 8, got 24 rows"), ((x, _bf16(0, 16)), "got 0 rows"), ((_bf16(4), wt), "x must have shape"),
                      ((x, wt, 9), "activation must be 0")):
        with pytest.raises(ValueError, match=why):
            ffn.gated_linear(*args)
    with pytest.raises(ValueError, match="x must be a CUDA tensor"):
        ffn.gated_linear(x.requires_grad_(), wt)
    x = _bf16(4, 16)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ffn.gated_linear_backward(_bf16(4, 8), torch.zeros(4, 16), x, wt)
    ids, a, b = torch.zeros(4, dtype=torch.int32), _bf16(2, 8, 16), _bf16(2, 16, 8)
    for args, why in (((x, wt, ids, a, b), "x must be a CUDA tensor"), ((x, wt, ids, _bf16(2, 12, 16), b), "multiple of 8 up to 128"),
                      ((x, wt, ids, _bf16(0, 8, 16), b), "at least one adapter"), ((x, _bf16(12, 16), ids, a, b), "positive multiples of 8"),
                      ((x, wt, ids, _bf16(2, 8, 8), b), "a must have shape")):
        with pytest.raises(ValueError, match=why):
            adapters.linear_adapters(*args)
    with pytest.raises(TypeError, match="ids must be a tensor"):
        adapters.linear_adapters(x, wt, [0] * 4, a, b)


def test_the_c_interface_checks_before_it_launches(cuda_lib):
    lib = cuda_lib
    p = C.c_void_p(4096)
    assert lib.fp4ar_gated_linear(p, p, 4, 8, 12, 0, p, None, None) == 1            # K
    assert lib.fp4ar_gated_linear(p, p, 4, 12, 16, 0, p, None, None) == 1           # F
    assert lib.fp4ar_gated_linear(p, p, -1, 8, 16, 0, p, None, None) == 1
    assert lib.fp4ar_gated_linear(p, p, 4, 8, 16, 3, p, None, None) == 1            # activation
    assert lib.fp4ar_gated_linear(p, None, 4, 8, 16, 0, p, None, None) == 1
    assert lib.fp4ar_gated_linear(p, C.c_void_p(4104), 4, 8, 16, 0, p, None, None) == 1      # alignment
    assert lib.fp4ar_gated_linear(None, None, 0, 8, 16, 0, None, None, None) == 0   # no rows: nothing to do
    assert lib.fp4ar_gated_linear(p, p, 4, 1 << 30, 16, 0, p, None, None) == 1      # 2 F beyond 32 bits
    assert lib.fp4ar_gated_backward(p, p, p, None, 4, 8, 16, 0, p, p, None, None) == 1       # dx needs wt
    assert lib.fp4ar_gated_backward(p, p, None, p, 4, 8, 16, 0, p, None, p, None) == 1       # dwt needs x
    assert lib.fp4ar_linear_adapters(p, p, p, p, p, None, 4, 16, 16, 136, 2, p, p, None) == 1      # rank
    assert lib.fp4ar_linear_adapters(p, p, p, p, p, None, 4, 16, 16, 8, 0, p, p, None) == 1        # no adapter
    assert lib.fp4ar_linear_adapters(p, p, None, p, p, None, 4, 16, 16, 8, 2, p, p, None) == 1
    assert lib.fp4ar_linear_adapters(p, p, p, p, p, None, 4, 16, 16, 8, 2, None, p, None) == 1     # workspace
    assert lib.fp4ar_linear_adapters(p, p, p, p, p, None, 4, 8192, 16, 8, 1 << 18, p, p, None) == 1   # adapters x N beyond 32 bits
    assert lib.fp4ar_linear_adapters(p, p, p, p, p, None, 4, 8, 8, 128, 1 << 25, p, p, None) == 1     # adapters x R beyond 32 bits
    assert lib.fp4ar_linear_adapters(None, None, None, None, None, None, 0, 16, 16, 8, 2, None, None, None) == 0
    # the workspace holds V (two BF16 halves per rank, ranks in blocks of 32) and a list of up to 256 adapters per 256 rows
    assert lib.fp4ar_adapters_workspace(1000, 40, 7) >= 1000 * 64 * 4 + 4 * 257 * 4
    assert lib.fp4ar_adapters_workspace(-1, 8, 1) == 0


def test_fake_kernels(ops):
    m = torch.device("meta")
    x, wt = torch.empty(5, 16, dtype=torch.bfloat16, device=m), torch.empty(48, 16, dtype=torch.bfloat16, device=m)
    h, pre = torch.ops.fp4ar.gated_linear_pre(x, wt, 0)
    assert h.shape == (5, 24) and h.dtype == torch.bfloat16 and pre.shape == (5, 48) and pre.dtype == torch.float32
    assert torch.ops.fp4ar.gated_linear(x, wt, 0).shape == (5, 24)
    dx, dw = torch.ops.fp4ar.gated_linear_backward(h, pre, x, wt, 0, True, False)
    assert dx.shape == x.shape and dw.shape == (0,)
    y = torch.ops.fp4ar.linear_adapters(x, wt, torch.empty(5, dtype=torch.int32, device=m), torch.empty(2, 8, 16, dtype=torch.bfloat16, device=m),
                                        torch.empty(2, 48, 8, dtype=torch.bfloat16, device=m), None)
    assert y.shape == (5, 48) and y.dtype == torch.bfloat16
