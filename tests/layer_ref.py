"""64-bit references of the feed-forward ops with bounds of what the kernels' arithmetic may add.

Bounds: half a BF16 step is 2^-8 of a value.  An FP32 sum over K products in steps of 16 on the tensor cores is off by at most
2 (K / 16 + 1) 2^-23 of the sum of the products' magnitudes (one rounding, possibly by truncation, per step and one inside it)."""
import math

import torch

BF16 = 2.0 ** -8


def sum_error(k: int) -> float:
    return 2 * (k / 16 + 1) * 2.0 ** -23


def act(g, kind):
    if kind == 0:
        return g * torch.sigmoid(g)
    if kind == 1:
        return 0.5 * g * torch.special.erfc(-g / math.sqrt(2))      # (ndtr cancels for negative g: 0 instead of 1.1e-19 at -9)
    return g * torch.sigmoid(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))      # (1 + tanh z) / 2 without its cancellation


def act_grad(g, kind):
    g = g.detach().clone().requires_grad_()
    return torch.autograd.grad(act(g, kind).sum(), g)[0]


def gated(x, wt, kind):
    """(h, gate, up, bound of h, bounds of the projections)"""
    x, wt = x.detach().double(), wt.detach().double()
    f = wt.shape[0] // 2
    pre = x @ wt.t()
    dpre = sum_error(x.shape[1]) * (x.abs() @ wt.abs().t())
    g, u, eg, eu = pre[:, :f], pre[:, f:], dpre[:, :f], dpre[:, f:]
    h = act(g, kind) * u
    # |a'| <= 1.13 for all three; 2^-18 for the FP32 exponential and division
    return h, g, u, (BF16 + 2.0 ** -18) * h.abs() + 1.13 * eg * (u.abs() + eu) + act(g, kind).abs() * eu + 1e-30, eg, eu


def gated_grads(dh, x, wt, kind):
    """(dx, dwt, their bounds).  |a'| <= 1.13 and |a''| <= 0.8; dpre is rounded to BF16, the results too."""
    _, g, u, _, eg, eu = gated(x, wt, kind)
    x, wt, dh = x.detach().double(), wt.detach().double(), dh.double()
    dg, du = dh * u * act_grad(g, kind), dh * act(g, kind)
    dpre = torch.cat([dg, du], 1)
    small = 2.0 ** -18
    edg = dh.abs() * (0.8 * eg * (u.abs() + eu) + 1.13 * eu) + (BF16 + small) * dg.abs() + small * dh.abs() * u.abs()
    edu = dh.abs() * 1.13 * eg + (BF16 + small) * du.abs()
    e = torch.cat([edg, edu], 1) * (1 + BF16)
    m, f2 = dpre.shape
    dx, dw = dpre @ wt, dpre.t() @ x
    bx = e @ wt.abs() + sum_error(f2) * (dpre.abs() @ wt.abs()) + BF16 * dx.abs() + 1e-30
    bw = e.t() @ x.abs() + sum_error(m) * (dpre.abs().t() @ x.abs()) + BF16 * dw.abs() + 1e-30
    return dx, dw, bx, bw


def adapters(x, wt, ids, a, b, scales):
    """(y, bound): every row by itself."""
    x, wt, a, b = x.double(), wt.double(), a.double(), b.double()
    n, r, k = a.shape
    sc = torch.ones(n, dtype=torch.float64, device=x.device) if scales is None else scales.double()
    y = x @ wt.t()
    e = sum_error(k + 2 * r) * (x.abs() @ wt.abs().t())
    for j in range(n):
        at = (ids == j).nonzero()[:, 0]
        if at.numel():
            v, va = sc[j] * (x[at] @ a[j].t()), sc[j].abs() * (x[at].abs() @ a[j].abs().t())
            y[at] += v @ b[j].t()
            # V: FP32 sums of K products, one by one at the worst, then 16 bits of mantissa
            ev = (k + 4) * 2.0 ** -24 * va + 2.0 ** -16 * v.abs()
            e[at] += (ev + sum_error(k + 2 * r) * v.abs()) @ b[j].abs().t()
    return y, e + BF16 * y.abs() + 1e-30
