"""The feed-forward half of a tensor-parallel layer, as cases that can be timed and compared on one B200.

A case is a dict of plain values; `op` names what is run:

* `gated`      `ops.ffn.gated_linear` under inference: act(x Wg^T) * (x Wu^T), the column-parallel projections of a gated
               feed-forward block (their output is the input of the row-parallel linear).
* `train`      the same with gradients: the forward pass and the gradients of x and of the weights.
* `adapters`   `ops.adapters.linear_adapters`: the row-parallel linear whose rows belong to requests with low-rank adapters of
               their own.

Row counts run from one token to 8192-token chunks, K of the gated projections is the hidden size (6144) or a smaller layer's,
F is an intermediate width over the tensor-parallel degree, K of the row-parallel linear likewise.

`own` selects what `run` computes with: the plain form (torch products and elementwise operations in 32 bits, one rounding at
the end) or the framework's operators.
"""
from __future__ import annotations

import math

import torch

own = False

HIDDEN = 6144
ACTS = ["silu", "gelu", "gelu_tanh"]          # in the order of _native.ACT_SILU, ACT_GELU, ACT_GELU_TANH
MAX_FLOPS = 4 * 4096 * HIDDEN * 8192          # of the largest listed case


def listed() -> list[dict]:
    return [
        # One token of one sequence: the weights are read once, latency counts.
        {"name": "gated_1", "op": "gated", "rows": 1, "k": 6144, "f": 2048, "act": "silu"},
        # A decode step of 48 sequences.
        {"name": "gated_48", "op": "gated", "rows": 48, "k": 6144, "f": 2048, "act": "silu"},
        # A ragged chunk, a width that no tile divides, the other activation.
        {"name": "gated_1031_f1368", "op": "gated", "rows": 1031, "k": 6144, "f": 1368, "act": "gelu_tanh"},
        # A prefill chunk with a whole layer's width on one GPU: the largest.
        {"name": "gated_4096_f8192", "op": "gated", "rows": 4096, "k": 6144, "f": 8192, "act": "silu"},
        # A small training step: launches and the host path.
        {"name": "train_64_k1024", "op": "train", "rows": 64, "k": 1024, "f": 1024, "act": "silu"},
        # A ragged micro-batch of a smaller layer, exact GELU.
        {"name": "train_333_k2048", "op": "train", "rows": 333, "k": 2048, "f": 2056, "act": "gelu"},
        # One sequence of 2048 tokens per step, one rank's share of the width.
        {"name": "train_2048", "op": "train", "rows": 2048, "k": 6144, "f": 2048, "act": "silu"},
        # One token of one request with an adapter.
        {"name": "adapters_1", "op": "adapters", "rows": 1, "k": 2048, "n": 6144, "rank": 16, "pool": 8, "requests": 1},
        # A decode step of 64 requests over 48 adapters, every eighth request without one.
        {"name": "adapters_64", "op": "adapters", "rows": 64, "k": 2048, "n": 6144, "rank": 16, "pool": 48, "requests": 64},
        # Eleven requests of odd lengths in one chunk, K that no tile divides.
        {"name": "adapters_1031_k1992", "op": "adapters", "rows": 1031, "k": 1992, "n": 6144, "rank": 32, "pool": 16, "requests": 11},
        # A prefill chunk of a few long requests.
        {"name": "adapters_4096", "op": "adapters", "rows": 4096, "k": 2048, "n": 6144, "rank": 16, "pool": 8, "requests": 6},
        # The largest chunk and the largest rank, the whole layer's width on one GPU.
        {"name": "adapters_8192_k8192", "op": "adapters", "rows": 8192, "k": 8192, "n": 6144, "rank": 64, "pool": 16, "requests": 16},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng) -> dict:
    """Any row count from 1 up, widths that are multiples of 8, all activations, ranks from 8 to 64, any mix of requests."""
    op = rng.choice(["gated", "train", "adapters"])
    while True:
        rows, k = _log_int(rng, 1, 8192), 8 * _log_int(rng, 64, 1024)
        if op == "adapters":
            c = {"op": op, "rows": rows, "k": k, "n": rng.choice([HIDDEN, 8 * _log_int(rng, 64, 1024)]),
                 "rank": rng.choice([8, 16, 24, 32, 64]), "pool": _log_int(rng, 1, 64), "requests": _log_int(rng, 1, min(rows, 256))}
        else:
            c = {"op": op, "rows": rows, "k": k, "f": 8 * _log_int(rng, 32, 1024), "act": rng.choice(ACTS)}
        if work(c)["flops"] <= MAX_FLOPS:
            return c


def _used(case: dict) -> tuple[int, int]:
    """(adapters in use, requests that have one): request r has adapter r modulo the pool, every eighth request none."""
    with_one = [r for r in range(case["requests"]) if r % 8 != 7]
    return len({r % case["pool"] for r in with_one}), len(with_one)


def work(case: dict) -> dict:
    """Inputs read once, outputs written once; of the adapters, those that are in use."""
    rows, k = case["rows"], case["k"]
    if case["op"] == "adapters":
        n, rank = case["n"], case["rank"]
        used, with_one = _used(case)
        return {"bytes": 2 * (rows * k + n * k + rows * n + used * rank * (k + n)) + 4 * rows,
                "flops": 2 * rows * n * k + 2 * rows * with_one // case["requests"] * rank * (k + n)}
    f = case["f"]
    if case["op"] == "gated":
        return {"bytes": 2 * (rows * k + 2 * f * k + rows * f), "flops": 4 * rows * f * k}
    return {"bytes": 2 * 2 * (rows * k + 2 * f * k + rows * f), "flops": 12 * rows * f * k}


def _requests(case: dict, g: torch.Generator) -> torch.Tensor:
    """Adapter ids of the rows: contiguous requests of random lengths, at least one row each."""
    rows, n = case["rows"], case["requests"]
    cuts = torch.randperm(rows - 1, generator=g, device="cuda")[:n - 1].sort().values + 1 if n > 1 else torch.zeros(0, dtype=torch.long, device="cuda")
    req = (torch.arange(rows, device="cuda")[:, None] >= cuts[None, :]).sum(1)
    return torch.where(req % 8 == 7, -1, req % case["pool"]).to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, rows, k = case["op"], case["rows"], case["k"]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)

    s: dict = {"case": case}
    if op == "adapters":
        n, rank, pool = case["n"], case["rank"], case["pool"]
        s["x"], s["wt"] = normal(rows, k), normal(n, k, std=k ** -0.5)
        s["ids"] = _requests(case, g)
        s["a"], s["b"] = normal(pool, rank, k, std=k ** -0.5), normal(pool, n, rank, std=0.1)
        s["scales"] = 0.5 + 1.5 * torch.rand(pool, generator=g, device="cuda")
        return s
    s["x"], s["wt"] = normal(rows, k), normal(2 * case["f"], k, std=k ** -0.5)
    if op == "train":
        s["dh"] = normal(rows, case["f"])
        s["x"].requires_grad_()
        s["wt"].requires_grad_()
    return s


def _act(t: torch.Tensor, kind: str) -> torch.Tensor:
    if kind == "silu":
        return t / (1 + torch.exp(-t))
    if kind == "gelu":
        return t * 0.5 * (1 + torch.erf(t * math.sqrt(0.5)))
    return t * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t * t * t)))


def _act_grad(t: torch.Tensor, kind: str) -> torch.Tensor:
    if kind == "silu":
        s = 1 / (1 + torch.exp(-t))
        return s * (1 + t * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(t * math.sqrt(0.5))) + t * torch.exp(-0.5 * t * t) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (t + 0.044715 * t * t * t))
    return 0.5 * (1 + th) + 0.5 * t * (1 - th * th) * c * (1 + 3 * 0.044715 * t * t)


def _run_plain(s: dict):
    case = s["case"]
    x, wt = s["x"].detach().float(), s["wt"].detach().float()
    if case["op"] == "adapters":
        y = x @ wt.t()
        ids, rank, pool = s["ids"].long(), case["rank"], case["pool"]
        a, b, sc = s["a"].float(), s["b"].float(), s["scales"]
        if case["rows"] * rank * (case["k"] + case["n"]) <= 1 << 26:       # few rows: each gathers its own adapter
            at = ids.clamp(min=0)
            v = torch.bmm(a[at], x[:, :, None]) * sc[at][:, None, None]
            y = y + torch.where(ids[:, None] >= 0, torch.bmm(b[at], v)[:, :, 0], 0.0)
        else:
            for i in range(pool):
                v = torch.where((ids == i)[:, None], x @ a[i].t() * sc[i], 0.0)
                y = y + v @ b[i].t()
        return y.to(torch.bfloat16)
    f, act = case["f"], case["act"]
    pre = x @ wt.t()
    gate, up = pre[:, :f], pre[:, f:]
    h = _act(gate, act) * up
    if case["op"] == "gated":
        return h.to(torch.bfloat16)
    dh = s["dh"].float()
    dpre = torch.cat([dh * up * _act_grad(gate, act), dh * _act(gate, act)], dim=1)
    return h.to(torch.bfloat16), (dpre @ wt).to(torch.bfloat16), (dpre.t() @ x).to(torch.bfloat16)


def run(s: dict):
    if not own:
        return _run_plain(s)
    case = s["case"]
    if case["op"] == "adapters":
        from fp4_all_reduce_b200.ops import adapters

        return adapters.linear_adapters(s["x"], s["wt"], s["ids"], s["a"], s["b"], s["scales"])
    from fp4_all_reduce_b200.ops import ffn

    h = ffn.gated_linear(s["x"], s["wt"], ACTS.index(case["act"]))
    if case["op"] == "gated":
        return h
    dx, dwt = torch.autograd.grad(h, (s["x"], s["wt"]), s["dh"])
    return h.detach(), dx, dwt


def exact(case: dict, seed: int):
    """From the definitions in 64 bits: sums over K by 64-bit products, sigmoid, the normal distribution's functions."""
    s = prepare(case, seed)
    x, wt = s["x"].detach().double(), s["wt"].detach().double()
    if case["op"] == "adapters":
        y = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=x.device)
        merged = {-1: wt}
        for a in sorted(set(s["ids"].tolist())):                  # W + s B A, one request's weights at a time
            if a >= 0:
                merged[a] = torch.addmm(wt, s["b"][a].double(), s["a"][a].double(), alpha=float(s["scales"][a].double()))
            at = (s["ids"] == a).nonzero()[:, 0]
            y[at] = x[at] @ merged.pop(a).t()
        return y
    f, kind = case["f"], case["act"]
    wg, wu = wt[:f], wt[f:]
    gate, up = x @ wg.t(), x @ wu.t()
    if kind == "silu":
        p = torch.sigmoid(gate)
        slope = p + gate * p * torch.sigmoid(-gate)
    elif kind == "gelu":
        p = torch.special.ndtr(gate)
        slope = p + gate * torch.exp(gate * gate * -0.5) * (2 * math.pi) ** -0.5
    else:
        c = (8 / math.pi) ** 0.5                                   # 0.5 (1 + tanh z) = sigmoid(2 z)
        p = torch.sigmoid(c * gate * (1 + 0.044715 * gate ** 2))
        slope = p + gate * p * (1 - p) * c * (1 + 0.134145 * gate ** 2)
    h = gate * p * up
    if case["op"] == "gated":
        return h
    dh = s["dh"].double()
    dgate, dup = dh * up * slope, dh * gate * p
    return h, dgate @ wg + dup @ wu, torch.cat([dgate.t() @ x, dup.t() @ x])
