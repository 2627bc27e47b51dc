"""The measured cases of the orthogonalised optimiser update and the grouped expert products.

Three operators, as a training or serving program calls them:

* ``orth``: ``orthogonalize(x)``, the Newton-Schulz approximation of the polar factor of each
  matrix of a batch: ``X = x / (||x||_F + eps)``, then five times
  ``X <- a X + (b A + c A^2) X`` with ``A = X X^T`` (or the same from the right);
* ``muon``: ``muon_update_(param, grad, momentum, ...)``, the optimiser step around it: the
  momentum average, the orthogonalised direction, the weights;
* ``grouped``: ``grouped_matmul(x, w, offsets)``, rows sorted by expert times their expert's
  matrix, alone (serving) or with both gradients (training).

With ``own`` false, ``run`` computes them from elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
COEFFS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7
LR, BETA, DECAY = 0.02, 0.95, 0.1
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # many small matrices (attention heads or blocks treated apart): latency and HBM
        dict(name="orth_b1024n64", op="orth", batch=1024, m=64, n=64, type="bf16"),
        # the smallest call: a single small matrix, launch latency only
        dict(name="orth_b1n128", op="orth", batch=1, m=128, n=128, type="bf16"),
        # a block-partitioned update, one tile per matrix
        dict(name="orth_b64n256", op="orth", batch=64, m=256, n=256, type="bf16"),
        # the same at full throughput
        dict(name="orth_b640n512", op="orth", batch=640, m=512, n=512, type="bf16"),
        # 32-bit matrices of odd sizes, taller than wide
        dict(name="orth_fp32_b3_1001x601", op="orth", batch=3, m=1001, n=601, type="fp32"),
        # one large projection's step, bf16 weights and a 32-bit momentum
        dict(name="muon_4096x4096", op="muon", batch=1, m=4096, n=4096, type="bf16"),
        # the experts' up projections of one layer in a single call
        dict(name="muon_e16_1024x2048", op="muon", batch=16, m=1024, n=2048, type="bf16"),
        # 32-bit weights of a small layer
        dict(name="muon_fp32_512x128", op="muon", batch=1, m=512, n=128, type="fp32"),
        # serving, a few tokens spread over many experts: reading the weights is all there is
        dict(name="grouped_decode_t48", op="grouped", rows=48, tail=0, experts=32, k=1024, n=2048, empty=0,
             transposed=False, train=False, type="bf16"),
        # serving a prompt batch, weights stored (out, in), the last rows padding
        dict(name="grouped_prefill_t8192", op="grouped", rows=8192, tail=300, experts=16, k=2048, n=1024, empty=1,
             transposed=True, train=False, type="bf16"),
        # a training step's expert products, forward and both gradients
        dict(name="grouped_train_t16384", op="grouped", rows=16384, tail=0, experts=16, k=2048, n=4096, empty=0,
             transposed=False, train=True, type="bf16"),
        # the same at odd sizes with experts that got nothing
        dict(name="grouped_train_odd", op="grouped", rows=1777, tail=5, experts=9, k=520, n=779, empty=3,
             transposed=False, train=True, type="fp16"),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["orth", "muon", "grouped"])
    if op == "grouped":
        train = rng.random() < 0.6
        case = dict(op=op, rows=_spread(rng, 1, 16384), tail=rng.choice([0, 0, 1, 77]), experts=_spread(rng, 1, 64),
                    k=_spread(rng, 64, 4096), n=_spread(rng, 64, 4096), empty=0, transposed=rng.random() < 0.5,
                    train=train, type=rng.choice(["bf16", "bf16", "fp16"]))
        case["empty"] = rng.randrange(case["experts"]) // 2
        if rng.random() < 0.6:  # most models' widths are multiples of 8
            case["k"], case["n"] = case["k"] // 8 * 8, case["n"] // 8 * 8
        most = 8.2e11
        while work(case)["flops"] > most or work(case)["bytes"] > 1.2e9:
            case["rows"], case["k"] = max(1, case["rows"] // 2), max(64, case["k"] * 3 // 4)
        return case
    kind = rng.choice(["bf16", "bf16", "fp32"])
    case = dict(op=op, batch=_spread(rng, 1, 640 if op == "orth" else 16), m=_spread(rng, 32, 4096),
                n=_spread(rng, 32, 4096), type=kind)
    most = 1.3e12 if kind == "bf16" else 2e11
    while work(case)["flops"] > most:
        if case["batch"] > 1:
            case["batch"] = case["batch"] // 2
        else:
            case["m"], case["n"] = max(32, case["m"] * 3 // 4), max(32, case["n"] * 3 // 4)
    return case


def _randn(seed, *shape):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(*shape, device=DEV, generator=g)


def _gradients(seed, batch, m, n):
    """Noise with a few stronger directions, at the scale of a gradient."""
    rank = min(4, m, n)
    noise = _randn(seed, batch, m, n)
    strong = _randn(seed + 1, batch, m, rank) @ _randn(seed + 2, batch, rank, n)
    return (noise + strong * (0.5 / math.sqrt(rank))) * 1e-3


def _counts(rows, experts, empty, seed):
    """How many rows each expert gets: uneven, `empty` of the experts none (host numbers)."""
    g = torch.Generator().manual_seed(seed)
    share = torch.rand(experts, generator=g) + 0.25
    share[torch.randperm(experts, generator=g)[:empty]] = 0
    ends = torch.cumsum(share, 0) / share.sum() * rows
    return torch.diff(ends.round().long(), prepend=torch.zeros(1, dtype=torch.long)).tolist()


def prepare(case, seed):
    kind = TYPES[case["type"]]
    seed = seed * 16
    if case["op"] == "orth":
        return {"op": "orth", "x": _gradients(seed, case["batch"], case["m"], case["n"]).to(kind)}
    if case["op"] == "muon":
        b, m, n = case["batch"], case["m"], case["n"]
        return {"op": "muon", "grad": _gradients(seed, b, m, n).to(kind), "momentum": _gradients(seed + 4, b, m, n),
                "param": (_randn(seed + 8, b, m, n) / math.sqrt(n)).to(kind)}
    t, e, k, n = case["rows"], case["experts"], case["k"], case["n"]
    counts = _counts(t, e, case["empty"], seed)
    total = t + case["tail"]
    shape = (e, n, k) if case["transposed"] else (e, k, n)
    w = (_randn(seed, *shape) / math.sqrt(k)).to(kind)
    state = {"op": "grouped", "train": case["train"], "x": _randn(seed + 1, total, k).to(kind),
             "w": w.transpose(1, 2) if case["transposed"] else w,
             "offsets": torch.tensor([0] + counts, device=DEV).cumsum(0).to(torch.int32),
             "most": max(counts + [case["tail"]])}  # the capacity of a program that pads
    if case["train"]:
        state["dy"] = _randn(seed + 2, total, n).to(kind)
        state["x"].requires_grad_()
        state["w"] = state["w"].requires_grad_()
    return state


def _newton_schulz(x):
    """Five steps in 32 bits; the smaller side carries the Gram matrix."""
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    a, b, c = COEFFS
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(STEPS):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


def _scale(m, n):
    return math.sqrt(max(1.0, m / n))


def _muon(s):
    grad, param, momentum = s["grad"].float(), s["param"], s["momentum"]
    momentum.copy_(BETA * momentum + (1 - BETA) * grad)
    o = _newton_schulz(BETA * momentum + (1 - BETA) * grad)
    param.copy_(param.float() * (1 - LR * DECAY) - LR * _scale(*param.shape[-2:]) * o)
    return {"param": param, "momentum": momentum}


def _grouped(s):
    """Every expert's rows padded to the largest group, then batched products."""
    x, w, off = s["x"].detach().float(), s["w"].detach().float(), s["offsets"].long()
    experts, total = w.shape[0], x.shape[0]
    row = torch.arange(total, device=x.device)
    expert = torch.searchsorted(off[1:], row, right=True)  # rows behind the last group: one more
    place = row - off[expert]
    padded = x.new_zeros(experts + 1, s["most"], x.shape[1])
    padded[expert, place] = x
    padded = padded[:experts]
    inside = (row < off[-1])[:, None]
    at = expert.clamp(max=experts - 1)
    kind = s["x"].dtype

    def rows_of(p):
        return torch.where(inside, p[at, torch.where(inside[:, 0], place, 0)], 0).to(kind)

    y = rows_of(padded @ w)
    if not s["train"]:
        return {"y": y}
    dy = s["dy"].float()
    padded_dy = dy.new_zeros(experts + 1, s["most"], dy.shape[1])
    padded_dy[expert, place] = dy
    padded_dy = padded_dy[:experts]
    return {"y": y, "dx": rows_of(padded_dy @ w.transpose(1, 2)),
            "dw": (padded.transpose(1, 2) @ padded_dy).to(kind)}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        if state["op"] == "orth":
            return _newton_schulz(state["x"].float()).to(state["x"].dtype)
        return _muon(state) if state["op"] == "muon" else _grouped(state)


def _own(state):
    from linalg_kernels_b200.grouped import grouped_matmul
    from linalg_kernels_b200.orthogonal import muon_update_, orthogonalize

    if state["op"] == "orth":
        return orthogonalize(state["x"], steps=STEPS, coefficients=COEFFS, eps=EPS)
    if state["op"] == "muon":
        muon_update_(state["param"], state["grad"], state["momentum"], lr=LR, beta=BETA, nesterov=True,
                     weight_decay=DECAY, steps=STEPS, coefficients=COEFFS, eps=EPS)
        return {"param": state["param"], "momentum": state["momentum"]}
    if not state["train"]:
        return {"y": grouped_matmul(state["x"], state["w"], state["offsets"])}
    y = grouped_matmul(state["x"], state["w"], state["offsets"])
    dx, dw = torch.autograd.grad(y, (state["x"], state["w"]), state["dy"])
    return {"y": y.detach(), "dx": dx, "dw": dw}


def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "grouped":
        t, e, k, n = case["rows"], case["experts"] - case["empty"], case["k"], case["n"]
        used = min(e, t)
        rows, weights = t * (k + n) * size, used * k * n * size
        if not case["train"]:
            return {"bytes": rows + weights, "flops": 2 * t * k * n}
        # x, dy, w in; y, dx, dw (every expert's) out
        return {"bytes": 2 * rows + weights + case["experts"] * k * n * size, "flops": 6 * t * k * n}
    b, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    # of the two symmetric products (the Gram matrix and its square) one half is enough
    flops = STEPS * b * (m * m * n + m ** 3 + 2 * m * m * n)
    if case["op"] == "orth":
        return {"bytes": 2 * b * m * n * size, "flops": flops}
    return {"bytes": b * m * n * (3 * size + 8), "flops": flops}


def _polar64(x):
    """The same polynomial in 64 bits, its terms nested and applied to X one Gram factor at a time."""
    x = x.double()
    x = x / (torch.linalg.vector_norm(x, dim=(-2, -1), keepdim=True) + EPS)
    a, b, c = COEFFS
    for _ in range(STEPS):
        if x.shape[-2] <= x.shape[-1]:
            gram = torch.matmul(x, x.mT)
            x = a * x + torch.matmul(gram, b * x + c * torch.matmul(gram, x))
        else:
            gram = torch.matmul(x.mT, x)
            x = a * x + torch.matmul(b * x + c * torch.matmul(x, gram), gram)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "orth":
            return _polar64(s["x"])
        if case["op"] == "muon":
            grad = s["grad"].double()
            momentum = torch.lerp(grad, s["momentum"].double(), BETA)
            o = _polar64(torch.lerp(grad, momentum, BETA))
            param = s["param"].double()
            return {"param": param - LR * (DECAY * param + _scale(case["m"], case["n"]) * o), "momentum": momentum}
        off = s["offsets"].tolist()
        x, w = s["x"].double(), s["w"]
        y = x.new_zeros(x.shape[0], w.shape[2])
        out = {"y": y}
        if case["train"]:
            dy = s["dy"].double()
            out["dx"], out["dw"] = torch.zeros_like(x), x.new_zeros(w.shape)
        for e, (i, j) in enumerate(zip(off, off[1:])):
            y[i:j] = x[i:j] @ w[e].double()
            if case["train"]:
                out["dx"][i:j] = dy[i:j] @ w[e].double().T
                out["dw"][e] = x[i:j].T @ dy[i:j]
        return out
