"""Measured cases of the block-scaled FP8 operators: values in e4m3 with one fp32 scale for each 128 values of a row
(activations) or each 128 x 128 tile (weights), the products that read them, and the same product grouped by expert.

    quant_blocks          bf16 rows -> e4m3 and a scale per row and 128 columns
    quant_weight_blocks   bf16 weights (one matrix, or one per expert) -> e4m3 and a scale per 128 x 128 tile
    silu_mul_quant_blocks bf16 gate | up rows -> silu(gate) * up -> e4m3 and a scale per row and 128 columns
    fp8_gemm_blocks       y = a w^T with both scales, bf16
    fp8_gemm_grouped      the same with rows sorted by expert and one weight matrix per expert

``run`` computes the plain form (elementary torch, 32 bits) unless ``own`` is set, which makes the framework's calls.
"""
import math
import random

import torch

own = False

FP8_MAX = 448.0
MIN_SCALE = 1.0 / (FP8_MAX * 512.0)
E4M3 = torch.float8_e4m3fn
BLOCK = 128


def listed():
    return [
        # quantisation of one token's hidden row before a projection (decode, or a conditioning token)
        {"name": "quant, one token", "op": "quant", "rows": 1, "k": 5120},
        # one rank's rows of the 124,992-token video sequence at two ranks
        {"name": "quant, 62,496 tokens", "op": "quant", "rows": 62_496, "k": 5120},
        # the qkv projection's weight, quantised when a model is loaded
        {"name": "weight quant, qkv", "op": "weight_quant", "experts": 1, "n": 15_360, "k": 5120},
        # sixteen experts whose width is no multiple of the tile
        {"name": "weight quant, 16 experts", "op": "weight_quant", "experts": 16, "n": 1544, "k": 5120},
        # the FFN's activation for a handful of tokens
        {"name": "silu-mul quant, 17 tokens", "op": "silu", "rows": 17, "k": 13_824},
        # the FFN's activation for one rank's rows at four ranks
        {"name": "silu-mul quant, 31,248 tokens", "op": "silu", "rows": 31_248, "k": 13_824},
        # one token through the qkv projection: the weight is read once for one row
        {"name": "product, one token", "op": "gemm", "rows": 1, "n": 15_360, "k": 5120},
        # a ragged number of text rows through the FFN's second projection
        {"name": "product, 777 rows", "op": "gemm", "rows": 777, "n": 5120, "k": 13_824},
        # the qkv projection of one rank's rows at two ranks
        {"name": "product, 62,496 rows", "op": "gemm", "rows": 62_496, "n": 15_360, "k": 5120},
        # a decode step of a mixture of experts: 48 routed rows over 64 experts, many without a row
        {"name": "grouped, 48 rows, 64 experts", "op": "grouped", "rows": 48, "experts": 64, "n": 4096, "k": 5120,
         "split": 1},
        # a short prompt: ragged groups of about a tile, expert width no multiple of the tile
        {"name": "grouped, 4,111 rows, 32 experts", "op": "grouped", "rows": 4111, "experts": 32, "n": 1544, "k": 5120,
         "split": 2},
        # one rank's rows at four ranks over few wide experts
        {"name": "grouped, 31,248 rows, 16 experts", "op": "grouped", "rows": 31_248, "experts": 16, "n": 10_240,
         "k": 5120, "split": 3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "weight_quant", "silu", "gemm", "gemm", "grouped", "grouped"])
    k = 16 * _log(rng, 16, 864)
    if op == "quant":
        return {"op": op, "rows": min(_log(rng, 1, 62_496), 62_496 * 5120 // k), "k": k}
    if op == "weight_quant":
        e = _log(rng, 1, 32)
        return {"op": op, "experts": e, "n": max(1, min(_log(rng, 64, 27_648), 120_000_000 // (e * k))), "k": k}
    if op == "silu":
        return {"op": op, "rows": min(_log(rng, 1, 31_248), 31_248 * 13_824 // k), "k": k}
    n = _log(rng, 64, 27_648)
    if op == "gemm":
        rows = min(_log(rng, 1, 62_496), 62_496 * 15_360 // n, 62_496 * 15_360 * 5120 // (n * k))
        return {"op": op, "rows": max(1, rows), "n": n, "k": k}
    e = _log(rng, 2, 128)
    n = max(1, min(n, 64 * 4096 * 5120 // (e * k)))
    rows = min(_log(rng, 1, 31_248), 31_248 * 10_240 // n, 31_248 * 10_240 * 5120 // (n * k))
    return {"op": op, "rows": max(1, rows), "experts": e, "n": n, "k": k, "split": rng.randrange(1 << 20)}


def _groups(case):
    """Rows of each expert: independent choices with uneven popularity, as a router makes them."""
    r = random.Random(case["split"])
    popular = [math.exp(r.gauss(0.0, 0.7)) for _ in range(case["experts"])]
    sizes = [0] * case["experts"]
    for e in r.choices(range(case["experts"]), popular, k=case["rows"]):
        sizes[e] += 1
    return sizes


def _blocks(n):
    return -(-n // BLOCK)


def _row_scales(rows, k, device):
    """A [rows, k / 128] scale tensor whose columns lie one after the other, as the products read them."""
    return torch.empty_strided((rows, _blocks(k)), (1, -(-rows // 4) * 4), dtype=torch.float32, device=device)


def _plain_quant(x):
    """x [rows, k] fp32 -> (e4m3 [rows, k], scale [rows, k / 128])."""
    rows, k = x.shape
    b = torch.nn.functional.pad(x, (0, _blocks(k) * BLOCK - k)).view(rows, -1, BLOCK)
    scale = (b.abs().amax(dim=2) / FP8_MAX).clamp_min(MIN_SCALE)
    q = (b * (1.0 / scale)[:, :, None]).clamp(-FP8_MAX, FP8_MAX).view(rows, -1)[:, :k]
    return q.to(E4M3), scale


def _plain_weight_quant(w):
    """w [experts, n, k] fp32 -> (e4m3 [experts, n, k], scale [experts, n / 128, k / 128])."""
    e, n, k = w.shape
    b = torch.nn.functional.pad(w, (0, _blocks(k) * BLOCK - k, 0, _blocks(n) * BLOCK - n))
    b = b.view(e, _blocks(n), BLOCK, _blocks(k), BLOCK)
    scale = (b.abs().amax(dim=(2, 4)) / FP8_MAX).clamp_min(MIN_SCALE)
    q = (b * (1.0 / scale)[:, :, None, :, None]).clamp(-FP8_MAX, FP8_MAX)
    return q.view(e, _blocks(n) * BLOCK, -1)[:, :n, :k].to(E4M3), scale


def _activations(rows, k, g):
    """Hidden rows with a few channels much larger than the others."""
    x = torch.randn(rows, k, generator=g, device="cuda")
    return x.mul_((torch.randn(k, generator=g, device="cuda") * 0.8).exp())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, k = case["op"], case["k"]
    if op == "quant":
        return {"op": op, "x": _activations(case["rows"], k, g).to(torch.bfloat16)}
    if op == "weight_quant":
        shape = (case["experts"], case["n"], k)
        w = (torch.randn(shape, generator=g, device="cuda") * 0.02).to(torch.bfloat16)
        return {"op": op, "w": w if case["experts"] > 1 else w[0]}
    if op == "silu":
        x = torch.randn(case["rows"], 2 * k, generator=g, device="cuda", dtype=torch.bfloat16)
        return {"op": op, "x": x.mul_(1.5)}
    a, s = _plain_quant(_activations(case["rows"], k, g))
    state = {"op": op, "a": a.contiguous(), "sa": _row_scales(case["rows"], k, "cuda").copy_(s)}
    experts = case.get("experts", 1)
    w = torch.randn(experts, case["n"], k, generator=g, device="cuda") * 0.02
    w, s = _plain_weight_quant(w)
    state["w"], state["sb"] = w.contiguous(), s.contiguous()
    if op == "gemm":
        state["w"], state["sb"] = state["w"][0], state["sb"][0]
        return state
    sizes = _groups(case)
    ends = [0]
    for m in sizes:
        ends.append(ends[-1] + m)
    state["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    state["most"] = max(sizes)
    return state


def _rows_f32(a, sa):
    return a.float() * sa.repeat_interleave(BLOCK, dim=1)[:, :a.shape[1]]


def _weights_f32(w, sb):
    s = sb.repeat_interleave(BLOCK, dim=-2)[..., :w.shape[-2], :]
    return w.float() * s.repeat_interleave(BLOCK, dim=-1)[..., :w.shape[-1]]


def _plain(state):
    op = state["op"]
    if op == "quant":
        return _plain_quant(state["x"].float())
    if op == "weight_quant":
        w = state["w"].float()
        q, s = _plain_weight_quant(w if w.dim() == 3 else w[None])
        return (q, s) if w.dim() == 3 else (q[0], s[0])
    if op == "silu":
        gate, up = state["x"].float().chunk(2, dim=1)
        return _plain_quant(gate / (1.0 + torch.exp(-gate)) * up)
    a, w = _rows_f32(state["a"], state["sa"]), _weights_f32(state["w"], state["sb"])
    if op == "gemm":
        return (a @ w.t()).to(torch.bfloat16)
    # every group padded to the longest one, one batched product, and the rows taken back out of it
    first, end = state["offsets"][:-1].long(), state["offsets"][1:].long()
    at = first[:, None] + torch.arange(state["most"], device=a.device)
    y = torch.bmm(a[at.clamp_max(a.shape[0] - 1)], w.transpose(1, 2))
    row = torch.arange(a.shape[0], device=a.device)
    expert = (row[:, None] >= end[None, :]).sum(dim=1)
    return y[expert, row - first[expert]].to(torch.bfloat16)


def _framework(state):
    import sys

    package = "minimax-h3-2x-dgx-spark-tp2_b200"
    if package not in sys.path:
        sys.path.insert(0, package)
    from h3b import ops

    op = state["op"]
    if op == "quant":
        return ops.quant_blocks(state["x"])
    if op == "weight_quant":
        return ops.quant_weight_blocks(state["w"])
    if op == "silu":
        return ops.silu_mul_quant_blocks(state["x"])
    if op == "gemm":
        return ops.fp8_gemm_blocks(state["a"], state["w"], state["sa"], state["sb"])
    return ops.fp8_gemm_grouped(state["a"], state["w"], state["sa"], state["sb"], state["offsets"])


def run(state):
    if own:
        return _framework(state)
    return _plain(state)


def work(case):
    op, k, kb = case["op"], case["k"], _blocks(case["k"])
    if op in ("quant", "silu"):
        read = 2 if op == "quant" else 4
        return {"bytes": case["rows"] * ((read + 1) * k + 4 * kb), "flops": (4 if op == "quant" else 8) * case["rows"] * k}
    n, nb = case["n"], _blocks(case["n"])
    if op == "weight_quant":
        return {"bytes": case["experts"] * (3 * n * k + 4 * nb * kb), "flops": 4 * case["experts"] * n * k}
    used = 1 if op == "gemm" else sum(m > 0 for m in _groups(case))
    rows = case["rows"]
    offsets = 0 if op == "gemm" else 4 * (case["experts"] + 1)
    return {"bytes": rows * (k + 4 * kb + 2 * n) + used * (n * k + 4 * nb * kb) + offsets, "flops": 2 * rows * n * k}


def _round_e4m3(x):
    """The nearest e4m3 value (ties to even) of each 64-bit value of at most 448, computed on the exponents."""
    _, e = torch.frexp(x)
    step = torch.exp2((e.double() - 4).clamp_min(-9.0))
    return torch.round(x / step) * step


def exact(case, seed):
    state = prepare(case, seed)
    op = state["op"]
    if op in ("quant", "silu"):
        x = state["x"].double()
        if op == "silu":
            half = x.shape[1] // 2
            x = x[:, :half] * torch.sigmoid(x[:, :half]) * x[:, half:]
        q, s = torch.empty_like(x), []
        for c in range(0, x.shape[1], BLOCK):
            part = x[:, c:c + BLOCK]
            s.append((part.abs().max(dim=1).values / FP8_MAX).clamp_min(MIN_SCALE))
            q[:, c:c + BLOCK] = _round_e4m3(part / s[-1][:, None])
        return q, torch.stack(s, dim=1)
    if op == "weight_quant":
        w = state["w"].double()
        three = w if w.dim() == 3 else w[None]
        q = torch.empty_like(three)
        s = torch.empty(three.shape[0], _blocks(w.shape[-2]), _blocks(w.shape[-1]), dtype=torch.float64, device=w.device)
        for j in range(s.shape[2]):
            cols = slice(BLOCK * j, BLOCK * (j + 1))
            for i in range(s.shape[1]):
                rows = slice(BLOCK * i, BLOCK * (i + 1))
                part = three[:, rows, cols]
                s[:, i, j] = (part.abs().amax(dim=(1, 2)) / FP8_MAX).clamp_min(MIN_SCALE)
                q[:, rows, cols] = _round_e4m3(part / s[:, i, j, None, None])
        return (q, s) if w.dim() == 3 else (q[0], s[0])
    n, k = state["w"].shape[-2:]
    row_block = torch.arange(n, device="cuda") // BLOCK
    col_block = torch.arange(k, device="cuda") // BLOCK
    a = state["a"].double().mul_(state["sa"].double()[:, col_block])
    if op == "gemm":
        return a @ state["w"].double().mul_(state["sb"].double()[row_block][:, col_block]).t()
    y = torch.empty(a.shape[0], n, dtype=torch.float64, device="cuda")
    ends = state["offsets"].tolist()
    for e in range(len(ends) - 1):
        if ends[e + 1] > ends[e]:
            w = state["w"][e].double().mul_(state["sb"][e].double()[row_block][:, col_block])
            y[ends[e]:ends[e + 1]] = a[ends[e]:ends[e + 1]] @ w.t()
    return y
