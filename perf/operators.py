"""The operators of a few-token pass through a model whose weights are held in few bits, as timed cases: top-k routing of
an MoE layer (forward, and with its gradient), 4-bit weights (quantising them, and products of a few rows with them), and a
whole MoE feed-forward layer for a handful of tokens.

Sizes are those of ``bench.py`` and the tests (expert shapes 1536 x 2048 and 4096 x 7168, projections 14336 x 4096,
8192 x 8192, 5760 x 2880), or generic.  Kinds of case (``"op"``):

  router   ``topk_router`` / ``topk_routing_map``: logits -> the k experts of a token and their probabilities, and back
  int4     ``gemm_int4``: rows of activations times a 4-bit weight with group scales
  quant    ``quantize_int4`` followed by ``dequantize_int4``
  moe      ``moe_few_tokens``: gate + up projection, SwiGLU, down projection and weighted sum over a token's experts
"""

import math

import torch

own = False

DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 128  # FP8 weights: one scale per 128 x 128 tile


def _router(name, tokens, experts, topk, score, bias, groups, topk_groups, normalize, scaling, dtype, dense, train):
    return {"name": name, "op": "router", "tokens": tokens, "experts": experts, "topk": topk, "score": score, "bias": bias,
            "groups": groups, "topk_groups": topk_groups, "normalize": normalize, "scaling": scaling, "dtype": dtype,
            "dense": dense, "train": train}


def _int4(name, m, n, k, group, zeros, bias=False, dtype="bf16"):
    return {"name": name, "op": "int4", "m": m, "n": n, "k": k, "group": group, "zeros": zeros, "bias": bias, "dtype": dtype}


def _quant(name, experts, n, k, group, zeros, dtype="bf16"):
    return {"name": name, "op": "quant", "experts": experts, "n": n, "k": k, "group": group, "zeros": zeros, "dtype": dtype}


def _moe(name, tokens, experts, topk, hidden, inter, weights, group=0, dtype="bf16"):
    return {"name": name, "op": "moe", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inter": inter,
            "weights": weights, "group": group, "dtype": dtype}


def listed():
    return [
        # one token of a decoding step finds its experts: the smallest call, all latency
        _router("router_token", 1, 128, 8, "softmax", False, 1, 1, True, 1.0, "bf16", False, False),
        # a training micro-batch with expert groups and a selection bias, as the dense tables that the permutation takes
        _router("router_train_groups", 16384, 256, 8, "sigmoid", True, 8, 4, True, 2.5, "fp32", True, True),
        # one token through a down projection of a dense layer
        _int4("int4_token", 1, 4096, 14336, 128, False),
        # a small ragged batch against a width that is no multiple of the tiles, small groups with zero points
        _int4("int4_ragged", 13, 5760, 2880, 32, True, bias=True, dtype="fp16"),
        # a full decoding batch, or the drafts of a speculative step, against a large square projection
        _int4("int4_batch", 64, 8192, 8192, 128, False),
        # a projection's weight packed when the model is loaded
        _quant("quant_projection", 1, 14336, 4096, 128, False),
        # the down projections of a layer's experts, small groups with zero points
        _quant("quant_experts", 64, 2048, 768, 32, True),
        # one token through a layer of many narrow experts in 4 bits: the smallest of these, latency counts
        _moe("moe_token_int4", 1, 128, 8, 2048, 768, "int4", 128),
        # one token through one rank's wide experts in FP8
        _moe("moe_token_fp8", 1, 32, 8, 7168, 2048, "fp8"),
        # a small decoding batch over many narrow experts in FP8: most experts have one to four rows
        _moe("moe_batch_fp8", 24, 128, 8, 2048, 768, "fp8"),
        # a decoding batch over wide experts in 4 bits with small groups
        _moe("moe_batch_int4", 48, 32, 6, 7168, 2048, "int4", 32),
        # a larger batch over few unquantised experts: a dozen rows each
        _moe("moe_batch_bf16", 64, 16, 4, 2880, 1440, "raw"),
    ]


def _size(rng, lo, hi, step):
    """A multiple of ``step`` in [lo, hi], even over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return int(min(hi, max(lo, round(v / step) * step)))


def draw(rng):
    op = rng.choice(["router"] * 3 + ["int4"] * 4 + ["quant"] * 2 + ["moe"] * 5)
    dtype = rng.choice(["bf16"] * 3 + ["fp16"])
    if op == "router":
        experts = _size(rng, 8, 512, 1)
        topk = rng.randint(1, min(16, experts))
        groups = topk_groups = 1
        if rng.random() < 0.4:
            groups = rng.choice([2, 4, 8])
            experts = -(-experts // (2 * groups)) * 2 * groups
            topk_groups = rng.randint(1, groups)
            topk = min(topk, experts // groups * topk_groups)
        tokens = _size(rng, 1, 16384 * 256 // max(256, experts), 1)
        normalize = topk > 1 and rng.random() < 0.7  # a single normalised probability is one, and has no gradient
        return {"op": op, "tokens": tokens, "experts": experts, "topk": topk, "score": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.4, "groups": groups, "topk_groups": topk_groups, "normalize": normalize,
                "scaling": rng.choice([1.0, 2.5]), "dtype": rng.choice(["bf16", "fp16", "fp32"]), "dense": rng.random() < 0.5,
                "train": rng.random() < 0.5}
    if op == "int4":
        m = _size(rng, 1, 64, 1)
        n, k = _size(rng, 256, 14336, rng.choice([1, 16, 64])), _size(rng, 256, 14336, rng.choice([8, 64]))
        while m * n * k > 64 * 8192 * 8192 or n * k > 14336 * 4096:
            n, k = n // 2, max(256, k // 16 * 8)
        return {"op": op, "m": m, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
                "bias": rng.random() < 0.3, "dtype": dtype}
    if op == "quant":
        experts, n, k = rng.choice([1, 1, 8, 32]), _size(rng, 64, 14336, 1), _size(rng, 256, 14336, rng.choice([8, 64]))
        while experts * n * k > 64 * 2048 * 768:
            n //= 2
        return {"op": op, "experts": experts, "n": n, "k": k, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
                "dtype": dtype}
    weights = rng.choice(["int4", "fp8", "fp8", "raw"])
    step = 16 if weights == "fp8" else 8
    experts, hidden, inter = _size(rng, 8, 128, 1), _size(rng, 512, 7168, rng.choice([step, 128])), _size(rng, 256, 2048, rng.choice([step, 128]))
    while experts * hidden * inter > 32 * 7168 * 2048 // (4 if weights == "raw" else 2):
        experts = max(4, experts // 2)
        inter = max(256, inter // 2 // step * step)
    return {"op": op, "tokens": _size(rng, 1, 64, 1), "experts": experts, "topk": rng.randint(1, min(8, experts)), "hidden": hidden,
            "inter": inter, "weights": weights, "group": rng.choice([32, 64, 128]) if weights == "int4" else 0, "dtype": dtype}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _weight4(gen, shape, group, zeros, deviation):
    """A 4-bit weight [..., N, K] as codes 0 .. 15, one bf16 scale (and one zero point) per ``group`` columns of a row."""
    dev = gen.device
    groups = (*shape[:-1], -(-shape[-1] // group))
    codes = (torch.randn(shape, generator=gen, device=dev) * 2.7 + 8).round_().clamp_(0, 15).to(torch.uint8)
    scale = ((torch.rand(groups, generator=gen, device=dev) * 0.6 + 0.7) * (deviation / 2.7)).to(torch.bfloat16)
    zero = torch.randint(6, 11, groups, generator=gen, device=dev, dtype=torch.uint8) if zeros else None
    return {"codes": codes, "scale": scale, "zero": zero, "group": group}


def _weight8(gen, shape, deviation):
    """An FP8 (e4m3) weight [E, N, K] with one fp32 inverse scale per 128 x 128 tile."""
    dev = gen.device
    data = torch.empty(shape, dtype=torch.float8_e4m3fn, device=dev)
    data.copy_((torch.randn(shape, generator=gen, device=dev, dtype=torch.bfloat16) * 100).clamp_(-448, 448))
    tiles = (shape[0], -(-shape[1] // BLOCK), -(-shape[2] // BLOCK))
    return {"data": data, "scale": (torch.rand(tiles, generator=gen, device=dev) * 0.6 + 0.7) * (deviation / 100)}


def _handle(weight, dtype):
    """The framework's own handle of a weight, as a program makes it when it loads the model."""
    if "codes" in weight:
        from primus_turbo_b200.pytorch.core.int4_weight import Int4Weight

        return Int4Weight.from_codes(weight["codes"], weight["scale"], weight["zero"], group_size=weight["group"])
    if "data" in weight:
        from primus_turbo_b200.pytorch.core.low_precision import ScalingGranularity, ScalingRecipe
        from primus_turbo_b200.pytorch.core.quantized_tensor import QuantizedTensor

        return QuantizedTensor(weight["data"], weight["scale"], shape=weight["data"].shape, orig_dtype=dtype,
                               dest_dtype=weight["data"].dtype, granularity=ScalingGranularity.BLOCKWISE, block_size=BLOCK,
                               scaling_recipe=ScalingRecipe(use_2d_block=True), quantized_axis=-1)
    return weight["raw"]


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPE[case["dtype"]]

    def randn(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale).to(dtype)

    state = {"case": case}
    if case["op"] == "router":
        t, e = case["tokens"], case["experts"]
        # some experts are more popular than others
        popular = torch.randn(e, generator=gen, device=dev) * 0.5
        state["logits"] = (torch.randn((t, e), generator=gen, device=dev) * 1.5 + popular).to(dtype)
        state["bias"] = torch.randn(e, generator=gen, device=dev) * 0.05 if case["bias"] else None
        if case["train"]:
            state["logits"].requires_grad_(True)
            state["grad"] = torch.randn((t, e if case["dense"] else case["topk"]), generator=gen, device=dev)
    elif case["op"] == "int4":
        state["x"] = randn(case["m"], case["k"])
        state["w"] = _weight4(gen, (case["n"], case["k"]), case["group"], case["zeros"], case["k"] ** -0.5)
        state["bias"] = randn(case["n"], scale=0.1) if case["bias"] else None
    elif case["op"] == "quant":
        shape = (case["n"], case["k"]) if case["experts"] == 1 else (case["experts"], case["n"], case["k"])
        # rows of unlike size, as trained weights have them
        rows = torch.rand((*shape[:-1], 1), generator=gen, device=dev) * 0.03 + 0.005
        state["w"] = (torch.randn(shape, generator=gen, device=dev) * rows).to(dtype)
    else:
        t, e, k, h, i = (case[n] for n in ("tokens", "experts", "topk", "hidden", "inter"))
        state["x"] = randn(t, h)
        logits = torch.randn((t, e), generator=gen, device=dev) + torch.randn(e, generator=gen, device=dev) * 0.5
        top = torch.sort(logits, dim=1, descending=True, stable=True)
        state["ids"] = top.indices[:, :k].contiguous()
        state["probs"] = torch.softmax(top.values[:, :k], dim=1)
        for name, shape in (("w1", (e, 2 * i, h)), ("w2", (e, h, i))):
            deviation = shape[2] ** -0.5
            if case["weights"] == "int4":
                state[name] = _weight4(gen, shape, case["group"], False, deviation)
            elif case["weights"] == "fp8":
                state[name] = _weight8(gen, shape, deviation)
            else:
                state[name] = {"raw": randn(*shape, scale=deviation)}
    if own:
        for name in {"int4": ("w",), "moe": ("w1", "w2")}.get(case["op"], ()):
            state["own_" + name] = _handle(state[name], dtype)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    return {"router": _run_router, "int4": _run_int4, "quant": _run_quant, "moe": _run_moe}[case["op"]](case, state)


def _run_router(case, state):
    options = dict(score_function=case["score"], expert_bias=state["bias"], num_groups=case["groups"],
                   topk_groups=case["topk_groups"], normalize=case["normalize"], scaling_factor=case["scaling"])
    if own:
        from primus_turbo_b200.pytorch.ops.moe import topk_router, topk_routing_map

        probs, chosen = (topk_routing_map if case["dense"] else topk_router)(state["logits"], case["topk"], **options)
    else:
        probs, chosen = _plain_router(case, state)
    if not case["train"]:
        return probs, chosen
    (grad,) = torch.autograd.grad(probs, state["logits"], state["grad"])
    return probs.detach(), chosen, grad


def _plain_router(case, state):
    logits = state["logits"]
    with torch.no_grad():
        # which experts are taken hangs on values that lie next to each other: in 64 bits
        wide = logits.double()
        if case["score"] == "softmax":
            e = torch.exp(wide - wide.amax(1, keepdim=True))
            score = e / e.sum(1, keepdim=True)
        else:
            score = 1 / (1 + torch.exp(-wide))
        choice = score if state["bias"] is None else score + state["bias"].double()
        if case["groups"] > 1:
            t, n = choice.shape[0], case["groups"]
            per_group = torch.sort(choice.view(t, n, -1), dim=2, descending=True).values[:, :, :2].sum(2)
            kept = torch.sort(per_group, dim=1, descending=True, stable=True).indices[:, : case["topk_groups"]]
            keep = torch.zeros((t, n), dtype=torch.bool, device=choice.device).scatter_(1, kept, True)
            choice = torch.where(keep.repeat_interleave(choice.shape[1] // n, dim=1), choice, -math.inf)
        ids = torch.sort(choice, dim=1, descending=True, stable=True).indices[:, : case["topk"]]
    x = logits.float()
    if case["score"] == "softmax":
        e = torch.exp(x - x.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    probs = score.gather(1, ids)
    if case["normalize"]:
        probs = probs / (probs.sum(1, keepdim=True) + 1e-20)
    probs = probs * case["scaling"]
    if not case["dense"]:
        return probs, ids
    table = torch.zeros_like(score).scatter(1, ids, probs)
    return table, torch.zeros_like(score, dtype=torch.bool).scatter_(1, ids, True)


def _values4(weight, rows=None):
    """The fp32 values of a 4-bit weight (of some experts of it)."""
    codes, scale, zero = (v if v is None or rows is None else v[rows] for v in (weight["codes"], weight["scale"], weight["zero"]))
    k, group = codes.shape[-1], weight["group"]
    step = scale.float().repeat_interleave(group, dim=-1)[..., :k]
    start = 8.0 if zero is None else zero.float().repeat_interleave(group, dim=-1)[..., :k]
    return (codes.float() - start) * step


def _run_int4(case, state):
    if own:
        from primus_turbo_b200.pytorch.ops import gemm_int4

        return gemm_int4(state["x"], state["own_w"], bias=state["bias"])
    y = state["x"].float() @ _values4(state["w"]).T
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def _run_quant(case, state):
    w, group = state["w"], case["group"]
    if own:
        from primus_turbo_b200.pytorch.ops import dequantize_int4, quantize_int4

        q = quantize_int4(w, group_size=group, symmetric=not case["zeros"])
        return dequantize_int4(q, w.dtype), q.scale, q.zero
    k = w.shape[-1]
    wide = torch.nn.functional.pad(w.float(), (0, -k % group)).unflatten(-1, (-1, group))
    seven, fifteen = (torch.full((), v, device=w.device) for v in (7.0, 15.0))  # divided by, not multiplied with an inverse
    if case["zeros"]:
        lo, hi = wide.amin(-1).clamp(max=0), wide.amax(-1).clamp(min=0)
        scale = (hi / fifteen - lo / fifteen).to(torch.bfloat16)
        s = scale.float()
        zero = torch.round(-lo / s).nan_to_num().clamp(0, 15)
    else:
        scale = (wide.abs().amax(-1) / seven).to(torch.bfloat16)
        s = scale.float()
        zero = torch.full_like(s, 8.0)
    codes = (torch.round(wide / s[..., None]).nan_to_num() + zero[..., None]).clamp(0, 15)
    values = ((codes - zero[..., None]) * s[..., None]).flatten(-2)[..., :k].to(w.dtype)
    return values, scale, zero.to(torch.uint8) if case["zeros"] else None


def _values(weight, rows=None):
    """The fp32 values of experts' weights [E, N, K], or of the experts ``rows``."""
    if "codes" in weight:
        return _values4(weight, rows)
    if "raw" in weight:
        return (weight["raw"] if rows is None else weight["raw"][rows]).float()
    data, scale = weight["data"].view(torch.uint8), weight["scale"]
    if rows is not None:
        data, scale = data[rows], scale[rows]
    n, k = data.shape[1:]
    tiles = scale.repeat_interleave(BLOCK, dim=1)[:, :n].repeat_interleave(BLOCK, dim=2)[:, :, :k]
    return data.view(torch.float8_e4m3fn).float() * tiles


def _run_moe(case, state):
    if own:
        from primus_turbo_b200.pytorch.ops.moe import moe_few_tokens

        return moe_few_tokens(state["x"], state["ids"], state["probs"], state["own_w1"], state["own_w2"])
    x, ids, probs, i = state["x"].float(), state["ids"], state["probs"], case["inter"]
    t, k = ids.shape
    if t * k <= case["experts"]:  # the weights of each token's experts
        flat = ids.flatten()
        gate_up = torch.bmm(_values(state["w1"], flat), x.repeat_interleave(k, dim=0)[:, :, None])[:, :, 0]
        gate, up = gate_up[:, :i], gate_up[:, i:]
        act = gate / (1 + torch.exp(-gate)) * up
        rows = torch.bmm(_values(state["w2"], flat), act[:, :, None])[:, :, 0]
        y = (rows.view(t, k, -1) * probs[:, :, None]).sum(1)
    else:  # every expert on every token, and what the router gives to each
        gate_up = torch.matmul(x, _values(state["w1"]).transpose(1, 2))
        gate, up = gate_up[..., :i], gate_up[..., i:]
        act = gate / (1 + torch.exp(-gate)) * up
        rows = torch.bmm(act, _values(state["w2"]).transpose(1, 2))
        table = torch.zeros((t, case["experts"]), device=x.device).scatter_(1, ids, probs)
        y = (rows * table.T[:, :, None]).sum(0)
    return y.to(state["x"].dtype)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def _bytes4(n, k, group, zeros):
    return n * k / 2 + n * -(-k // group) * (3 if zeros else 2)


def work(case):
    size = DTYPE[case["dtype"]].itemsize
    if case["op"] == "router":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        moved = t * e * size + (t * e * 5 if case["dense"] else t * k * 12) + (4 * e if case["bias"] else 0)
        if case["train"]:
            moved += t * e * size * 2 + t * (e if case["dense"] else k) * 4
        return {"bytes": moved, "flops": t * e * (16 if case["train"] else 8)}
    if case["op"] == "int4":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": _bytes4(n, k, case["group"], case["zeros"]) + size * (m * (n + k) + (n if case["bias"] else 0)), "flops": 2 * m * n * k}
    if case["op"] == "quant":
        n, k = case["experts"] * case["n"], case["k"]
        # the weight in, the codes out; the codes in, the values out
        return {"bytes": 2 * n * k * size + 2 * _bytes4(n, k, case["group"], case["zeros"]), "flops": 6 * n * k}
    t, e, k, h, i = (case[n] for n in ("tokens", "experts", "topk", "hidden", "inter"))
    hit = e * (1 - (1 - k / e) ** t)  # experts that at least one token goes to
    if case["weights"] == "int4":
        weight = _bytes4(2 * i, h, case["group"], False) + _bytes4(h, i, case["group"], False)
    else:
        weight = 3 * h * i * (1 if case["weights"] == "fp8" else size)
    return {"bytes": hit * weight + t * (2 * h * size + 12 * k), "flops": 6 * t * k * h * i}


# ---- the definition, in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"router": _exact_router, "int4": _exact_int4, "quant": _exact_quant, "moe": _exact_moe}[case["op"]](case, state)


def _exact_router(case, state):
    l = state["logits"].detach().double()
    t, e = l.shape
    s = torch.softmax(l, 1) if case["score"] == "softmax" else torch.sigmoid(l)
    order = s if state["bias"] is None else s + state["bias"].double()
    if case["groups"] > 1:
        best = order.reshape(t, case["groups"], -1).topk(2, dim=2).values.sum(2)
        place = best.argsort(dim=1, descending=True, stable=True).argsort(dim=1)
        order = order.masked_fill((place >= case["topk_groups"]).repeat_interleave(e // case["groups"], 1), -torch.inf)
    rank = order.argsort(dim=1, descending=True, stable=True)
    ids = rank[:, : case["topk"]]
    taken = torch.zeros_like(s).scatter(1, ids, 1.0)
    a = case["scaling"]
    total = (s * taken).sum(1, keepdim=True) + 1e-20 if case["normalize"] else torch.ones((t, 1), device=s.device, dtype=s.dtype)
    table = a * taken * s / total
    probs = table if case["dense"] else table.gather(1, ids)
    if not case["train"]:
        return probs, None
    g = state["grad"].double()
    g = g * taken if case["dense"] else torch.zeros_like(s).scatter(1, ids, g)
    ds = a * g / total
    if case["normalize"]:
        ds = ds - taken * a * (g * s).sum(1, keepdim=True) / total**2
    if case["score"] == "softmax":
        dl = s * (ds - (ds * s).sum(1, keepdim=True))
    else:
        dl = ds * s * (1 - s)
    return probs, None, dl


def _exact_values(weight):
    if "raw" in weight:
        return weight["raw"].double()
    if "data" in weight:
        d = weight["data"].double()
        r, c = torch.arange(d.shape[1], device=d.device) // BLOCK, torch.arange(d.shape[2], device=d.device) // BLOCK
        return d * weight["scale"].double()[:, r][:, :, c]
    q = weight["codes"].double()
    c = torch.arange(q.shape[-1], device=q.device) // weight["group"]
    return (q - (8 if weight["zero"] is None else weight["zero"].double()[..., c])) * weight["scale"].double()[..., c]


def _exact_int4(case, state):
    y = torch.einsum("mk,nk->mn", state["x"].double(), _exact_values(state["w"]))
    return y if state["bias"] is None else y + state["bias"].double()


def _exact_quant(case, state):
    w = state["w"].double()
    c = torch.arange(w.shape[-1], device=w.device) // case["group"]
    index = c.expand(w.shape)
    none = torch.zeros((*w.shape[:-1], int(c[-1]) + 1), device=w.device, dtype=w.dtype)
    hi = none.scatter_reduce(-1, index, w, "amax", include_self=True)
    lo = none.scatter_reduce(-1, index, w, "amin", include_self=True)
    if case["zeros"]:
        scale = ((hi - lo) / 15).to(torch.bfloat16).double()
        zero = (-lo / scale).round().clamp(0, 15)
    else:
        scale = (torch.maximum(hi, -lo) / 7).to(torch.bfloat16).double()
        zero = torch.full_like(scale, 8.0)
    z, s = zero.gather(-1, index), scale.gather(-1, index)
    return ((w / s).round() + z).clamp(0, 15).sub(z) * s, scale, None


def _exact_moe(case, state):
    x, i = state["x"].double(), case["inter"]
    y = torch.zeros_like(x)
    for e in state["ids"].unique().tolist():  # an expert's weights at a time: all of them in 64 bits take the card's memory
        row, slot = (state["ids"] == e).nonzero(as_tuple=True)
        w1, w2 = (_exact_values({n: v if n == "group" or v is None else v[e : e + 1] for n, v in state[m].items()})[0] for m in ("w1", "w2"))
        u = x[row] @ w1.T
        a = u[:, :i] * torch.sigmoid(u[:, :i]) * u[:, i:]
        y.index_add_(0, row, state["probs"][row, slot].double()[:, None] * (a @ w2.T))
    return y
