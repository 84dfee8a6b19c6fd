"""The operators of a mixture-of-experts layer and of 4-bit linear layers, in their plain form and through the library.

Five kinds of work:

``route``    ``ops.router.route``: scores, top-k choice, gates, per-expert counts and balance loss; with ``train`` the backward pass too
``quant``    ``ops.fp4.quantize_fp4`` and back: microscaled 4-bit values (e2m1, blocks of 32, one power of two each)
``linear``   ``quantize_fp4`` of the activations, ``gemm_fp4`` with weights held in 4 bits
``experts``  fp8 rows as the exchange delivers them, requantised, through the gate and up projections of their experts with SwiGLU
``down``     bf16 rows grouped by expert, quantised, through the down projections of their experts

Widths are those of ``models.llama.CONFIGS``, of one rank's share of them under tensor parallelism over eight ranks, and of
the expert-parallel benchmark (256 experts, 8 per token, hidden 7168; 32 experts on one of eight ranks).
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# (out features, in features): the projections of llama3_70b, of one of eight ranks' share of it, of llama3_8b and of small, odd ones
LINEARS = [(28672, 8192), (8192, 28672), (3584, 8192), (8192, 3584), (14336, 4096), (4096, 14336), (4096, 4096), (1024, 4096), (4096, 1024), (1000, 2080), (136, 96)]
# (experts, per token) of the exchange's tests and benchmark
ROUTERS = [(8, 2), (64, 6), (128, 4), (256, 8)]
# (experts on this rank, hidden, intermediate)
EXPERTS = [(32, 7168, 2048), (32, 4096, 1536), (8, 4096, 14336), (16, 2048, 1408), (8, 1024, 4096)]


def listed():
    return [
        # one decoding step of a small batch: nothing but latency; sigmoid scores with a selection bias, as served
        {"name": "route-decode-16", "kind": "route", "tokens": 16, "experts": 256, "topk": 8, "dtype": "fp32", "scoring": "sigmoid",
         "renormalize": True, "biased": True, "masked": False, "train": False},
        # the benchmark's tokens of one rank, a training step
        {"name": "route-train-4096", "kind": "route", "tokens": 4096, "experts": 256, "topk": 8, "dtype": "bf16", "scoring": "softmax",
         "renormalize": True, "biased": False, "masked": False, "train": True},
        # a long packed batch with padding in it and experts that are switched off
        {"name": "route-train-65003", "kind": "route", "tokens": 65003, "experts": 64, "topk": 6, "dtype": "fp32", "scoring": "softmax",
         "renormalize": False, "biased": False, "masked": True, "train": True},
        # activations of a few tokens of the 70B model's down projection
        {"name": "quant-decode-16", "kind": "quant", "rows": 16, "cols": 28672, "dtype": "bf16"},
        # weights of one projection, quantised when a model is loaded
        {"name": "quant-weights-8192", "kind": "quant", "rows": 8192, "cols": 28672, "dtype": "bf16"},
        # decoding with a batch of 16: the weights are read for a handful of rows
        {"name": "linear-decode-16", "kind": "linear", "m": 16, "n": 28672, "k": 8192, "dtype": "bf16"},
        # one chunk of a prefill on one rank's share, as long as the prompt's rest happens to be
        {"name": "linear-chunk-777", "kind": "linear", "m": 777, "n": 3584, "k": 8192, "dtype": "bf16"},
        # a prefill through the whole up projection
        {"name": "linear-prefill-8192", "kind": "linear", "m": 8192, "n": 28672, "k": 8192, "dtype": "bf16"},
        # one rank's experts while decoding: 64 tokens from each of eight ranks
        {"name": "experts-decode-512", "kind": "experts", "rows": 512, "experts": 32, "hidden": 7168, "inter": 2048},
        # one rank's experts in a prefill: every expert has a ragged thousand of rows
        {"name": "experts-prefill-32768", "kind": "experts", "rows": 32768, "experts": 32, "hidden": 7168, "inter": 2048},
        # their down projections while decoding a single token
        {"name": "down-decode-8", "kind": "down", "rows": 8, "experts": 32, "hidden": 7168, "inter": 2048},
        # and for a batch of prompts of no round length
        {"name": "down-prefill-5003", "kind": "down", "rows": 5003, "experts": 32, "hidden": 7168, "inter": 2048},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread evenly over their logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(["route"] * 3 + ["quant"] + ["linear"] * 3 + ["experts"] * 2 + ["down"])
    if kind == "route":
        experts, topk = rng.choice(ROUTERS)
        scoring = rng.choice(["softmax", "sigmoid"])
        return {"kind": kind, "tokens": _log(rng, 1, 65536), "experts": experts, "topk": topk, "dtype": rng.choice(["bf16", "fp16", "fp32"]), "scoring": scoring,
                "renormalize": rng.random() < 0.6, "biased": scoring == "sigmoid" and rng.random() < 0.5, "masked": rng.random() < 0.4, "train": rng.random() < 0.6}
    if kind == "quant":
        return {"kind": kind, "rows": _log(rng, 1, 8192), "cols": 32 * _log(rng, 1, 896), "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if kind == "linear":
        n, k = rng.choice(LINEARS)
        return {"kind": kind, "m": _log(rng, 1, 8192), "n": n, "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    experts, hidden, inter = rng.choice(EXPERTS)
    return {"kind": kind, "rows": _log(rng, 1, 16384), "experts": experts, "hidden": hidden, "inter": inter}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = case["kind"]
    if kind == "route":
        return _prepare_route(case, g)
    if kind == "quant":
        return {"case": case, "x": _activations(g, case["rows"], case["cols"], DTYPES[case["dtype"]])}
    if kind == "linear":
        state = {"case": case, "x": _activations(g, case["m"], case["k"], DTYPES[case["dtype"]])}
        return _weights(state, g, "w", (case["n"], case["k"]))
    rows, experts, hidden, inter = case["rows"], case["experts"], case["hidden"], case["inter"]
    # some experts are asked for more often than others; rows are grouped by expert
    share = torch.softmax(0.5 * torch.randn(experts, device="cuda", generator=g), 0)
    counts = torch.bincount(torch.multinomial(share, rows, replacement=True, generator=g), minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
    capacity = rows + 64            # the buffers are longer than what a step fills
    if kind == "experts":
        x = _activations(g, capacity, hidden, torch.float32).view(capacity, hidden // 128, 128)
        amax = x.abs().amax(-1, keepdim=True).clamp_min(1e-4)
        scales = amax / torch.full_like(amax, 448.0)
        state = {"case": case, "x": (x / scales).to(torch.float8_e4m3fn).view(capacity, hidden), "x_scales": scales.view(capacity, hidden // 128).contiguous()}
        out = torch.zeros(capacity, inter, device="cuda", dtype=torch.bfloat16)
        _weights(_weights(state, g, "gate", (experts, inter, hidden)), g, "up", (experts, inter, hidden))
    else:
        state = {"case": case, "x": _activations(g, capacity, inter, torch.bfloat16)}
        out = torch.zeros(capacity, hidden, device="cuda", dtype=torch.bfloat16)
        _weights(state, g, "down", (experts, hidden, inter))
    state.update(offsets=offsets, out=out)
    return state


def _activations(g, rows, cols, dtype):
    """Values of about one, with a few channels that are ten times as large, as hidden states have them."""
    x = torch.randn(rows, cols, device="cuda", generator=g)
    x *= 1 + 9 * (torch.rand(cols, device="cuda", generator=g) < 0.01)
    return x.to(dtype)


def _weights(state, g, name, shape):
    """4-bit weights as a checkpoint holds them: two values a byte, one power of two for every 32."""
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.randint(118, 122, (*shape[:-1], shape[-1] // 32), device="cuda", generator=g, dtype=torch.uint8)
    state[name] = (codes, scales)
    if own:
        from hcomm_b200.ops.fp4 import Fp4Tensor
        state[name + "_fp4"] = Fp4Tensor.from_parts(codes, scales)
    return state


def _prepare_route(case, g):
    tokens, experts = case["tokens"], case["experts"]
    logits = 1.5 * torch.randn(tokens, experts, device="cuda", generator=g) + 0.5 * torch.randn(experts, device="cuda", generator=g)
    state = {"case": case, "valid": None, "bias": None}
    if case["masked"]:
        logits[:, torch.rand(experts, device="cuda", generator=g) < 0.05] = float("-inf")       # experts that are switched off
        logits[torch.rand(tokens, device="cuda", generator=g) < 0.002] = float("-inf")          # a mask that leaves a token nothing
        state["valid"] = torch.rand(tokens, device="cuda", generator=g) < 0.85                  # padding
    if case["biased"]:
        state["bias"] = 0.2 * torch.randn(experts, device="cuda", generator=g)
    state["logits"] = logits.to(DTYPES[case["dtype"]])
    if case["train"]:
        state["logits"].requires_grad_(own)
        lift = 1024.0 if case["dtype"] == "fp16" else 1.0           # training in fp16 scales its loss, or its gradients are too small for the type
        state["dgates"] = torch.randn(tokens, case["topk"], device="cuda", generator=g) * (lift / tokens)
        state["dloss"] = torch.full((), lift, device="cuda")
    return state


SCALE = 2.5             # of the gates
BALANCE = 0.01          # coefficient of the balance loss


def run(state):
    kind = state["case"]["kind"]
    if kind == "route":
        return _route_own(state) if own else _route_plain(state)
    if own:
        return _fp4_own(state)
    if kind == "quant":
        return _quantised(state["x"].float()).to(torch.bfloat16)
    if kind == "linear":
        return (_quantised(state["x"].float()) @ _dequantised(*state["w"]).t()).to(torch.bfloat16)
    out, bounds = torch.zeros_like(state["out"]), state["offsets"].tolist()
    for e, (lo, hi) in enumerate(zip(bounds, bounds[1:])):
        if lo == hi:
            continue
        x = state["x"][lo:hi].float()
        if kind == "experts":
            x = (x.view(hi - lo, -1, 128) * state["x_scales"][lo:hi].unsqueeze(-1)).view(hi - lo, -1)
        x = _quantised(x)
        if kind == "experts":
            gate, up = (x @ _dequantised(state[n][0][e], state[n][1][e]).t() for n in ("gate", "up"))
            out[lo:hi] = (gate / (1 + torch.exp(-gate)) * up).to(torch.bfloat16)
        else:
            out[lo:hi] = (x @ _dequantised(state["down"][0][e], state["down"][1][e]).t()).to(torch.bfloat16)
    return out


# ------------------------------------------------------------------------------------------------ through the library

def _route_own(state):
    from hcomm_b200.ops.router import route
    case = state["case"]
    r = route(state["logits"], case["topk"], scoring=case["scoring"], renormalize=case["renormalize"], scale=SCALE, bias=state["bias"], valid=state["valid"],
              balance=BALANCE if case["train"] else 0.0)
    if not case["train"]:
        return r.topk_idx, r.gates, r.counts
    (dlogits,) = torch.autograd.grad((r.gates, r.loss), state["logits"], (state["dgates"], state["dloss"]))
    return r.topk_idx, r.gates.detach(), r.counts, r.loss.detach(), dlogits


def _fp4_own(state):
    from hcomm_b200.ops.fp4 import dequantize_fp4, gemm_fp4, gemm_fp4_swiglu, quantize_fp4
    kind, x = state["case"]["kind"], state["x"]
    if kind == "quant":
        return dequantize_fp4(quantize_fp4(x))
    if kind == "linear":
        return gemm_fp4(quantize_fp4(x), state["w_fp4"])
    if kind == "experts":
        return gemm_fp4_swiglu(quantize_fp4(x, state["x_scales"], offsets=state["offsets"]), state["gate_fp4"], state["up_fp4"], state["out"])
    return gemm_fp4(quantize_fp4(x, offsets=state["offsets"]), state["down_fp4"], state["out"])


# ------------------------------------------------------------------------------------------------ plain forms

def _route_plain(state):
    case, logits, valid = state["case"], state["logits"].float(), state["valid"]
    tokens, experts, k = case["tokens"], case["experts"], case["topk"]
    softmax = case["scoring"] == "softmax"
    # log of the score; a sigmoid next to 0 keeps its logarithm
    z = logits if softmax else torch.minimum(logits, torch.zeros_like(logits)) - torch.log(1 + torch.exp(-logits.abs()))
    key = logits.double() if state["bias"] is None else 1 / (1 + torch.exp(-logits.double())) + state["bias"].double()
    key = key.masked_fill(logits == float("-inf"), float("-inf"))
    idx = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = logits.gather(1, idx) != float("-inf")
    alive = torch.ones(tokens, dtype=torch.bool, device=logits.device) if valid is None else valid
    chosen = chosen & alive.unsqueeze(1)
    p = _softmax(z, alive)
    if case["renormalize"]:
        share = _softmax(z.gather(1, idx).masked_fill(~chosen, float("-inf")), alive)
    else:
        share = torch.where(chosen, (p if softmax else torch.exp(z)).gather(1, idx), torch.zeros((), device=z.device))
    gates = SCALE * share
    hits = torch.zeros(tokens, experts, device=z.device).scatter_(1, idx, chosen.float())
    counts = hits.sum(0, dtype=torch.float64).to(torch.int32)
    idx = idx.masked_fill(~chosen, -1).to(torch.int32)
    if not case["train"]:
        return idx, gates, counts
    total = alive.sum()
    total32 = total.float().clamp_min(1)
    load = counts.float() / (total32 * k)
    loss = BALANCE * experts * (load * (p.sum(0, dtype=torch.float64) / total32).float()).sum()
    # backward
    safe = idx.clamp_min(0).long()
    dgates = torch.where(chosen, SCALE * state["dgates"], torch.zeros((), device=z.device))
    u = (state["dloss"] * BALANCE * experts * load / total32).expand(tokens, experts)
    dz = torch.zeros_like(z)
    if case["renormalize"]:
        d = share * (dgates - (share * dgates).sum(1, keepdim=True))
        dz.scatter_add_(1, safe, d)
    elif softmax:
        u = u.clone().scatter_add_(1, safe, dgates)
    dz += p * (u - (p * u).sum(1, keepdim=True))
    if not softmax:
        if not case["renormalize"]:
            dz.scatter_add_(1, safe, share * dgates)
        dz = dz / (1 + torch.exp(logits))
    return idx, gates, counts, loss, dz.to(state["logits"].dtype)


def _softmax(z, alive):
    """Rows that hold nothing, or do not count, are zero."""
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    return e / e.sum(1, keepdim=True).clamp_min(1e-30) * alive.unsqueeze(1)


def _quantised(x):
    """The values that x stands for in microscaled 4 bits, in 32 bits."""
    blocks = x.view(*x.shape[:-1], -1, 32)
    amax = blocks.abs().amax(-1, keepdim=True)
    power = (torch.frexp(amax).exponent - 3).masked_fill(amax == 0, -127).clamp(-127, 127)
    a = blocks.abs() * _power_of_two(-power)
    half = ((a > 0.25).to(torch.float32) + (a >= 0.75) + (a > 1.25) + (a >= 1.75)) * 0.5
    value = half + (a > 2.5) + (a >= 3.5) + 2.0 * (a > 5)
    return (value * _power_of_two(power) * torch.sign(blocks)).view(x.shape)


def _power_of_two(n):
    """2^n in 32 bits from its exponent field, n from -127 to 127; torch.ldexp takes a power that CUDA rounds."""
    return torch.where(n > -127, (n + 127) << 23, 1 << 22).int().view(torch.float32)


def _dequantised(codes, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, 0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    pairs = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1)
    values = pairs.view(*scales.shape, 32)
    return (values * _power_of_two(scales.int() - 127).unsqueeze(-1)).view(*codes.shape[:-1], -1)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    kind = case["kind"]
    if kind == "route":
        t, e, k = case["tokens"], case["experts"], case["topk"]
        size = DTYPES[case["dtype"]].itemsize
        forward = t * e * size + 8 * t * k + 4 * e + (4 * e if case["biased"] else 0) + (t if case["masked"] else 0)
        backward = 2 * t * e * size + 4 * t * k if case["train"] else 0
        return {"bytes": forward + backward, "flops": t * e * (18 if case["train"] else 8)}
    if kind == "quant":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (DTYPES[case["dtype"]].itemsize + 2) + n * 17 // 32, "flops": 4 * n}
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k * DTYPES[case["dtype"]].itemsize + n * k * 17 // 32 + 2 * m * n, "flops": 2 * m * n * k}
    rows, experts, hidden, inter = case["rows"], case["experts"], case["hidden"], case["inter"]
    active = experts * (1 - (1 - 1 / experts) ** rows)          # experts that any row asks for
    if kind == "experts":
        return {"bytes": int(rows * hidden * 33 / 32 + active * 2 * inter * hidden * 17 / 32 + 2 * rows * inter), "flops": 4 * rows * hidden * inter}
    return {"bytes": int(2 * rows * inter + active * inter * hidden * 17 / 32 + 2 * rows * hidden), "flops": 2 * rows * hidden * inter}


# ------------------------------------------------------------------------------------------------ 64 bits, from the definition

def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "route":
        return _route_exact(state)
    if kind == "quant":
        return _nearest(state["x"].double())
    if kind == "linear":
        return _nearest(state["x"].double()) @ _held(*state["w"]).t()
    out, offsets = state["out"].double(), state["offsets"].tolist()
    for e in range(case["experts"]):
        rows = slice(offsets[e], offsets[e + 1])
        x = state["x"][rows].float()
        if not len(x):
            continue
        if kind == "experts":           # the exchange's values are their products in 32 bits
            x = x * state["x_scales"][rows].repeat_interleave(128, dim=1)
        x = _nearest(x.double())
        if kind == "down":
            out[rows] = x @ _held(state["down"][0][e], state["down"][1][e]).t()
        else:
            gate = x @ _held(state["gate"][0][e], state["gate"][1][e]).t()
            out[rows] = gate * torch.sigmoid(gate) * (x @ _held(state["up"][0][e], state["up"][1][e]).t())
    return out


def _nearest(x):
    """Every value to the nearest of its block's sixteen, the even one of two that are as near."""
    blocks = x.reshape(-1, 32)
    top = blocks.abs().amax(1)
    power = ((top.view(torch.int64) >> 52) - 1023 - 2).clamp(-127, 127)         # the exponent field is the logarithm's whole part; 0 has the least
    unit = _unit(power).unsqueeze(1)
    a = blocks.abs() / unit
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    value = (torch.round(a / step) * step).clamp_max(6.0)           # torch.round: halves go to the even one
    return (torch.copysign(value, blocks) * unit).view(x.shape)


def _unit(n):
    return ((n + 1023) << 52).view(torch.float64)


def _held(codes, scales):
    nibbles = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    magnitude = nibbles % 8
    value = torch.where(magnitude < 4, magnitude / 2, torch.where(magnitude < 6, magnitude - 2, 2 * magnitude - 8))
    unit = _unit(scales.long() - 127).repeat_interleave(32, dim=-1)
    return torch.where(nibbles >= 8, -value, value) * unit


def _route_exact(state):
    case, valid = state["case"], state["valid"]
    x = state["logits"].detach().double()
    tokens, experts = x.shape
    k, softmax, renorm = case["topk"], case["scoring"] == "softmax", case["renormalize"]
    if valid is not None:
        x = torch.where(valid.unsqueeze(1), x, -torch.inf)
    x.requires_grad_(case["train"])
    off = torch.isneginf(x)
    score = torch.sigmoid(x)
    key = (x if state["bias"] is None else score + state["bias"].double()).detach().clone()
    key[off] = -torch.inf
    picks, ids = [], torch.arange(experts, device=x.device)
    for _ in range(k):
        best = key.amax(1, keepdim=True)
        i = torch.where(key == best, ids, experts).amin(1, keepdim=True)
        picks.append(torch.where(torch.isneginf(best), -1, i))
        key.scatter_(1, i, -torch.inf)
    idx = torch.cat(picks, 1)
    live = idx >= 0
    at = idx.clamp_min(0)
    weight = torch.exp(x - torch.nan_to_num(x.detach().amax(1, keepdim=True), neginf=0.0)) if softmax else score
    whole = weight.sum(1, keepdim=True)
    p = weight / torch.where(whole > 0, whole, 1.0)
    gates = torch.where(live, (p if softmax else score).gather(1, at), 0.0)
    if renorm:
        part = gates.sum(1, keepdim=True)
        gates = gates / torch.where(part > 0, part, 1.0)
    gates = SCALE * gates
    counts = torch.bincount(idx[live], minlength=experts)
    if not case["train"]:
        return idx.to(torch.int32), gates, counts.to(torch.int32)
    total = max(1, tokens if valid is None else int(valid.sum()))
    loss = BALANCE * experts * (counts.double() / (total * k) * p.sum(0) / total).sum()
    (dx,) = torch.autograd.grad((gates, loss), x, (state["dgates"].double(), state["dloss"].double()))
    dx = torch.where(off, 0.0, torch.nan_to_num(dx))
    return idx.to(torch.int32), gates.detach(), counts.to(torch.int32), loss.detach(), dx
