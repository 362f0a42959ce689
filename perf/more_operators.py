"""What a serving program runs around and inside an MoE block beside its router and prompt-sized products.

Three operators: `add_norm` (a block's output normed, gated, scaled and joined to the residual stream, and the norm
before the next block), `adapter_linear` and `adapter_gated_linear` (the dense products with the low-rank adapters
of many requests beside the shared weight) and `token_experts` (the routed experts of a layer for a few tokens).
`run` computes a case in plain torch operations in 32 bits or, where `own` is true, by the framework's operators.
Hidden rows are ~N(0, 1), the residual stream ~N(0, 2), weights and adapters ~N(0, 0.02), expert choices those of
random logits with softmax weights.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-6
_OPS = None


def _ops():
    global _OPS
    if _OPS is None:
        sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "uniserve-v1_amd"))
        from uniserve_moe import ops

        _OPS = ops
    return _OPS


def _norm(tokens, width, dtype="bf16", stream="same", norm="rms", post=False, gate=False, channels=False, bias=False,
          offset=0.0, scale=1.0, residual_scale=1.0):
    return {"op": "add_norm", "tokens": tokens, "width": width, "dtype": dtype, "stream": stream, "norm": norm,
            "post": post, "gate": gate, "channels": channels, "bias": bias, "offset": offset, "scale": scale,
            "residual_scale": residual_scale}


def _adapted(op, tokens, width, rows, rank, adapters, requests=0, dtype="bf16", bias=False, activation="none",
             gate=False, residual=False, without=False):
    """`requests` runs of consecutive tokens, one adapter each; 0: every token a request of its own."""
    return {"op": op, "tokens": tokens, "width": width, "rows": rows, "rank": rank, "adapters": adapters,
            "requests": requests, "dtype": dtype, "bias": bias, "activation": activation, "gate": gate,
            "residual": residual, "without": without}


def _experts(tokens, hidden, intermediate, experts, top, dtype="bf16", activation="silu", residual=False):
    return {"op": "token_experts", "tokens": tokens, "hidden": hidden, "intermediate": intermediate,
            "experts": experts, "top": top, "dtype": dtype, "activation": activation, "residual": residual}


def listed():
    return [
        # One user's decode step between attention and the block: the plain residual join and norm.
        dict(_norm(1, 2048), name="norm-one"),
        # A decode batch normed on both sides of the block, on an FP32 residual stream, with a row gate.
        dict(_norm(64, 4096, stream="f32", post=True, gate=True, offset=1.0), name="norm-decode"),
        # Odd extents, the whole of the layer norm: biases, a scale per channel, both residual scales.
        dict(_norm(333, 1000, dtype="f16", norm="layer", post=True, channels=True, bias=True, scale=0.5,
                   residual_scale=1.5), name="norm-odd"),
        # Whole prompts normed on both sides of the block.
        dict(_norm(8192, 4096, post=True, scale=0.25), name="norm-prompt"),
        # One user's token with its own adapter beside an attention projection.
        dict(_adapted("adapter_linear", 1, 2048, 4096, 16, 8), name="adapt-one"),
        # The benchmark's decode batch, every request with another adapter, some with none, onto the residual stream.
        dict(_adapted("adapter_linear", 64, 4096, 2048, 16, 64, residual=True, without=True), name="adapt-decode"),
        # A chunk of a few requests' prompts through a shared expert's up and gate halves.
        dict(_adapted("adapter_gated_linear", 777, 2048, 1408, 8, 16, requests=5, dtype="f16", bias=True,
                      activation="gelu_tanh"), name="adapt-gated-chunk"),
        # Odd extents and an odd rank.
        dict(_adapted("adapter_linear", 333, 1000, 1001, 5, 7, requests=19, dtype="f16", bias=True, without=True),
             name="adapt-odd"),
        # Whole prompts of twelve requests with adapters of a large rank.
        dict(_adapted("adapter_linear", 8192, 2048, 4096, 64, 16, requests=12, residual=True, without=True),
             name="adapt-prompt"),
        # The benchmark's layer for one token.
        dict(_experts(1, 2048, 768, 128, 8), name="experts-one"),
        # A few tokens of a smaller layer of f16 weights, joined to a shared expert's output.
        dict(_experts(5, 2048, 704, 64, 6, dtype="f16", activation="gelu_tanh", residual=True), name="experts-few"),
        # The benchmark's layer for its decode batch: nearly every expert is named.
        dict(_experts(64, 2048, 768, 128, 8), name="experts-batch"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.random()
    tokens = _log(rng, 1, 8192)
    if kind < 0.33:
        width = _log(rng, 64, 8192)
        width = width if rng.random() < 0.3 else -(-width // 8) * 8
        tokens = max(1, min(tokens, 8192 * 4096 // (width * 2)))
        norm = rng.choice(["rms", "rms", "layer"])
        return _norm(tokens, width, rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["same", "f32"]), norm,
                     rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.3, norm == "layer",
                     rng.choice([0.0, 1.0]), rng.choice([1.0, 0.25]), rng.choice([1.0, 1.5]))
    dtype, activation = rng.choice(["bf16", "bf16", "f16"]), rng.choice(["silu", "gelu_tanh"])
    if kind < 0.7:
        # Widths are whole 8 elements for the most part, some of them whole 128; ranks are mostly powers of two.
        width = _log(rng, 64, 5632)
        width = {0: width, 1: -(-width // 128) * 128, 2: -(-width // 128) * 128}.get(rng.randrange(5), -(-width // 8) * 8)
        rows = _log(rng, 16, 5632)
        rows = rows if rng.random() < 0.3 else -(-rows // 16) * 16
        rank = rng.choice([4, 8, 16, 16, 32, 64, rng.randint(1, 64)])
        gated = rng.random() < 0.4
        tokens = max(1, min(tokens, 8192 * 2048 * 4096 // (width * rows * (2 if gated else 1))))
        requests = 0 if tokens <= 256 and rng.random() < 0.6 else rng.randint(1, min(tokens, 16))
        adapters = _log(rng, 1, 64)
        if gated:
            return _adapted("adapter_gated_linear", tokens, width, rows, rank, adapters, requests, dtype,
                            rng.random() < 0.3, activation, without=rng.random() < 0.5)
        return _adapted("adapter_linear", tokens, width, rows, rank, adapters, requests, dtype, rng.random() < 0.4,
                        rng.choice(["none", "none", activation]), rng.random() < 0.3, rng.random() < 0.5,
                        rng.random() < 0.5)
    experts = _log(rng, 4, 128)
    top = rng.randint(1, min(8, experts))
    hidden, intermediate = _log(rng, 128, 2048), _log(rng, 64, 768)
    if rng.random() < 0.7:
        hidden, intermediate = -(-hidden // 64) * 64, -(-intermediate // 32) * 32
    return _experts(_log(rng, 1, 64), hidden, intermediate, experts, top, dtype, activation, rng.random() < 0.5)


def _normal(generator, shape, std, dtype, mean=0.0):
    values = torch.randn(shape, generator=generator, device="cuda", dtype=torch.float32).mul_(std)
    return (values.add_(mean) if mean else values).to(dtype)


def _prepare_norm(case, generator):
    dtype, tokens, width = _TYPES[case["dtype"]], case["tokens"], case["width"]
    stream = dtype if case["stream"] == "same" else torch.float32
    mean = 1.0 - case["offset"]
    state = {"x": _normal(generator, (tokens, width), 1.0, dtype),
             "residual": _normal(generator, (tokens, width), 2.0, stream),
             "weight": _normal(generator, (width,), 0.1, dtype, mean),
             "post": _normal(generator, (width,), 0.1, dtype, mean) if case["post"] else None,
             "gate": _normal(generator, (tokens, 1), 1.0, dtype) if case["gate"] else None,
             "channels": _normal(generator, (width,), 0.3, dtype) if case["channels"] else None,
             "bias": _normal(generator, (width,), 0.3, dtype) if case["bias"] else None,
             "post_bias": _normal(generator, (width,), 0.3, dtype) if case["bias"] and case["post"] else None}
    return state


def _runs(case, seed):
    """(first token, end, adapter) of each run; adapter -1: none. As many adapters are in use as there can be."""
    rng = random.Random(seed)
    tokens, requests = case["tokens"], case["requests"] or case["tokens"]
    ends = sorted(rng.sample(range(1, tokens), requests - 1)) + [tokens]
    order = rng.sample(range(case["adapters"]), case["adapters"])
    runs, first = [], 0
    for i, end in enumerate(ends):
        runs.append((first, end, -1 if case["without"] and i % 8 == 5 else order[i % len(order)]))
        first = end
    return runs


def _prepare_adapted(case, generator, seed):
    dtype, tokens, width = _TYPES[case["dtype"]], case["tokens"], case["width"]
    halves = 2 if case["op"] == "adapter_gated_linear" else 1
    rows, rank, adapters = case["rows"] * halves, case["rank"], case["adapters"]
    runs = _runs(case, seed)
    index = torch.empty(tokens, dtype=torch.int32)
    for first, end, adapter in runs:
        index[first:end] = adapter
    state = {"runs": runs, "adapter": index.cuda(),
             "x": _normal(generator, (tokens, width), 1.0, dtype),
             "weight": _normal(generator, (rows, width), 0.02, dtype),
             "down": _normal(generator, (adapters, halves * rank, width), 0.02, dtype),
             "up": _normal(generator, (adapters, rows, rank), 0.02, dtype),
             "scales": torch.rand(adapters, generator=generator, device="cuda") * 2.0 + 0.5,
             "bias": _normal(generator, (rows,), 0.5, dtype) if case["bias"] else None,
             "gate": _normal(generator, (tokens, 1), 1.0, dtype) if case["gate"] else None,
             "residual": _normal(generator, (tokens, rows), 1.0, dtype) if case["residual"] else None,
             "workspace": None}
    if own:
        # A serving program keeps one for its largest batch.
        state["workspace"] = torch.empty(_ops().adapter_workspace(tokens, halves * rank), dtype=torch.uint8, device="cuda")
    return state


def _prepare_experts(case, generator):
    dtype, tokens, hidden, width = _TYPES[case["dtype"]], case["tokens"], case["hidden"], case["intermediate"]
    logits = torch.randn((tokens, case["experts"]), generator=generator, device="cuda") * 1.5
    values, ids = torch.topk(logits, case["top"], dim=1)
    state = {"x": _normal(generator, (tokens, hidden), 1.0, dtype), "ids": ids.to(torch.int32),
             "weights": torch.softmax(values, dim=1),
             "up_gate": _normal(generator, (case["experts"], 2 * width, hidden), 0.02, dtype),
             "down": _normal(generator, (case["experts"], hidden, width), 0.02, dtype),
             "residual": _normal(generator, (tokens, hidden), 1.0, dtype) if case["residual"] else None,
             "workspace": None}
    if own:
        size = _ops().token_experts_workspace(tokens, case["top"], width)
        state["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")
    return state


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "add_norm":
        state = _prepare_norm(case, generator)
    elif case["op"] == "token_experts":
        state = _prepare_experts(case, generator)
    else:
        state = _prepare_adapted(case, generator, seed)
    state["case"] = case
    return state


def _own_run(state):
    ops, case = _ops(), state["case"]
    if case["op"] == "add_norm":
        return ops.add_norm(state["x"], state["weight"], residual=state["residual"], post=state["post"],
                            gate=state["gate"], channels=state["channels"], scale=case["scale"],
                            residual_scale=case["residual_scale"], norm=case["norm"], bias=state["bias"],
                            post_bias=state["post_bias"], offset=case["offset"], eps=_EPS)
    if case["op"] == "token_experts":
        return ops.token_experts(state["x"], state["ids"], state["weights"], state["up_gate"], state["down"],
                                 activation=case["activation"], residual=state["residual"],
                                 workspace=state["workspace"])
    if case["op"] == "adapter_gated_linear":
        return ops.adapter_gated_linear(state["x"], state["weight"], state["down"], state["up"], state["adapter"],
                                        scales=state["scales"], bias=state["bias"], activation=case["activation"],
                                        workspace=state["workspace"])
    activation = None if case["activation"] == "none" else case["activation"]
    return ops.adapter_linear(state["x"], state["weight"], state["down"], state["up"], state["adapter"],
                              scales=state["scales"], bias=state["bias"], activation=activation, gate=state["gate"],
                              residual=state["residual"], workspace=state["workspace"])


def _plain_activation(y, activation):
    if activation == "silu":
        return y / (1.0 + torch.exp(-y))
    if activation == "gelu_tanh":
        return 0.5 * y * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain_norm(v, case, weight, bias):
    if case["norm"] == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(dim=1, keepdim=True) + _EPS) * (weight.float() + case["offset"])
    return v if bias is None else v + bias.float()


def _plain_add_norm(state):
    case, v = state["case"], state["x"].float()
    if state["post"] is not None:
        v = _plain_norm(v, case, state["post"], state["post_bias"])
    if state["channels"] is not None:
        v = v * state["channels"].float()
    if state["gate"] is not None:
        v = v / (1.0 + torch.exp(-state["gate"].float()))
    total = state["residual"].float() * case["residual_scale"] + v * case["scale"]
    out = _plain_norm(total, case, state["weight"], state["bias"])
    return out.to(state["x"].dtype), total.to(state["residual"].dtype)


def _plain_low_rank(state, halves):
    """The adapters' part of the product: run by run where there are few, else token by token from gathered stacks."""
    case, x, rank = state["case"], state["x"].float(), state["case"]["rank"]
    rows = case["rows"]
    if case["requests"]:
        parts = []
        for first, end, adapter in state["runs"]:
            if adapter < 0:
                parts.append(x.new_zeros(end - first, halves * rows))
                continue
            down, up = state["down"][adapter].float(), state["up"][adapter].float()
            low = (x[first:end] @ down.t()) * state["scales"][adapter]
            parts += [torch.cat([low[:, h * rank:(h + 1) * rank] @ up[h * rows:(h + 1) * rows].t() for h in range(halves)], dim=1)]
        return torch.cat(parts)
    index = state["adapter"].long()
    kept = index.clamp(min=0)
    factor = torch.where(index >= 0, state["scales"][kept], 0.0)
    low = (state["down"][kept].float() * x[:, None, :]).sum(dim=2) * factor[:, None]
    up = state["up"][kept].float()
    return torch.cat([(up[:, h * rows:(h + 1) * rows] * low[:, None, h * rank:(h + 1) * rank]).sum(dim=2) for h in range(halves)], dim=1)


def _plain_adapted(state):
    case, x = state["case"], state["x"]
    halves, rows = (2 if case["op"] == "adapter_gated_linear" else 1), case["rows"]
    y = x.float() @ state["weight"].float().t() + _plain_low_rank(state, halves)
    if state["bias"] is not None:
        y = y + state["bias"].float()
    if halves == 2:
        return (y[:, :rows] * _plain_activation(y[:, rows:], case["activation"])).to(x.dtype)
    y = _plain_activation(y, case["activation"])
    if state["gate"] is not None:
        y = y / (1.0 + torch.exp(-state["gate"].float()))
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(x.dtype)


def _plain_experts(state):
    """Token by token, its experts' rows gathered."""
    case, x = state["case"], state["x"]
    width, hidden = case["intermediate"], case["hidden"]
    out = []
    for t in range(case["tokens"]):
        ids = state["ids"][t].long()
        product = state["up_gate"][ids].float().reshape(-1, hidden) @ x[t].float()
        product = product.reshape(-1, 2 * width)
        gated = product[:, :width] * _plain_activation(product[:, width:], case["activation"])
        gated = gated * state["weights"][t][:, None]
        out.append((state["down"][ids].float() * gated[:, None, :]).sum(dim=(0, 2)))
    y = torch.stack(out)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(x.dtype)


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op == "add_norm":
        return _plain_add_norm(state)
    return _plain_experts(state) if op == "token_experts" else _plain_adapted(state)


def work(case):
    """Inputs and outputs once each - of the adapters and experts those in use (experts: as many as uniform choices
    name on average) - and the products' multiplications and additions, or a norm's few operations."""
    element, tokens = _TYPES[case["dtype"]].itemsize, case["tokens"]
    if case["op"] == "add_norm":
        width = case["width"]
        stream = element if case["stream"] == "same" else 4
        vectors = 1 + sum((case["post"], case["channels"], case["bias"], case["bias"] and case["post"]))
        moved = tokens * width * 2 * (element + stream) + vectors * width * element + (tokens * element if case["gate"] else 0)
        return {"bytes": moved, "flops": tokens * width * (12 if case["post"] else 7)}
    if case["op"] == "token_experts":
        hidden, width, experts, top = case["hidden"], case["intermediate"], case["experts"], case["top"]
        named = experts * (1.0 - (1.0 - top / experts) ** tokens)
        moved = int(named * 3 * width * hidden * element) + tokens * (hidden * element * (3 if case["residual"] else 2) + top * 8)
        return {"bytes": moved, "flops": 6 * tokens * top * hidden * width}
    halves = 2 if case["op"] == "adapter_gated_linear" else 1
    width, rows, rank = case["width"], case["rows"], case["rank"]
    used = min(case["adapters"], case["requests"] or tokens)
    moved = (tokens + halves * rows) * width * element + tokens * rows * element * (2 if case["residual"] else 1)
    moved += used * halves * rank * (width + rows) * element + (halves * rows * element if case["bias"] else 0)
    moved += tokens * 4 + case["adapters"] * 4 + (tokens * element if case["gate"] else 0)
    return {"bytes": moved, "flops": 2 * tokens * halves * (width * rows + rank * (width + rows))}


def _exact_activation(y, activation):
    if activation == "silu":
        return y * torch.special.expit(y)
    if activation == "gelu_tanh":
        return torch.nn.functional.gelu(y, approximate="tanh")
    return y


def _exact_norm(v, case, weight, bias):
    centre = v.mean(dim=1) if case["norm"] == "layer" else torch.zeros_like(v[:, 0])
    spread = torch.sqrt(torch.square(v - centre[:, None]).sum(dim=1) / v.shape[1] + _EPS)
    y = (v - centre[:, None]) / spread[:, None]
    y = y * weight.double() + y * case["offset"]
    return y + bias.double() if bias is not None else y


def _exact_add_norm(case, state):
    block = state["x"].double()
    if state["post"] is not None:
        block = _exact_norm(block, case, state["post"], state["post_bias"])
    factor = torch.full_like(block, case["scale"])
    if state["gate"] is not None:
        factor *= torch.special.expit(state["gate"].double())
    if state["channels"] is not None:
        factor *= state["channels"].double()[None, :]
    total = case["residual_scale"] * state["residual"].double() + factor * block
    return _exact_norm(total, case, state["weight"], state["bias"]), total


def _exact_adapted(case, state):
    gated = case["op"] == "adapter_gated_linear"
    x, rank, rows = state["x"].double(), case["rank"], case["rows"]
    product = torch.matmul(state["weight"].double(), x.t()).t().contiguous()
    for adapter in range(case["adapters"]):
        at = torch.nonzero(state["adapter"] == adapter).flatten()
        if at.numel() == 0:
            continue
        factor = state["scales"][adapter].double()
        for half in range(2 if gated else 1):
            down = state["down"][adapter, half * rank:(half + 1) * rank].double()
            up = state["up"][adapter, half * rows:(half + 1) * rows].double()
            part = torch.matmul(torch.matmul(x[at], down.t()), up.t()) * factor
            product[at, half * rows:(half + 1) * rows] += part
    if state["bias"] is not None:
        product += state["bias"].double()
    if gated:
        up, gate = torch.split(product, rows, dim=1)
        return (up * _exact_activation(gate, case["activation"])).contiguous()
    product = _exact_activation(product, case["activation"])
    if state["gate"] is not None:
        product = product * torch.special.expit(state["gate"].double())
    return product if state["residual"] is None else product + state["residual"].double()


def _exact_experts(case, state):
    x, width = state["x"].double(), case["intermediate"]
    out = torch.zeros_like(x) if state["residual"] is None else state["residual"].double()
    for expert in range(case["experts"]):
        at = torch.nonzero(state["ids"] == expert)
        if at.shape[0] == 0:
            continue
        rows, places = at[:, 0], at[:, 1]
        up, gate = torch.split(torch.matmul(x[rows], state["up_gate"][expert].double().t()), width, dim=1)
        product = torch.matmul(up * _exact_activation(gate, case["activation"]), state["down"][expert].double().t())
        out.index_add_(0, rows, product * state["weights"][rows, places].double()[:, None])
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "add_norm":
        return _exact_add_norm(case, state)
    if case["op"] == "token_experts":
        return _exact_experts(case, state)
    return _exact_adapted(case, state)
