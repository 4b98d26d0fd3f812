"""Cases of the products whose weight matrix is chosen by the row: grouped_matmul, its weight gradient, lora_matmul.

``own`` false: the operators in their plain form (padded batches and torch.bmm in 32 bits, rounded once);
``own`` true: the library's kernels, called as a user calls them.
"""

import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One token of a mixture-of-experts layer while it is being generated: two experts' matrices, one row each.
        {"name": "experts_one_token", "op": "forward", "rows": 2, "groups": 8, "used": 2, "k": 4096, "n": 2048,
         "type": "bf16", "padding": 0},
        # A batch of 64 generated tokens, four of 64 experts each, on a buffer sized for 96 tokens; some experts idle.
        {"name": "experts_batch", "op": "forward", "rows": 256, "groups": 64, "used": 60, "k": 2048, "n": 1024,
         "type": "bf16", "padding": 128},
        # A prompt, or the forward pass of a training step: 8192 tokens to two of 16 experts each.
        {"name": "experts_prompt", "op": "forward", "rows": 16384, "groups": 16, "used": 16, "k": 2048, "n": 4096,
         "type": "bf16", "padding": 0},
        # Ragged in every size, in the other type.
        {"name": "experts_ragged", "op": "forward", "rows": 5001, "groups": 32, "used": 29, "k": 1544, "n": 1160,
         "type": "fp16", "padding": 7},
        # Backward of a layer of small experts, towards its input: the same weights, read as transposed views.
        {"name": "experts_input_gradient", "op": "input_gradient", "rows": 16384, "groups": 64, "used": 64, "k": 1024,
         "n": 2048, "type": "bf16", "padding": 0},
        # Backward of the prompt-sized layer towards its weights.
        {"name": "experts_weight_gradient", "op": "weight_gradient", "rows": 16384, "groups": 16, "used": 16, "k": 2048,
         "n": 4096, "type": "bf16", "padding": 0},
        # The same with short groups: the gradient's own size is most of the work.
        {"name": "experts_weight_gradient_few", "op": "weight_gradient", "rows": 2003, "groups": 64, "used": 61,
         "k": 1024, "n": 776, "type": "fp16", "padding": 5},
        # One request with an adapter, one token.
        {"name": "adapters_one_token", "op": "adapters", "rows": 1, "requests": 1, "bare": 0, "adapters": 16, "k": 4096,
         "n": 4096, "rank": 16, "type": "bf16", "padding": 0},
        # 64 requests, a token each, under 32 adapters, eight requests without one.
        {"name": "adapters_batch", "op": "adapters", "rows": 64, "requests": 64, "bare": 8, "adapters": 32, "k": 4096,
         "n": 4096, "rank": 16, "type": "bf16", "padding": 0},
        # A few prompts at once, one of them without an adapter.
        {"name": "adapters_prompts", "op": "adapters", "rows": 8192, "requests": 6, "bare": 1, "adapters": 4, "k": 4096,
         "n": 4096, "rank": 32, "type": "bf16", "padding": 0},
        # Prompts and generated tokens mixed, ragged in every size, in the other type.
        {"name": "adapters_ragged", "op": "adapters", "rows": 1533, "requests": 40, "bare": 5, "adapters": 8, "k": 1000,
         "n": 2056, "rank": 24, "type": "fp16", "padding": 3},
        # Backward of a layer under adapters towards its input: transposed views of all three matrices.
        {"name": "adapters_input_gradient", "op": "adapters_input_gradient", "rows": 4096, "requests": 4, "bare": 0,
         "adapters": 4, "k": 4096, "n": 2048, "rank": 64, "type": "bf16", "padding": 0},
    ]


def _spread(rng, low, high, step=1):
    """A whole multiple of `step` in [low, high], spread over the logarithm."""
    value = low * (high / low) ** rng.random()
    return min(high, max(low, int(round(value / step)) * step))


def draw(rng):
    op = rng.choice(["forward", "forward", "input_gradient", "weight_gradient", "adapters", "adapters",
                     "adapters_input_gradient"])
    kind = rng.choice(["bf16", "fp16"])
    k, n = _spread(rng, 256, 4096, 8), _spread(rng, 256, 4096, 8)
    padding = rng.choice([0, 0, rng.randint(1, 40)])
    if op.startswith("adapters"):
        rows = _spread(rng, 1, 8192)
        requests = _spread(rng, 1, min(rows, 128))
        return {"op": op, "rows": rows, "requests": requests, "bare": rng.randint(0, requests // 4),
                "adapters": rng.randint(1, 32), "k": k, "n": n, "rank": _spread(rng, 8, 128, 8), "type": kind,
                "padding": padding}
    groups = _spread(rng, 2, 128)
    rows = _spread(rng, 1, 16384)
    used = max(1, min(rows, groups) - rng.randint(0, groups // 8))
    # no costlier than the largest listed case, in products and in bytes of weights (in 32 bits, as the plain form has them)
    while rows * k * n > 16384 * 2048 * 4096 or groups * k * n > 64 * 2048 * 1024:
        k, n = max(256, k // 2 // 8 * 8), max(256, n // 2 // 8 * 8)
    return {"op": op, "rows": rows, "groups": groups, "used": used, "k": k, "n": n, "type": kind, "padding": padding}


def _lengths(rng, rows, parts):
    """`rows` dealt to `parts` runs, one at least to each, uneven like a router's choices or a batch of prompts."""
    weights = [rng.uniform(0.5, 1.5) for _ in range(parts)]
    spare, total = rows - parts, sum(weights)
    lengths = [1 + int(spare * w / total) for w in weights]
    for i in range(rows - sum(lengths)):
        lengths[i % parts] += 1
    return lengths


def _offsets(lengths):
    bounds = [0]
    for length in lengths:
        bounds.append(bounds[-1] + length)
    return bounds


def _inputs(case, seed):
    """Tensors of a case, made from the seed alone (also what `exact` starts from)."""
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]
    rows, k, n = case["rows"], case["k"], case["n"]
    total = rows + case["padding"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(kind)

    if case["op"].startswith("adapters"):
        lengths = _lengths(rng, rows, case["requests"])
        dressed = case["requests"] - case["bare"]
        ids = rng.sample(range(case["adapters"]), min(dressed, case["adapters"]))
        ids += [rng.randrange(case["adapters"]) for _ in range(dressed - len(ids))] + [-1] * case["bare"]
        rng.shuffle(ids)
        rank = case["rank"]
        state = {
            # the projection's weight and the adapters' two, as a model holds them
            "weight": normal(k, n, scale=k ** -0.5),
            "down": normal(case["adapters"], k, rank, scale=k ** -0.5),
            "up": normal(case["adapters"], rank, n, scale=rank ** -0.5),
            "scales": torch.rand(case["adapters"], generator=g, device="cuda") + 0.5,
            "adapters": torch.tensor(ids, dtype=torch.int32, device="cuda"),
        }
        inner = k if case["op"] == "adapters" else n
    else:
        counts = _lengths(rng, rows, case["used"])
        lengths = [0] * case["groups"]
        for place, count in zip(rng.sample(range(case["groups"]), case["used"]), counts):
            lengths[place] = count
        state = {}
        if case["op"] == "weight_gradient":
            state["grad"] = normal(total, n)
        else:
            state["weight"] = normal(case["groups"], k, n, scale=k ** -0.5)
        inner = n if case["op"] == "input_gradient" else k
    state["x"] = normal(total, inner)
    state["offsets"] = torch.tensor(_offsets(lengths), dtype=torch.int32, device="cuda")
    state["lengths"] = lengths
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["op"], state["rows"] = case["op"], case["rows"]
    state["longest"] = max(state["lengths"])
    kind, total = state["x"].dtype, state["x"].shape[0]
    if case["op"] == "weight_gradient":
        shape = (case["groups"], case["k"], case["n"])
    else:
        shape = (total, case["k"] if case["op"].endswith("input_gradient") else case["n"])
    state["output"] = torch.zeros(shape, dtype=kind, device="cuda")  # rows behind the last group stay zero
    return state


def run(state):
    if own:
        return _call(state)
    return _plain(state)


def _call(state):
    from ninetoothed_b200.torch_ops import ops

    x, offsets, output = state["x"], state["offsets"], state["output"]
    if state["op"] == "forward":
        ops.grouped_matmul(x, state["weight"], offsets, output)
    elif state["op"] == "input_gradient":
        ops.grouped_matmul(x, state["weight"].transpose(1, 2), offsets, output)
    elif state["op"] == "weight_gradient":
        ops.grouped_matmul_rhs_grad(x, state["grad"], offsets, output)
    elif state["op"] == "adapters":
        ops.lora_matmul(x, state["weight"], state["down"], state["up"], state["scales"], offsets, state["adapters"],
                        output)
    else:
        ops.lora_matmul(x, state["weight"].t(), state["up"].transpose(1, 2), state["down"].transpose(1, 2),
                        state["scales"], offsets, state["adapters"], output)
    return output


def _plain(state):
    x, offsets, rows = state["x"], state["offsets"].long(), state["rows"]
    # rows of every run side by side, padded to the longest run
    place = offsets[:-1, None] + torch.arange(state["longest"], device=x.device)
    held = place < offsets[1:, None]
    place = torch.where(held, place, 0)
    runs = torch.where(held[..., None], x[place].float(), 0.0)
    if state["op"] == "weight_gradient":
        grads = torch.where(held[..., None], state["grad"][place].float(), 0.0)
        return torch.bmm(runs.transpose(1, 2), grads).to(x.dtype)
    if state["op"] in ("forward", "input_gradient"):
        weight = state["weight"].float()
        products = torch.bmm(runs, weight if state["op"] == "forward" else weight.transpose(1, 2))[held]
    else:
        weight, first, second = state["weight"], state["down"], state["up"]
        if state["op"] != "adapters":
            weight, first, second = weight.t(), second.transpose(1, 2), first.transpose(1, 2)
        ids = state["adapters"].long()
        which = ids.clamp(min=0)
        scales = torch.where(ids >= 0, state["scales"][which], 0.0)
        low = torch.bmm(runs, first[which].float()) * scales[:, None, None]
        products = torch.matmul(x[:rows].float(), weight.float()) + torch.bmm(low, second[which].float())[held]
    output = torch.zeros_like(state["output"])
    output[:rows] = products.to(x.dtype)
    return output


def exact(case, seed):
    """The operators from their definitions in 64 bits, run by run."""
    state = _inputs(case, seed)
    x = state["x"].double()
    bounds = _offsets(state["lengths"])
    spans = list(zip(bounds[:-1], bounds[1:]))
    if case["op"] == "weight_gradient":
        grad = state["grad"].double()
        return torch.stack([x[a:b].t() @ grad[a:b] for a, b in spans])
    if case["op"] in ("forward", "input_gradient"):
        width = case["n"] if case["op"] == "forward" else case["k"]
        result = torch.zeros(x.shape[0], width, dtype=torch.float64, device=x.device)
        for group, (a, b) in enumerate(spans):
            matrix = state["weight"][group].double()
            result[a:b] = x[a:b] @ (matrix if case["op"] == "forward" else matrix.t())
        return result
    weight = state["weight"].double()
    forward = case["op"] == "adapters"
    result = torch.zeros(x.shape[0], case["n"] if forward else case["k"], dtype=torch.float64, device=x.device)
    for (a, b), adapter in zip(spans, state["adapters"].tolist()):
        result[a:b] = x[a:b] @ (weight if forward else weight.t())
        if adapter >= 0:
            down, up = state["down"][adapter].double(), state["up"][adapter].double()
            low = x[a:b] @ down @ up if forward else x[a:b] @ up.t() @ down.t()
            result[a:b] += state["scales"][adapter].double() * low
    return result


def work(case):
    rows, k, n = case["rows"], case["k"], case["n"]
    if case["op"].startswith("adapters"):
        dressed = case["requests"] - case["bare"]
        with_adapter = rows * dressed // case["requests"]
        weights = k * n + min(dressed, case["adapters"]) * case["rank"] * (k + n)
        return {"bytes": 2 * (rows * (k + n) + weights), "flops": 2 * rows * k * n + 2 * with_adapter * case["rank"] * (k + n)}
    if case["op"] == "weight_gradient":
        return {"bytes": 2 * (rows * (k + n) + case["groups"] * k * n), "flops": 2 * rows * k * n}
    return {"bytes": 2 * (rows * (k + n) + case["used"] * k * n), "flops": 2 * rows * k * n}
