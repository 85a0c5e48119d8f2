"""The operators of an optimiser step behind the gradient exchange, at the sizes their users bring.

  momentum   momentum_update: a gradient bucket (dense, as the hook returns it) goes into the momentum, and the update
             that the step applies comes out.
  lists      momentum_update_sparse: the same from ascending (index, value) lists, as the merge and the second exchange
             leave them: several of one length each, or one whose length is known on the device alone.
  product    product: alpha a b + beta c, with b stored either way round; `symmetric` for a matrix with its own transpose.
  orthogonal orthogonalize: an update made orthogonal by five Newton-Schulz steps; one matrix, or a stack of them.
  step       orthogonal_step: the same, applied to the weights.

Everything is drawn from a seeded generator on the GPU.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "int32": 4, "int64": 8}
_STEPS = 5
_A, _B, _C = 3.4445, -4.7750, 2.0315
_EPS = 1e-7
_MU = 0.95


def listed():
    return [
        # one small matrix's gradient, dense fp32: latency only
        {"name": "momentum_590k_fp32", "kind": "momentum", "n": 768 * 768, "grad": "fp32", "state": "fp32", "nesterov": True},
        # a 128 MB bucket of bf16 gradients, as the hook returns it
        {"name": "momentum_62m_bf16", "kind": "momentum", "n": 61953360, "grad": "bf16", "state": "fp32", "nesterov": True},
        # the same bucket from the sixteen lists of the second exchange: int64 indices, bf16 values, 5 % of the elements
        {"name": "lists_62m_x16", "kind": "lists", "n": 61953360, "lists": 16, "density": 0.05, "index": "int64",
         "values": "bf16", "state": "fp32", "known": True, "nesterov": True},
        # an embedding and a decoder layer of an 8B model as one bucket, one merged list: its length is on the device
        {"name": "lists_743m_x1", "kind": "lists", "n": 743440384, "lists": 1, "density": 0.004, "index": "int32",
         "values": "fp32", "state": "fp32", "known": False, "nesterov": True},
        # odd sizes, rows that no wide load divides
        {"name": "product_odd_fp16", "kind": "product", "m": 257, "n": 511, "k": 1023, "type": "fp16", "result": "fp32",
         "b_rows": "n", "residual": True, "symmetric": False},
        # a square weight's product with a residual, b stored as it is multiplied
        {"name": "product_4096_bf16", "kind": "product", "m": 4096, "n": 4096, "k": 4096, "type": "bf16", "result": "bf16",
         "b_rows": "k", "residual": True, "symmetric": False},
        # a wide update with its own transpose
        {"name": "product_gram_4096x14336", "kind": "product", "m": 4096, "n": 4096, "k": 14336, "type": "fp16",
         "result": "fp16", "b_rows": "n", "residual": False, "symmetric": True},
        # a small tall matrix of odd sizes in fp32: latency
        {"name": "orthogonal_1023x65_fp32", "kind": "orthogonal", "stack": 1, "m": 1023, "n": 65, "type": "fp32"},
        # one projection of each of the twelve layers of a small model
        {"name": "orthogonal_12x768x768", "kind": "orthogonal", "stack": 12, "m": 768, "n": 768, "type": "bf16"},
        # a wide projection of an 8B model's feed-forward
        {"name": "orthogonal_4096x14336", "kind": "orthogonal", "stack": 1, "m": 4096, "n": 14336, "type": "bf16"},
        # key and value projection of an 8B model, fp32 weights (and so fp32 precision throughout)
        {"name": "step_1024x4096_fp32", "kind": "step", "stack": 1, "m": 1024, "n": 4096, "type": "fp32", "decay": 0.1},
        # query and output projection of an 8B model, bf16 weights
        {"name": "step_4096x4096_bf16", "kind": "step", "stack": 1, "m": 4096, "n": 4096, "type": "bf16", "decay": 0.1},
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["momentum", "lists", "product", "orthogonal", "orthogonal", "step"])
    if kind == "momentum":
        return {"kind": kind, "n": _spread(rng, 100_000, 400_000_000), "grad": rng.choice(["fp32", "bf16"]),
                "state": rng.choice(["fp32", "fp32", "bf16"]), "nesterov": rng.random() < 0.7}
    if kind == "lists":
        n = _spread(rng, 100_000, 400_000_000)
        return {"kind": kind, "n": n, "lists": rng.choice([1, 2, 4, 8, 16, 32]),
                "density": math.exp(rng.uniform(math.log(0.002), math.log(0.1))), "index": rng.choice(["int32", "int64"]),
                "values": rng.choice(["fp32", "bf16"]), "state": "fp32", "known": rng.random() < 0.5,
                "nesterov": rng.random() < 0.7}
    if kind == "product":
        m, n, k = (_spread(rng, 64, 6000) for _ in range(3))
        if rng.random() < 0.5:
            m, n, k = (-(-v // 64) * 64 for v in (m, n, k))
        symmetric = rng.random() < 0.3
        return {"kind": kind, "m": m, "n": m if symmetric else n, "k": k, "type": rng.choice(["bf16", "fp16"]),
                "result": rng.choice(["bf16", "fp16", "fp32"]), "b_rows": "n" if symmetric else rng.choice(["n", "k"]),
                "residual": rng.random() < 0.6 and not symmetric, "symmetric": symmetric}
    m, n = _spread(rng, 48, 4096), _spread(rng, 48, 6000)
    if rng.random() < 0.5:
        m, n = -(-m // 64) * 64, -(-n // 64) * 64
    if rng.random() < 0.5:
        m, n = n, m
    stack = max(1, min(rng.choice([1, 1, 2, 5, 12]), 24_000_000 // (m * n)))
    case = {"kind": kind, "stack": stack, "m": m, "n": n, "type": rng.choice(["bf16", "bf16", "fp32", "fp16"])}
    return case if kind == "orthogonal" else {**case, "type": rng.choice(["bf16", "fp32"]), "decay": rng.choice([0.0, 0.1])}


# ------------------------------------------------------------------ inputs


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, gen, dtype, scale=1.0):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def _update(stack, m, n, gen):
    """What a momentum holds: a few directions that many batches agree on, and noise of about the same size."""
    r = max(1, min(m, n) // 32)
    strong = torch.randn(stack, m, r, generator=gen, device="cuda") * torch.logspace(0, -1, r, device="cuda")
    x = torch.bmm(strong, torch.randn(stack, r, n, generator=gen, device="cuda"))
    x /= x.square().mean(dim=(1, 2), keepdim=True).sqrt()
    x += torch.randn(stack, m, n, generator=gen, device="cuda")
    return x * 1e-3


def prepare(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "momentum":
        n = case["n"]
        return {**case, "grads": _normal(n, gen, _TYPES[case["grad"]], 1e-3),
                "momentum": _normal(n, gen, _TYPES[case["state"]], 4e-3)}
    if kind == "lists":
        n, lists = case["n"], case["lists"]
        # every list holds indices of its own, as the partitions' do: list p those that are p modulo the lists' number,
        # ascending, one in every stretch of `gap`
        per = max(1, int(n * case["density"] / lists))
        gap = n // lists // per
        at = torch.randint(0, gap, (lists, per), generator=gen, device="cuda") + torch.arange(per, device="cuda") * gap
        index = at * lists + torch.arange(lists, device="cuda")[:, None]
        state = {**case, "index": list(index.to(getattr(torch, case["index"]))),
                 "values": list(_normal((lists, per), gen, _TYPES[case["values"]], 1e-3)), "counts": None,
                 "momentum": _normal(n, gen, _TYPES[case["state"]], 4e-3)}
        if not case["known"]:  # the lists' last entries are room that was not needed
            used = torch.randint(max(1, per * 3 // 4), per + 1, (lists,), generator=gen, device="cuda")
            state["counts"] = used
            for p in range(lists):
                unused = torch.arange(per, device="cuda") >= used[p]
                state["index"][p].masked_fill_(unused, -1)
                state["values"][p].masked_fill_(unused, float("nan"))
        return state
    if kind == "product":
        m, n, k, dtype = case["m"], case["n"], case["k"], _TYPES[case["type"]]
        a = _normal((m, k), gen, dtype)
        if case["symmetric"]:
            b = a.t()
        else:
            b = _normal((n, k), gen, dtype).t() if case["b_rows"] == "n" else _normal((k, n), gen, dtype)
        c = _normal((m, n), gen, _TYPES[case["result"]]) if case["residual"] else None
        return {**case, "a": a, "b": b, "c": c, "alpha": 0.5 / math.sqrt(k), "beta": 0.75}
    stack, m, n, dtype = case["stack"], case["m"], case["n"], _TYPES[case["type"]]
    state = {**case, "update": _update(stack, m, n, gen).to(dtype)}
    if kind == "step":
        state["weight"] = _normal((stack, m, n), gen, dtype, 0.02)
        state["lr"] = 0.02
        state["scale"] = 0.2 * math.sqrt(max(m, n))
    return state


# -------------------------------------------------------------- plain forms


def _plain_momentum(momentum, g, nesterov):
    moved = momentum.float() * _MU + g
    momentum.copy_(moved)
    return {"momentum": momentum, "update": (g + moved * _MU if nesterov else moved).to(torch.bfloat16)}


def _plain_lists(state):
    index, value = torch.stack(state["index"]).long(), torch.stack(state["values"]).float()
    if state["counts"] is not None:
        there = torch.arange(index.shape[1], device=index.device)[None] < state["counts"][:, None]
        index, value = torch.where(there, index, 0), torch.where(there, value, 0.0)
    g = torch.zeros(state["n"], dtype=torch.float32, device=index.device)
    return g.index_add_(0, index.reshape(-1), value.reshape(-1))


def _plain_product(state):
    d = torch.matmul(state["a"].float(), state["b"].float()) * state["alpha"]
    if state["c"] is not None:
        d += state["c"].float() * state["beta"]
    return d.to(_TYPES[state["result"]])


def _plain_orthogonal(update):
    x = update.float()
    turned = x.shape[1] > x.shape[2]
    if turned:
        x = x.transpose(1, 2).contiguous()
    x = x / (torch.sqrt(torch.sum(x * x, dim=(1, 2), keepdim=True)) + _EPS)
    for _ in range(_STEPS):
        gram = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = _A * x + torch.matmul(_B * gram + _C * torch.matmul(gram, gram), x)
    return x.transpose(1, 2) if turned else x


def run(state):
    kind = state["kind"]
    if own:
        import zen_repro_amd as zen
        if kind == "momentum":
            u = zen.momentum_update(state["momentum"], state["grads"], _MU, state["nesterov"], dtype=torch.bfloat16)
            return {"momentum": state["momentum"], "update": u}
        if kind == "lists":
            u, _ = zen.momentum_update_sparse(state["momentum"], state["index"], state["values"], _MU, state["nesterov"],
                                              counts=state["counts"], dtype=torch.bfloat16)
            return {"momentum": state["momentum"], "update": u}
        if kind == "product":
            return zen.product(state["a"], state["b"], residual=state["c"], alpha=state["alpha"], beta=state["beta"],
                               symmetric=state["symmetric"], dtype=_TYPES[state["result"]])
        if kind == "orthogonal":
            return zen.orthogonalize(state["update"], steps=_STEPS, coefficients=(_A, _B, _C), eps=_EPS)
        return zen.orthogonal_step(state["weight"], state["update"], state["lr"], weight_decay=state["decay"],
                                   scale=state["scale"], steps=_STEPS, coefficients=(_A, _B, _C), eps=_EPS)
    if kind == "momentum":
        return _plain_momentum(state["momentum"], state["grads"].float(), state["nesterov"])
    if kind == "lists":
        return _plain_momentum(state["momentum"], _plain_lists(state), state["nesterov"])
    if kind == "product":
        return _plain_product(state)
    o = _plain_orthogonal(state["update"])
    if kind == "orthogonal":
        return o.to(state["update"].dtype).contiguous()
    w = state["weight"]
    w.copy_(w.float() * (1.0 - state["lr"] * state["decay"]) - o * (state["lr"] * state["scale"]))
    return w


# ------------------------------------------------------------- 64-bit answers


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("momentum", "lists"):
        if kind == "momentum":
            g = s["grads"].double()
        else:
            g = torch.zeros(case["n"], dtype=torch.float64, device="cuda")
            for p in range(case["lists"]):
                used = case["n"] if s["counts"] is None else int(s["counts"][p])
                g[s["index"][p][:used].long()] += s["values"][p][:used].double()
        m = torch.add(g, s["momentum"].double(), alpha=_MU)
        return {"momentum": m, "update": torch.add(g, m, alpha=_MU) if case["nesterov"] else m}
    if kind == "product":
        d = s["alpha"] * (s["a"].double() @ s["b"].double())
        return d if s["c"] is None else d + s["beta"] * s["c"].double()
    answer = []
    for u in s["update"].double():
        x = u if u.shape[0] <= u.shape[1] else u.T.contiguous()
        x = x / (torch.linalg.matrix_norm(x) + _EPS)
        for _ in range(_STEPS):
            xx = x @ x.T.contiguous()
            p = _C * (xx @ xx) + _B * xx
            p.diagonal().add_(_A)
            x = p @ x
        answer.append(x if u.shape[0] <= u.shape[1] else x.T.contiguous())
    o = torch.stack(answer)
    if kind == "orthogonal":
        return o
    return s["weight"].double() * (1.0 - s["lr"] * case["decay"]) - s["lr"] * s["scale"] * o


# ------------------------------------------------------------------- the floor


def work(case):
    kind = case["kind"]
    if kind == "momentum":
        return {"bytes": case["n"] * (2 * _BYTES[case["state"]] + _BYTES[case["grad"]] + 2), "flops": 4 * case["n"]}
    if kind == "lists":
        entries = int(case["n"] * case["density"] / case["lists"]) * case["lists"] * (1.0 if case["known"] else 0.875)
        return {"bytes": case["n"] * (2 * _BYTES[case["state"]] + 2)
                + entries * (_BYTES[case["index"]] + _BYTES[case["values"]]), "flops": 3 * case["n"]}
    if kind == "product":
        m, n, k = case["m"], case["n"], case["k"]
        size, out = _BYTES[case["type"]], _BYTES[case["result"]]
        return {"bytes": (m * k + (0 if case["symmetric"] else k * n)) * size + m * n * out * (2 if case["residual"] else 1),
                "flops": m * n * k * (1 if case["symmetric"] else 2)}  # a symmetric result is one half and its mirror image
    small, large = sorted((case["m"], case["n"]))
    size = _BYTES[case["type"]] * case["stack"] * small * large
    return {"bytes": size * (2 if kind == "orthogonal" else 3),
            "flops": case["stack"] * _STEPS * (3 * small * small * large + small ** 3)}
