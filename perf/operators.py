"""Operators on points held in 8 bits and the teacher's loss: the cases that are timed, their plain forms and their definitions in 64 bits.

  write    rows into a store of points in 8 bits: e4m3 codes, one power-of-two scale for each block of 128 coordinates of a row
  read     rows of the store as the values they stand for
  product  rows (quantised as `write` would) with the stored points: the logits of an encoder's batch against the bank
  dproduct the gradient of `product` to its rows
  loss     cross entropy of a row's logits against a teacher's top list (a graph row with its probabilities, or top logits), in one pass with its gradient
  train    the same loss forward, then its gradient from the kept statistics and each row's own upstream gradient

`own = False` computes elementary torch operations in 32 bits; `own = True` makes the framework's calls."""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 128


def listed():
    return [
        # one new point of 784 coordinates takes the place of an older one: latency counts
        {"name": "write one row", "op": "write", "n": 1, "dim": 784, "type": "f32", "capacity": 4096, "slots": True},
        # a scattered batch of short points, an odd number of them
        {"name": "write scattered", "op": "write", "n": 8191, "dim": 128, "type": "f16", "capacity": 60000, "slots": True},
        # a bank laid out in one go from an encoder's outputs
        {"name": "write bank", "op": "write", "n": 262144, "dim": 1024, "type": "bf16", "capacity": 262144, "slots": False},
        # the neighbours of a few points fetched by their ids
        {"name": "read gathered", "op": "read", "n": 1013, "dim": 784, "type": "f32", "capacity": 60000, "slots": True},
        # the whole bank read back
        {"name": "read bank", "op": "read", "n": 200000, "dim": 784, "type": "bf16", "capacity": 200000, "slots": False},
        # one query against a bank of 60 000 points of 784 coordinates
        {"name": "product one query", "op": "product", "m": 1, "n": 60000, "dim": 784, "type": "f32", "out": "f32"},
        # the logits of an odd batch against the same bank
        {"name": "product batch", "op": "product", "m": 300, "n": 60000, "dim": 784, "type": "bf16", "out": "bf16"},
        # a large batch of wide vectors against a large bank
        {"name": "product large", "op": "product", "m": 8192, "n": 16384, "dim": 4096, "type": "bf16", "out": "bf16"},
        # the batch's gradient through the bank of 60 000
        {"name": "dproduct batch", "op": "dproduct", "m": 300, "n": 60000, "dim": 784, "type": "bf16", "out": "f32"},
        # a small batch's gradient kept in 32 bits throughout
        {"name": "dproduct f32", "op": "dproduct", "m": 64, "n": 10007, "dim": 128, "type": "f32", "out": "f32"},
        # a training step's loss and gradient together, twelve neighbours a row
        {"name": "loss and gradient", "op": "loss", "rows": 4096, "cols": 32768, "k": 12, "type": "bf16", "teacher": "proba", "temperature": 1.0, "grad": True},
        # loss, then gradient under each row's own upstream gradient, from a teacher's top logits; some rows are padding
        {"name": "loss then gradient", "op": "train", "rows": 300, "cols": 60000, "k": 32, "type": "f32", "teacher": "logits", "temperature": 2.0},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["write", "read", "product", "product", "dproduct", "loss", "train"])
    kind = rng.choice(["f32", "bf16", "f16"])
    if op in ("write", "read"):
        dim = _log_int(rng, 16, 4096)
        n = _log_int(rng, 1, min(262144, (1 << 28) // dim // BYTES[kind] * 2))
        return {"op": op, "n": n, "dim": dim, "type": kind, "capacity": n + rng.randrange(1, 1000), "slots": rng.random() < 0.5}
    if op in ("product", "dproduct"):
        dim = _log_int(rng, 16, 4096)
        n = _log_int(rng, 100, 100000)
        most = (1 << 39 if op == "product" else 1 << 37) // (n * dim)
        m = _log_int(rng, 1, max(1, min(8192, most, (1 << 27) // n)))
        return {"op": op, "m": m, "n": n, "dim": dim, "type": kind, "out": rng.choice(["f32", "bf16", "f16"])}
    cols = _log_int(rng, 100, 130000)
    rows = _log_int(rng, 1, max(1, min(8192, (1 << 26) // cols)))
    case = {"op": op, "rows": rows, "cols": cols, "k": rng.randrange(1, 65), "type": kind, "teacher": rng.choice(["proba", "logits"]),
            "temperature": rng.choice([0.5, 1.0, 2.0, 4.0])}
    if op == "loss":
        case["grad"] = rng.random() < 0.7
    return case


def work(case):
    op = case["op"]
    if op in ("write", "read"):
        held = case["n"] * (case["dim"] + -(-case["dim"] // BLOCK))
        return {"bytes": held + case["n"] * case["dim"] * BYTES[case["type"]] + (4 * case["n"] if case["slots"] else 0), "flops": 0}
    if op in ("product", "dproduct"):
        m, n, dim = case["m"], case["n"], case["dim"]
        given, made = (m * dim, m * n) if op == "product" else (m * n, m * dim)
        return {"bytes": n * (dim + -(-dim // BLOCK)) + given * BYTES[case["type"]] + made * BYTES[case["out"]], "flops": 2 * m * n * dim}
    size = case["rows"] * case["cols"]
    lists = case["rows"] * (8 * case["k"] + 16)
    passes = 3 if op == "train" else 2 if case["grad"] else 1
    return {"bytes": passes * size * BYTES[case["type"]] + lists, "flops": 4 * size * (2 if passes > 1 else 1)}


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def _vectors(n, dim, kind, g):
    """Vectors of a few clusters, coordinates of unequal size: an encoder's outputs."""
    centres = torch.randn(16, dim, generator=g, device="cuda")
    spread = torch.exp(0.7 * torch.randn(dim, generator=g, device="cuda"))
    x = torch.randn(n, dim, generator=g, device="cuda").mul_(0.6)
    x += centres[torch.randint(0, 16, (n,), generator=g, device="cuda")]
    return (x * spread).to(TYPES[kind])


def _bank(x):
    """The bank as a program keeps it: the framework's store, or its codes and scale bytes."""
    if own:
        import annembed_amd as A
        store = A.Points8(x.shape[0], x.shape[1])
        store.write(x)
        return store
    codes, scales = _quantise(x)
    return {"codes": codes.view(torch.uint8), "scales": scales}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    state = dict(case)
    if op in ("write", "read"):
        n, dim, cap = case["n"], case["dim"], case["capacity"]
        if op == "write":
            state["x"] = _vectors(n, dim, case["type"], g)
            if own:
                import annembed_amd as A
                state["bank"] = A.Points8(cap, dim)
            else:
                state["bank"] = {"codes": torch.zeros(cap, dim, dtype=torch.uint8, device="cuda"),
                                 "scales": torch.zeros(cap, -(-dim // BLOCK), dtype=torch.uint8, device="cuda")}
        else:
            state["bank"] = _bank(_vectors(cap, dim, "bf16", g))
        state["ids"] = torch.randperm(cap, generator=g, device="cuda")[:n].to(torch.int32) if case["slots"] else None
    elif op == "product":
        state["bank"] = _bank(_vectors(case["n"], case["dim"], "bf16", g))
        state["x"] = _vectors(case["m"], case["dim"], case["type"], g)
    elif op == "dproduct":
        state["bank"] = _bank(_vectors(case["n"], case["dim"], "bf16", g))
        # a gradient of logits: small everywhere, larger at a few places of every row
        d = torch.randn(case["m"], case["n"], generator=g, device="cuda").mul_(1e-3)
        at = torch.randint(0, case["n"], (case["m"], 12), generator=g, device="cuda")
        state["dc"] = d.scatter_(1, at, -0.1).to(TYPES[case["type"]])
    else:
        rows, cols, k = case["rows"], case["cols"], case["k"]
        s = torch.randn(rows, cols, generator=g, device="cuda").mul_(2.0)
        state["idx"] = torch.stack([torch.randint(cols * j // k, max(cols * j // k + 1, cols * (j + 1) // k), (rows,), generator=g, device="cuda") for j in range(k)], 1).to(torch.int32)
        s.scatter_add_(1, state["idx"].long(), 6.0 * torch.rand(rows, k, generator=g, device="cuda"))
        state["logits"] = s.to(TYPES[case["type"]])
        t = torch.randn(rows, k, generator=g, device="cuda").mul_(2.0).sort(1, descending=True)[0]
        state["list"] = torch.softmax(t, 1) if case["teacher"] == "proba" else t
        # rows of a padded batch weigh nothing
        state["weight"] = (torch.rand(rows, generator=g, device="cuda") > 0.1).float() if rows > 8 else torch.ones(rows, device="cuda")
        if op == "train":
            state["dloss"] = torch.rand(rows, generator=g, device="cuda") / rows * state["weight"]
    return state


# ---- plain forms --------------------------------------------------------------------------------------------------------------


def _quantise(x):
    """e4m3 codes and scale bytes of rows: the block's scale is the smallest power of two that brings its largest magnitude to 448 or less."""
    n, dim = x.shape
    nb = -(-dim // BLOCK)
    y = torch.nn.functional.pad(x.float(), (0, nb * BLOCK - dim)).view(n, nb, BLOCK)
    fine = torch.isfinite(y)
    bits = torch.where(fine, y.abs(), 0.0).amax(2).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000).int()).clamp(min=1)
    shrink = ((254 - byte) << 23).view(torch.float32)
    y = torch.where(fine, y * shrink[:, :, None], float("nan"))
    return y.view(n, nb * BLOCK)[:, :dim].contiguous().to(torch.float8_e4m3fn), byte.to(torch.uint8)


def _values(codes, scales):
    """The values that codes and scale bytes stand for, in 32 bits."""
    scale = (scales.int() << 23).view(torch.float32).repeat_interleave(BLOCK, 1)[:, : codes.shape[1]]
    return codes.view(torch.float8_e4m3fn).float() * scale


def _softmax(state):
    """max, ln sum exp((s - max) / T) and the rows that count, in 32 bits."""
    s = state["logits"].float()
    big = s.amax(1)
    counts = (state["weight"] != 0) & (big > float("-inf"))
    safe = torch.where(counts, big, 0.0)
    lnsum = torch.log(torch.exp((s - safe[:, None]) / state["temperature"]).sum(1))
    return s, torch.where(counts, big, float("-inf")), torch.where(counts, lnsum, 0.0), counts


def _teacher(state):
    t = state["list"]
    if state["teacher"] == "proba":
        return t
    e = torch.exp((t - t.amax(1, keepdim=True)) / state["temperature"])
    return e / e.sum(1, keepdim=True)


def _loss(state, s, big, lnsum, counts):
    p = _teacher(state)
    picked = s.gather(1, state["idx"].long())
    lnq = (picked.double() - big.double()[:, None]) / state["temperature"] - lnsum.double()[:, None]
    lnp = torch.log(p.double())
    return torch.where(counts, state["weight"] * (p.double() * (lnp - lnq)).sum(1), 0.0).float()


def _gradient(state, s, big, lnsum, counts, up):
    p = _teacher(state)
    q = torch.exp((s - torch.where(counts, big, 0.0)[:, None]) / state["temperature"] - lnsum[:, None])
    d = q * p.sum(1, keepdim=True)
    d.scatter_add_(1, state["idx"].long(), -p)
    d *= (up / state["temperature"])[:, None]
    return torch.where(counts[:, None], d, 0.0).to(state["logits"].dtype)


def _plain(state):
    op = state["op"]
    if op == "write":
        codes, scales = _quantise(state["x"])
        bank, ids = state["bank"], state["ids"]
        at = slice(0, state["n"]) if ids is None else ids.long()
        bank["codes"][at] = codes.view(torch.uint8)
        bank["scales"][at] = scales
        return {"codes": bank["codes"].view(torch.float8_e4m3fn), "scales": bank["scales"]}
    if op == "read":
        bank, ids = state["bank"], state["ids"]
        at = slice(0, state["n"]) if ids is None else ids.long()
        return {"x": _values(bank["codes"][at], bank["scales"][at]).to(TYPES[state["type"]])}
    if op == "product":
        x = _values(*_quantise(state["x"]))
        return {"c": (x @ _values(**state["bank"]).T).to(TYPES[state["out"]])}
    if op == "dproduct":
        return {"dx": (state["dc"].float() @ _values(**state["bank"])).to(TYPES[state["out"]])}
    parts = _softmax(state)
    out = {"loss": _loss(state, *parts)}
    if op == "train":
        out["grad"] = _gradient(state, *parts, state["dloss"])
    elif state["grad"]:
        out["grad"] = _gradient(state, *parts, state["weight"])
    return out


def _own(state):
    import annembed_amd as A
    op = state["op"]
    if op == "write":
        store = state["bank"]
        store.write(state["x"], slots=state["ids"])
        return {"codes": store.codes(), "scales": store.scales()}
    if op == "read":
        return {"x": state["bank"].read(n=state["n"], slots=state["ids"], dtype=TYPES[state["type"]])}
    if op == "product":
        return {"c": state["bank"].product(state["x"], dtype=TYPES[state["out"]])}
    if op == "dproduct":
        return {"dx": state["bank"].product_grad(state["dc"], dtype=TYPES[state["out"]])}
    said = dict(teacher=state["teacher"], temperature=state["temperature"], row_weight=state["weight"])
    if op == "loss" and state["grad"]:
        loss, _, grad = A.teacher_loss(state["logits"], state["idx"], state["list"], grad=True, **said)
        return {"loss": loss, "grad": grad}
    loss, stats = A.teacher_loss(state["logits"], state["idx"], state["list"], **said)
    out = {"loss": loss}
    if op == "train":
        out["grad"] = A.teacher_grad(state["logits"], stats, state["idx"], state["list"], state["dloss"], teacher=state["teacher"],
                                     temperature=state["temperature"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------------------


def _power(e):
    """2^e in 64 bits, from its bits: a power computed on the GPU is off in the last of them."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _exact_points(x):
    """(values of the codes, exponents) of rows, in 64 bits: codes are the multiples of the e4m3 spacing nearest to x / 2^e, ties to even."""
    n, dim = x.shape
    values = torch.empty(n, dim, dtype=torch.float64, device=x.device)
    powers = torch.empty(n, -(-dim // BLOCK), dtype=torch.int64, device=x.device)
    for b, lo in enumerate(range(0, dim, BLOCK)):
        y = x[:, lo:lo + BLOCK].double()
        part, power = torch.frexp(y.abs().amax(1) / 448.0)
        power = torch.where(part == 0.5, power - 1, power).clamp(min=-126)
        power = torch.where(part == 0.0, -126, power)
        scale = _power(power)
        y = y / scale[:, None]
        spacing = _power((torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
        values[:, lo:lo + BLOCK] = torch.round(y / spacing) * spacing
        powers[:, b] = power
    return values, powers


def _exact_values(x):
    values, powers = _exact_points(x)
    for b in range(powers.shape[1]):
        values[:, b * BLOCK:(b + 1) * BLOCK] *= _power(powers[:, b])[:, None]
    return values


def exact(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    if op in ("write", "read"):
        n, dim, cap = case["n"], case["dim"], case["capacity"]
        x = _vectors(n, dim, case["type"], g) if op == "write" else _vectors(cap, dim, "bf16", g)
        ids = torch.randperm(cap, generator=g, device="cuda")[:n] if case["slots"] else torch.arange(n, device="cuda")
        if op == "read":
            return {"x": _exact_values(x[ids])}
        values, powers = _exact_points(x)
        codes = torch.zeros(cap, dim, dtype=torch.float64, device="cuda")
        codes[ids] = values
        scales = torch.zeros(cap, powers.shape[1], dtype=torch.int64, device="cuda")
        scales[ids] = powers + 127
        return {"codes": codes, "scales": scales}
    if op == "product":
        y = _exact_values(_vectors(case["n"], case["dim"], "bf16", g))
        x = _exact_values(_vectors(case["m"], case["dim"], case["type"], g))
        return {"c": torch.matmul(x, y.T)}
    if op == "dproduct":
        global own
        kept, own = own, False
        try:
            state = prepare(case, seed)
        finally:
            own = kept
        g.manual_seed(seed)
        y = _exact_values(_vectors(case["n"], case["dim"], "bf16", g))
        return {"dx": torch.matmul(state["dc"].double(), y)}
    state = prepare(case, seed)
    z = state["logits"].double() / case["temperature"]
    lnq = z - torch.logsumexp(z, 1, keepdim=True)
    t = state["list"].double()
    p = t if case["teacher"] == "proba" else torch.softmax(t / case["temperature"], 1)
    at = state["idx"].long()
    out = {"loss": state["weight"].double() * (p * (torch.log(p) - lnq.gather(1, at))).sum(1)}
    if op == "train" or case["grad"]:
        up = state["dloss"] if op == "train" else state["weight"]
        full = torch.zeros_like(z).scatter_add_(1, at, p)
        out["grad"] = (torch.exp(lnq) * p.sum(1, keepdim=True) - full) * (up.double() / case["temperature"])[:, None]
    return out
