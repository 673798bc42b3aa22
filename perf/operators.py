"""The parts of an int8 mixture-of-experts layer, as cases that can be timed and compared.

``kind`` says which operator a case calls:

  linear     ``w8a8_int8_matmul``: int8 activations with one scale per token times an int8 weight with one
             scale per output channel
  grouped    ``w8a8_int8_grouped_mm``: the same for rows that are sorted by expert, one weight per expert
  permute    ``moe_permute``: every token's row copied to the places of its experts; with ``train`` the gradient too
  unpermute  ``moe_unpermute``: the experts' rows weighted and summed per token; with ``train`` the gradients too

Activations are N(0, 1) and weights N(0, 0.02) before they are quantised; experts are drawn evenly, as a router
with a balancing term does; router weights are a softmax over the chosen experts.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "int8": torch.int8}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4, "int8": 1}
# (outputs, inputs) of the linear layers: Llama-3-8B, and the projections of DeepSeek-V3
LINEAR = ((6144, 4096), (4096, 4096), (28672, 4096), (4096, 14336), (2112, 7168), (24576, 7168), (7168, 2048))
# hidden size, intermediate size, experts, experts per token
DEEPSEEK = (7168, 2048, 256, 8)
MIXTRAL = (4096, 14336, 8, 2)


def listed():
    return [
        # One token through a qkv projection: launches, the host path and the stream of the weight.
        {"name": "linear_1x6144", "kind": "linear", "m": 1, "n": 6144, "k": 4096, "dtype": "bf16", "bias": False},
        # A decode batch through a gate_up projection: the weight has to be streamed.
        {"name": "linear_16x28672", "kind": "linear", "m": 16, "n": 28672, "k": 4096, "dtype": "bf16", "bias": False},
        # A short prompt of odd length through a projection with bias.
        {"name": "linear_1037x6144", "kind": "linear", "m": 1037, "n": 6144, "k": 4096, "dtype": "fp16", "bias": True},
        # A prefill batch through a down projection: tensor cores.
        {"name": "linear_8192x4096", "kind": "linear", "m": 8192, "n": 4096, "k": 14336, "dtype": "bf16", "bias": False},
        # A decode batch of 32 tokens in the first product of 256 experts: a row or two for each of many weights.
        {"name": "grouped_256x4096", "kind": "grouped", "m": 256, "n": 4096, "k": 7168, "groups": 256, "dtype": "bf16"},
        # A prefill chunk of odd length, sorted, in the second product of 8 large experts.
        {"name": "grouped_16382x4096", "kind": "grouped", "m": 16382, "n": 4096, "k": 14336, "groups": 8, "dtype": "bf16"},
        # A decode batch sorted for its experts: latency.
        {"name": "permute_64", "kind": "permute", "tokens": 64, "hidden": 7168, "experts": 256, "topk": 8,
         "dtype": "bf16", "train": False},
        # A prefill batch that was quantised per token, sorted with its scales.
        {"name": "permute_int8_8192", "kind": "permute", "tokens": 8192, "hidden": 7168, "experts": 256, "topk": 8,
         "dtype": "int8", "train": False},
        # A training batch of odd length, forward and backward.
        {"name": "permute_train_4093", "kind": "permute", "tokens": 4093, "hidden": 4096, "experts": 8, "topk": 2,
         "dtype": "bf16", "train": True},
        # A decode batch back in token order: latency.
        {"name": "unpermute_64", "kind": "unpermute", "tokens": 64, "hidden": 7168, "experts": 256, "topk": 8,
         "dtype": "bf16", "train": False},
        # A prefill chunk of odd length back in token order.
        {"name": "unpermute_16381", "kind": "unpermute", "tokens": 16381, "hidden": 4096, "experts": 8, "topk": 2,
         "dtype": "fp16", "train": False},
        # A training batch of a model with many experts, forward and backward: gradients of rows and router weights.
        {"name": "unpermute_train_8192", "kind": "unpermute", "tokens": 8192, "hidden": 7168, "experts": 256, "topk": 8,
         "dtype": "bf16", "train": True},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("linear", "linear", "grouped", "grouped", "permute", "permute", "unpermute", "unpermute"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind == "linear":
        n, k = rng.choice(LINEAR)
        if rng.random() < 0.3:  # outputs and inputs of no tile's size
            n, k = _log_int(rng, 1, 16384), 16 * _log_int(rng, 1, 512)
        return {"kind": kind, "m": _log_int(rng, 1, 8192), "n": n, "k": k, "dtype": dtype, "bias": rng.random() < 0.3}
    hidden, inter, experts, topk = rng.choice((DEEPSEEK, MIXTRAL))
    if kind == "grouped":
        n, k = rng.choice(((2 * inter, hidden), (hidden, inter)))
        most = min(16384, int(1.9e12 / (2.0 * n * k)))
        return {"kind": kind, "m": _log_int(rng, 1, most), "n": n, "k": k,
                "groups": experts if rng.random() < 0.7 else _log_int(rng, 1, experts), "dtype": dtype}
    if rng.random() < 0.4:  # other layers: odd numbers of experts, any number of experts per token
        hidden, experts = 8 * _log_int(rng, 8, 1024), _log_int(rng, 1, 320)
        topk = rng.randint(1, min(10, experts))
    train = rng.random() < 0.5
    if kind == "permute" and not train and rng.random() < 0.4:
        dtype = "int8"
    most = 8192 * 7168 * 8 * 2 // (hidden * topk * BYTES[dtype])
    return {"kind": kind, "tokens": _log_int(rng, 1, min(16384, most)), "hidden": hidden, "experts": experts,
            "topk": topk, "dtype": dtype, "train": train}


# ---- inputs ---------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _quantized(x):
    """fp32 [rows, k] -> int8 values and one fp32 scale per row."""
    s = x.abs().amax(-1).clamp_min(1e-10) / 127.0
    return (x / s[:, None]).round().clamp(-128, 127).to(torch.int8), s


def _route(g, tokens, experts, topk):
    """Distinct experts of every token, int32 [tokens, topk]."""
    return torch.rand(tokens, experts, device="cuda", generator=g).topk(topk, dim=1).indices.to(torch.int32)


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "linear":
        a, a_s = _quantized(_randn(g, case["m"], case["k"]))
        b, b_s = _quantized(_randn(g, case["n"], case["k"]) * 0.02)
        bias = _randn(g, case["n"]).to(DTYPES[case["dtype"]]) if case["bias"] else None
        return {"case": case, "a": a, "b": b, "a_s": a_s[:, None], "b_s": b_s, "bias": bias}
    if kind == "grouped":
        m, n, k, groups = case["m"], case["n"], case["k"], case["groups"]
        a, a_s = _quantized(_randn(g, m, k))
        b = torch.empty(groups, n, k, dtype=torch.int8, device="cuda")
        b_s = torch.empty(groups, n, device="cuda")
        for e in range(groups):
            b[e], b_s[e] = _quantized(_randn(g, n, k) * 0.02)
        rows = torch.randint(0, groups, (m,), device="cuda", generator=g)
        offs = torch.bincount(rows, minlength=groups).cumsum(0).to(torch.int32)
        return {"case": case, "a": a, "b": b, "a_s": a_s[:, None], "b_s": b_s, "offs": offs}
    tokens, hidden, experts, topk = case["tokens"], case["hidden"], case["experts"], case["topk"]
    dtype, train = DTYPES[case["dtype"]], case["train"]
    ids = _route(g, tokens, experts, topk)
    state = {"case": case, "ids": ids}
    if kind == "permute":
        x = _randn(g, tokens, hidden)
        state["scale"] = None
        if dtype == torch.int8:
            x, s = _quantized(x)
            state["scale"] = s[:, None]
        state["x"] = x.to(dtype).requires_grad_(train)
        if train:
            state["d_rows"] = _randn(g, tokens * topk, hidden).to(dtype)
        return state
    state["rows"] = _randn(g, tokens * topk, hidden).to(dtype).requires_grad_(train)
    state["weights"] = _randn(g, tokens, topk).softmax(1).requires_grad_(train)
    if train:
        state["d_out"] = _randn(g, tokens, hidden).to(dtype)
    if own:
        import flag_gems

        # the plan that the tokens were sorted with, kept until their way back
        state["plan"] = flag_gems.moe_permute(torch.zeros(tokens, 16, dtype=torch.int8, device="cuda"), ids, experts)[2]
    else:
        state["plan"] = _plan(ids, experts)[1]
    return state


# ---- the operators in plain torch -------------------------------------------------------------
def _plan(ids, experts):
    """The ends of the experts' rows, the row of every route slot, and the slot of every row."""
    flat = ids.reshape(-1).long()
    slot_of_row = torch.argsort(flat, stable=True)
    row_of_slot = torch.empty_like(slot_of_row)
    row_of_slot[slot_of_row] = torch.arange(flat.numel(), device=flat.device)
    ends = torch.bincount(flat, minlength=experts).cumsum(0).to(torch.int32)
    return ends, row_of_slot.reshape(ids.shape), slot_of_row


def _product(a, b, a_s, b_s, bias, dtype):
    # sums of int8 products pass 2^24: held in 64 bits, where they are whole
    c = (a.double() @ b.double().t()).float() * a_s * b_s
    if bias is not None:
        c = c + bias.float()
    return c.to(dtype)


def _run_plain(state):
    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "linear":
        return _product(state["a"], state["b"], state["a_s"], state["b_s"], state["bias"], dtype)
    if kind == "grouped":
        out = torch.empty(case["m"], case["n"], dtype=dtype, device="cuda")
        begin = 0
        for e, end in enumerate(state["offs"].tolist()):
            if end > begin:
                out[begin:end] = _product(state["a"][begin:end], state["b"][e], state["a_s"][begin:end], state["b_s"][e],
                                          None, dtype)
            begin = end
        return out
    topk = case["topk"]
    if kind == "permute":
        x = state["x"].detach()
        ends, row_of_slot, slot_of_row = _plan(state["ids"], case["experts"])
        source = slot_of_row // topk
        out = {"rows": x[source], "offs": ends, "row_of_slot": row_of_slot.to(torch.int32)}
        if state["scale"] is not None:
            out["scale"] = state["scale"][source]
        if case["train"]:
            out["d_x"] = state["d_rows"][row_of_slot].float().sum(1).to(dtype)
        return out
    rows, weights, row_of_slot = state["rows"].detach(), state["weights"].detach(), state["plan"]
    taken = rows[row_of_slot].float()
    out = {"out": (taken * weights[:, :, None]).sum(1).to(dtype)}
    if case["train"]:
        d_out = state["d_out"].float()
        out["d_weights"] = (taken * d_out[:, None, :]).sum(2).to(weights.dtype)
        d_rows = torch.empty_like(rows)
        d_rows[row_of_slot] = (weights[:, :, None] * d_out[:, None, :]).to(dtype)
        out["d_rows"] = d_rows
    return out


# ---- the framework's operators ------------------------------------------------------------------
def _run_own(state):
    import flag_gems

    case = state["case"]
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "linear":
        return flag_gems.w8a8_int8_matmul(state["a"], state["b"], state["a_s"], state["b_s"], state["bias"], dtype)
    if kind == "grouped":
        return flag_gems.w8a8_int8_grouped_mm(state["a"], state["b"], state["a_s"], state["b_s"], state["offs"], None, dtype)
    if kind == "permute":
        rows, scale, plan = flag_gems.moe_permute(state["x"], state["ids"], case["experts"], scale=state["scale"])
        out = {"rows": rows, "offs": plan.offs, "row_of_slot": plan.row_of_slot}
        if scale is not None:
            out["scale"] = scale
        if case["train"]:
            out["d_x"], = torch.autograd.grad(rows, state["x"], state["d_rows"])
        return out
    out = {"out": flag_gems.moe_unpermute(state["rows"], state["plan"], state["weights"])}
    if case["train"]:
        out["d_rows"], out["d_weights"] = torch.autograd.grad(out["out"], (state["rows"], state["weights"]), state["d_out"])
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- floors -----------------------------------------------------------------------------------
def work(case):
    kind, size = case["kind"], BYTES[case["dtype"]]
    if kind == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + size * m * n + 4 * (m + n) + (size * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    if kind == "grouped":
        m, n, k, groups = case["m"], case["n"], case["k"], case["groups"]
        used = groups * (1.0 - (1.0 - 1.0 / groups) ** m)  # weights that some row needs, on average
        return {"bytes": int(m * k + used * n * (k + 4) + size * m * n + 4 * m + 4 * groups), "flops": 2 * m * n * k}
    tokens, hidden, topk = case["tokens"], case["hidden"], case["topk"]
    few, many = tokens * hidden, tokens * hidden * topk  # values in token order, values in expert order
    slots = 4 * tokens * topk  # bytes of one 32-bit value per route slot
    if kind == "permute":
        moved = size * (few + many) + 2 * slots + 4 * case["experts"]
        if case["dtype"] == "int8":
            moved += 4 * tokens + slots
        if case["train"]:
            return {"bytes": 2 * size * (few + many) + 2 * slots + 4 * case["experts"], "flops": many}
        return {"bytes": moved, "flops": 0}
    if case["train"]:
        # forward: rows in, sums out; backward: the sums' gradient and the rows in, the rows' gradient out
        return {"bytes": size * (few + many) + size * (few + 2 * many) + 5 * slots, "flops": 5 * many}
    return {"bytes": size * (few + many) + 2 * slots, "flops": 2 * many}


# ---- the definition in 64 bits ------------------------------------------------------------------
def exact(case, seed):
    global own
    as_own, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = as_own
    kind = case["kind"]
    if kind in ("linear", "grouped"):
        m = case["m"]
        a = s["a"].double() * s["a_s"].double()
        if kind == "linear":
            out = torch.matmul(a, (s["b"].double() * s["b_s"].double()[:, None]).transpose(0, 1))
            return out if s["bias"] is None else out + s["bias"].double()
        out = torch.zeros(m, case["n"], dtype=torch.float64, device="cuda")
        group = torch.searchsorted(s["offs"], torch.arange(m, dtype=torch.int32, device="cuda"), right=True)
        for e in group.unique().tolist():
            at = (group == e).nonzero()[:, 0]
            out[at] = torch.einsum("mk,nk->mn", a[at], s["b"][e].double()) * s["b_s"][e].double()
        return out
    tokens, topk, experts = case["tokens"], case["topk"], case["experts"]
    flat = s["ids"].cpu().reshape(-1).tolist()
    count = [0] * experts
    for e in flat:
        count[e] += 1
    end, ends = 0, []
    for c in count:
        end += c
        ends.append(end)
    at = [e - c for e, c in zip(ends, count)]
    row_of = []
    for e in flat:
        row_of.append(at[e])
        at[e] += 1
    row_of = torch.tensor(row_of, device="cuda").view(tokens, topk)
    if kind == "permute":
        x = s["x"].detach()
        rows = torch.empty(tokens * topk, case["hidden"], dtype=torch.int8 if case["dtype"] == "int8" else torch.float64,
                           device="cuda")
        for j in range(topk):
            rows[row_of[:, j]] = x.to(rows.dtype)
        out = {"rows": rows, "offs": torch.tensor(ends, dtype=torch.int32, device="cuda"), "row_of_slot": row_of.to(torch.int32)}
        if s["scale"] is not None:
            out["scale"] = torch.empty(tokens * topk, 1, dtype=torch.float64, device="cuda")
            for j in range(topk):
                out["scale"][row_of[:, j]] = s["scale"].double()
        if case["train"]:
            out["d_x"] = torch.zeros(tokens, case["hidden"], dtype=torch.float64, device="cuda")
            for j in range(topk):
                out["d_x"] += s["d_rows"].double()[row_of[:, j]]
        return out
    w = s["weights"].detach().double()
    total = torch.zeros(tokens, case["hidden"], dtype=torch.float64, device="cuda")
    out = {"out": total}
    if case["train"]:
        out["d_weights"] = torch.empty(tokens, topk, dtype=torch.float64, device="cuda")
        out["d_rows"] = torch.empty(tokens * topk, case["hidden"], dtype=torch.float64, device="cuda")
    for j in range(topk):
        taken = s["rows"].detach()[row_of[:, j]].double()
        total += taken * w[:, j:j + 1]
        if case["train"]:
            d_out = s["d_out"].double()
            out["d_weights"][:, j] = torch.einsum("th,th->t", taken, d_out)
            out["d_rows"][row_of[:, j]] = w[:, j:j + 1] * d_out
    return out
