"""Operators around the grouped GEMM of a mixture-of-experts layer: routing, rows sorted by expert and back, dense products.

Four operators, each through its public entry point when ``own`` is true and in elementary torch operations when it is not:

  route     nvfp4_gemm.route_tokens    top-k experts of every token and their weights from the router's logits
  sort      nvfp4_gemm.sort_tokens     token rows into the grouped GEMM's contiguous layout, everything on the device
  unsort    nvfp4_gemm.unsort_tokens   the expert outputs of every token, weighted and summed
  linear    nvfp4_gemm.linear          activation(x w^T + bias) + residual

``listed()`` gives fixed cases, ``draw(rng)`` others out of the same ranges.  A case with ``"train"`` runs forward and backward and
returns the gradients too.
"""
import math

import torch

own = False

DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # one decode step of 64 sequences: the router's logits of a 128-expert model, a call bound by its launch
        {"name": "route_step", "op": "route", "tokens": 64, "experts": 128, "k": 8, "scores": "softmax", "renormalize": True,
         "masked": False, "dtype": "float32", "train": False},
        # a training micro-batch whose padding tokens and switched-off experts have logits of -inf
        {"name": "route_train", "op": "route", "tokens": 16384, "experts": 128, "k": 8, "scores": "softmax", "renormalize": False,
         "masked": True, "dtype": "bfloat16", "train": True},
        # a decode step ahead of the grouped GEMM in its decode orientation (groups padded to 32 rows)
        {"name": "sort_step", "op": "sort", "tokens": 16, "experts": 128, "k": 8, "hidden": 4096, "alignment": 32, "dropped": False,
         "dtype": "bfloat16", "train": False},
        # prefill: every token's row goes to eight groups padded to the GEMM's 128-row tile
        {"name": "sort_prefill", "op": "sort", "tokens": 8192, "experts": 128, "k": 8, "hidden": 4096, "alignment": 128, "dropped": False,
         "dtype": "bfloat16", "train": False},
        # training of a smaller model in float16, a ragged number of tokens, some of them routed nowhere (padding)
        {"name": "sort_train", "op": "sort", "tokens": 4099, "experts": 64, "k": 6, "hidden": 2048, "alignment": 128, "dropped": True,
         "dtype": "float16", "train": True},
        # the other end of the decode step
        {"name": "unsort_step", "op": "unsort", "tokens": 16, "experts": 128, "k": 8, "hidden": 4096, "alignment": 32, "dropped": False,
         "dtype": "bfloat16", "train": False},
        # the other end of a training micro-batch: the gradients of the expert outputs and of the routing weights
        {"name": "unsort_train", "op": "unsort", "tokens": 8192, "experts": 128, "k": 8, "hidden": 4096, "alignment": 128, "dropped": False,
         "dtype": "bfloat16", "train": True},
        # one token through a dense projection of the attention block, added to the residual stream: bound by the weights' bytes
        {"name": "linear_token", "op": "linear", "m": 1, "n": 4096, "k": 4096, "activation": "none", "bias": False, "residual": True,
         "out": None, "dtype": "bfloat16", "train": False},
        # a decode batch of 33 through a shared expert's up projection, odd output width
        {"name": "linear_decode", "op": "linear", "m": 33, "n": 1411, "k": 2048, "activation": "gelu_tanh", "bias": True, "residual": False,
         "out": None, "dtype": "float16", "train": False},
        # the router: FP32 logits of a prefill's tokens, a narrow product bound by the activations' bytes
        {"name": "linear_router", "op": "linear", "m": 16384, "n": 128, "k": 4096, "activation": "none", "bias": True, "residual": False,
         "out": "float32", "dtype": "bfloat16", "train": False},
        # prefill through a wide dense layer, bound by the tensor cores
        {"name": "linear_prefill", "op": "linear", "m": 8192, "n": 4096, "k": 4096, "activation": "silu", "bias": True, "residual": True,
         "out": None, "dtype": "bfloat16", "train": False},
        # a training step of a dense layer with a ragged number of tokens: the output and four gradients
        {"name": "linear_train", "op": "linear", "m": 4099, "n": 4096, "k": 2048, "activation": "gelu", "bias": True, "residual": True,
         "out": None, "dtype": "bfloat16", "train": True},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi // step * step, max(-(-lo // step) * step, int(v / step + 0.5) * step))


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


def _draw(rng):
    op = rng.choice(["route", "sort", "unsort", "linear", "linear"])
    if op == "route":
        experts = _log_int(rng, 4, 512)
        return {"op": op, "tokens": _log_int(rng, 1, 32768), "experts": experts, "k": rng.randint(1, min(12, experts)),
                "scores": rng.choice(["softmax", "sigmoid"]), "renormalize": rng.random() < 0.5, "masked": rng.random() < 0.5,
                "dtype": rng.choice(["bfloat16", "float16", "float32"]), "train": rng.random() < 0.5}
    if op in ("sort", "unsort"):
        experts = _log_int(rng, 4, 256)
        hidden = _log_int(rng, 64, 8192, 8) if rng.random() < 0.8 else _log_int(rng, 64, 4096)
        return {"op": op, "tokens": _log_int(rng, 1, 16384), "experts": experts, "k": rng.randint(1, min(10, experts)), "hidden": hidden,
                "alignment": rng.choice([16, 32, 64, 128]), "dropped": rng.random() < 0.3,
                "dtype": rng.choice(["bfloat16", "bfloat16", "float16", "float32"]), "train": rng.random() < 0.5}
    return {"op": op, "m": _log_int(rng, 1, 16384), "n": _log_int(rng, 8, 8192), "k": _log_int(rng, 64, 8192, 8),
            "activation": rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"]), "bias": rng.random() < 0.5,
            "residual": rng.random() < 0.5, "out": rng.choice([None, None, "float32"]), "dtype": rng.choice(["bfloat16", "float16"]),
            "train": rng.random() < 0.3}


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6e12, w["flops"] / 1.5e15)


def _rows(case):
    """Rows of the sorted buffer: the bound on the padded groups that the host knows without the routing."""
    pairs, a = case["tokens"] * case["k"], case["alignment"]
    return (pairs + min(case["experts"], pairs) * (a - 1)) // a * a


def work(case):
    size = {"bfloat16": 2, "float16": 2, "float32": 4}[case["dtype"]]
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["k"]
        forward = t * e * size + t * k * 12
        backward = t * e * size + t * k * 4 if case["train"] else 0                # the gradient of the logits, the incoming one
        return {"bytes": forward + backward, "flops": t * e * (8 if case["train"] else 4)}
    if case["op"] in ("sort", "unsort"):
        t, k, h, m = case["tokens"], case["k"], case["hidden"], _rows(case)
        pairs = t * k
        if case["op"] == "sort":
            forward = t * h * size + m * h * size + pairs * 16 + m * 8            # x, ids in; rows, place, source, m_indices out
            backward = pairs * h * size + t * h * size if case["train"] else 0
            return {"bytes": forward + backward, "flops": pairs * h if case["train"] else 0}
        forward = pairs * h * size + pairs * 12 + t * h * size
        backward = t * h * size + m * h * size + pairs * 4 if case["train"] else 0  # dy in; gradients of the rows and of the weights out
        return {"bytes": forward + backward, "flops": pairs * h * (5 if case["train"] else 2)}
    m, n, k = case["m"], case["n"], case["k"]
    out = 4 if case["out"] else size
    forward = (m * k + n * k) * size + m * n * out + (n * size if case["bias"] else 0) + (m * n * out if case["residual"] else 0)
    backward = m * n * out + (m * k + n * k) * size + (n * size if case["bias"] else 0) if case["train"] else 0
    return {"bytes": forward + backward, "flops": 2 * m * n * k * (3 if case["train"] else 1)}


# ---- inputs ------------------------------------------------------------------------------------------------------

def _router_logits(g, tokens, experts):
    """Logits as a trained router gives them: spread of about one and a half, some experts more popular than others."""
    popular = torch.randn(experts, generator=g, device="cuda") * 0.5
    return torch.randn(tokens, experts, generator=g, device="cuda") * 1.5 + popular


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    randn = lambda *shape: torch.randn(*shape, generator=g, device="cuda")
    if case["op"] == "route":
        logits = _router_logits(g, case["tokens"], case["experts"])
        if case["masked"]:                       # experts switched off for a token, and padding tokens without any expert
            off = torch.rand(logits.shape, generator=g, device="cuda") < 0.1
            off |= torch.rand(case["tokens"], 1, generator=g, device="cuda") < 0.02
            logits = logits.masked_fill(off, float("-inf"))
        state = {"case": case, "logits": logits.to(dtype).requires_grad_(case["train"])}
        if case["train"]:
            state["grad"] = randn(case["tokens"], case["k"])
        return state
    if case["op"] in ("sort", "unsort"):
        t, e, k, h = case["tokens"], case["experts"], case["k"], case["hidden"]
        top, ids = torch.topk(_router_logits(g, t, e), k, dim=1)
        if case["dropped"]:                      # padding tokens, and pairs that a router with limited groups has left out
            off = (torch.rand(t, k, generator=g, device="cuda") < 0.05) | (torch.rand(t, 1, generator=g, device="cuda") < 0.05)
            ids = ids.masked_fill(off, -1)
        if case["op"] == "sort":
            state = {"case": case, "ids": ids, "x": randn(t, h).to(dtype).requires_grad_(case["train"])}
            if case["train"]:
                state["grad"] = randn(_rows(case), h).to(dtype)
            return state
        # what a program holds before it adds up the experts' outputs: the order of the rows, the rows and the weights
        weights = torch.softmax(top, dim=1).masked_fill(ids < 0, 0.0).requires_grad_(case["train"])
        place, source, m_indices = _order(ids, e, case["alignment"], _rows(case))
        state = {"case": case, "place": place, "source": source, "m_indices": m_indices, "weights": weights,
                 "rows": randn(_rows(case), h).to(dtype).requires_grad_(case["train"])}
        if own:
            from nvfp4_gemm import TokenOrder
            state["order"] = TokenOrder(place, source, m_indices)
        if case["train"]:
            state["grad"] = randn(t, h).to(dtype)
        return state
    m, n, k = case["m"], case["n"], case["k"]
    out = DTYPES[case["out"]] if case["out"] else dtype
    state = {"case": case, "x": randn(m, k).to(dtype), "w": (randn(n, k) * k ** -0.5).to(dtype), "out": out,
             "bias": (randn(n) * 0.2).to(dtype) if case["bias"] else None, "residual": randn(m, n).to(out) if case["residual"] else None}
    if case["train"]:
        state["leaves"] = [state[name].requires_grad_() for name in ("x", "w", "bias", "residual") if state[name] is not None]
        state["grad"] = randn(m, n).to(out)
    return state


# ---- one pass ----------------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    import nvfp4_gemm

    case = state["case"]
    if case["op"] == "route":
        ids, weights = nvfp4_gemm.route_tokens(state["logits"], case["k"], scores=case["scores"], renormalize=case["renormalize"])
        if not case["train"]:
            return ids, weights
        return ids, weights.detach(), torch.autograd.grad(weights, state["logits"], state["grad"])[0]
    if case["op"] == "sort":
        rows, order = nvfp4_gemm.sort_tokens(state["x"], state["ids"], case["experts"], alignment=case["alignment"])
        if not case["train"]:
            return rows, order.place, order.source, order.m_indices
        dx = torch.autograd.grad(rows, state["x"], state["grad"])[0]
        return rows.detach(), order.place, order.source, order.m_indices, dx
    if case["op"] == "unsort":
        y = nvfp4_gemm.unsort_tokens(state["rows"], state["order"], state["weights"])
        if not case["train"]:
            return y
        return (y.detach(), *torch.autograd.grad(y, (state["rows"], state["weights"]), state["grad"]))
    y = nvfp4_gemm.linear(state["x"], state["w"], bias=state["bias"], residual=state["residual"], activation=case["activation"],
                          out_dtype=state["out"])
    if not case["train"]:
        return y
    return (y.detach(), *torch.autograd.grad(y, state["leaves"], state["grad"]))


def _plain(state):
    case = state["case"]
    with torch.no_grad():
        return {"route": _plain_route, "sort": _plain_sort, "unsort": _plain_unsort, "linear": _plain_linear}[case["op"]](case, state)


def _plain_route(case, state):
    l = state["logits"].float()
    top, ids = torch.sort(l, dim=1, descending=True, stable=True)
    top, ids = top[:, :case["k"]], ids[:, :case["k"]]
    live = top > float("-inf")
    ids = torch.where(live, ids, -1)
    at = ids.clamp(min=0)
    zero = torch.zeros((), device=l.device)
    if case["scores"] == "softmax":
        biggest = torch.where(live[:, :1], top[:, :1], zero)
        p = torch.exp(l - biggest)
        total = p.sum(dim=1, keepdim=True)
        p = torch.where(total > 0, p / total, zero)
        chosen = torch.where(live, torch.exp(top - biggest) / total, zero)
    else:
        chosen = torch.where(live, 1 / (1 + torch.exp(-top)), zero)
    if case["renormalize"]:
        part = chosen.sum(dim=1, keepdim=True)
        weights = torch.where(part > 0, chosen / part, zero)
    else:
        weights = chosen
    if not case["train"]:
        return ids, weights
    g = torch.where(live, state["grad"], zero)
    if case["renormalize"]:
        dchosen = weights * (g - (g * weights).sum(dim=1, keepdim=True))          # times the chosen score, over it below
        dsel = dchosen if case["scores"] == "softmax" else dchosen * (1 - chosen)
    elif case["scores"] == "sigmoid":
        dsel = g * chosen * (1 - chosen)
    else:
        dsel = g * chosen
    dsel = torch.where(live, dsel, zero)
    dlogits = torch.zeros_like(l).scatter_add_(1, at, dsel)
    if case["scores"] == "softmax" and not case["renormalize"]:
        dlogits = dlogits - p * (g * chosen).sum(dim=1, keepdim=True)
    return ids, weights, dlogits.to(state["logits"].dtype)


def _order(ids, experts, alignment, m):
    """(place, source, m_indices): row of every (token, choice) pair in the sorted buffer, -1 for none; pair of every row, -1 for a row
    of padding; expert of every row, -1 behind the last group."""
    flat = ids.reshape(-1)
    n = flat.numel()
    valid = (flat >= 0) & (flat < experts)
    key = torch.where(valid, flat, experts)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    padded = (counts[:experts] + alignment - 1) // alignment * alignment
    ends = torch.cumsum(padded, 0)
    order = torch.sort(key, stable=True)[1]
    first = torch.cumsum(counts, 0) - counts
    sorted_key = key[order]
    starts = torch.cat([ends - padded, ends.new_zeros(1)])
    row = starts[sorted_key] + torch.arange(n, device=flat.device) - first[sorted_key]
    row = torch.where(sorted_key < experts, row, -1)
    place = torch.empty_like(row)
    place[order] = row
    source = torch.full((m + 1,), -1, dtype=torch.int32, device=flat.device)
    source[torch.where(row >= 0, row, m)] = order.to(torch.int32)                 # the last entry takes what has no row
    at = torch.arange(m, device=flat.device)
    expert = torch.bucketize(at, ends, right=True)
    m_indices = torch.where(at < ends[-1], expert, -1).to(torch.int32)
    return place.reshape(ids.shape), source[:m], m_indices


def _gather(rows, index):
    """rows[index] in FP32, zeros where the index is -1."""
    return torch.where(index[..., None] >= 0, rows[index.clamp(min=0)].float(), torch.zeros((), device=rows.device))


def _plain_sort(case, state):
    x, ids = state["x"], state["ids"]
    k = case["k"]
    place, source, m_indices = _order(ids, case["experts"], case["alignment"], _rows(case))
    token = torch.where(source >= 0, source.long() // k, -1)
    rows = _gather(x, token).to(x.dtype)
    if not case["train"]:
        return rows, place, source, m_indices
    dx = torch.zeros(x.shape, device=x.device)
    for j in range(k):
        dx += _gather(state["grad"], place[:, j])
    return rows, place, source, m_indices, dx.to(x.dtype)


def _plain_unsort(case, state):
    rows, place, w = state["rows"], state["place"], state["weights"]
    y = torch.zeros(place.shape[0], rows.shape[1], device=rows.device)
    for j in range(case["k"]):
        y += _gather(rows, place[:, j]) * w[:, j, None]
    if not case["train"]:
        return y.to(rows.dtype)
    dy = state["grad"].float()
    source = state["source"].long()
    pair = source.clamp(min=0)
    drows = torch.where(source[:, None] >= 0, dy[pair // case["k"]] * w.reshape(-1)[pair][:, None], torch.zeros((), device=dy.device))
    dw = torch.stack([(_gather(rows, place[:, j]) * dy).sum(dim=1) for j in range(case["k"])], dim=1)
    return y.to(rows.dtype), drows.to(rows.dtype), dw


def _plain_linear(case, state):
    x, w = state["x"].float(), state["w"].float()
    z = x @ w.t()
    if state["bias"] is not None:
        z = z + state["bias"].float()
    act = case["activation"]
    if act == "none":
        y, slope = z, None
    elif act == "relu":
        y, slope = torch.where(z > 0, z, 0.0), (z > 0).float()
    elif act == "silu":
        s = 1 / (1 + torch.exp(-z))
        y, slope = z * s, s * (1 + z * (1 - s))
    elif act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
        y, slope = z * cdf, cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    else:
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z * z * z))
        y, slope = 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    y = y.to(state["out"])
    if not case["train"]:
        return y
    dz = state["grad"].float()
    if slope is not None:
        dz = dz * slope
    out = [y, (dz @ w).to(state["x"].dtype), (dz.t() @ x).to(state["w"].dtype)]
    if state["bias"] is not None:
        out.append(dz.sum(dim=0).to(state["bias"].dtype))
    if state["residual"] is not None:
        out.append(state["grad"])
    return tuple(out)


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "sort": _exact_sort, "unsort": _exact_unsort, "linear": _exact_linear}[case["op"]](case, state)


def _exact_route(case, state):
    l = state["logits"].detach().double()
    left, ids = l.clone(), []
    for _ in range(case["k"]):
        best = left.max(dim=1, keepdim=True).values
        first = (left == best).int().argmax(dim=1, keepdim=True)          # the lowest index among equals
        ids.append(torch.where(best > -math.inf, first, -1))
        left.scatter_(1, first, -math.inf)
    ids = torch.cat(ids, dim=1)
    live = ids >= 0
    chosen_logit = torch.where(live, l.gather(1, ids.clamp(min=0)), -math.inf)
    if case["scores"] == "softmax":
        log_score = l - torch.logsumexp(l, dim=1, keepdim=True)
    else:
        log_score = torch.nn.functional.logsigmoid(l)
    chosen = torch.where(live, log_score.gather(1, ids.clamp(min=0)), -math.inf)
    if case["renormalize"]:
        weights = torch.where(live, torch.exp(chosen - torch.logsumexp(chosen, dim=1, keepdim=True)), 0.0)
    else:
        weights = torch.where(live, torch.exp(chosen), 0.0)
    if not case["train"]:
        return ids, weights
    # d weights / d logits by the chain rule on logarithms: d w_j = w_j d(log w_j)
    h = torch.where(live, state["grad"].double() * weights, 0.0)           # gradient of log w_j
    if case["renormalize"]:
        h = h - weights * h.sum(dim=1, keepdim=True)                       # log w_j = log s_j - logsumexp(log s)
    if case["scores"] == "sigmoid":
        h = torch.where(live, h * torch.sigmoid(-chosen_logit), 0.0)       # d log sigmoid(l) = sigmoid(-l)
    dlogits = torch.zeros_like(l).scatter_add_(1, ids.clamp(min=0), h)
    if case["scores"] == "softmax":
        p = torch.where(live[:, :1], torch.softmax(l, dim=1), 0.0)
        dlogits = dlogits - p * h.sum(dim=1, keepdim=True)                 # the total is zero where the weights were renormalised
    return ids, weights, dlogits


def _exact_order(case, ids):
    """The order of the rows, expert by expert on the host."""
    flat = ids.reshape(-1).cpu()
    a, m = case["alignment"], _rows(case)
    place = torch.full((flat.numel(),), -1, dtype=torch.int64)
    source = torch.full((m,), -1, dtype=torch.int32)
    m_indices = torch.full((m,), -1, dtype=torch.int32)
    at = 0
    for e in range(case["experts"]):
        pairs = (flat == e).nonzero().reshape(-1)
        place[pairs] = at + torch.arange(pairs.numel())
        source[at:at + pairs.numel()] = pairs.int()
        end = at + -(-pairs.numel() // a) * a
        m_indices[at:end] = e
        at = end
    return place.reshape(ids.shape).cuda(), source.cuda(), m_indices.cuda()


def _exact_sort(case, state):
    x = state["x"].detach()
    place, source, m_indices = _exact_order(case, state["ids"])
    rows = torch.zeros(_rows(case), x.shape[1], dtype=x.dtype, device=x.device)
    live = source >= 0
    rows[live] = x[source[live].long() // case["k"]]                        # copies: exact in the type itself
    if not case["train"]:
        return rows, place, source, m_indices
    dx = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dx.index_add_(0, source[live].long() // case["k"], state["grad"][live].double())
    return rows, place, source, m_indices, dx


def _exact_unsort(case, state):
    rows, w, place = state["rows"].detach(), state["weights"].detach().double(), state["place"]
    t, k = place.shape
    y = torch.zeros(t, rows.shape[1], dtype=torch.float64, device=rows.device)
    dw = torch.zeros(t, k, dtype=torch.float64, device=rows.device)
    drows = torch.zeros(rows.shape, dtype=torch.float64, device=rows.device) if case["train"] else None
    for j in range(k):
        live = place[:, j] >= 0
        here = rows[place[live, j]].double()
        y[live] += here * w[live, j, None]
        if case["train"]:
            dy = state["grad"][live].double()
            dw[live, j] = (here * dy).sum(dim=1)
            drows[place[live, j]] = dy * w[live, j, None]
    return (y, drows, dw) if case["train"] else y


def _exact_linear(case, state):
    x, w = state["x"].detach().double(), state["w"].detach().double()
    z = torch.matmul(x, w.t())
    if state["bias"] is not None:
        z += state["bias"].detach().double()
    z.requires_grad_(case["train"])
    with torch.enable_grad():
        f = {"none": lambda v: v * 1.0, "relu": torch.relu, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["activation"]]
        a = f(z)
        if case["train"]:
            dz = torch.autograd.grad(a, z, state["grad"].double())[0]
    y = a.detach()
    if state["residual"] is not None:
        y = y + state["residual"].detach().double()
    if not case["train"]:
        return y
    out = [y, torch.matmul(dz, w), torch.matmul(dz.t(), x)]
    if state["bias"] is not None:
        out.append(dz.sum(dim=0))
    if state["residual"] is not None:
        out.append(state["grad"].double())
    return tuple(out)
