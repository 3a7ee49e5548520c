"""The operators around a language model's feed-forward blocks, as a user's program calls them, with their plain forms.

  linear            out = act(x W^T + b) + r, or with a gate act(x Wg^T + bg) * (x Wu^T + bu) + r; for training it also
                    keeps z, the product before the activation
  linear_backward   dz = dy act'(z), dx = dz W, dW = dz^T x, db = sum of dz over the tokens
  route             top-k experts of each token from its logits: softmax or sigmoid scores, a bias that takes part in the
                    choice only, groups of experts of which the best are kept, weights scaled to a sum of one
  route_backward    the gradient of those weights with respect to the logits
  expert_in         rows of the tokens sorted by expert, and each row's product with its expert's matrices (gathered
                    straight from the tokens), with bias, activation and gate
  expert_out        each sorted row's product with its expert's matrix, then the weighted sum of every token's rows
  expert_backward   the gradients of one such product: sorted rows in, sorted rows out, one dW and db per expert

Every expert's rows keep the order of the tokens; an id outside [0, experts) drops its row.
"""
import math

import torch

own = False

_DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


def listed():
    return [
        # one token through an attention output projection, residual added: decoding, bound by reading W
        {"name": "linear, 1 token", "op": "linear", "dtype": "bfloat16", "tokens": 1, "k": 4096, "n": 4096,
         "act": "none", "gated": False, "bias": True, "residual": True, "keep": False},
        # 48 sequences decoding together through a gated feed-forward's first matrices
        {"name": "linear, 48 tokens gated", "op": "linear", "dtype": "float16", "tokens": 48, "k": 2048, "n": 8192,
         "act": "silu", "gated": True, "bias": False, "residual": False, "keep": False},
        # a ragged training step of a GELU layer that keeps z: no size is a multiple of a tile
        {"name": "linear, 1237 tokens ragged", "op": "linear", "dtype": "bfloat16", "tokens": 1237, "k": 1000, "n": 2051,
         "act": "gelu", "gated": False, "bias": True, "residual": True, "keep": True},
        # a long prompt through a gated feed-forward: bound by the matrix product
        {"name": "linear, 8192 tokens gated", "op": "linear", "dtype": "bfloat16", "tokens": 8192, "k": 4096, "n": 8192,
         "act": "silu", "gated": True, "bias": False, "residual": False, "keep": False},
        # fine-tuning on a short batch: launches and the sums over tokens count
        {"name": "linear backward, 200 tokens", "op": "linear_backward", "dtype": "float16", "tokens": 200, "k": 512,
         "n": 1003, "act": "silu", "gated": True, "bias": True},
        # a training step's layer
        {"name": "linear backward, 4096 tokens", "op": "linear_backward", "dtype": "bfloat16", "tokens": 4096, "k": 4096,
         "n": 4096, "act": "gelu_tanh", "gated": False, "bias": True},
        # the router of a decoding batch
        {"name": "route, 16 tokens", "op": "route", "dtype": "float32", "tokens": 16, "experts": 64, "top_k": 6,
         "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renorm": True},
        # the router of a long prompt: balancing bias, half of the groups kept
        {"name": "route, 16384 tokens grouped", "op": "route", "dtype": "float32", "tokens": 16384, "experts": 256,
         "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renorm": True},
        # the same in training, softmax over all experts without scaling: every logit has a gradient
        {"name": "route backward, 8192 tokens", "op": "route_backward", "dtype": "bfloat16", "tokens": 8192, "experts": 128,
         "top_k": 8, "scoring": "softmax", "renorm": False},
        # 8 tokens decoding: most experts have no row or one, bound by reading the chosen experts
        {"name": "expert_in, 8 tokens", "op": "expert_in", "dtype": "bfloat16", "tokens": 8, "experts": 64, "top_k": 8,
         "k": 2048, "n": 1024, "act": "silu", "gated": True, "bias": False, "drop": False},
        # a prompt's down projection with its padding dropped: bound by the matrix products
        {"name": "expert_out, 4096 tokens", "op": "expert_out", "dtype": "bfloat16", "tokens": 4096, "experts": 32,
         "top_k": 4, "k": 2048, "n": 2048, "drop": True},
        # a training step of the gated product, uneven rows per expert
        {"name": "expert backward, 2000 tokens", "op": "expert_backward", "dtype": "bfloat16", "tokens": 2000, "experts": 16,
         "top_k": 2, "k": 1024, "n": 1400, "act": "silu", "gated": True, "bias": True, "drop": False},
    ]


def _log(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_backward", "route", "route_backward", "expert_in", "expert_out",
                     "expert_backward"])
    kind = rng.choice(["bfloat16", "float16"])
    act = rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu"])
    if op in ("linear", "linear_backward"):
        top = 8192 if op == "linear" else 4096
        case = {"op": op, "dtype": kind, "tokens": _log(rng, 1, top), "k": 8 * _log(rng, 8, 512),
                "n": _log(rng, 64, 8192 if op == "linear" else 4096), "act": act, "gated": rng.random() < 0.4,
                "bias": rng.random() < 0.5}
        if op == "linear":
            case["residual"] = rng.random() < 0.5
            case["keep"] = rng.random() < 0.3
        return case
    if op in ("route", "route_backward"):
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log(rng, 4, 320 // groups)
        case = {"op": op, "dtype": rng.choice(["float32", "bfloat16", "float16"]), "tokens": _log(rng, 1, 16384),
                "experts": experts, "top_k": rng.randint(1, min(10, experts // groups)),
                "scoring": rng.choice(["softmax", "sigmoid"]), "renorm": rng.random() < 0.6}
        if op == "route":
            case["bias"] = rng.random() < 0.5
            case["groups"] = groups
            case["top_groups"] = rng.randint(1, groups)
        return case
    experts = _log(rng, 4, 128)
    case = {"op": op, "dtype": kind, "tokens": _log(rng, 1, 4096), "experts": experts,
            "top_k": rng.randint(1, min(8, experts)), "k": 8 * _log(rng, 16, 256), "n": 8 * _log(rng, 16, 256)}
    if op != "expert_out":
        case.update(act=act, gated=rng.random() < 0.6, bias=rng.random() < 0.4)
    case["drop"] = rng.random() < 0.3
    return case


# ------------------------------------------------------------------------------------------------ inputs
def _ids(gen, case):
    """Expert ids of every token, some experts wanted more than others; `drop`: the last tokens are padding."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    wish = torch.randn(t, e, generator=gen, device="cuda") + 0.5 * torch.randn(e, generator=gen, device="cuda")
    ids = wish.topk(k, dim=1).indices.to(torch.int32)
    if case["drop"]:
        ids[t - t // 16:] = -1
    return ids.contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    dtype = _DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, kind=dtype):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)

    def empty(*shape, kind=dtype):
        return torch.zeros(*shape, device="cuda", dtype=kind)

    s = {"case": dict(case)}
    op, t = case["op"], case["tokens"]
    if op in ("route", "route_backward"):
        e, k = case["experts"], case["top_k"]
        s["logits"] = normal(t, e, scale=1.5)
        if op == "route":
            s["bias"] = normal(e, scale=0.1, kind=torch.float32) if case["bias"] else None
            s["ids"], s["weights"] = empty(t, k, kind=torch.int32), empty(t, k, kind=torch.float32)
        else:
            s["ids"] = s["logits"].float().sort(dim=1, descending=True, stable=True).indices[:, :k].to(torch.int32).contiguous()
            s["dweights"], s["dlogits"] = normal(t, k, kind=torch.float32), empty(t, e)
        return s
    k, n = case["k"], case["n"]
    wide = n * (2 if case.get("gated") else 1)
    if op in ("linear", "linear_backward"):
        s["x"], s["w"] = normal(t, k), normal(wide, k, scale=k ** -0.5)
        bias = normal(wide, scale=0.1) if case["bias"] else None
        if op == "linear":
            s["bias"] = bias
            s["residual"] = normal(t, n) if case["residual"] else None
            s["out"], s["z"] = empty(t, n), empty(t, wide) if case["keep"] else None
        else:
            s["z"] = normal(t, wide)
            s["dy"] = normal(t, n)
            s["dx"], s["dw"], s["db"] = empty(t, k), empty(wide, k), empty(wide) if case["bias"] else None
        return s
    e, top = case["experts"], case["top_k"]
    rows = t * top
    s["ids"] = _ids(gen, case)
    s["w"] = normal(e, wide, k, scale=k ** -0.5)
    if op == "expert_in":
        s["x"] = normal(t, k)
        s["bias"] = normal(e, wide, scale=0.1) if case["bias"] else None
        s["out"] = empty(rows, n)
    elif op == "expert_out":
        s["x"] = normal(rows, k)
        s["weights"] = torch.rand(t, top, generator=gen, device="cuda")
        s["residual"] = normal(t, n)
        s["y"], s["out"] = empty(rows, n), empty(t, n)
    else:
        s["x"], s["z"], s["dy"] = normal(rows, k), normal(rows, wide), normal(rows, n)
        s["dx"], s["dw"], s["db"] = empty(rows, k), empty(e, wide, k), empty(e, wide) if case["bias"] else None
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _act(z, name):
    if name == "relu":
        return torch.clamp(z, min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        h = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + h) + 0.5 * z * (1 - h * h) * c * (1 + 3 * 0.044715 * z * z)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _through(z, case):
    if not case.get("gated"):
        return _act(z, case.get("act", "none"))
    n = z.shape[1] // 2
    return _act(z[:, :n], case["act"]) * z[:, n:]


def _before(dy, z, case):
    """dz from dy and z."""
    if not case["gated"]:
        return dy * _slope(z, case["act"])
    n = z.shape[1] // 2
    gate, up = z[:, :n], z[:, n:]
    return torch.cat([dy * up * _slope(gate, case["act"]), dy * _act(gate, case["act"])], dim=1)


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    out = _through(z, case)
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return [out.to(dtype)] + ([z.to(dtype)] if case["keep"] else [])


def _plain_linear_backward(s):
    case, dtype = s["case"], s["x"].dtype
    dz = _before(s["dy"].float(), s["z"].float(), case)
    out = [(dz @ s["w"].float()).to(dtype), (dz.t() @ s["x"].float()).to(dtype)]
    return out + ([dz.sum(dim=0).to(dtype)] if case["bias"] else [])


def _choose(logits, bias, case):
    """Indices of the chosen experts, best first, equal ones in the order of their index; scores in 64 bits."""
    t, e = logits.shape
    score = logits.double()
    if bias is not None or case["groups"] > 1:
        score = torch.softmax(score, dim=1) if case["scoring"] == "softmax" else torch.sigmoid(score)
        if bias is not None:
            score = score + bias.double()
    if case["groups"] > 1:
        split = score.view(t, case["groups"], e // case["groups"])
        best = split.sort(dim=2, descending=True).values[:, :, :2].sum(dim=2)
        kept = best.sort(dim=1, descending=True, stable=True).indices[:, :case["top_groups"]]
        mask = torch.zeros(t, case["groups"], dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        score = torch.where(mask[:, :, None].expand_as(split).reshape(t, e), score, -math.inf)
    return score.sort(dim=1, descending=True, stable=True).indices[:, :case["top_k"]]


def _plain_route(s):
    case, x = s["case"], s["logits"].float()
    ids = _choose(s["logits"], s["bias"], case)
    if case["scoring"] == "softmax":
        p = torch.exp(x - x.max(dim=1, keepdim=True).values)
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    w = p.gather(1, ids)
    if case["renorm"]:
        w = w / w.sum(dim=1, keepdim=True)
    return [ids.to(torch.int32), w]


def _plain_route_backward(s):
    case, x, ids, g = s["case"], s["logits"].float(), s["ids"].long(), s["dweights"]
    if case["scoring"] == "softmax":
        p = torch.exp(x - x.max(dim=1, keepdim=True).values)
        p = p / p.sum(dim=1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    if case["renorm"]:
        w = p.gather(1, ids)
        total = w.sum(dim=1, keepdim=True)
        g = (g - (g * w).sum(dim=1, keepdim=True) / total) / total
    dp = torch.zeros_like(x).scatter_(1, ids, g)
    if case["scoring"] == "softmax":
        dx = p * (dp - (dp * p).sum(dim=1, keepdim=True))
    else:
        dx = dp * p * (1 - p)
    return [dx.to(s["logits"].dtype)]


def _sorted_rows(ids, experts):
    """offsets [experts + 1], order (sorted place -> token * top_k + slot, -1 past the last) and its inverse slots."""
    flat = ids.reshape(-1).long()
    rows = flat.numel()
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)
    order = key.sort(stable=True).indices
    offsets = (key[None, :] < torch.arange(experts + 1, device=ids.device)[:, None]).sum(dim=1)
    place = torch.arange(rows, device=ids.device)
    slots = torch.empty_like(place).scatter_(0, order, place)
    slots = torch.where(key < experts, slots, -1)
    order = torch.where(place < offsets[experts], order, -1)
    return offsets.to(torch.int32), order.to(torch.int32), slots.to(torch.int32)


def _plain_expert_in(s):
    case, dtype = s["case"], s["x"].dtype
    offsets, order, slots = _sorted_rows(s["ids"], case["experts"])
    out = torch.zeros(order.numel(), case["n"], device="cuda")
    ends = offsets.tolist()
    for e in range(case["experts"]):  # one product per expert that has rows
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        z = s["x"][order[a:b].long() // case["top_k"]].float() @ s["w"][e].float().t()
        if s["bias"] is not None:
            z = z + s["bias"][e].float()
        out[a:b] = _through(z, case)
    return [offsets, order, slots, out.to(dtype)]


def _plain_expert_out(s):
    case, dtype = s["case"], s["x"].dtype
    offsets, order, slots = _sorted_rows(s["ids"], case["experts"])
    y = torch.zeros(order.numel() + 1, case["n"], device="cuda")  # the last row, of zeros, stands for dropped ones
    ends = offsets.tolist()
    for e in range(case["experts"]):  # one product per expert that has rows
        a, b = ends[e], ends[e + 1]
        if a < b:
            y[a:b] = s["x"][a:b].float() @ s["w"][e].float().t()
    part = y[slots.long()].view(case["tokens"], case["top_k"], case["n"])
    return [(s["residual"].float() + (part * s["weights"][:, :, None]).sum(dim=1)).to(dtype)]


def _plain_expert_backward(s):
    case, dtype = s["case"], s["x"].dtype
    ends = _sorted_rows(s["ids"], case["experts"])[0].tolist()
    dx = torch.zeros(s["x"].shape, device="cuda")
    dw = torch.zeros(s["w"].shape, device="cuda")
    db = torch.zeros(s["w"].shape[:2], device="cuda")
    for e in range(case["experts"]):  # one product per expert that has rows
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        dz = _before(s["dy"][a:b].float(), s["z"][a:b].float(), case)
        dx[a:b] = dz @ s["w"][e].float()
        dw[e] = dz.t() @ s["x"][a:b].float()
        db[e] = dz.sum(dim=0)
    return [dx.to(dtype), dw.to(dtype)] + ([db.to(dtype)] if case["bias"] else [])


_PLAIN = {"linear": _plain_linear, "linear_backward": _plain_linear_backward, "route": _plain_route,
          "route_backward": _plain_route_backward, "expert_in": _plain_expert_in, "expert_out": _plain_expert_out,
          "expert_backward": _plain_expert_backward}


# ------------------------------------------------------------------------------------------------ the framework's calls
def _own(s):
    from flextensor_b200 import backend
    case, op = s["case"], s["case"]["op"]
    if op == "linear":
        backend.linear(s["x"], s["w"], s["out"], bias=s["bias"], residual=s["residual"], activation=case["act"],
                       gated=case["gated"], preact=s["z"])
        return [s["out"]] + ([s["z"]] if case["keep"] else [])
    if op == "linear_backward":
        if "workspace" not in s:  # kept by the program from step to step
            s["workspace"] = torch.empty(backend.linear_backward_workspace_bytes(
                case["tokens"], case["n"], case["k"], case["gated"]), dtype=torch.uint8, device="cuda")
        backend.linear_backward(s["x"], s["w"], s["dy"], dx=s["dx"], dweight=s["dw"], dbias=s["db"], preact=s["z"],
                                activation=case["act"], gated=case["gated"], workspace=s["workspace"])
        return [s["dx"], s["dw"]] + ([s["db"]] if case["bias"] else [])
    if op == "route":
        backend.route_experts(s["logits"], s["ids"], s["weights"], bias=s["bias"], scoring=case["scoring"],
                              groups=case["groups"], top_groups=case["top_groups"], renormalize=case["renorm"])
        return [s["ids"], s["weights"]]
    if op == "route_backward":
        backend.route_experts_backward(s["logits"], s["ids"], s["dweights"], s["dlogits"], scoring=case["scoring"],
                                       renormalize=case["renorm"])
        return [s["dlogits"]]
    if "plan" not in s:  # its buffers, kept from step to step; expert_plan fills them anew in every pass
        s["plan"] = backend.ExpertPlan(case["tokens"], case["top_k"], case["experts"], device=s["ids"].device)
    plan = s["plan"]
    backend.expert_plan(s["ids"], plan)
    if op == "expert_in":
        backend.expert_linear(s["x"], s["w"], plan, s["out"], bias=s["bias"], activation=case["act"], gated=case["gated"],
                              gather=True)
        return [plan.offsets, plan.order, plan.slots, s["out"]]
    if op == "expert_out":
        backend.expert_linear(s["x"], s["w"], plan, s["y"])
        backend.expert_combine(s["y"], plan, s["out"], weights=s["weights"], residual=s["residual"])
        return [s["out"]]
    if "workspace" not in s:
        s["workspace"] = torch.empty(backend.expert_linear_backward_workspace_bytes(plan, case["n"], case["k"], case["gated"]),
                                     dtype=torch.uint8, device="cuda")
    backend.expert_linear_backward(s["x"], s["w"], plan, s["dy"], dx=s["dx"], dweight=s["dw"], dbias=s["db"],
                                   preact=s["z"], activation=case["act"], gated=case["gated"], workspace=s["workspace"])
    return [s["dx"], s["dw"]] + ([s["db"]] if case["bias"] else [])


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    op, t = case["op"], case["tokens"]
    if op in ("route", "route_backward"):
        e, k = case["experts"], case["top_k"]
        if op == "route":
            return {"bytes": t * e * size + (4 * e if case["bias"] else 0) + 8 * t * k, "flops": 5 * t * e}
        return {"bytes": 2 * t * e * size + 8 * t * k, "flops": 6 * t * e}
    k, n = case["k"], case["n"]
    wide = n * (2 if case.get("gated") else 1)
    if op == "linear":
        moved = t * k + wide * k + t * n + (wide if case["bias"] else 0) + (t * n if case["residual"] else 0)
        moved += t * wide if case["keep"] else 0
        return {"bytes": 2 * moved, "flops": 2 * t * k * wide}
    if op == "linear_backward":
        z = t * wide if case["act"] != "none" or case["gated"] else 0
        return {"bytes": 2 * (2 * t * k + 2 * wide * k + t * n + z + (wide if case["bias"] else 0)),
                "flops": 4 * t * k * wide}
    e, rows = case["experts"], t * case["top_k"]
    if case["drop"]:
        rows = (t - t // 16) * case["top_k"]
    busy = min(e, rows)
    if op in ("expert_in", "expert_out"):
        moved = busy * wide * k + ((t if op == "expert_in" else rows) * k)
        moved += rows * n if op == "expert_in" else 2 * t * n + 2 * t * case["top_k"]
        return {"bytes": 2 * moved + 4 * t * case["top_k"], "flops": 2 * rows * k * wide}
    z = rows * wide if case["act"] != "none" or case["gated"] else 0
    return {"bytes": 2 * (2 * rows * k + rows * n + z + busy * wide * k + e * wide * k) + 4 * t * case["top_k"],
            "flops": 4 * rows * k * wide}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """What run() returns, from the definitions in 64 bits; whole numbers are left to the plain form."""
    s = prepare(case, seed)
    up = {name: v.double() for name, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    op = case["op"]

    def f(z):
        return {"none": lambda: z, "relu": lambda: z * (z > 0), "gelu": lambda: z * torch.special.ndtr(z),
                "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)),
                "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()

    def forward(z):
        if not case.get("gated"):
            return f(z) if "act" in case else z
        gate, rest = z.split(case["n"], dim=1)
        return f(gate) * rest

    def pull(z, dy):
        z = z.clone().requires_grad_(True)
        with torch.enable_grad():
            return torch.autograd.grad(forward(z), z, dy)[0]

    if op == "linear":
        z = torch.einsum("tk,nk->tn", up["x"], up["w"])
        z = z + up["bias"] if case["bias"] else z
        out = forward(z) + (up["residual"] if case["residual"] else 0)
        return [out] + ([z] if case["keep"] else [])
    if op == "linear_backward":
        dz = pull(up["z"], up["dy"])
        got = [torch.einsum("tn,nk->tk", dz, up["w"]), torch.einsum("tn,tk->nk", dz, up["x"])]
        return got + ([torch.einsum("tn->n", dz)] if case["bias"] else [])
    if op in ("route", "route_backward"):
        def weights(x, ids):
            p = torch.softmax(x, 1) if case["scoring"] == "softmax" else torch.sigmoid(x)
            w = torch.take_along_dim(p, ids, 1)
            return w / w.sum(1, keepdim=True) if case["renorm"] else w

        x = up["logits"]
        if op == "route_backward":
            x.requires_grad_(True)
            with torch.enable_grad():
                return [torch.autograd.grad(weights(x, s["ids"].long()), x, up["dweights"])[0]]
        left = torch.softmax(x, 1) if case["scoring"] == "softmax" else torch.sigmoid(x)
        left = left + up["bias"] if case["bias"] else (left if case["groups"] > 1 else x.clone())
        if case["groups"] > 1:
            parts = torch.stack(left.split(case["experts"] // case["groups"], dim=1), dim=1)
            value = parts.topk(min(2, parts.shape[2]), dim=2).values.sum(2)
            bar = value.topk(case["top_groups"], dim=1).values[:, -1:]
            left = torch.where(value[:, :, None] >= bar[:, :, None], parts, -math.inf).flatten(1)
        picked = []
        for _ in range(case["top_k"]):
            best = left.max(dim=1, keepdim=True).values
            place = torch.arange(case["experts"], device=x.device).expand_as(left)
            at = torch.where(left == best, place, case["experts"]).min(dim=1, keepdim=True).values
            picked.append(at)
            left = left.scatter(1, at, -math.inf)
        return [None, weights(x, torch.cat(picked, dim=1))]
    # experts: the rows of each in the order of the tokens, found one expert at a time
    flat = s["ids"].flatten()
    if op == "expert_in":
        token = torch.arange(case["tokens"], device="cuda").repeat_interleave(case["top_k"])
        got = []
        for e in range(case["experts"]):
            z = up["x"][token[flat == e]] @ up["w"][e].T
            got.append(forward(z + up["bias"][e] if case["bias"] else z))
        got.append(torch.zeros(flat.numel() - sum(len(g) for g in got), case["n"], device="cuda", dtype=torch.float64))
        return [None, None, None, torch.cat(got)]
    first, out, grads = 0, torch.zeros_like(up["out"]) if op == "expert_out" else None, []
    for e in range(case["experts"]):
        mine = (flat == e).nonzero().flatten()
        rows = slice(first, first + len(mine))
        first += len(mine)
        if op == "expert_out":
            y = up["x"][rows] @ up["w"][e].T
            out.index_add_(0, mine // case["top_k"], y * up["weights"].flatten()[mine][:, None])
        else:
            dz = pull(up["z"][rows], up["dy"][rows])
            grads.append((dz @ up["w"][e], dz.T @ up["x"][rows], dz.sum(0)))
    if op == "expert_out":
        return [out + up["residual"]]
    rest = torch.zeros(flat.numel() - first, case["k"], device="cuda", dtype=torch.float64)
    got = [torch.cat([g[0] for g in grads] + [rest]), torch.stack([g[1] for g in grads])]
    return got + ([torch.stack([g[2] for g in grads])] if case["bias"] else [])
