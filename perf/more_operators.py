"""What the operators of an attention and expert layer of a message-passing potential are measured on, called through the public
entry points, over rows [owned | ghost] as the exchange gives them.

A case is one of these kinds:

  rotary   queries and keys normalised per head and turned by the positions of their rows (``rotary_heads``), in front of
           ``neighbor_attention``; with ``grad`` also the gradients of queries, keys, positions (forces) and of the norms' weights
  route    a few experts for every row from its logits (``route_experts``) and the rows by expert; with ``grad`` also the
           gradient of the logits
  expert   rows times the matrices of their experts, with offset and activation (``expert_linear``), from rows to (row, choice)
           pairs or from pairs to pairs; with ``grad`` also the gradients of rows, matrices and offsets
  combine  weighted sums of the pairs of a row on top of its residual (``expert_combine``); with ``grad`` also all gradients

``run`` makes the framework's calls where ``own`` is true and computes the plain forms otherwise.
"""

import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "f64": torch.float64}
EPS = 1e-6


def listed():
    return [
        # a molecule box, energies alone: launches and host time are all there is
        {"name": "rotary_500", "kind": "rotary", "rows": 500, "owned": 1.0, "heads": 8, "kv_heads": 8, "dim": 16, "dtype": "f32",
         "pos": "f32", "axes": 3, "periodic": True, "interleaved": False, "norm": True, "grad": False},
        # a rank's layer in an MD step in 16 bits: forces, heads that share keys, odd sizes
        {"name": "rotary_grad_owned_90k", "kind": "rotary", "rows": 90_001, "owned": 0.7, "heads": 8, "kv_heads": 2, "dim": 64,
         "dtype": "bf16", "pos": "f32", "axes": 3, "periodic": False, "interleaved": True, "norm": True, "grad": True},
        # the 128-wide embeddings of the configurations' million atoms in single precision, forces and training
        {"name": "rotary_grad_1m", "kind": "rotary", "rows": 1_000_000, "owned": 1.0, "heads": 8, "kv_heads": 8, "dim": 16,
         "dtype": "f32", "pos": "f32", "axes": 3, "periodic": True, "interleaved": False, "norm": True, "grad": True},
        # a molecule box: two of eight experts, energies alone
        {"name": "route_1k", "kind": "route", "rows": 1000, "experts": 8, "choices": 2, "score": "softmax", "bias": False, "groups": 1,
         "kept": 1, "renormalize": True, "closed": 0.0, "dtype": "f32", "grad": False},
        # a rank's rows, balanced by a bias, half of the groups kept, training
        {"name": "route_grad_groups_200k", "kind": "route", "rows": 200_003, "experts": 64, "choices": 6, "score": "sigmoid", "bias": True,
         "groups": 8, "kept": 4, "renormalize": True, "closed": 0.0, "dtype": "f32", "grad": True},
        # a million atoms, 16-bit logits (many equal ones), experts that some rows may not use
        {"name": "route_grad_1m", "kind": "route", "rows": 1_000_000, "experts": 32, "choices": 2, "score": "softmax", "bias": False,
         "groups": 1, "kept": 1, "renormalize": False, "closed": 0.3, "dtype": "bf16", "grad": True},
        # first product of a molecule box, single precision, training
        {"name": "expert_grad_1k", "kind": "expert", "rows": 1003, "experts": 8, "choices": 2, "paired": False, "inner": 128, "outer": 256,
         "activation": "silu", "offset": True, "absent": 0.0, "dtype": "f32", "grad": True},
        # second product, 16 bits, energies alone, ragged shares of 64 experts
        {"name": "expert_bf16_pairs_150k", "kind": "expert", "rows": 150_001, "experts": 64, "choices": 2, "paired": True, "inner": 512,
         "outer": 256, "activation": "none", "offset": False, "absent": 0.0, "dtype": "bf16", "grad": False},
        # first product, 16 bits, training, some places without an expert
        {"name": "expert_grad_bf16_150k", "kind": "expert", "rows": 150_000, "experts": 64, "choices": 2, "paired": False, "inner": 256,
         "outer": 512, "activation": "silu", "offset": True, "absent": 0.05, "dtype": "bf16", "grad": True},
        # second product in single precision, hidden rows of 512, forces and training
        {"name": "expert_grad_f32_100k", "kind": "expert", "rows": 100_000, "experts": 16, "choices": 2, "paired": True, "inner": 512,
         "outer": 128, "activation": "none", "offset": True, "absent": 0.0, "dtype": "f32", "grad": True},
        # a molecule box, energies alone
        {"name": "combine_1k", "kind": "combine", "rows": 1003, "choices": 2, "width": 128, "residual": True, "absent": 0.0, "dtype": "f32",
         "grad": False},
        # a rank's rows, forces and training
        {"name": "combine_grad_300k", "kind": "combine", "rows": 300_007, "choices": 4, "width": 256, "residual": True, "absent": 0.05,
         "dtype": "bf16", "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo + 1))))))


def draw(rng):
    kind = rng.choice(["rotary", "route", "expert", "expert", "combine"])
    dtype, grad = rng.choice(["f32", "f32", "bf16", "f16"]), rng.random() < 0.6
    if kind == "rotary":
        shared, kv = rng.choice([1, 1, 1, 2, 4]), rng.choice([1, 2, 4, 5, 8])
        dim = 2 * rng.choice([4, 8, 8, 16, 32, _log(rng, 2, 64)])
        width = (shared + 1) * kv * dim
        return {"kind": kind, "rows": _log(rng, 100, min(1_000_000, 1_000_000 * 256 // max(width, 256))), "owned": rng.choice([1.0, 1.0, 0.5, 0.8]),
                "heads": shared * kv, "kv_heads": kv, "dim": dim, "dtype": dtype, "pos": "f32" if grad else rng.choice(["f32", "f64"]), "axes": rng.choice([1, 2, 3, 3]),
                "periodic": rng.random() < 0.5, "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.7, "grad": grad}
    if kind == "route":
        groups, size = rng.choice([1, 1, 2, 4, 8]), rng.choice([2, 4, 4, 8, 8, 16, 5, 32])
        experts = groups * size
        kept = rng.randint(1, groups)
        return {"kind": kind, "rows": _log(rng, 200, min(1_000_000, 16_000_000 // experts)), "experts": experts, "choices": rng.randint(1, min(8, kept * size)),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "kept": kept,
                "renormalize": rng.random() < 0.6, "closed": rng.choice([0.0, 0.0, 0.3]), "dtype": dtype, "grad": grad}
    choices = rng.choice([1, 2, 2, 3, 4])
    absent = rng.choice([0.0, 0.0, 0.1])
    if kind == "combine":
        width = rng.choice([64, 128, 128, 256, _log(rng, 8, 600)])
        return {"kind": kind, "rows": _log(rng, 200, min(1_000_000, 300_000 * 4 * 128 // (choices * width))), "choices": choices, "width": width,
                "residual": rng.random() < 0.7, "absent": absent, "dtype": dtype, "grad": grad}
    inner, outer = (rng.choice([64, 128, 128, 256, 512, _log(rng, 16, 600)]) for _ in range(2))
    pairs = _log(rng, 200, min(600_000, 150_000 * 128 * 512 // (inner * outer)))
    return {"kind": kind, "rows": max(pairs // choices, 1), "experts": rng.choice([4, 8, 8, 16, 37, 64]), "choices": choices, "paired": rng.random() < 0.5,
            "inner": inner, "outer": outer, "activation": rng.choice(["none", "silu", "silu", "gelu"]), "offset": rng.random() < 0.6, "absent": absent,
            "dtype": dtype, "grad": grad}


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _by_expert(experts, count):
    """(row, choice) pairs by expert, ascending inside one, those without an expert behind the last; where every expert begins."""
    flat = experts.reshape(-1).long()
    key = torch.where(flat >= 0, flat, count)
    start = torch.zeros(count + 1, dtype=torch.int32, device=flat.device)
    start[1:] = torch.cumsum(torch.bincount(key, minlength=count + 1)[:count], 0)
    return torch.argsort(key, stable=True).to(torch.int32), start


def prepare(case, seed):
    gen = _generator(seed)
    kind, state = case["kind"], dict(case)
    rows, dtype = case["rows"], TYPES[case["dtype"]]

    def uniform(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    def normal(*shape, kind=dtype, scale=1.0, leaf=True):
        t = (torch.randn(*shape, generator=gen, device="cuda") * scale).to(kind)
        return t.requires_grad_(bool(leaf and case["grad"]))

    if kind == "rotary":
        dim, axes, targets = case["dim"], case["axes"], max(int(rows * case["owned"]), 1)
        pairs = torch.arange(dim // 2, device="cuda")
        if case["periodic"]:
            # fractional coordinates, some atoms in images of the box; whole waves over the box
            at = uniform(rows, axes).double() + torch.randint(-2, 3, (rows, axes), generator=gen, device="cuda")
            wave = torch.randint(-4, 5, (dim // 2, axes), generator=gen, device="cuda").float()
        else:
            # Cartesian coordinates of a box at 0.1 atoms per cubic Angstrom; each pair turns with one axis, from 3 to 600 Angstrom a turn
            at = uniform(rows, axes).double() * (rows / 0.1) ** (1.0 / 3.0)
            wave = torch.zeros(dim // 2, axes, device="cuda")
            wave[pairs, pairs % axes] = 0.3 * 200.0 ** (-pairs.float() / max(dim // 2 - 1, 1))
        state["at"] = at.to(TYPES[case["pos"]]).requires_grad_(bool(case["grad"]))
        state["wave"] = wave
        state["q"] = normal(targets, case["heads"], dim)
        state["k"] = normal(rows, case["kv_heads"], dim)
        for name in ("q_weight", "k_weight"):
            state[name] = (1.0 + 0.2 * torch.randn(dim, generator=gen, device="cuda")).requires_grad_(bool(case["grad"])) if case["norm"] else None
        state["d_q"] = normal(targets, case["heads"], dim, leaf=False)
        state["d_k"] = normal(rows, case["kv_heads"], dim, leaf=False)
        return state
    if kind == "route":
        # some experts liked more than others by all rows
        logits = normal(rows, case["experts"], kind=torch.float32, scale=1.5, leaf=False) + normal(case["experts"], kind=torch.float32, scale=0.7, leaf=False)
        logits[uniform(rows, case["experts"]) < case["closed"]] = -math.inf
        state["logits"] = logits.to(dtype).requires_grad_(bool(case["grad"]))
        state["balance"] = normal(case["experts"], kind=torch.float32, scale=0.1, leaf=False) if case["bias"] else None
        state["d_weights"] = normal(rows, case["choices"], kind=torch.float32, leaf=False)
        return state
    # a routing in hand: experts by shares 1 / (e + 1), different ones for a row, some places without one
    choices, count = case["choices"], case.get("experts", 16)
    share = -torch.log(torch.arange(1, count + 1, device="cuda").float())
    experts = (share - torch.log(-torch.log(uniform(rows, count).clamp(1e-7, 1 - 1e-7)))).topk(choices, 1).indices
    experts = torch.where(uniform(rows, choices) < case["absent"], -1, experts).to(torch.int32)
    weights = torch.where(experts >= 0, uniform(rows, choices), 0.0)
    state["experts_of"], state["weights"] = experts, weights.requires_grad_(bool(case["grad"] and kind == "combine"))
    state["order"], state["start"] = _by_expert(experts, count)
    if kind == "combine":
        state["z"] = normal(rows, choices, case["width"])
        state["residual_rows"] = normal(rows, case["width"]) if case["residual"] else None
        state["d_y"] = normal(rows, case["width"], leaf=False)
        return state
    state["bounds"] = state["start"].tolist()
    shape = (rows, choices) if case["paired"] else (rows,)
    state["x"] = normal(*shape, case["inner"])
    state["weight"] = normal(count, case["inner"], case["outer"], scale=case["inner"] ** -0.5)
    state["offset_rows"] = normal(count, case["outer"], scale=0.3) if case["offset"] else None
    state["d_z"] = normal(rows, choices, case["outer"], leaf=False)
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _pair(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _join(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def _rotary(s):
    along, mixed = s["at"].detach().double(), s["interleaved"]
    turns = along @ s["wave"].double().T      # angles of far rows: 64 bits
    angle = 2 * math.pi * (turns - turns.round())
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    result, d_angle = {}, torch.zeros_like(turns, dtype=torch.float32)
    for name in ("q", "k"):
        x = s[name].detach().float()
        n, c, t = x.size(0), cos[:x.size(0)], sin[:x.size(0)]
        if s["norm"]:
            g = s[name + "_weight"].detach()
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            unit = x * r
        else:
            unit, g = x, 1.0
        a, b = _pair(unit * g, mixed)
        result[name] = _join(a * c - b * t, a * t + b * c, mixed).to(s[name].dtype)
        if s["grad"]:
            da, db = _pair(s["d_" + name].float(), mixed)
            da, db = da * c + db * t, db * c - da * t
            d_angle[:n] += (db * a - da * b).sum(1)
            dn = _join(da, db, mixed)
            if s["norm"]:
                result[f"d_{name}_weight"] = (dn * unit).double().sum((0, 1)).float()     # sums over all rows: 64 bits
                dn = dn * g
                dn = r * (dn - unit * (dn * unit).mean(-1, keepdim=True))
            result["d_" + name] = dn.to(s[name].dtype)
    if s["grad"]:
        result["d_at"] = (2 * math.pi * (d_angle @ s["wave"])).to(s["at"].dtype)
    return {n: result[n] for n in ("q", "k", "d_q", "d_k", "d_at", "d_q_weight", "d_k_weight") if n in result}


def _route(s):
    logits = s["logits"].detach()
    wide = logits.double()                    # which expert comes first: 64 bits
    rows, count = logits.shape
    if s["score"] == "softmax":
        top = wide.max(1, keepdim=True).values.clamp(min=-1e300)
        score = torch.exp(wide - top)
        score = score / score.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        score = 1 / (1 + torch.exp(-wide))
    key = score if s["balance"] is None else score + s["balance"].double()
    key = torch.where(wide > -math.inf, key, -math.inf)
    if s["groups"] > 1:
        best = key.view(rows, s["groups"], -1).topk(min(2, count // s["groups"]), 2).values
        group = best[..., 0] + (torch.where(best[..., 1] > -math.inf, best[..., 1], 0.0) if best.size(2) > 1 else 0.0)
        kept = torch.sort(group, dim=1, descending=True, stable=True).indices[:, :s["kept"]]
        out = torch.ones_like(group, dtype=torch.bool).scatter_(1, kept, False)
        key = torch.where(out.repeat_interleave(count // s["groups"], 1), -math.inf, key)
    value, at = torch.sort(key, dim=1, descending=True, stable=True)
    value, at = value[:, :s["choices"]], at[:, :s["choices"]]
    live = value > -math.inf
    chosen = torch.where(live, score.gather(1, at), 0.0).float()
    total = chosen.sum(1, keepdim=True)
    weights = chosen / torch.where(total > 0, total, 1.0) if s["renormalize"] else chosen
    experts = torch.where(live, at, -1).to(torch.int32)
    order, start = _by_expert(experts, count)
    result = {"experts": experts, "weights": weights, "order": order, "start": start}
    if s["grad"]:
        g = torch.where(live, s["d_weights"], 0.0)
        if s["renormalize"]:
            d = weights * (g - (g * weights).sum(1, keepdim=True))
            if s["score"] == "sigmoid":
                d = d * (1 - chosen)
            full = torch.zeros(rows, count, device=d.device).scatter_add_(1, at, d)
        elif s["score"] == "sigmoid":
            full = torch.zeros(rows, count, device=g.device).scatter_add_(1, at, g * chosen * (1 - chosen))
        else:
            full = torch.zeros(rows, count, device=g.device).scatter_add_(1, at, g)
            full = score.float() * (full - (g * chosen).sum(1, keepdim=True))
        result["d_logits"] = full.to(logits.dtype)
    return result


def _activation(u, name):
    """The activation and its slope."""
    if name == "silu":
        p = 1 / (1 + torch.exp(-u))
        return u * p, p * (1 + u * (1 - p))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(u * math.sqrt(0.5)))
        return u * p, p + u * torch.exp(-0.5 * u * u) * (1 / math.sqrt(2 * math.pi))
    return u, torch.ones_like(u)


def _expert(s):
    x, weight, order = s["x"].detach().float(), s["weight"].detach().float(), s["order"].long()
    choices, count, dtype = s["choices"], weight.size(0), s["x"].dtype
    flat, wide = x.reshape(-1, x.size(-1)), weight.size(2)
    z = x.new_zeros(order.numel(), wide)
    if s["grad"]:
        d_z = s["d_z"].float().view(-1, wide)
        dx, dw, db = torch.zeros_like(flat), torch.zeros_like(weight), torch.zeros_like(weight[:, 0])
    for e in range(count):
        pairs = order[s["bounds"][e]:s["bounds"][e + 1]]
        rows = pairs if s["paired"] else pairs // choices
        xe = flat[rows]
        u = xe @ weight[e]
        if s["offset"]:
            u = u + s["offset_rows"][e].detach().float()
        z[pairs], slope = _activation(u, s["activation"])
        if s["grad"]:
            du = d_z[pairs] * slope
            dx.index_add_(0, rows, du @ weight[e].T)
            dw[e] = xe.T @ du
            db[e] = du.sum(0)
    result = {"z": z.view(-1, choices, wide).to(dtype)}
    if s["grad"]:
        result.update(d_x=dx.view(x.shape).to(dtype), d_weight=dw.to(dtype))
        if s["offset"]:
            result["d_offset"] = db.to(dtype)
    return result


def _combine(s):
    z, w = s["z"].detach().float(), s["weights"].detach()
    live = s["experts_of"] >= 0
    w = torch.where(live, w, 0.0)
    y = (w[..., None] * z).sum(1)
    if s["residual"]:
        y = y + s["residual_rows"].detach().float()
    result = {"y": y.to(s["z"].dtype)}
    if s["grad"]:
        d_y = s["d_y"].float()[:, None]
        result["d_z"] = (w[..., None] * d_y).to(s["z"].dtype)
        result["d_weights"] = torch.where(live, (d_y * z).sum(-1), 0.0)
        if s["residual"]:
            result["d_residual"] = s["d_y"].clone()
    return result


def run(state):
    if not own:
        with torch.no_grad():
            return {"rotary": _rotary, "route": _route, "expert": _expert, "combine": _combine}[state["kind"]](state)
    import dynamis_b200 as D

    s, kind, grad = state, state["kind"], state["grad"]
    if kind == "rotary":
        q, k = D.rotary_heads(s["q"], s["k"], s["at"], s["wave"], s["q_weight"], s["k_weight"], eps=EPS if s["norm"] else None, interleaved=s["interleaved"])
        result = {"q": q.detach(), "k": k.detach()}
        if grad:
            names = ["q", "k", "at"] + (["q_weight", "k_weight"] if s["norm"] else [])
            grads = torch.autograd.grad([q, k], [s[n] for n in names], [s["d_q"], s["d_k"]])
            result.update(zip(("d_" + n for n in names), grads))
        return result
    if kind == "route":
        routing = D.route_experts(s["logits"], s["choices"], score=s["score"], bias=s["balance"], groups=s["groups"], kept_groups=s["kept"],
                                  renormalize=s["renormalize"])
        result = {"experts": routing.experts, "weights": routing.weights.detach(), "order": routing.order, "start": routing.start}
        if grad:
            result["d_logits"], = torch.autograd.grad(routing.weights, [s["logits"]], s["d_weights"])
        return result
    routing = D.Routing(experts=s["experts_of"], weights=s["weights"], order=s["order"], start=s["start"])
    if kind == "expert":
        z = D.expert_linear(s["x"], s["weight"], routing, s["offset_rows"], activation=None if s["activation"] == "none" else s["activation"])
        result = {"z": z.detach()}
        if grad:
            leaves = [s["x"], s["weight"]] + ([s["offset_rows"]] if s["offset"] else [])
            result.update(zip(("d_x", "d_weight", "d_offset"), torch.autograd.grad(z, leaves, s["d_z"])))
        return result
    y = D.expert_combine(s["z"], routing, s["residual_rows"])
    result = {"y": y.detach()}
    if grad:
        leaves = [s["z"], s["weights"]] + ([s["residual_rows"]] if s["residual"] else [])
        result.update(zip(("d_z", "d_weights", "d_residual"), torch.autograd.grad(y, leaves, s["d_y"])))
    return result


# ---------------------------------------------------------------------------------------------- measures
def work(case):
    kind, n, grad, size = case["kind"], case["rows"], case["grad"], (4 if case["dtype"] == "f32" else 2)
    if kind == "rotary":
        dim, place = case["dim"], (8 if case["pos"] == "f64" else 4) * case["axes"] * n
        values = max(int(n * case["owned"]), 1) * case["heads"] * dim + n * case["kv_heads"] * dim
        fixed = 4 * (dim // 2) * case["axes"] + (8 * dim if case["norm"] else 0)
        moved, flops = 2 * size * values + place + fixed, 7 * values
        if grad:      # the results' gradients in, three kinds of gradients out
            moved, flops = moved + 2 * size * values + place + (8 * dim if case["norm"] else 0), flops + 16 * values
        return {"bytes": int(moved), "flops": int(flops)}
    if kind == "route":
        e, c = case["experts"], case["choices"]
        moved, flops = size * n * e + 12 * n * c + 4 * e + (4 * e if case["bias"] else 0), n * e * (6 + c)
        if grad:
            moved, flops = moved + 4 * n * c + size * n * e, flops + 4 * n * e
        return {"bytes": int(moved), "flops": int(flops)}
    c = case["choices"]
    pairs = n * c
    if kind == "combine":
        values = pairs * case["width"] + n * case["width"] * (2 if case["residual"] else 1)
        moved, flops = size * values + 8 * pairs, 2 * pairs * case["width"]
        if grad:      # the result's gradient in; those of pairs, weights and residuals out
            moved, flops = moved + size * values + 4 * pairs, 3 * flops
        return {"bytes": int(moved), "flops": int(flops)}
    a, b, e = case["inner"], case["outer"], case["experts"]
    rows_in = pairs if case["paired"] else n
    weights = e * a * b + (e * b if case["offset"] else 0)
    moved, flops = size * (rows_in * a + pairs * b + weights) + 4 * pairs, 2 * pairs * a * b
    if grad:
        moved, flops = 2 * moved - 4 * pairs, 3 * flops
    return {"bytes": int(moved), "flops": int(flops)}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_rotary(s):
    """The rotation as a product of complex numbers, gradients by differentiation."""
    leaves = {n: s[n].detach().double().requires_grad_() for n in ("q", "k", "at", "q_weight", "k_weight") if s[n] is not None}
    at = s["at"].detach().double()
    whole = (at @ s["wave"].double().T).round()                       # whole turns are left out
    phase = leaves["at"] @ s["wave"].double().T - whole
    turn = torch.polar(torch.ones_like(phase), 2 * math.pi * phase)
    result, outs, grads = {}, [], []
    half = s["dim"] // 2
    for name in ("q", "k"):
        x = leaves[name]
        if s["norm"]:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / s["dim"] + EPS) * leaves[name + "_weight"]
        pair = x.unflatten(-1, (half, 2)) if s["interleaved"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
        y = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn[:x.size(0), None])
        y = (y if s["interleaved"] else y.transpose(-1, -2)).flatten(-2)
        result[name] = y.detach()
        outs.append(y)
        grads.append(s["d_" + name].double())
    if s["grad"]:
        result.update(zip(("d_" + n for n in leaves), torch.autograd.grad(outs, list(leaves.values()), grads)))
    return result


def _exact_route(s):
    """One choice after the other, each the first of the largest keys; gradients by differentiation of logarithms."""
    logits = s["logits"].detach().double().requires_grad_()
    rows, count = logits.shape
    fixed = logits.detach()
    shut = fixed == -math.inf
    if s["score"] == "softmax":
        all_shut = shut.all(1, keepdim=True)
        log_score = torch.log_softmax(torch.where(all_shut, 0.0, logits), 1)
    else:
        log_score = torch.nn.functional.logsigmoid(logits)
    log_score = torch.where(shut, -math.inf, log_score)
    key = log_score.detach().exp() + (0.0 if s["balance"] is None else s["balance"].double())
    key = key.masked_fill(shut, -math.inf)
    number = torch.arange(count, device=key.device)

    def first_of_largest(t):
        best = t.max(1, keepdim=True).values
        return best[:, 0], torch.where(t == best, torch.arange(t.size(1), device=t.device), t.size(1)).min(1).values

    if s["groups"] > 1:
        per = count // s["groups"]
        parts = []
        for g in range(s["groups"]):
            part = key[:, g * per:(g + 1) * per]
            best, where = first_of_largest(part)
            rest = part.masked_fill(number[:per] == where[:, None], -math.inf).max(1).values
            parts.append(best + torch.where(rest == -math.inf, 0.0, rest))
        left, keep = torch.stack(parts, 1), torch.zeros(rows, s["groups"], dtype=torch.bool, device=key.device)
        for _ in range(s["kept"]):
            best, where = first_of_largest(torch.where(keep, -math.inf, left))
            none = best == -math.inf      # groups without an open expert come behind all others; of those the first not yet kept
            spare = torch.where(keep, s["groups"], torch.arange(s["groups"], device=key.device)).min(1).values
            keep[torch.arange(rows, device=key.device), torch.where(none, spare, where)] = True
        key = torch.where(keep.repeat_interleave(per, 1), key, -math.inf)
    experts, logs = [], []
    for _ in range(s["choices"]):
        best, where = first_of_largest(key)
        none = best == -math.inf
        experts.append(torch.where(none, -1, where))
        logs.append(torch.where(none, -math.inf, log_score.gather(1, where[:, None])[:, 0]))
        key = key.masked_fill(number == where[:, None], -math.inf)
    experts, logs = torch.stack(experts, 1), torch.stack(logs, 1)
    live = experts >= 0
    safe = torch.where(live, logs, -1e4)
    if s["renormalize"]:
        weights = torch.where(live, torch.softmax(safe, 1), 0.0)
    else:
        weights = torch.where(live, torch.exp(safe), 0.0)
    lists = [torch.nonzero(experts.reshape(-1) == e)[:, 0] for e in [*range(count), -1]]
    start = torch.tensor([0] + [t.numel() for t in lists[:-1]], device=key.device).cumsum(0)
    result = {"experts": experts.to(torch.int32), "weights": weights.detach(), "order": torch.cat(lists).to(torch.int32), "start": start.to(torch.int32)}
    if s["grad"]:
        grad, = torch.autograd.grad(weights, [logits], torch.where(live, s["d_weights"].double(), 0.0))
        result["d_logits"] = torch.nan_to_num(grad, nan=0.0)
    return result


def _exact_expert(s, chunk=1 << 16):
    flat, weight = s["x"].detach().double().reshape(-1, s["inner"]), s["weight"].detach().double()
    of = s["experts_of"].reshape(-1).long()
    offset = s["offset_rows"].detach().double() if s["offset"] else weight.new_zeros(weight.size(0), s["outer"])
    z = weight.new_zeros(of.numel(), s["outer"])
    d_z = s["d_z"].double().view(-1, s["outer"])
    dx, dw, db = torch.zeros_like(flat), torch.zeros_like(weight), torch.zeros_like(offset)
    act = {"none": lambda u: u, "silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu}[s["activation"]]
    for e in range(weight.size(0)):
        for pairs in torch.nonzero(of == e)[:, 0].split(chunk):
            rows = pairs if s["paired"] else torch.div(pairs, s["choices"], rounding_mode="floor")
            u = (flat[rows] @ weight[e] + offset[e]).requires_grad_()
            with torch.enable_grad():
                out = act(u)
            z[pairs] = out.detach()
            if s["grad"]:
                du, = torch.autograd.grad(out, [u], d_z[pairs])
                dx.index_add_(0, rows, du @ weight[e].T)
                dw[e] += flat[rows].T @ du
                db[e] += du.sum(0)
    result = {"z": z.view(-1, s["choices"], s["outer"])}
    if s["grad"]:
        result.update(d_x=dx.view(s["x"].shape), d_weight=dw)
        if s["offset"]:
            result["d_offset"] = db
    return result


def _exact_combine(s):
    live = (s["experts_of"] >= 0).double()
    z, w = s["z"].detach().double(), s["weights"].detach().double() * live
    y = torch.einsum("nc,ncw->nw", w, z)
    if s["residual"]:
        y = y + s["residual_rows"].detach().double()
    result = {"y": y}
    if s["grad"]:
        d_y = s["d_y"].double()
        result["d_z"] = torch.einsum("nc,nw->ncw", w, d_y)
        result["d_weights"] = torch.einsum("nw,ncw->nc", d_y, z) * live
        if s["residual"]:
            result["d_residual"] = d_y
    return result


def exact(case, seed):
    state = prepare(case, seed)
    return {"rotary": _exact_rotary, "route": _exact_route, "expert": _exact_expert, "combine": _exact_combine}[case["kind"]](state)
