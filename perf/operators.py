"""What the model-side operators are measured on: the work between two halo exchanges of a message-passing potential, called
through the public entry points, over rows [owned | ghost] and edge lists as the radius graph gives them (edges of a target
behind one another, targets in cell order, sources anywhere).

A case is one of these kinds:

  index      lists of a graph by target and by source (``neighbor_index``), once per MD step, shared by all layers
  attention  every target attends to its neighbours (``neighbor_attention``); with ``grad`` also all gradients, as every MD
             step needs them for the forces
  bias       learned bias of the logits from the distances, smooth at the cutoff (``distance_bias``); with ``grad`` also the
             gradients of the table (training) and of the distances (forces)
  linear     rows times the matrix of their atom type (``type_linear``); with ``grad`` also the gradients of rows, matrices
             and offsets

``run`` makes the framework's calls where ``own`` is true and computes the plain forms otherwise.
"""

import math

import torch

own = False

DENSITY = 0.1            # atoms per cubic Angstrom of the liquid in the repository's configurations
DILUTE = 0.004           # a thin gas, where many atoms have one neighbour or none
BUCKETS = 64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a small molecule box: launches and host time are all there is
        {"name": "index_liquid_1k", "kind": "index", "atoms": 1000, "owned": 1.0, "radius": 5.0, "density": DENSITY},
        # a rank's graph over [owned | ghost], odd size
        {"name": "index_owned_200k", "kind": "index", "atoms": 200_003, "owned": 0.77, "radius": 5.0, "density": DENSITY},
        # energies of a molecule box, no forces asked for
        {"name": "attention_500", "kind": "attention", "atoms": 500, "owned": 1.0, "radius": 5.0, "density": DENSITY, "heads": 8,
         "kv_heads": 8, "dim": 16, "dtype": "f32", "bias": True, "grad": False},
        # forces of a thin gas in half precision: lists of one edge and of none, a head size that is no multiple of 16 bytes
        {"name": "attention_grad_gas_9k", "kind": "attention", "atoms": 9001, "owned": 1.0, "radius": 5.0, "density": DILUTE,
         "heads": 6, "kv_heads": 3, "dim": 20, "dtype": "f16", "bias": True, "grad": True},
        # 256-wide embeddings, heads that share keys and values, no forces
        {"name": "attention_bf16_150k", "kind": "attention", "atoms": 150_000, "owned": 1.0, "radius": 5.0, "density": DENSITY,
         "heads": 8, "kv_heads": 2, "dim": 32, "dtype": "bf16", "bias": True, "grad": False},
        # one layer of a rank in an MD step: forces, a list with a skin whose far pairs the bias masks
        {"name": "attention_grad_owned_60k", "kind": "attention", "atoms": 60_001, "owned": 0.7, "radius": 5.5, "density": DENSITY,
         "heads": 4, "kv_heads": 4, "dim": 64, "dtype": "bf16", "bias": True, "grad": True},
        # the 128-wide embeddings of the configurations in single precision, the largest
        {"name": "attention_grad_200k", "kind": "attention", "atoms": 200_000, "owned": 1.0, "radius": 5.0, "density": DENSITY,
         "heads": 8, "kv_heads": 8, "dim": 16, "dtype": "f32", "bias": True, "grad": True},
        # biases of a molecule box's edges
        {"name": "bias_26k", "kind": "bias", "edges": 26_177, "heads": 8, "grad": False},
        # the edges of the 200 k atoms above, forces and the table's gradient
        {"name": "bias_grad_10m", "kind": "bias", "edges": 10_471_003, "heads": 8, "grad": True},
        # a molecule box, organic elements
        {"name": "linear_grad_1k", "kind": "linear", "rows": 1003, "types": 5, "inner": 128, "outer": 128, "dtype": "f32", "grad": True},
        # many elements with ragged shares, 256-wide embeddings, forward alone
        {"name": "linear_bf16_400k", "kind": "linear", "rows": 400_001, "types": 89, "inner": 256, "outer": 256, "dtype": "bf16", "grad": False},
        # a million atoms of the configurations, all gradients
        {"name": "linear_grad_1m", "kind": "linear", "rows": 1_000_000, "types": 5, "inner": 128, "outer": 128, "dtype": "f32", "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(hi, lo + 1))))))


def draw(rng):
    kind = rng.choice(["index", "attention", "attention", "attention", "bias", "linear", "linear"])
    if kind == "bias":
        return {"kind": kind, "edges": _log(rng, 1000, 10_000_000), "heads": rng.choice([1, 4, 5, 8, 8, 16]) if rng.random() < 0.5 else 8,
                "grad": rng.random() < 0.6}
    if kind == "linear":
        inner, outer = (rng.choice([64, 128, 128, 256, _log(rng, 16, 400)]) for _ in range(2))
        rows = _log(rng, 200, min(1_000_000, 1_000_000 * 128 * 128 // (inner * outer)))
        return {"kind": kind, "rows": rows, "types": rng.choice([1, 2, 5, 10, 89]), "inner": inner, "outer": outer,
                "dtype": rng.choice(["f32", "f32", "bf16", "f16"]), "grad": rng.random() < 0.6}
    case = {"kind": kind, "owned": rng.choice([1.0, 1.0, 0.5, 0.8]), "radius": rng.choice([4.5, 5.0, 5.5]),
            "density": rng.choice([DENSITY, DENSITY, DENSITY, DILUTE])}
    if kind == "index":
        return {**case, "atoms": _log(rng, 200, 200_000)}
    shared = rng.choice([1, 1, 1, 2, 4])
    kv = rng.choice([1, 2, 2, 3, 4]) if shared > 1 else rng.choice([1, 4, 8, 8, 5])
    dim = rng.choice([8, 16, 16, 32, 64, _log(rng, 5, 64)])
    width = shared * kv * dim
    atoms = _log(rng, 100, min(200_000, 200_000 * 90 // max(width, 90)))
    return {**case, "atoms": atoms, "heads": shared * kv, "kv_heads": kv, "dim": dim, "dtype": rng.choice(["f32", "f32", "bf16", "f16"]),
            "bias": rng.random() < 0.75, "grad": rng.random() < 0.6}


# ---------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _graph(case, gen):
    """Uniform atoms in a periodic box, the first ``owned`` part of it owned, and the pairs within the radius whose target is
    owned: ``edge_index`` [2, E], distances, number of targets and of rows.  The seed numbers the atoms: every seed has as many edges."""
    n, r = case["atoms"], case["radius"]
    length = (n / case["density"]) ** (1.0 / 3.0)
    pos = torch.rand(n, 3, generator=_generator(1002), device="cuda") * length
    side = max(int(length / r), 1)
    mine, rest = (torch.nonzero(t)[:, 0] for t in ((pos[:, 0] < length * case["owned"]), (pos[:, 0] >= length * case["owned"])))
    targets = mine.numel()
    pos = pos[torch.cat([t[torch.randperm(t.numel(), generator=gen, device="cuda")] for t in (mine, rest)])]
    at = (pos * (side / length)).long().clamp_(max=side - 1)
    flat = (at[:, 0] * side + at[:, 1]) * side + at[:, 2]
    order = torch.argsort(flat, stable=True)
    held = torch.bincount(flat, minlength=side ** 3)
    begin = torch.cumsum(held, 0) - held
    deep = int(held.max())
    slot = torch.arange(deep, device="cuda")
    near = range(-1, 2) if side >= 3 else range(side)
    mine = order[order < targets]
    src, dst = [], []
    for dx in near:
        for dy in near:
            for dz in near:
                shift = torch.tensor([dx, dy, dz], device="cuda")
                there = (at[mine] + shift) % side if side >= 3 else shift.expand(mine.numel(), 3)
                cell = (there[:, 0] * side + there[:, 1]) * side + there[:, 2]
                place = begin[cell][:, None] + slot
                ok = slot < held[cell][:, None]
                other = order[place.clamp_(max=n - 1)]
                d = pos[other] - pos[mine][:, None]
                d = d - length * torch.round(d / length)
                ok &= ((d * d).sum(-1) <= r * r) & (other != mine[:, None])
                i, j = torch.nonzero(ok, as_tuple=True)
                src.append(other[i, j])
                dst.append(i)
    src, dst = torch.cat(src), torch.cat(dst)
    by = torch.argsort(dst, stable=True)
    src, dst = src[by], mine[dst[by]]
    d = pos[src] - pos[dst]
    d = d - length * torch.round(d / length)
    return torch.stack([src, dst]).contiguous(), torch.sqrt((d * d).sum(-1)), targets, n


def _lists(edge_index, targets, sources):
    """The index of a graph from elementary operations: edges by target as they stand, and by source."""
    src, dst = edge_index[0], edge_index[1]
    edges, dev = src.numel(), src.device
    used, counts = torch.unique_consecutive(dst, return_counts=True)
    seen = torch.zeros(targets, dtype=torch.bool, device=dev)
    seen[used] = True
    rows = torch.cat([used, torch.nonzero(~seen)[:, 0]])
    row_start = torch.full((targets + 1,), edges, dtype=torch.int64, device=dev)
    row_start[0] = 0
    row_start[1:1 + used.numel()] = torch.cumsum(counts, 0)
    first = torch.full((sources,), edges, dtype=torch.int64, device=dev)
    first.scatter_reduce_(0, src, torch.arange(edges, device=dev), "amin")
    cols = torch.argsort(first, stable=True)
    place = torch.empty_like(cols)
    place[cols] = torch.arange(sources, device=dev)
    key = place[src]
    in_edge = torch.argsort(key, stable=True)
    col_start = torch.zeros(sources + 1, dtype=torch.int64, device=dev)
    col_start[1:] = torch.cumsum(torch.bincount(key, minlength=sources), 0)
    out = {"rows": rows, "row_start": row_start, "src": src, "cols": cols, "col_start": col_start, "in_edge": in_edge, "in_dst": dst[in_edge]}
    return {name: t.to(torch.int32) for name, t in out.items()}


def prepare(case, seed):
    gen = _generator(seed)
    kind, state = case["kind"], dict(case)

    def normal(*shape, dtype=torch.float32, scale=1.0, leaf=True):
        t = (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)
        return t.requires_grad_(bool(leaf and case.get("grad")))

    if kind in ("index", "attention"):
        edge_index, dist, targets, sources = _graph(case, gen)
        state.update(edge_index=edge_index, targets=targets, sources=sources)
        if kind == "index":
            return state
        dtype, dim = TYPES[case["dtype"]], case["dim"]
        state["index"] = _lists(edge_index, targets, sources)
        state["q"] = normal(targets, case["heads"], dim, dtype=dtype)
        state["k"] = normal(sources, case["kv_heads"], dim, dtype=dtype)
        state["v"] = normal(sources, case["kv_heads"], dim, dtype=dtype)
        state["bias"] = None
        if case["bias"]:
            # as the distances give it: decays towards the cutoff of 5 A, pairs of the skin behind it take no part
            u = (dist / 5.0).clamp(max=1.0)[:, None]
            learned = torch.randn(dist.numel(), case["heads"], generator=gen, device="cuda") * 0.5
            bias = torch.where(u < 1.0, learned + 3.0 * torch.log1p(-u.clamp(max=0.999)), -math.inf)
            state["bias"] = bias.requires_grad_(bool(case["grad"]))
        state["d_out"] = normal(targets, case["heads"], dim, dtype=dtype, leaf=False)
    elif kind == "bias":
        # distances of a liquid's pairs within 5.5 A, list and skin, for a cutoff of 5 A
        r = 5.5 * torch.rand(case["edges"], generator=gen, device="cuda") ** (1.0 / 3.0)
        state["dist"] = r.requires_grad_(bool(case["grad"]))
        state["table"] = normal(BUCKETS, case["heads"])
        state["d_bias"] = normal(case["edges"], case["heads"], leaf=False)
    else:
        dtype, types = TYPES[case["dtype"]], case["types"]
        # shares of the elements as 1 / (k + 1): one element common, most of them rare
        share = 1.0 / torch.arange(1, types + 1, device="cuda")
        kinds = torch.multinomial(share, case["rows"], replacement=True, generator=gen)
        state["order"] = torch.argsort(kinds, stable=True).to(torch.int32)
        state["start"] = torch.zeros(types + 1, dtype=torch.int32, device="cuda")
        state["start"][1:] = torch.cumsum(torch.bincount(kinds, minlength=types), 0)
        state["bounds"] = state["start"].tolist()
        state["x"] = normal(case["rows"], case["inner"], dtype=dtype)
        state["weight"] = normal(types, case["inner"], case["outer"], dtype=dtype, scale=case["inner"] ** -0.5)
        state["offset"] = normal(types, case["outer"], dtype=dtype)
        state["d_y"] = normal(case["rows"], case["outer"], dtype=dtype, leaf=False)
    return state


# ---------------------------------------------------------------------------------------------- plain forms
def _attention(s):
    src, dst = s["edge_index"][0], s["edge_index"][1]
    q, k, v = s["q"].detach().float(), s["k"].detach().float(), s["v"].detach().float()
    heads, shared, targets = q.size(1), q.size(1) // k.size(1), q.size(0)
    scale = q.size(2) ** -0.5
    k, v = k.repeat_interleave(shared, 1), v.repeat_interleave(shared, 1)
    ke, ve, qe = k[src], v[src], q[dst]
    logit = (qe * ke).sum(-1) * scale
    if s["bias"] is not None:
        bias = s["bias"].detach()
        logit = torch.where(bias == -math.inf, bias, logit + bias)
    top = logit.new_full((targets, heads), -math.inf).scatter_reduce_(0, dst[:, None].expand_as(logit), logit, "amax")
    p = torch.where(logit == -math.inf, 0.0, torch.exp(logit - top[dst]))
    total = p.new_zeros(targets, heads).index_add_(0, dst, p)
    p = p / torch.where(total > 0, total, 1.0)[dst]
    out = q.new_zeros(q.shape).index_add_(0, dst, p[..., None] * ve)
    result = {"out": out.to(s["q"].dtype)}
    if s["grad"]:
        do = s["d_out"].float()
        doe = do[dst]
        dp = (doe * ve).sum(-1)
        ds = p * (dp - (do * out).sum(-1)[dst])
        group = lambda t: t.view(t.size(0), -1, shared, t.size(2)).sum(2)  # noqa: E731
        result["dq"] = (q.new_zeros(q.shape).index_add_(0, dst, ds[..., None] * ke) * scale).to(s["q"].dtype)
        result["dk"] = group(k.new_zeros(k.shape).index_add_(0, src, ds[..., None] * qe) * scale).to(s["k"].dtype)
        result["dv"] = group(v.new_zeros(v.shape).index_add_(0, src, p[..., None] * doe)).to(s["v"].dtype)
        if s["bias"] is not None:
            result["d_bias"] = ds
    return result


def _spline(t):
    """The four cubic B-spline weights of a place t in [0, 1] between two buckets, and their derivatives."""
    w = torch.stack([(1 - t) ** 3, 3 * t ** 3 - 6 * t ** 2 + 4, -3 * t ** 3 + 3 * t ** 2 + 3 * t + 1, t ** 3], 1) / 6
    dw = torch.stack([-(1 - t) ** 2, 3 * t ** 2 - 4 * t, -3 * t ** 2 + 2 * t + 1, t ** 2], 1) / 2
    return w, dw


def _bias(s, cutoff=5.0):
    r, table = s["dist"].detach(), s["table"].detach()
    pieces = table.size(0) - 3
    x = (r.double() / cutoff * pieces).float()
    at = x.long().clamp(0, pieces - 1)
    w, dw = _spline(x - at)
    inside = r < cutoff
    u = r / cutoff
    rest = torch.where(inside, (cutoff - r) / cutoff, 1.0)   # exact next to the cutoff, where the logarithm is steep
    poly = 1 + 3 * u + 6 * u * u
    place = at[:, None] + torch.arange(4, device=r.device)
    rows = table[place]
    value = (w[..., None] * rows).sum(1) + (3 * torch.log(rest) + torch.log(poly))[:, None]
    result = {"bias": torch.where(inside[:, None], value, -math.inf)}
    if s["grad"]:
        g = torch.where(inside[:, None], s["d_bias"], 0.0)
        slope = (dw[..., None] * rows).sum(1) * pieces - (30 * u * u / (rest * poly))[:, None]
        result["d_dist"] = (g * slope).sum(1) / cutoff
        add = (w[..., None] * g[:, None]).reshape(-1, table.size(1)).double()   # 64 bits: sums over all edges of a bucket
        result["d_table"] = torch.zeros_like(table, dtype=torch.float64).index_add_(0, place.reshape(-1), add).float()
    return result


def _linear(s):
    x, weight, order, dtype = s["x"].detach().float(), s["weight"].detach().float(), s["order"].long(), s["x"].dtype
    y = x.new_empty(x.size(0), weight.size(2))
    if s["grad"]:
        d_y, dx = s["d_y"].float(), torch.empty_like(x)
        dw, db = torch.zeros_like(weight), torch.zeros_like(weight[:, 0])
    for t in range(weight.size(0)):
        rows = order[s["bounds"][t]:s["bounds"][t + 1]]
        xt = x[rows]
        y[rows] = xt @ weight[t] + s["offset"][t].detach().float()
        if s["grad"]:
            gt = d_y[rows]
            dx[rows] = gt @ weight[t].T
            dw[t] = xt.T @ gt
            db[t] = gt.sum(0)
    if not s["grad"]:
        return {"y": y.to(dtype)}
    return {"y": y.to(dtype), "dx": dx.to(dtype), "d_weight": dw.to(dtype), "d_offset": db.to(dtype)}


def run(state):
    if not own:
        with torch.no_grad():
            if state["kind"] == "index":
                return _lists(state["edge_index"], state["targets"], state["sources"])
            return {"attention": _attention, "bias": _bias, "linear": _linear}[state["kind"]](state)
    import dynamis_b200 as D

    s, kind = state, state["kind"]
    if kind == "index":
        index = D.neighbor_index(s["edge_index"], s["targets"], s["sources"])
        return {name: getattr(index, name) for name in ("rows", "row_start", "src", "cols", "col_start", "in_edge", "in_dst")}
    if kind == "attention":
        index = D.NeighborIndex(**s["index"])
        out = D.neighbor_attention(s["q"], s["k"], s["v"], index, s["bias"])
        result = {"out": out.detach()}
        if s["grad"]:
            leaves = [s["q"], s["k"], s["v"]] + ([s["bias"]] if s["bias"] is not None else [])
            result.update(zip(("dq", "dk", "dv", "d_bias"), torch.autograd.grad(out, leaves, s["d_out"])))
        return result
    if kind == "bias":
        bias = D.distance_bias(s["dist"], s["table"], 5.0)
        result = {"bias": bias.detach()}
        if s["grad"]:
            result.update(zip(("d_dist", "d_table"), torch.autograd.grad(bias, [s["dist"], s["table"]], s["d_bias"])))
        return result
    y = D.type_linear(s["x"], s["weight"], D.TypeIndex(order=s["order"], start=s["start"]), s["offset"])
    result = {"y": y.detach()}
    if s["grad"]:
        result.update(zip(("dx", "d_weight", "d_offset"), torch.autograd.grad(y, [s["x"], s["weight"], s["offset"]], s["d_y"])))
    return result


# ---------------------------------------------------------------------------------------------- measures
def _edges(case):
    """Edges that a uniform system has on average."""
    per = 4.0 / 3.0 * math.pi * case["radius"] ** 3 * case["density"]
    return case["owned"] * case["atoms"] * per


def work(case):
    kind = case["kind"]
    if kind in ("index", "attention"):
        e, rows, cols = _edges(case), case["owned"] * case["atoms"], case["atoms"]
        if kind == "index":   # endpoints in, three entries an edge and two a row out
            return {"bytes": int(16 * e + 12 * e + 8 * (rows + cols)), "flops": int(4 * e)}
        size, wide, kv = (4 if case["dtype"] == "f32" else 2), case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
        per_edge = 4 + (4 * case["heads"] if case["bias"] else 0)
        moved, flops = size * (2 * wide * rows + 2 * kv * cols) + per_edge * e + 8 * rows, 4 * wide * e
        if case["grad"]:   # the output's gradient in, three gradients out, the bias's gradient, the lists by source
            moved += size * (2 * wide * rows + 2 * kv * cols) + 8 * e + 8 * cols + (4 * case["heads"] * e if case["bias"] else 0)
            flops += 10 * wide * e
        return {"bytes": int(moved), "flops": int(flops)}
    if kind == "bias":
        e, h = case["edges"], case["heads"]
        moved, flops = 4 * e + 4 * h * e + 4 * BUCKETS * h, e * (8 * h + 30)
        if case["grad"]:
            moved, flops = moved + 4 * e + 4 * h * e + 4 * BUCKETS * h, flops + e * (18 * h + 30)
        return {"bytes": int(moved), "flops": int(flops)}
    n, a, b, t, size = case["rows"], case["inner"], case["outer"], case["types"], (4 if case["dtype"] == "f32" else 2)
    moved, flops = size * (n * (a + b) + t * (a * b + b)) + 4 * n, 2 * n * a * b
    if case["grad"]:
        moved, flops = moved + size * (n * (a + b) + t * (a * b + b)), 3 * flops
    return {"bytes": int(moved), "flops": int(flops)}


# ---------------------------------------------------------------------------------------------- 64 bits
def _exact_attention(s, chunk=4096):
    """Target by target on lists padded to the longest, a few thousand targets at a time."""
    rows, start, src = (s["index"][n].long() for n in ("rows", "row_start", "src"))
    q, k, v, do = (s[n].detach().double() for n in ("q", "k", "v", "d_out"))
    heads, shared, dim = q.size(1), q.size(1) // k.size(1), q.size(2)
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    d_bias = torch.zeros(src.numel(), heads, dtype=torch.float64, device=q.device)
    for c in range(0, rows.numel(), chunk):
        r = rows[c:c + chunk]
        b = start[c:c + r.numel()]
        n = start[c + 1:c + 1 + r.numel()] - b
        edge = b[:, None] + torch.arange(max(int(n.max()), 1), device=q.device)
        live = edge < (b + n)[:, None]
        edge = torch.where(live, edge, 0)
        if src.numel() == 0:
            continue
        who = src[edge]
        ks, vs = (t[who].unsqueeze(3).expand(-1, -1, -1, shared, -1).reshape(*who.shape, heads, dim) for t in (k, v))
        z = torch.einsum("thd,tnhd->tnh", q[r], ks) / math.sqrt(dim)
        if s["bias"] is not None:
            z = z + s["bias"].detach().double()[edge]
        z = z.masked_fill(~live[..., None], -math.inf)
        a = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
        out[r] = torch.einsum("tnh,tnhd->thd", a, vs)
        if s["grad"]:
            g = torch.einsum("thd,tnhd->tnh", do[r], vs)
            ds = a * (g - (a * g).sum(1, keepdim=True))
            dq[r] = torch.einsum("tnh,tnhd->thd", ds, ks) / math.sqrt(dim)
            to_k = torch.einsum("tnh,thd->tnhd", ds, q[r]) / math.sqrt(dim)
            to_v = torch.einsum("tnh,thd->tnhd", a, do[r])
            for grad, part in ((dk, to_k), (dv, to_v)):
                grad.index_add_(0, who[live], part.reshape(*who.shape, -1, shared, dim).sum(3)[live])
            d_bias[edge[live]] = ds[live]
    result = {"out": out}
    if s["grad"]:
        result.update(dq=dq, dk=dk, dv=dv)
        if s["bias"] is not None:
            result["d_bias"] = d_bias
    return result


def _exact_bias(s, cutoff=5.0):
    """The spline by its recursion over degrees, one bucket after the other, with gradients by differentiation."""
    r = s["dist"].detach().double().requires_grad_()
    table = s["table"].detach().double().requires_grad_()
    pieces = table.size(0) - 3
    x = r / cutoff * pieces
    inside = (s["dist"].detach() < cutoff)[:, None]
    value = 0.0
    for j in range(table.size(0)):     # bucket j stands over [j - 3, j + 1]
        y = (x - (j - 3)).clamp(0, 4)
        hat = ((y ** 3) - 4 * (y - 1).clamp(min=0) ** 3 + 6 * (y - 2).clamp(min=0) ** 3 - 4 * (y - 3).clamp(min=0) ** 3) / 6
        value = value + hat[:, None] * table[j]
    u = (r / cutoff)[:, None]
    u = torch.where(inside, u, 0.0)
    value = value + 3 * torch.log1p(-u) + torch.log1p(3 * u + 6 * u * u)
    result = {"bias": torch.where(inside, value, -math.inf).detach()}
    if s["grad"]:
        g = torch.where(inside, s["d_bias"].double(), 0.0)
        result["d_dist"], result["d_table"] = torch.autograd.grad(torch.where(inside, value, 0.0), [r, table], g)
    return result


def _exact_linear(s, chunk=1 << 16):
    x, weight, offset, d_y = (s[n].detach().double() for n in ("x", "weight", "offset", "d_y"))
    kinds = torch.empty(x.size(0), dtype=torch.int64, device=x.device)
    kinds[s["order"].long()] = torch.repeat_interleave(torch.arange(weight.size(0), device=x.device), (s["start"][1:] - s["start"][:-1]).long())
    y, dx = x.new_zeros(x.size(0), weight.size(2)), torch.zeros_like(x)
    dw, db = torch.zeros_like(weight), torch.zeros_like(offset)
    for t in range(weight.size(0)):
        mine = torch.nonzero(kinds == t)[:, 0]
        for rows in mine.split(chunk):
            y[rows] = x[rows] @ weight[t] + offset[t]
            dx[rows] = d_y[rows] @ weight[t].T
            dw[t] += x[rows].T @ d_y[rows]
            db[t] += d_y[rows].sum(0)
    result = {"y": y, "dx": dx, "d_weight": dw, "d_offset": db}
    return result if s["grad"] else {"y": y}


def exact(case, seed):
    if case["kind"] == "index":
        return None
    state = prepare(case, seed)
    if case["kind"] == "bias":
        return _exact_bias(state) if case["edges"] <= 2_000_000 else None
    return {"attention": _exact_attention, "linear": _exact_linear}[case["kind"]](state)
