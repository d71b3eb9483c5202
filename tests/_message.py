"""Plain forms in 64 bits of the message-passing operators, with bounds on what 32-bit kernels may be off.

u = 2^-24 is half a step of fp32 relative to the value.  A sum of n products in any order is off by at most (n + 1) u times the sum of the
products' magnitudes; a result rounded to a type is off by half a step of the type more (and for fp16 by 2^-25 where it is subnormal)."""

from __future__ import annotations

import torch

U = 2.0 ** -24
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def rounding(ref: torch.Tensor, dtype) -> torch.Tensor:
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150
    return torch.finfo(dtype).eps / 2 * ref.abs() + tiny


def check(got: torch.Tensor, ref: torch.Tensor, slack: torch.Tensor, what: str):
    """|got - ref| within slack before and half a step of got's type behind the rounding."""
    assert got.shape == ref.shape, f"{what}: {tuple(got.shape)} for {tuple(ref.shape)}"
    ok_inf = torch.isinf(ref) & (got.double() == ref)
    off = torch.where(ok_inf, 0.0, (got.double() - ref).abs())
    limit = torch.where(ok_inf, 0.0, slack * (1 + torch.finfo(got.dtype).eps) + rounding(ref, got.dtype))
    bad = ~(off <= limit)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / limit.clamp(min=1e-300))[bad].max()):.3g} of the limit "
                           f"at {torch.nonzero(bad)[0].tolist()}")


def attention(q, k, v, src, dst, bias, scale, d_out=None):
    """{name: (value, bound)} of out, and with d_out of dq, dk, dv, d_bias; edges in any order.  What a masked edge's rows hold is not
    used.  The bounds follow the formula step by step:
      z: dot of dim products, scale and bias;   p = exp(z - top) / sum: relative error 2 (dz_e + largest dz of the target) for
      numerator and denominator, |z - top| 3 u for the exponent's argument, 8 u for two exponentials, the division and products, n u for
      the sum;   dp, delta: dots of dim products;   ds = p (dp - delta);   sums over lists of n edges."""
    q, k, v = (t.detach().double() for t in (q, k, v))
    T, H, D = q.shape
    shared = H // k.size(1)
    kk, vv = k.repeat_interleave(shared, 1), v.repeat_interleave(shared, 1)
    E, dev = src.numel(), q.device
    b = torch.zeros(E, H, dtype=torch.float64, device=dev) if bias is None else bias.detach().double()
    live = b != -float("inf")

    def rows(t, at):
        return torch.where(live[..., None], t[at], 0.0)

    def add(n, at, what):
        return torch.zeros((n,) + what.shape[1:], dtype=torch.float64, device=dev).index_add_(0, at, what)

    qe, ke, ve = rows(q, dst), rows(kk, src), rows(vv, src)
    dots, mags = (qe * ke).sum(-1) * scale, (qe * ke).abs().sum(-1) * abs(scale)
    z = torch.where(live, dots + b, -float("inf"))
    n = add(T, dst, torch.ones(E, 1, dtype=torch.float64, device=dev))
    top = torch.full((T, H), -float("inf"), dtype=torch.float64, device=dev).scatter_reduce_(0, dst[:, None].expand(E, H), z, "amax")
    fall = torch.where(live, z - top[dst], 0.0)
    p = torch.where(live, torch.exp(fall), 0.0)
    total = add(T, dst, p)
    p = p / torch.where(total > 0, total, 1.0)[dst]
    dz = torch.where(live, (D + 4) * U * mags + 2 * U * torch.where(live, b.abs() + z.abs(), 0.0), 0.0)
    dz_top = torch.zeros(T, H, dtype=torch.float64, device=dev).scatter_reduce_(0, dst[:, None].expand(E, H), dz, "amax")
    rel = 2 * (dz + dz_top[dst]) + 3 * U * fall.abs() + (8 + n[dst]) * U
    rel = torch.expm1(rel)
    dp_abs = p * rel + 2.0 ** -126     # an exponential below the smallest normal number may be flushed
    out = add(T, dst, p[..., None] * ve)
    out_off = add(T, dst, (dp_abs + (n[dst] + 2) * U * p)[..., None] * ve.abs())
    result = {"out": (out, out_off)}
    if d_out is None:
        return result
    g = d_out.double()
    ge = rows(g, dst)
    dp, dp_mag = (ge * ve).sum(-1), (ge * ve).abs().sum(-1)
    delta = (g * out).sum(-1)
    delta_off = (g.abs() * (out_off + U * out.abs())).sum(-1) + (D + 2) * U * (g * out).abs().sum(-1)
    diff = torch.where(live, dp - delta[dst], 0.0)
    diff_off = (D + 2) * U * dp_mag + delta_off[dst] + 2 * U * diff.abs()
    ds = p * diff
    ds_off = dp_abs * (diff.abs() + diff_off) + p * diff_off + 4 * U * ds.abs()
    m = add(kk.size(0), src, torch.ones(E, 1, dtype=torch.float64, device=dev))

    def kv(t):
        return t.view(t.size(0), -1, shared, D).sum(2)

    nd, ms = (n[dst] + 6) * U, (m[src] * shared + 6) * U
    result["dq"] = (add(T, dst, ds[..., None] * ke) * scale, add(T, dst, (ds_off + nd * ds.abs())[..., None] * ke.abs()) * abs(scale))
    result["dk"] = (kv(add(kk.size(0), src, ds[..., None] * qe) * scale), kv(add(kk.size(0), src, (ds_off + ms * ds.abs())[..., None] * qe.abs()) * abs(scale)))
    result["dv"] = (kv(add(kk.size(0), src, p[..., None] * ge)), kv(add(kk.size(0), src, (dp_abs + ms * p)[..., None] * ge.abs())))
    result["d_bias"] = (ds, ds_off)
    return result


def spline(dist, table, cutoff, smooth=True):
    """The bias in 64 bits, differentiable (dist, table: float64), by the recursion of truncated powers."""
    K = table.size(0)
    x = dist / cutoff * (K - 3)
    value = torch.zeros(dist.numel(), table.size(1), dtype=torch.float64, device=dist.device)
    for j in range(K):
        y = (x - (j - 3)).clamp(0, 4)
        hat = (y ** 3 - 4 * (y - 1).clamp(min=0) ** 3 + 6 * (y - 2).clamp(min=0) ** 3 - 4 * (y - 3).clamp(min=0) ** 3) / 6
        value = value + hat[:, None] * table[j]
    inside = dist < cutoff
    if smooth:
        u = torch.where(inside, dist / cutoff, 0.0)
        value = value + (3 * torch.log1p(-u) + torch.log1p(3 * u + 6 * u * u))[:, None]
    return torch.where(inside[:, None], value, -float("inf"))


def ragged_graph(degrees, sources, seed, dev, apart=False):
    """Edges of targets in a scattered order, ``degrees[t]`` of them from random sources: (edge_index, src, dst)."""
    gen = torch.Generator().manual_seed(seed)
    deg = torch.as_tensor(degrees, dtype=torch.int64)
    order = torch.randperm(deg.numel(), generator=gen)
    dst = torch.repeat_interleave(order, deg[order])
    src = torch.randint(0, max(sources, 1), (dst.numel(),), generator=gen)
    if apart:
        dst = dst[torch.randperm(dst.numel(), generator=gen)]
    ei = torch.stack([src, dst]).to(dev)
    return ei, ei[0], ei[1]


def index_lists(src, dst, T, S):
    """The seven lists by a walk over the edges (CPU)."""
    src, dst = src.tolist(), dst.tolist()
    rows, row_start, seen = [], [], set()
    cols, into = [], {}
    for e, (s, d) in enumerate(zip(src, dst)):
        if d not in seen:
            seen.add(d)
            rows.append(d)
            row_start.append(e)
        if s not in into:
            into[s] = []
            cols.append(s)
        into[s].append(e)
    E = len(src)
    empty = [t for t in range(T) if t not in seen]
    rows, row_start = rows + empty, row_start + [E] * (len(empty) + 1)
    if not rows:
        row_start = [E]
    cols = cols + [s for s in range(S) if s not in into]
    col_start, in_edge = [0], []
    for s in cols:
        in_edge += into.get(s, [])
        col_start.append(len(in_edge))
    return {"rows": rows, "row_start": row_start, "src": src, "cols": cols, "col_start": col_start, "in_edge": in_edge,
            "in_dst": [dst[e] for e in in_edge]}
