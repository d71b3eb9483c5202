"""Plain forms in 64 bits of rotary heads, routing and the experts' products, with bounds on what 32-bit kernels may be off.

u = 2^-24 is half a step of fp32 relative to the value.  A sum of n products in any order is off by at most (n + 1) u times the sum of the
products' magnitudes; results that are rounded to a type are off by half a step of it more (tests/_message.py: check)."""

from __future__ import annotations

import math

import torch

from tests import _message as M

U = M.U


def _pair(x, interleaved):
    return (x[..., 0::2], x[..., 1::2]) if interleaved else x.chunk(2, -1)


def _join(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def rotary(q, k, pos, wave, q_weight, k_weight, eps, interleaved, d_q, d_k):
    """{name: (value, bound)} of q, k, d_q, d_k, d_pos and with a norm d_q_weight, d_k_weight.  Step by step:
      r = 1 / sqrt(mean + eps): the mean of D squares is off by (D + 2) u, relative; root, division and the addition bring 4 u more, and the root halves what
        was there before it: (D / 2 + 6) u
      n = x r w: two products more;   cosine and sine: the angle is left with at most half a turn, rounded to 32 bits (pi u at most), sincospif adds 2 ulp
        (2 u at most), and 64 bits lose (axes + 1) 2^-53 of the turns' magnitudes
      results: two products and a sum of two terms that share the error of the cosine.
    Gradients follow the formulas; sums over n terms bring (n + 8) u of the magnitudes."""
    axes = pos.size(1)
    p64, w64 = pos.detach().double(), wave.double()
    turns = p64 @ w64.T
    angle = 2 * math.pi * (turns - turns.round())
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    off_c = ((math.pi + 2 + 1) * U + 2 * math.pi * (axes + 1) * 2.0 ** -53 * (p64.abs() @ w64.abs().T))[:, None]
    d_theta = torch.zeros_like(turns)
    off_theta, mag_theta = torch.zeros_like(turns), torch.zeros_like(turns)
    result = {}
    for name, x, w, g in (("q", q, q_weight, d_q), ("k", k, k_weight, d_k)):
        x, g = x.detach().double(), g.double()
        n, D = x.size(0), x.size(2)
        w = torch.ones(D, dtype=torch.float64, device=x.device) if w is None else w.detach().double()
        r, rel_r = (torch.ones_like(x[..., :1]), 0.0) if eps is None else (torch.rsqrt((x * x).mean(-1, keepdim=True) + eps), (D / 2 + 6) * U)
        cc, ss, oc = c[:n], s[:n], off_c[:n]
        na, nb = _pair(x * r * w, interleaved)
        mag = na.abs() + nb.abs()
        bound = mag * (rel_r + 5 * U + oc)
        result[name] = (_join(na * cc - nb * ss, na * ss + nb * cc, interleaved), _join(bound, bound, interleaved))
        ga, gb = _pair(g, interleaved)
        da, db = ga * cc + gb * ss, gb * cc - ga * ss
        off_d = (ga.abs() + gb.abs()) * (oc + 3 * U)
        dn, off_dn = _join(da, db, interleaved), _join(off_d, off_d, interleaved)
        both = (db * na).abs() + (da * nb).abs()
        d_theta[:n] += (db * na - da * nb).sum(1)
        mag_theta[:n] += both.sum(1)
        off_theta[:n] += (off_d * mag + both * (rel_r + 4 * U)).sum(1)
        if eps is None:
            result["d_" + name] = (dn, off_dn)
            continue
        result[f"d_{name}_weight"] = ((dn * x * r).sum((0, 1)), (off_dn * (x * r).abs() + (dn * x * r).abs() * (rel_r + (n * x.size(1) + 8) * U)).sum((0, 1)))
        m = (w * dn * x).mean(-1, keepdim=True)
        off_m = ((w * x).abs() * off_dn + (D + 8) * U * (w * dn * x).abs()).mean(-1, keepdim=True)
        part = x.abs() * r * r
        value = r * (w * dn - x * r * r * m)
        off = r * (w.abs() * (off_dn + 3 * U * dn.abs()) + part * (off_m + m.abs() * (2 * rel_r + 6 * U))) + r * ((w * dn).abs() + part * m.abs()) * (rel_r + 4 * U)
        result["d_" + name] = (value, off)
    heads = q.size(1) + k.size(1)
    terms = heads + wave.size(0) + 40
    result["d_pos"] = (2 * math.pi * d_theta @ w64, 2 * math.pi * (off_theta + terms * U * mag_theta) @ w64.abs())
    return result


def route(logits, choices, score="softmax", bias=None, groups=1, kept_groups=1, renormalize=True, scale=1.0, d_weights=None):
    """Experts, order and start by a walk over the rows (CPU, 64 bits), weights and the logits' gradient with bounds."""
    l64 = logits.detach().double().cpu()
    rows, count = l64.shape
    per = count // groups
    experts = torch.full((rows, choices), -1, dtype=torch.int32)
    s = torch.softmax(l64, 1) if score == "softmax" else torch.sigmoid(l64)
    s = torch.where(l64 == -math.inf, 0.0, s)
    plain = bias is None and groups == 1
    key = l64.clone() if plain else torch.where(l64 == -math.inf, -math.inf, s + (0.0 if bias is None else bias.double().cpu()))
    rank = torch.where(torch.isnan(key), math.inf, key)
    for i, row in enumerate(rank.tolist()):
        group = []
        for g in range(groups):
            two = sorted((v for v in row[g * per:(g + 1) * per] if v > -math.inf), reverse=True)[:2]
            group.append(sum(two) if two else -math.inf)
        stay = set(sorted(range(groups), key=lambda g: (-group[g], g))[:kept_groups])
        open_ = [e for e in range(count) if row[e] > -math.inf and e // per in stay]
        for j, e in enumerate(sorted(open_, key=lambda e: (-row[e], e))[:choices]):
            experts[i, j] = e
    live, at = experts >= 0, experts.long().clamp(min=0)
    logit = l64.gather(1, at)
    if score == "softmax":
        z, top = logit, l64.max(1, keepdim=True).values.clamp(min=-1e300)
        fall = torch.where(live, top - z, 0.0)
        spread = torch.where(l64 == -math.inf, 0.0, torch.softmax(l64, 1) * (top - l64)).sum(1, keepdim=True)
        rel = (2 * fall + spread + count + 12) * U
    else:
        z = torch.nn.functional.logsigmoid(logit)
        rel = torch.full_like(z, 8 * U)
    chosen = torch.where(live, s.gather(1, at), 0.0)
    if renormalize:
        # log s is off by 3 u of its size and 3 u; the exponents are differences of two of them, the sum has `choices` terms
        zz = torch.where(live, z, -math.inf)
        p = torch.where(live, torch.softmax(torch.where(live, z, -1e9), 1), 0.0)
        far = torch.where(live, z.abs(), 0.0).max(1, keepdim=True).values
        rel = (8 * (far if score == "sigmoid" else torch.where(live, zz.max(1, keepdim=True).values - z, 0.0).max(1, keepdim=True).values) + choices + 24) * U
        rel = rel.expand_as(p)
    else:
        p = chosen
    flat = torch.where(live, experts, count).reshape(-1).long()
    order = torch.sort(flat, stable=True).indices.to(torch.int32)
    start = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(flat, minlength=count + 1)[:count].cumsum(0)]).to(torch.int32)
    result = {"experts": experts, "order": order, "start": start, "weights": (scale * p, scale * p * (rel + 3 * U))}
    if d_weights is not None:
        g = torch.where(live, d_weights.double().cpu() * scale, 0.0)
        r = rel + 4 * U
        dot, off_dot = (p * g).sum(1, keepdim=True), (p * g.abs() * (r + (choices + 8) * U)).sum(1, keepdim=True)
        if renormalize:
            d = p * (g - dot)
            off = p * (r * (g - dot).abs() + off_dot + 4 * U * (g.abs() + dot.abs()))
            if score == "sigmoid":      # 1 - s is off by 8 u
                off = off * (1 - chosen) + d.abs() * 10 * U
                d = d * (1 - chosen)
            full, off_full = (torch.zeros(rows, count, dtype=torch.float64).scatter_add_(1, at, torch.where(live, t, 0.0)) for t in (d, off))
        elif score == "sigmoid":
            d, off = g * chosen * (1 - chosen), g.abs() * chosen * 24 * U
            full, off_full = (torch.zeros(rows, count, dtype=torch.float64).scatter_add_(1, at, torch.where(live, t, 0.0)) for t in (d, off))
        else:
            full = s * (torch.zeros(rows, count, dtype=torch.float64).scatter_add_(1, at, g) - dot)
            size = torch.zeros(rows, count, dtype=torch.float64).scatter_add_(1, at, g.abs()) + dot.abs()
            rel_s = (2 * torch.where(l64 == -math.inf, 0.0, top - l64) + spread + count + 12) * U
            off_full = s * (size * (rel_s + 6 * U) + off_dot)
        result["d_logits"] = (full, off_full)
    return result


def _activate(u, name):
    if name == "silu":
        p = torch.sigmoid(u)
        return u * p, p * (1 + u * (1 - p))
    if name == "gelu":
        p = 0.5 * torch.erfc(-u * math.sqrt(0.5))
        return u * p, p + u * torch.exp(-0.5 * u * u) / math.sqrt(2 * math.pi)
    return u, torch.ones_like(u)


def linear(x, weight, experts, bias, activation, d_z):
    """{name: (value, bound)} of z, d_x, d_weight, d_bias.  Sums of n products on the tensor cores: (n + 17) u (three parts a number, and a cut every 16 products).
    The activations' slopes are at most 1.2, their derivatives at most 0.8; CUDA's exponential, normal distribution and division bring 16 u of what they
    multiply.  In 16 bits the slope is kept to within 2^-15 and du is rounded to the type before it is multiplied."""
    dtype, dev = x.dtype, x.device
    rows, choices = experts.shape
    E, inner, outer = weight.shape
    xp = (x if x.dim() == 3 else x[:, None].expand(rows, choices, inner)).detach().double().reshape(-1, inner)
    w, of, g = weight.detach().double(), experts.reshape(-1).long(), d_z.double().reshape(-1, outer)
    z, off_z, du, off_du = (torch.zeros(of.numel(), outer, dtype=torch.float64, device=dev) for _ in range(4))
    dx, off_x = (torch.zeros(of.numel(), inner, dtype=torch.float64, device=dev) for _ in range(2))
    dw, off_w = torch.zeros_like(w), torch.zeros_like(w)
    db, off_b = torch.zeros_like(w[:, 0]), torch.zeros_like(w[:, 0])
    for e in range(E):
        m = torch.nonzero(of == e)[:, 0]
        xe, size = xp[m], xp[m].abs() @ w[e].abs()
        u, off_u = xe @ w[e], (inner + 17) * U * size
        if bias is not None:
            u, off_u = u + bias[e].detach().double(), off_u + 2 * U * (bias[e].detach().double().abs() + size)
        z[m], slope = _activate(u, activation)
        if activation is None:
            off_z[m], off_s = off_u, torch.zeros_like(u)
        else:
            off_z[m] = 1.2 * off_u + 16 * U * u.abs()
            off_s = 0.8 * off_u + 16 * U * (1 + u.abs()) + (2.0 ** -15 if dtype != torch.float32 else 0.0)
        d = g[m] * slope
        off_d = g[m].abs() * off_s + 2 * U * d.abs()
        if activation is not None and dtype != torch.float32:
            off_d = off_d + M.rounding(d.abs() + off_d, dtype)
        du[m], off_du[m] = d, off_d
        dx[m], off_x[m] = d @ w[e].T, off_d @ w[e].abs().T + (outer + 17) * U * ((d.abs() + off_d) @ w[e].abs().T)
        dw[e], off_w[e] = xe.T @ d, xe.abs().T @ off_d + (m.numel() + 17) * U * (xe.abs().T @ (d.abs() + off_d))
        db[e], off_b[e] = d.sum(0), off_d.sum(0) + (m.numel() + 2) * U * (d.abs() + off_d).sum(0)
    if x.dim() == 2:
        dx, off_x = (t.view(rows, choices, inner) for t in (dx, off_x))
        dx, off_x = dx.sum(1), off_x.sum(1) + (choices + 1) * U * (dx.abs() + off_x).sum(1)
    shape = (rows, choices, outer)
    result = {"z": (z.view(shape), off_z.view(shape)), "d_x": (dx.view(x.shape), off_x.view(x.shape)), "d_weight": (dw, off_w)}
    if bias is not None:
        result["d_bias"] = (db, off_b)
    return result


def combine(z, weights, experts, residual, d_y):
    live = (experts >= 0).double()
    zz, w, g = torch.where(live[..., None] > 0, z.detach().double(), 0.0), torch.where(live > 0, weights.detach().double(), 0.0), d_y.double()
    y, size = torch.einsum("nc,ncw->nw", w, zz), torch.einsum("nc,ncw->nw", w.abs(), zz.abs())
    if residual is not None:
        y, size = y + residual.detach().double(), size + residual.detach().double().abs()
    d_z, d_w = w[..., None] * g[:, None], torch.einsum("nw,ncw->nc", g, zz) * live
    return {"y": (y, (z.size(1) + 2) * U * size), "d_z": (d_z, 2 * U * d_z.abs()),
            "d_weights": (d_w, (z.size(2) + 2) * U * torch.einsum("nw,ncw->nc", g.abs(), zz.abs()) * live)}


def routing_by_hand(rows, experts, choices, absent, seed, dev):
    """Experts by shares 1 / (e + 1), some places without one: (experts, weights, order, start)."""
    gen = torch.Generator().manual_seed(seed)
    share = 1.0 / torch.arange(1, experts + 1)
    chosen = torch.multinomial(share.expand(max(rows, 1), -1), choices, generator=gen)[:rows].to(torch.int32)
    chosen[torch.rand(rows, choices, generator=gen) < absent] = -1
    weights = torch.where(chosen >= 0, torch.rand(rows, choices, generator=gen), 0.0)
    flat = torch.where(chosen >= 0, chosen, experts).reshape(-1).long()
    start = torch.zeros(experts + 1, dtype=torch.int32)
    start[1:] = torch.bincount(flat, minlength=experts + 1)[:experts].cumsum(0)
    order = torch.sort(flat, stable=True).indices.to(torch.int32)
    return tuple(t.to(dev) for t in (chosen, weights, order, start))
