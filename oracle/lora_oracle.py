"""64-bit oracle of the low-rank adapters and of the balance loss, with the error
bounds of kernels that work as documented: operands in the op type, inner rows
rounded to it once, sums in 32 bits, one rounding of the output."""
from __future__ import annotations

import math

import torch

E32 = 2.0 ** -23   # of one 32-bit addition, whichever way it rounds


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def tiny(dtype: torch.dtype) -> float:
    """Half the least subnormal number: what a rounding can lose there."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def _inner(rows, ids, mats, scale):
    """scale_i * rows[t] @ mats[ids[t]], and the same of magnitudes."""
    out = torch.zeros(rows.shape[0], mats.shape[2], dtype=torch.float64)
    mag = torch.zeros_like(out)
    for i in range(mats.shape[0]):
        at = (ids == i).nonzero().view(-1)
        if at.numel():
            out[at] = scale[i] * (rows[at] @ mats[i])
            mag[at] = abs(scale[i]) * (rows[at].abs() @ mats[i].abs())
    return out, mag


def _outer(left, right, ids, n):
    out = torch.zeros(n, left.shape[1], right.shape[1], dtype=torch.float64)
    for i in range(n):
        at = (ids == i).nonzero().view(-1)
        if at.numel():
            out[i] = left[at].t() @ right[at]
    return out


def lora(x, ids, a, b, weight=None, base=None, scale=1.0, op=torch.float32, out_type=None):
    """(y, bound on |kernel - y|, inner rows, bound on those) for x [T, d_in] and
    ids [T]; operands already rounded to `op`.  Rows with infinities or NaN have no
    bound."""
    x, a, b = x.double(), a.double(), b.double()
    n, K, r = a.shape
    s = torch.full((n,), float(scale), dtype=torch.float64) if not torch.is_tensor(scale) else scale.double()
    h, hmag = _inner(x, ids, a, s)
    # K products of 32-bit sums, the scale's rounding and product, then the rounding to the op type
    hb = half_step(op) * h.abs() + (1 + half_step(op)) * (K + 3) * E32 * hmag + tiny(op)
    one = torch.ones(n, dtype=torch.float64)
    y, _ = _inner(h, ids, b, one)
    spread, _ = _inner(hb, ids, b.abs(), one)
    sums, _ = _inner(h.abs() + hb, ids, b.abs(), one)
    terms = r + 2
    if weight is not None:
        y = y + x @ weight.double()
        sums = sums + x.abs() @ weight.double().abs()
        terms += K
    if base is not None:
        y = y + base.double()
        sums = sums + base.double().abs()
    u = half_step(out_type or op)
    return y, u * y.abs() + (1 + u) * (spread + terms * E32 * sums) + tiny(out_type or op), h, hb


def lora_grads(x, ids, a, b, grad, weight=None, scale=1.0, op=torch.float32, a_type=None, b_type=None, x_type=None):
    """{name: (value, bound)} of the gradients of x, a and b for frozen weight."""
    n = a.shape[0]
    at, bt = a.transpose(1, 2), b.transpose(1, 2)
    gx, gxb, u, ub = lora(grad, ids, bt, at, None if weight is None else weight.t(), None, scale, op, op)
    if x_type is not None and x_type != op:
        gxb = gxb + half_step(x_type) * gx.abs()
    _, _, h, hb = lora(x, ids, a, b, None, None, scale, op)
    T = x.shape[0]
    res = {"x": (gx, gxb)}
    for name, left, lb, right, rb, t in (("a", x.double(), None, u, ub, a_type), ("b", h, hb, grad.double(), None, b_type)):
        v = _outer(left, right, ids, n)
        lm, rm = left.abs(), right.abs()
        err = _outer(lm, rb, ids, n) if lb is None else _outer(lb, rm, ids, n)
        full = _outer(lm if lb is None else lm + lb, rm if rb is None else rm + rb, ids, n)
        w = half_step(t or op)
        res[name] = (v, w * v.abs() + (1 + w) * (err + (T + 64) * E32 * full) + tiny(t or op))
    return res


def balance(logits, sel, kind="load", scores="softmax", mask=None, per_sequence=False, weight=1.0, z_weight=0.0):
    """(loss, terms, counts) from logits [S, T, E] in 64 bits (differentiable)."""
    S, T, E = logits.shape
    k = sel.shape[-1]
    live = torch.ones(S, T, dtype=torch.bool) if mask is None else mask
    groups = [[s] for s in range(S)] if per_sequence else [list(range(S))]
    groups = [g for g in groups if any(bool(live[s].any()) for s in g)]
    counts = torch.zeros(E, dtype=torch.int64)
    total = torch.zeros((), dtype=torch.float64)
    zs = []
    for g in groups:
        l = torch.cat([logits[s][live[s]] for s in g])
        ids = torch.cat([sel[s][live[s]].reshape(-1) for s in g])
        if scores == "softmax":
            p = torch.softmax(l, -1)
        else:
            sg = torch.sigmoid(l)
            p = sg / sg.sum(-1, keepdim=True).clamp_min(1e-20)
        P = p.mean(0)
        ids = ids[(ids >= 0) & (ids < E)]
        c = torch.bincount(ids.long(), minlength=E)
        counts += c
        if kind == "load":
            total = total + (E * c.double() / (k * l.shape[0]) * P).sum() / len(groups)
        else:
            total = total + torch.special.xlogy(P, P).sum() / len(groups)
        zs.append(torch.logsumexp(l, -1) ** 2)
    z = torch.cat(zs).mean() if zs else torch.zeros((), dtype=torch.float64)
    loss = torch.zeros((), dtype=torch.float64)
    if weight:
        loss = loss + weight * total
    if z_weight:
        loss = loss + z_weight * z
    return loss, torch.stack([total, z]).detach(), counts
