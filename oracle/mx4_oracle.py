"""64-bit oracle of the 4-bit operators and the router of balanced models,
written from their definitions on CPU tensors."""
from __future__ import annotations

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(t: torch.Tensor, dim: int = -1) -> torch.Tensor:
    """The microscaled 4-bit values of t, blocks of 32 along dim (float64)."""
    v = t.detach().cpu().double().movedim(dim, -1)
    n = v.shape[-1]
    v = torch.cat([v, v.new_zeros(*v.shape[:-1], -n % 32)], -1).unflatten(-1, (-1, 32))
    top = v.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(v).all(-1, keepdim=True)
    top = torch.where(bad, torch.zeros_like(top), top)
    # floor(log2 top) - 2 by its definition, not by a rounded logarithm
    s = torch.where(top > 0, torch.frexp(top).exponent.double() - 3, torch.full_like(top, -127.0)).clamp(min=-127)
    a = v / torch.exp2(s)
    d = (a.abs().unsqueeze(-1) - GRID).abs()
    # the nearest code, of two equally near ones the even
    near = d == d.amin(-1, keepdim=True)
    code = torch.arange(8)
    pick = torch.where(near, torch.where(code % 2 == 0, code, code + 8), torch.full_like(code, 99)).amin(-1) % 8
    q = GRID[pick] * torch.sign(a) * torch.exp2(s)
    q = torch.where(bad, torch.full_like(q, float("nan")), q)
    return q.flatten(-2)[..., :n].movedim(-1, dim)


def product(x, sel, keys, gates=None, grad=None):
    """rows times the chosen experts' weights, in float64: x [T, d_in] (token
    rows) or [T, k, d_in] (route rows); ids outside the experts give zeros.
    Returns y and, with grad, grad_x and grad_gates, each with the sum of its
    products' magnitudes (.._abs) and, for a sum over a token's routes, of its
    terms' (.._rows): what rounding bounds multiply."""
    T, k = sel.shape
    E, K, N = keys.shape
    route = x.dim() == 3
    rows = (x if route else x.unsqueeze(1).expand(T, k, K)).double().reshape(T * k, K)
    ids = sel.reshape(-1)

    def experts(a, transposed):
        """a[r] @ W of r's expert, and the same of the magnitudes."""
        out = a.new_zeros(T * k, K if transposed else N)
        mag = out.clone()
        for e in range(E):
            at = (ids == e).nonzero().view(-1)
            w = keys[e].double().t() if transposed else keys[e].double()
            out[at] = a[at] @ w
            mag[at] = a[at].abs() @ w.abs()
        return out, mag

    r, ra = (t.view(T, k, N) for t in experts(rows, False))
    g = None if gates is None else gates.double().unsqueeze(-1)
    res = {}
    if g is None:
        res["y"], res["y_abs"] = r, ra
    else:
        res["y"], res["y_abs"], res["y_rows"] = (g * r).sum(1), (g.abs() * ra).sum(1), (g * r).abs().sum(1)
    if grad is not None:
        gy = grad.double()
        gr = gy if g is None else gy.unsqueeze(1).expand(T, k, N)
        b, ba = (t.view(T, k, K) for t in experts(gr.reshape(T * k, N), True))
        if g is not None:
            rk = rows.view(T, k, K)
            res["grad_gates"], res["grad_gates_abs"] = (b * rk).sum(-1), (ba * rk.abs()).sum(-1)
            b, ba = g * b, g.abs() * ba
        if route:
            res["grad_x"], res["grad_x_abs"] = b, ba
        else:
            res["grad_x"], res["grad_x_abs"], res["grad_x_rows"] = b.sum(1), ba.sum(1), b.abs().sum(1)
    return res


def scores_of(logits, kind):
    l = logits.double()
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-l))
    e = torch.exp(l - l.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def route(logits, k, bias=None, scores="softmax", groups=1, topk_groups=None, renormalize=True, scale=1.0):
    """(weights, sel): float64 weights, ids by falling biased score."""
    s = scores_of(logits, scores)
    T, E = s.shape
    c = s if bias is None else s + bias.double()
    c = torch.where(torch.isnan(c), torch.full_like(c, -float("inf")), c)
    keep = torch.ones(T, E, dtype=torch.bool)
    if topk_groups is not None and topk_groups < groups:
        per = E // groups
        best = c.view(T, groups, per).sort(-1, descending=True).values[..., :2].sum(-1)
        best = torch.where(torch.isnan(best), torch.full_like(best, -float("inf")), best)
        order = best.argsort(dim=-1, descending=True, stable=True)[:, :topk_groups]
        kg = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, order, True)
        keep = kg.repeat_interleave(per, 1)
    # left-out experts after all others, whatever their scores
    rank = c.argsort(dim=-1, descending=True, stable=True)
    rank = rank.gather(1, (~keep).gather(1, rank).int().argsort(dim=-1, stable=True))
    sel = rank[:, :k].contiguous()
    w = s.gather(1, sel)
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total < 1e-20, torch.full_like(total, 1e-20), total)
    return scale * w, sel


def route_weights(logits, sel, scores, renormalize, scale):
    """The weights of a fixed choice: what the gradient differentiates."""
    w = scores_of(logits, scores).gather(1, sel)
    if renormalize:
        w = w / w.sum(-1, keepdim=True)
    return scale * w
