"""The operators of MoE serving and training in 4 bits whose speed is measured.

Three kinds of case:

- ``route``: the choice of experts as balanced MoE models make it.  Scores
  s = sigmoid(l) or softmax(l); a bias of the balance enters the choice alone;
  the experts stand in groups, and a group whose best biased scores sum to too
  little is left out; the k best remaining experts are chosen (ties to the
  lower id) and their scores, renormalised and scaled, are the routing
  weights.  The selection comes with it, sorted by expert.  ``train`` adds the
  logits' gradient.
- ``quantize``: a tensor to microscaled 4-bit values and back: blocks of 32
  values share a scale 2^s, s = floor(log2 max|v|) - 2, and each value is the
  nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6} * 2^s (ties to the even code, the
  largest where it lies beyond).  ``what`` "keys": expert weights [E, K, N] in
  blocks along K, as a checkpoint is laid out once; "rows": activations
  [T, K] in blocks along K.
- ``product``: rows times the experts' 4-bit weights.  ``mode`` "up" takes
  token rows and returns one row per route; "down" takes one row per route and
  returns the weighted sum per token.  ``inputs`` 16: the rows as they are; 4:
  the rows in microscaled 4-bit values too, quantised within the call.
  ``train`` adds the gradients of the rows (and of the routing weights): the
  weights are frozen, as in fine-tuning adapters around a quantised model.
"""
import math

import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _route(name, tokens, experts, k, scores, groups, kept, dtype, train):
    case = {"kind": "route", "tokens": tokens, "experts": experts, "k": k, "scores": scores, "groups": groups,
            "kept": kept, "dtype": dtype, "train": train}
    return {"name": name, **case} if name else case


def _quantize(name, what, batch, d_in, d_out, dtype):
    case = {"kind": "quantize", "what": what, "batch": batch, "d_in": d_in, "d_out": d_out, "dtype": dtype}
    return {"name": name, **case} if name else case


def _product(name, mode, tokens, d_in, d_out, experts, k, dtype, inputs, train=False):
    case = {"kind": "product", "mode": mode, "tokens": tokens, "d_in": d_in, "d_out": d_out, "experts": experts,
            "k": k, "dtype": dtype, "inputs": inputs, "train": train}
    return {"name": name, **case} if name else case


def listed():
    return [
        # a decode step of a served batch: sigmoid scores, balance bias, 4 of 8 groups
        _route("route_decode_32", 32, 256, 8, "sigmoid", 8, 4, "bfloat16", False),
        # prefill of the feed-forward stack: softmax scores with a balance bias, no groups
        _route("route_prefill_16384", 16384, 128, 8, "softmax", 1, 1, "bfloat16", False),
        # a training step's router in float32 logits, with the logits' gradient
        _route("route_train_8192", 8192, 64, 8, "sigmoid", 4, 2, "float32", True),
        # all expert weights of a projection, quantised once from float32 masters
        _quantize("quantize_keys_2048", "keys", 128, 2048, 512, "float32"),
        # a prompt's activations of a width that no block divides
        _quantize("quantize_rows_odd", "rows", 1999, 1000, 0, "bfloat16"),
        # sampling a few sequences: the call's latency
        _product("up_4", "up", 4, 1024, 128, 64, 8, "bfloat16", 16),
        # one decode step of a served batch, both projections
        _product("up_32", "up", 32, 2048, 512, 128, 8, "bfloat16", 16),
        _product("down_32", "down", 32, 512, 2048, 128, 8, "bfloat16", 16),
        # prefill of one prompt of odd length
        _product("up_1999", "up", 1999, 2048, 512, 128, 8, "bfloat16", 16),
        # fine-tuning around frozen experts: forward and the gradients of rows and routing weights
        _product("down_train_8192", "down", 8192, 128, 1024, 64, 8, "float16", 16, True),
        # the largest batches, activations in 4 bits as well
        _product("up_16384_4bit", "up", 16384, 2048, 512, 128, 8, "bfloat16", 4),
        _product("down_16384_4bit", "down", 16384, 512, 2048, 128, 8, "bfloat16", 4),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ones' ranges."""
    family = rng.choice(["route", "route", "quantize", "decode", "decode", "prefill", "4bit", "4bit", "train"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16"])
    if family == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_int(rng, max(2, 12 // groups), 256 // groups)
        kept = rng.randint(1, groups)
        k = rng.randint(1, min(8, kept * (experts // groups)))
        return _route("", _log_int(rng, 1, 16384), experts, k, rng.choice(["sigmoid", "softmax"]), groups, kept,
                      rng.choice(["bfloat16", "float16", "float32"]), rng.choice([False, True]))
    if family == "quantize":
        dtype = rng.choice(["bfloat16", "float16", "float32"])
        if rng.choice([False, True]):
            return _quantize("", "rows", _log_int(rng, 1, 16384), _log_int(rng, 32, 2048), 0, dtype)
        return _quantize("", "keys", _log_int(rng, 4, 128), _log_int(rng, 64, 2048), _log_int(rng, 64, 512), dtype)
    odd = rng.choice([False, True])
    step = 1 if odd else 32
    d_model, d_expert = step * _log_int(rng, 256 // step, 2048 // step), step * _log_int(rng, 64 // step, 512 // step)
    experts, k, mode = _log_int(rng, 8, 128), rng.choice([1, 2, 4, 8]), rng.choice(["up", "down"])
    lo, hi = {"decode": (1, 64), "prefill": (65, 4000), "4bit": (200, 16384), "train": (200, 8192)}[family]
    d_in, d_out = (d_model, d_expert) if mode == "up" else (d_expert, d_model)
    return _product("", mode, _log_int(rng, lo, hi), d_in, d_out, experts, k, dtype, 4 if family == "4bit" else 16,
                    family == "train")


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    state = {"case": case}
    if case["kind"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        # experts that the gate likes more or less, and the bias that has grown against that
        liked = 0.5 * _randn(g, E)
        state["logits"] = (1.5 * _randn(g, T, E) + liked).to(dtype)
        state["bias"] = -(0.1 if case["scores"] == "sigmoid" else 0.1 / E) * liked + 0.01 / E * _randn(g, E)
        if case["train"]:
            state["logits"].requires_grad_()
            state["grad"] = _randn(g, T, k)
        return state
    if case["kind"] == "quantize":
        n, d_in, d_out = case["batch"], case["d_in"], case["d_out"]
        if case["what"] == "keys":
            state["t"] = (_randn(g, n, d_in, d_out) / math.sqrt(d_in)).to(dtype)
        else:  # some channels of activations are far larger than the rest
            state["t"] = (_randn(g, n, d_in) * torch.exp(_randn(g, d_in))).to(dtype)
        return state
    T, E, k, d_in, d_out = case["tokens"], case["experts"], case["k"], case["d_in"], case["d_out"]
    # mild differences between the experts' loads, as a balanced router shows
    gates, ids = torch.softmax(_randn(g, T, E) + 0.3 * _randn(g, E), dim=-1).topk(k, dim=-1)
    state["sel"] = ids.contiguous()
    if case["mode"] == "up":
        state["x"] = _randn(g, T, d_in).to(dtype)
    else:
        state["x"] = torch.nn.functional.gelu(_randn(g, T, k, d_in)).to(dtype)
        state["gates"] = (gates / gates.sum(-1, keepdim=True)).contiguous()
    if case["train"]:
        state["x"].requires_grad_()
        if case["mode"] == "down":
            state["gates"].requires_grad_()
        state["grad"] = _randn(g, *((T, k, d_out) if case["mode"] == "up" else (T, d_out))).to(dtype)
    # frozen weights: values of the 4-bit grid, which packing them keeps as they are
    state["keys"] = _values(_randn(g, E, d_in, d_out) / math.sqrt(d_in), 1)
    if own:
        import cvmm_codex_amd as cvmm
        state["packed"] = cvmm.cvmm_mx4_quantize(state["keys"], dim=1)
    return state


def _values(t, dim):
    """The microscaled 4-bit values of t, blocks along `dim`, in float32."""
    t = t.detach().float().movedim(dim, -1)
    n = t.shape[-1]
    pad = -n % 32
    b = torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    s = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127)
    a = b * torch.ldexp(torch.ones_like(top), -s)
    # the grid's spacing: .5 up to 2, 1 up to 4, 2 beyond; round() takes ties to even
    grid = torch.where(a.abs() < 2, 0.5, torch.where(a.abs() < 4, 1.0, 2.0))
    q = (torch.round(a / grid) * grid).clamp(-6, 6) * torch.ldexp(torch.ones_like(top), s)
    return q.flatten(-2)[..., :n].movedim(-1, dim).contiguous()


def _experts(rows, ids, keys):
    """rows[r] @ keys[ids[r]]: the rows of each expert side by side, one product of all."""
    ids, order = torch.sort(ids, stable=True)
    load = torch.bincount(ids, minlength=keys.shape[0])
    at = torch.arange(ids.numel(), device=ids.device) - (load.cumsum(0) - load)[ids]
    padded = rows.new_zeros(keys.shape[0], int(load.max()), rows.shape[1])
    padded[ids, at] = rows[order]
    out = torch.bmm(padded, keys)[ids, at]
    return torch.empty_like(out).index_copy_(0, order, out)


def _plain_route(state):
    case = state["case"]
    E, k, G = case["experts"], case["k"], case["groups"]
    # in 64 bits: the choice between near scores is part of the answer
    l = state["logits"].detach().double()
    s = torch.sigmoid(l) if case["scores"] == "sigmoid" else torch.softmax(l, dim=-1)
    c = s + state["bias"].double()
    if G > 1:
        per = c.view(-1, G, E // G)
        best = per.topk(min(2, E // G), dim=-1).values.sum(-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :case["kept"]]
        out = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        c = per.masked_fill(out.unsqueeze(-1), -math.inf).view(-1, E)
    sel = torch.sort(c, dim=-1, descending=True, stable=True).indices[:, :k].contiguous()
    p = s.gather(1, sel)
    total = p.sum(-1, keepdim=True)
    w = 2.5 * p / total
    ids, order = torch.sort(sel.reshape(-1), stable=True)
    res = {"weights": w.float(), "sel": sel, "sorted": ids.int(), "order": order}
    if case["train"]:
        gw = state["grad"].double()
        gp = (2.5 * gw - (gw * w).sum(-1, keepdim=True)) / total
        if case["scores"] == "sigmoid":
            d = torch.zeros_like(s).scatter_(1, sel, gp * p * torch.sigmoid(-l).gather(1, sel))
        else:
            d = s * (torch.zeros_like(s).scatter_(1, sel, gp) - (gp * p).sum(-1, keepdim=True))
        res["grad_logits"] = d.to(state["logits"].dtype)
    return res


def _plain_product(state):
    case = state["case"]
    T, k = case["tokens"], case["k"]
    dtype, ids = _TYPES[case["dtype"]], state["sel"].reshape(-1)
    x = state["x"].detach()
    v = _values(x, -1) if case["inputs"] == 4 else x.float()
    rows = v.repeat_interleave(k, dim=0) if case["mode"] == "up" else v.view(T * k, -1)
    r = _experts(rows, ids, state["keys"])
    if case["mode"] == "up":
        res = {"y": r.view(T, k, -1).to(dtype)}
        if case["train"]:
            back = state["keys"].transpose(1, 2).contiguous()
            g = _experts(state["grad"].float().view(T * k, -1), ids, back)
            res["grad_x"] = g.view(T, k, -1).sum(1).to(dtype)
        return res
    w = state["gates"].detach().view(T, k, 1)
    res = {"y": (w * r.view(T, k, -1)).sum(1).to(dtype)}
    if case["train"]:
        back = state["keys"].transpose(1, 2).contiguous()
        g = _experts(state["grad"].float().repeat_interleave(k, dim=0), ids, back)
        res["grad_x"] = (w * g.view(T, k, -1)).to(dtype)
        res["grad_gates"] = (g.view(T, k, -1) * v).sum(-1)
    return res


def _own(state):
    import cvmm_codex_amd as cvmm
    case = state["case"]
    if case["kind"] == "route":
        with torch.set_grad_enabled(case["train"]):
            weights, sel, routed = cvmm.cvmm_route_scored(
                state["logits"], case["k"], bias=state["bias"], scores=case["scores"], groups=case["groups"],
                topk_groups=case["kept"], renormalize=True, scale=2.5)
        res = {"weights": weights.detach(), "sel": sel, "sorted": routed.sel.view(-1), "order": routed.out_index}
        if case["train"]:
            res["grad_logits"], = torch.autograd.grad(weights, [state["logits"]], state["grad"])
        return res
    if case["kind"] == "quantize":
        q = cvmm.cvmm_mx4_quantize(state["t"], dim=1 if case["what"] == "keys" else -1)
        return {"values": q.dequantize(torch.bfloat16)}
    up = case["mode"] == "up"
    with torch.set_grad_enabled(case["train"]), torch.autocast("cuda", dtype=_TYPES[case["dtype"]]):
        sel = cvmm.cvmm_prepare_sel2(state["sel"], None if up else state["gates"], route_input=not up)
        y = cvmm.cvmm_mx4(state["x"], sel, state["packed"], quantize_input=case["inputs"] == 4)
    res = {"y": y.detach()}
    if case["train"]:
        names = ["x"] if up else ["x", "gates"]
        grads = torch.autograd.grad(y, [state[n] for n in names], state["grad"])
        res.update({"grad_" + n: v for n, v in zip(names, grads)})
    return res


def run(state):
    if own:
        return _own(state)
    kind = state["case"]["kind"]
    if kind == "route":
        return _plain_route(state)
    if kind == "quantize":  # the values fit bfloat16: two digits and a power of two
        return {"values": _values(state["t"], 1 if state["case"]["what"] == "keys" else -1).to(torch.bfloat16)}
    return _plain_product(state)


def work(case):
    """Inputs once, outputs once, and the multiply-adds.  (A product reads the
    weights of the experts that its routes can reach at most; 17 bytes hold 32
    of them.  A router's few operations per score do not count.)"""
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "route":
        T, E, k = case["tokens"], case["experts"], case["k"]
        nbytes = size * T * E + 4 * E + T * k * (4 + 8 + 4 + 8)
        if case["train"]:
            nbytes += size * T * E + 4 * T * k
        return {"bytes": nbytes, "flops": 0}
    if case["kind"] == "quantize":
        n = case["batch"] * case["d_in"] * max(1, case["d_out"])
        return {"bytes": n * (size + 2), "flops": 0}
    T, E, k, d_in, d_out = case["tokens"], case["experts"], case["k"], case["d_in"], case["d_out"]
    R = T * k
    used = E * (1 - (1 - k / E) ** T)  # experts that some token chose, on average
    in_rows, out_rows = (T, R) if case["mode"] == "up" else (R, T)
    nbytes = size * (in_rows * d_in + out_rows * d_out) + int(used * d_out * -(-d_in // 32) * 17) + 8 * R
    flops = 2 * R * d_in * d_out
    if case["mode"] == "down":
        nbytes += 4 * R
    if case["train"]:  # the output's gradient in, the rows' out; the weights stay in reach between the two
        nbytes += size * (out_rows * d_out + in_rows * d_in) + (4 * R if case["mode"] == "down" else 0)
        flops *= 2
    return {"bytes": nbytes, "flops": flops}


def _values64(t, dim):
    """The same values from the definition: the codes by the midpoints between
    the grid's neighbours, a midpoint itself going to the even code."""
    t = t.detach().double().movedim(dim, -1)
    n = t.shape[-1]
    b = torch.cat([t, t.new_zeros(*t.shape[:-1], -n % 32)], dim=-1).unflatten(-1, (-1, 32))
    scale = torch.exp2(torch.floor(torch.log2(b.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -125))) - 2)
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64, device=t.device)
    low, high = (torch.bucketize(b.abs() / scale, mids, right=r) for r in (False, True))
    levels = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=t.device)
    v = torch.sign(b) * levels[torch.where(low % 2 == 0, low, high)] * scale
    return v.flatten(-2)[..., :n].movedim(-1, dim)


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "quantize":
        return {"values": _values64(state["t"], 1 if case["what"] == "keys" else -1)}
    T, k = case["tokens"], case["k"]
    if case["kind"] == "route":
        E, G = case["experts"], case["groups"]
        l = state["logits"].detach().double().requires_grad_()
        s = 1 / (1 + torch.exp(-l)) if case["scores"] == "sigmoid" else \
            torch.exp(l - torch.logsumexp(l, dim=-1, keepdim=True))
        c = s.detach() + state["bias"].double()
        rank = torch.argsort(c, dim=-1, descending=True, stable=True)
        if G > 1:  # the two best of each group, by the group that each rank's expert stands in
            best = torch.sort(c.view(T, G, -1), dim=-1, descending=True).values[..., :2].sum(-1)
            groups = torch.argsort(best, dim=-1, descending=True, stable=True)[:, :case["kept"]]
            of = rank // (E // G)
            good = (of.unsqueeze(-1) == groups.unsqueeze(1)).any(-1)
            rank = rank.gather(1, torch.argsort((~good).int(), dim=-1, stable=True))
        sel = rank[:, :k].contiguous()
        p = s.gather(1, sel)
        w = 2.5 * p / p.sum(-1, keepdim=True)
        order = torch.argsort(sel.reshape(-1), stable=True)
        res = {"weights": w.detach(), "sel": sel, "sorted": sel.reshape(-1)[order].int(), "order": order}
        if case["train"]:
            res["grad_logits"], = torch.autograd.grad(w, [l], state["grad"].double())
        return res
    x = state["x"].detach().double()
    v = (_values64(x, -1) if case["inputs"] == 4 else x).reshape(-1, case["d_in"])
    ids, up = state["sel"].reshape(-1), case["mode"] == "up"
    token = torch.arange(T * k, device=x.device) // k
    wt = None if up else state["gates"].detach().double().reshape(-1, 1)
    r = torch.zeros(T * k, case["d_out"], dtype=torch.float64, device=x.device)
    back = torch.zeros(T * k, case["d_in"], dtype=torch.float64, device=x.device) if case["train"] else None
    for e in torch.unique(ids).tolist():
        at = torch.nonzero(ids == e).view(-1)
        w = state["keys"][e].double()
        r[at] = v[token[at] if up else at] @ w
        if case["train"]:
            g = state["grad"].double().view(-1, case["d_out"])
            back[at] = g[at if up else token[at]] @ w.t().contiguous()
    if up:
        res = {"y": r.view(T, k, -1)}
        if case["train"]:
            res["grad_x"] = back.view(T, k, -1).sum(1)
        return res
    res = {"y": (wt * r).view(T, k, -1).sum(1)}
    if case["train"]:
        res["grad_x"] = (wt * back).view(T, k, -1)
        res["grad_gates"] = (back * v).sum(-1).view(T, k)
    return res
