"""Low-rank adapters where kernels of different kinds meet: infinities beside other
infinities, calls that compile without gradients, more adapters than a sort takes,
inner rows in 32 bits, matrices past 32-bit offsets."""
import ctypes

import pytest
import torch

import cvmm_codex_amd as C
from cvmm_codex_amd import _native as N
from oracle import lora_oracle as O

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")


def _make(T, d_in, d_out, r, n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    return {"ids": torch.randint(-1, n, (T,), generator=g), "x": rnd(T, d_in).to(dtype),
            "a": (rnd(n, d_in, r) / d_in ** 0.5).to(dtype), "b": (rnd(n, r, d_out) / r ** 0.5).to(dtype),
            "weight": (rnd(d_in, d_out) / d_in ** 0.5).to(dtype), "base": rnd(T, d_out).to(dtype),
            "grad": rnd(T, d_out).to(dtype)}


def _dev(t, *names):
    return [t[n].cuda() for n in names]


def _within(got, exp, bound):
    got = got.detach().cpu().double()
    assert got.shape == exp.shape
    over = (got - exp).abs() - bound
    assert bool((over <= 0).all()), f"over the bound by {float(over.max())} of {float(exp.abs().max())}"


def _ptr(t):
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


@pytest.mark.parametrize("T", [3, 600])
@pytest.mark.parametrize("d_in,d_out,r,pitch", [(64, 128, 4, 1 << 24), (1024, (1 << 20) + 1, 12, (1 << 20) + 1)])
def test_weights_past_32_bit_offsets(T, d_in, d_out, r, pitch):
    """A weight that spans 2^30 elements, with a rank or a width that copies would pad:
    nothing behind the output's rows and behind the inner rows is written."""
    n, g = 2, torch.Generator(device="cuda").manual_seed(8)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda").to(BF)
    x, a, b, ids = rnd(T, d_in), rnd(n, d_in, r) / 32, rnd(n, r, d_out), torch.arange(T, device="cuda") % 3 - 1
    w = torch.empty(d_in * pitch, dtype=BF, device="cuda").as_strided((d_in, d_out), (pitch, 1))
    w.copy_(rnd(d_in, d_out) / 8)
    base = rnd(T, d_out)
    out, ld = torch.full((T * d_out + 64,), 77.0, dtype=BF, device="cuda"), (T + 7) // 8 * 8
    inner = torch.full((r + 8, ld), 77.0, dtype=BF, device="cuda")
    lib = N.lib()
    size = lib.cvmm_lora_workspace_bytes(T, n, d_in, d_out, r, N.BF16, 1, 1)
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    rc = lib.cvmm_lora(_ptr(x), N.BF16, T, d_in, _ptr(w), pitch, 1, _ptr(a), d_in * r, r, 1, _ptr(b), r * d_out, d_out, 1,
                       n, d_in, d_out, r, _ptr(ids), 1, None, None, 0.5, _ptr(base), N.BF16, d_out, _ptr(out), d_out,
                       _ptr(inner), ld, _ptr(ws), size, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0
    at = torch.cat([torch.arange(40), torch.arange(d_out - 40, d_out)])
    ex = [v.cpu() for v in (x, ids, a, b[..., at.cuda()], w[:, at.cuda()], base[:, at.cuda()])]
    exp, bound, h, hb = O.lora(*ex, 0.5, BF)
    _within(out[:T * d_out].view(T, d_out)[:, at.cuda()], exp, bound)
    _within(inner[:r, :T], h.t(), hb.t())
    assert bool((out[T * d_out:] == 77.0).all()) and bool((inner[r:] == 77.0).all())


# one per tile size of the fused product, with and without the shared weight, and the few rows' path
@pytest.mark.parametrize("T,d_out,weight", [(200, 264, True), (777, 264, True), (3001, 1032, True), (12345, 1032, True),
                                            (777, 264, False)])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_infinities_beside_other_infinities(T, d_out, weight, dtype):
    """A tile's rows of several adapters, some of whose B hold an infinity: what base and
    projection hold beside it counts as it does in a sum."""
    d_in, r, n = 64, 8, 3
    t = _make(T, d_in, d_out, r, n, dtype, 3)
    t["ids"] = torch.arange(T) % 4 - 1
    t["x"], t["a"] = t["x"].abs(), t["a"].abs()   # inner rows above 0
    t["weight"][:, 16:24] = -1000.0                # about -51000 a row; in fp16 base takes it past the type's range
    b, base, ids = t["b"], t["base"], t["ids"]
    b[1, 2, 8:24] = INF
    b[2, 5, 10] = -INF
    for i in range(T):
        base[i, 8 + i // 4 % 3] = (NAN, -INF, INF)[i // 12 % 3]
        base[i, 16 + i % 8] = -60000.0
    x, a, bd, w, bs, idd = _dev(t, "x", "a", "b", "weight", "base", "ids")
    y = C.cvmm_lora(x, idd, a, bd, weight=w if weight else None, base=bs).cpu()
    exp, bound, _, _ = O.lora(t["x"], ids, t["a"], b, t["weight"] if weight else None, base, 1.0, dtype)
    e = exp.to(dtype)
    assert bool(e.isnan().any() and (e == INF).any() and (e == -INF).any())
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(y), f(e)), f"{int((f(y) != f(e)).sum())} places"
    at = e.isfinite() & bound.isfinite()
    _within(y[at], exp[at], bound[at])


@pytest.mark.parametrize("T,r,dtype", [(1, 16, BF), (40, 12, BF), (256, 64, F16), (500, 8, BF)])
@pytest.mark.parametrize("weight", [True, False])
def test_few_rows_hold_inner_rows_in_32_bits(T, r, dtype, weight):
    """Calls of few rows round nothing but their output."""
    t = _make(T, 320, 520, r, 7, dtype, 6)
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")
    y = C.cvmm_lora(x, ids, a, b, weight=w if weight else None, scale=1.5)
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"] if weight else None, None, 1.5, F32, dtype)
    _within(y, exp, bound)


def test_few_rows_inner_values_past_half_precision():
    t = _make(33, 64, 72, 8, 3, F16, 7)
    t["b"] *= 2.0 ** -12
    x, ids, a, b = _dev(t, "x", "ids", "a", "b")
    y = C.cvmm_lora(x, ids, a, b, scale=2.0 ** 18)
    exp, bound, h, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], None, None, 2.0 ** 18, F32, F16)
    assert float(h.abs().max()) > 65520 and float(exp.abs().max()) < 65000
    _within(y, exp, bound)


@pytest.mark.parametrize("wanted", ["nothing", "x"])
def test_compiled_without_gradients_of_adapters(wanted):
    """The same kernels, and so the same bits, as the eager call: no inner rows are made
    for a gradient that nobody asks for."""
    t = _make(200, 256, 192, 16, 5, BF, 4)
    x, ids, a, b, w, grad = _dev(t, "x", "ids", "a", "b", "weight", "grad")

    def f(x):
        return C.cvmm_lora(x, C.cvmm_prepare_sel2(ids, route_input=True), a, b, weight=w, scale=1.25)

    res = []
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        if wanted == "x":
            leaf = x.detach().requires_grad_()
            y = fn(leaf)
            res.append((y, *torch.autograd.grad(y, leaf, grad)))
        else:
            with torch.no_grad():
                res.append((fn(x),))
    for e, c in zip(*res):
        assert torch.equal(e, c)


def test_compiled_gradient_of_rows_needs_no_sort():
    """Only the adapters' gradients need one: more adapters than a sort takes."""
    t = _make(70, 16, 24, 8, 32768, BF, 9)
    x, ids, a, b, w, grad = _dev(t, "x", "ids", "a", "b", "weight", "grad")

    def f(x):
        return C.cvmm_lora(x, ids, a, b, weight=w)

    res = []
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        leaf = x.detach().requires_grad_()
        y = fn(leaf)
        res.append((y, *torch.autograd.grad(y, leaf, grad)))
    for e, c in zip(*res):
        assert torch.equal(e, c)


@pytest.mark.parametrize("how", ["new", "used", "compiled"])
@pytest.mark.parametrize("wanted", ["nothing", "x"])
def test_selection_beside_more_adapters_than_a_sort_takes(how, wanted):
    """Its ids are used as plain ones are; the adapters' gradients are refused."""
    t = _make(70, 16, 24, 8, 32768, BF, 5)
    x, ids, a, b, w, grad = _dev(t, "x", "ids", "a", "b", "weight", "grad")

    def call(fn):
        if wanted == "nothing":
            with torch.no_grad():
                return (fn(x),)
        leaf = x.detach().requires_grad_()
        y = fn(leaf)
        return (y, *torch.autograd.grad(y, leaf, grad))

    exp = call(lambda x: C.cvmm_lora(x, ids, a, b, weight=w))
    _within(exp[0], *O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"], None, 1.0, BF)[:2])
    sel = C.cvmm_prepare_sel2(ids.view(70, 1), route_input=True)
    if how == "used":
        C.cvmm(torch.zeros(70, 1, 64, device="cuda", dtype=BF), sel, torch.zeros(8, 64, 64, device="cuda", dtype=BF))

    def f(x):
        s = C.cvmm_prepare_sel2(ids, route_input=True) if how == "compiled" else sel
        return C.cvmm_lora(x, s, a, b, weight=w)

    got = call(torch.compile(f, backend="aot_eager", fullgraph=True) if how == "compiled" else f)
    for e, g in zip(exp, got):
        assert torch.equal(e, g)
    with pytest.raises(ValueError):
        C.cvmm_lora(x, sel, a.requires_grad_(), b)


@pytest.mark.parametrize("made", ["scored", "topk", "prepared", "prepared strided"])
@pytest.mark.parametrize("used", [False, True])
@pytest.mark.parametrize("n", [16, 20])
def test_ids_written_after_the_selection_was_made(made, used, n):
    """A selection is the routing that was recorded, whatever the tensor of ids that came or
    went with it holds by now: output, every gradient, counts."""
    T, k, E = 90, 4, 16
    g = torch.Generator().manual_seed(10)
    logits = torch.randn(T, E, generator=g).cuda()
    t = _make(T * k, 64, 72, 8, n, BF, 10)
    grad = t["grad"].cuda().view(T, k, 72)
    res = []
    for write in (False, True):
        if made == "scored":
            _, ids, sel = C.cvmm_route_scored(logits, k)
        elif made == "topk":
            _, ids, sel = C.cvmm_route_topk(logits, k)
        else:
            ids = logits.topk(k).indices
            if made.endswith("strided"):
                ids = ids.t().contiguous().t()
            ids[::5, 1] = -1
            ids[::7, 2] = n
            sel = C.cvmm_prepare_sel(ids, E)
        if used:
            C.cvmm(torch.zeros(T, k, 64, device="cuda", dtype=BF), C.cvmm_prepare_sel2(sel, route_input=True),
                   torch.zeros(E, 64, 64, device="cuda", dtype=BF))
        if write:
            ids.copy_((ids * 7 + 3) % E)
        x, a, b = (v.requires_grad_() for v in _dev(t, "x", "a", "b"))
        with torch.no_grad():
            quiet = C.cvmm_lora(x.view(T, k, 64), sel, a, b)
        y = C.cvmm_lora(x.view(T, k, 64), C.cvmm_prepare_sel2(sel, route_input=True), a, b)
        counts = C.cvmm_balance_loss(logits, sel)[2]
        res.append((quiet, y, *torch.autograd.grad(y, [x, a, b], grad), counts))
    for e, c in zip(*res):
        assert torch.equal(e, c)


@pytest.mark.parametrize("odd", ["rank", "x", "weight", "a", "b", "d_in", "d_out"])
def test_copies_have_their_room(odd):
    """Few rows hold the inner rows in 32 bits, which the kernels of whole pieces do alone:
    each operand that is none by itself or by its width is copied."""
    d_in, d_out, r = 320 - (odd == "d_in"), 520 - (odd == "d_out"), 16 - (odd == "rank")
    t = _make(40, d_in, d_out, r, 7, BF, 11)
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")

    def shifted(v):
        return torch.cat([v.flatten()[:1], v.flatten()])[1:].view(v.shape)

    x, w, a, b = (shifted(v) if odd == name else v for name, v in (("x", x), ("weight", w), ("a", a), ("b", b)))
    y = C.cvmm_lora(x, ids, a, b, weight=w, scale=1.5)
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"], None, 1.5, F32, BF)
    _within(y, exp, bound)


@pytest.mark.parametrize("T,d_out,weight", [(200, 264, True), (777, 264, True), (3001, 1032, True), (12345, 1032, True),
                                            (777, 264, False)])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_infinite_rows_beside_infinite_adapters(T, d_out, weight, dtype):
    """Inner rows that are infinite themselves where B is: an infinity by the definition, as
    in tiles of one adapter."""
    d_in, r, n = 64, 8, 3
    t = _make(T, d_in, d_out, r, n, dtype, 12)
    t["ids"] = torch.arange(T) % 4 - 1
    t["x"], t["a"], t["b"] = t["x"].abs(), t["a"].abs(), t["b"].abs()
    t["weight"] = t["weight"].abs()
    t["x"][1::5, 3] = INF
    t["b"][1, 2, 8:24] = INF
    t["b"][2, :, 20:30] = -INF
    t["b"][2, 4, 40] = 0   # infinity times 0
    t["base"][:, 9:12], t["base"][:, 21] = INF, -INF
    t["weight"][5, 9], t["weight"][5, 10] = NAN, -INF
    x, a, bd, w, bs, idd = _dev(t, "x", "a", "b", "weight", "base", "ids")
    y = C.cvmm_lora(x, idd, a, bd, weight=w if weight else None, base=bs).cpu()
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"] if weight else None, t["base"], 1.0, dtype)
    e = exp.to(dtype)
    assert bool(e.isnan().any() and (e == INF).any() and (e == -INF).any())
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(y), f(e)), f"{int((f(y) != f(e)).sum())} places"
    at = e.isfinite() & bound.isfinite()
    _within(y[at], exp[at], bound[at])


@pytest.mark.parametrize("T", [40, 777, 3001])
@pytest.mark.parametrize("r", [4, 12, 16])
@pytest.mark.parametrize("weight", [True, False])
def test_infinite_rows_at_ranks_that_are_padded(T, r, weight):
    """The ranks that a copy adds are zeros, not the NaN of infinity times zero."""
    t = _make(T, 64, 72, r, 3, BF, 13)
    for name in ("x", "a", "b", "weight"):
        t[name] = t[name].abs()
    t["x"][1::3, 7] = INF
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")
    y = C.cvmm_lora(x, ids, a, b, weight=w if weight else None).cpu()
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"] if weight else None, None, 1.0, BF)
    assert bool((exp == INF).any()) and not bool(exp.isnan().any())
    assert torch.equal(y == INF, exp == INF) and not bool(y.isnan().any())
    at = exp.isfinite()
    _within(y[at], exp[at], bound[at])


@pytest.mark.parametrize("written", [False, True])
@pytest.mark.parametrize("made", ["scored", "prepared", "lazy"])
def test_compiled_use_of_a_selection_made_before(made, written):
    """The eager call's bits, gradients too, and the selection stays as it was; so with ids
    that are written before the compiled call."""
    T, k, E = 90, 4, 16
    g = torch.Generator().manual_seed(14)
    logits = torch.randn(T, E, generator=g).cuda()
    t = _make(T * k, 64, 72, 8, E, BF, 14)
    x, a, b, grad = _dev(t, "x", "a", "b", "grad")
    ids = logits.topk(k).indices
    if made == "scored":
        _, ids, sel = C.cvmm_route_scored(logits, k)
    elif made == "prepared":
        sel = C.cvmm_prepare_sel(ids, E)
    else:
        sel = C.cvmm_prepare_sel2(ids, route_input=True)
    raw = sel._routing.raw

    def f(x, a, b):
        return C.cvmm_lora(x.view(T, k, 64), sel, a, b)

    res = []
    for fn in (f, torch.compile(f, backend="aot_eager"), f):
        if written and len(res) == 1:
            ids.copy_((ids * 5 + 2) % E)
        leaves = [v.detach().requires_grad_() for v in (x, a, b)]
        y = fn(*leaves)
        res.append((y, *torch.autograd.grad(y, leaves, grad.view(T, k, 72))))
        with torch.no_grad():
            res[-1] += (fn(x, a, b),)
    for e, *others in zip(*res):
        assert all(torch.equal(e, o) for o in others)
    assert written or (sel._routing.raw is raw and not sel._routing.restored)


@pytest.mark.parametrize("made", ["scored", "topk", "prepared"])
def test_compiled_ids_written_after_the_selection_was_made(made):
    T, k, E = 90, 4, 16
    g = torch.Generator().manual_seed(15)
    logits = torch.randn(T, E, generator=g).cuda()
    t = _make(T * k, 64, 72, 8, E, BF, 15)
    x, a, b = _dev(t, "x", "a", "b")

    def f(x, write):
        if made == "scored":
            _, ids, sel = C.cvmm_route_scored(logits, k)
        elif made == "topk":
            _, ids, sel = C.cvmm_route_topk(logits, k)
        else:
            ids = logits.topk(k).indices
            sel = C.cvmm_prepare_sel(ids, E)
        if write:
            ids.copy_((ids * 5 + 2) % E)
        return C.cvmm_lora(x.view(T, k, 64), sel, a, b), C.cvmm_balance_loss(logits, sel)[2], ids

    with torch.no_grad():
        exp = f(x, False)
        got = torch.compile(f, backend="aot_eager", fullgraph=True)(x, True)
    assert torch.equal(exp[0], got[0]) and torch.equal(exp[1], got[1])
    assert torch.equal(got[2], (exp[2] * 5 + 2) % E)
