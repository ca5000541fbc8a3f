"""Low-rank adapters beside a shared projection against the 64-bit oracle, whose
bounds count the documented roundings."""
import pytest
import torch

import cvmm_codex_amd as C
from oracle import lora_oracle as O

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")


def _ids(how, T, n, g):
    if how == "own":
        return torch.randint(-1, n, (T,), generator=g)
    if how == "runs":
        ends = torch.sort(torch.randint(0, T + 1, (2 * n,), generator=g)).values
        return torch.randperm(2 * n + 1, generator=g)[torch.bucketize(torch.arange(T), ends, right=True)] % (n + 1) - 1
    if how == "one":
        return torch.full((T,), n - 1)
    if how == "none":
        return torch.where(torch.arange(T) % 2 == 0, -1, n)
    return torch.arange(T) % n   # "alternate"


def _make(T, d_in, d_out, r, n, how, dtype, weight=True, base=False, seed=0):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g)
    t = {"ids": _ids(how, T, n, g), "x": rnd(T, d_in).to(dtype), "a": (rnd(n, d_in, r) / d_in ** 0.5).to(dtype),
         "b": (rnd(n, r, d_out) / r ** 0.5).to(dtype),
         "weight": (rnd(d_in, d_out) / d_in ** 0.5).to(dtype) if weight else None,
         "base": rnd(T, d_out).to(dtype) if base else None, "grad": rnd(T, d_out).to(dtype)}
    return t


def _dev(t, *names):
    return [None if t[n] is None else t[n].cuda() for n in names]


def _within(got, exp, bound):
    got = got.detach().cpu().double()
    assert got.shape == exp.shape
    over = (got - exp).abs() - bound
    assert bool((over <= 0).all()), f"over the bound by {float(over.max())} of {float(exp.abs().max())}"


# T, d_in, d_out, rank, adapters, ids, dtype, weight, base
CASES = [
    (1, 64, 64, 16, 3, "own", BF, True, False),
    (1, 1024, 1024, 16, 8, "one", BF, True, False),
    (2, 8, 8, 1, 1, "own", F16, True, True),
    (7, 33, 17, 5, 4, "own", BF, True, True),
    (16, 2048, 512, 16, 32, "own", BF, True, False),
    (32, 512, 2048, 32, 64, "own", F16, True, False),
    (64, 256, 128, 64, 9, "alternate", BF, True, True),
    (65, 128, 256, 8, 2, "runs", F32, True, False),
    (100, 1000, 518, 12, 5, "runs", BF, True, False),
    (129, 136, 264, 24, 7, "own", BF, False, True),
    (200, 64, 72, 40, 3, "runs", F16, False, False),
    (256, 320, 192, 16, 100, "own", BF, True, False),
    (257, 96, 640, 33, 2, "runs", F32, False, True),
    (300, 1024, 1024, 16, 4, "runs", BF, True, True),
    (511, 72, 1032, 64, 6, "alternate", F16, True, False),
    (777, 1000, 512, 16, 5, "runs", BF, True, False),
    (1000, 2048, 128, 256, 2, "runs", BF, True, False),
    (1031, 128, 1024, 16, 64, "alternate", BF, False, True),
    (1999, 512, 768, 32, 8, "runs", F16, True, False),
    (2500, 264, 520, 8, 3, "none", BF, True, True),
    (4099, 256, 320, 64, 16, "runs", BF, True, False),
    # the largest tiles: 192 and more of 256 x 256
    (12345, 96, 1032, 16, 40, "runs", BF, True, True),
    (12345, 40, 1280, 72, 3, "alternate", F16, True, False),
    (16000, 64, 1000, 8, 5, "own", BF, False, True),
    # and of 128 x 128
    (3001, 160, 1032, 40, 6, "runs", F16, True, True),
    (3100, 33, 1000, 6, 11, "alternate", BF, True, False),
    # copies of odd rows in a launch of their own
    (4001, 1001, 72, 16, 3, "runs", BF, True, False),
]


@pytest.mark.parametrize("T,d_in,d_out,r,n,how,dtype,weight,base", CASES)
def test_forward(T, d_in, d_out, r, n, how, dtype, weight, base):
    t = _make(T, d_in, d_out, r, n, how, dtype, weight, base)
    x, ids, a, b, w, bs = _dev(t, "x", "ids", "a", "b", "weight", "base")
    y = C.cvmm_lora(x, ids, a, b, weight=w, base=bs, scale=1.7)
    assert y.dtype == dtype and y.shape == (T, d_out)
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"], t["base"], torch.tensor(1.7).item(), dtype)
    _within(y, exp, bound)
    # twice the same bits; the sorted selection's order changes nothing but sums
    assert torch.equal(y, C.cvmm_lora(x, ids, a, b, weight=w, base=bs, scale=1.7))
    ys = C.cvmm_lora(x, C.cvmm_prepare_sel2(ids, route_input=True), a, b, weight=w, base=bs, scale=1.7)
    _within(ys, exp, bound)


@pytest.mark.parametrize("T,d_in,d_out,r,n,how,dtype,weight,base", CASES)
def test_gradients(T, d_in, d_out, r, n, how, dtype, weight, base):
    t = _make(T, d_in, d_out, r, n, how, dtype, weight, base, 1)
    x, ids, a, b, w, bs, grad = _dev(t, "x", "ids", "a", "b", "weight", "base", "grad")
    leaves = [v.requires_grad_() for v in (x, a, b)] + ([bs.requires_grad_()] if base else [])
    y = C.cvmm_lora(x, ids, a, b, weight=w, base=bs, scale=0.75)
    got = torch.autograd.grad(y, leaves, grad)
    exp = O.lora_grads(t["x"], t["ids"], t["a"], t["b"], t["grad"], t["weight"], 0.75, dtype)
    for name, v in zip(("x", "a", "b"), got):
        assert v.dtype == dtype
        _within(v, *exp[name])
    if base:
        assert torch.equal(got[3], grad)
    # adapters without rows: zeros, not left over memory
    idle = [i for i in range(n) if not bool((t["ids"] == i).any())]
    assert not got[1][idle].any() and not got[2][idle].any()
    # each by itself: the same bits
    for i, leaf in enumerate(leaves):
        for other in leaves:
            other.requires_grad_(other is leaf)
        alone, = torch.autograd.grad(C.cvmm_lora(x, ids, a, b, weight=w, base=bs, scale=0.75), [leaf], grad)
        if i != 0:   # (x alone takes its rows in the order given)
            assert torch.equal(alone, got[i])
        else:
            _within(alone, *exp["x"])


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("T", [3, 70, 600])
def test_strides_and_layouts(T, dtype):
    """Rows cut out of wider ones, a Linear's weight, adapters stored the other way
    round, matrices of no unit stride, leading dimensions, int32 ids, a scale per
    adapter."""
    d_in, d_out, r, n = 72, 136, 8, 5
    t = _make(T, d_in, d_out, r, n, "own", dtype, True, True, 2)
    scale = torch.tensor([0.5, -1.0, 2.0, 0.0, 1.5])
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"], t["base"], scale, dtype)
    x, ids, a, b, w, bs = _dev(t, "x", "ids", "a", "b", "weight", "base")
    wide = torch.full((T, d_in + 19), NAN, dtype=dtype, device="cuda")
    wide[:, 3:3 + d_in] = x
    wbase = torch.full((T, 2 * d_out), NAN, dtype=dtype, device="cuda")
    wbase[:, d_out:] = bs
    linear = w.t().contiguous().t()
    at, bt = a.transpose(1, 2).contiguous().transpose(1, 2), b.transpose(1, 2).contiguous().transpose(1, 2)
    spread = torch.full((n, d_in, r, 2), NAN, dtype=dtype, device="cuda")
    spread[..., 0] = a
    for args in ((wide[:, 3:3 + d_in], ids, a, b, linear, wbase[:, d_out:]), (x, ids.int(), at, bt, w, bs),
                 (x, ids, spread[..., 0], b.flip(0).flip(0), linear, bs), (x.t().contiguous().t(), ids, at, b, w, bs)):
        _within(C.cvmm_lora(*args[:4], weight=args[4], base=args[5], scale=scale.cuda()), exp, bound)
    if T % 3 == 0:
        y = C.cvmm_lora(x.view(3, -1, d_in), ids.view(3, -1), a, b, weight=w, base=bs.view(3, -1, d_out),
                        scale=scale.cuda())
        assert y.shape == (3, T // 3, d_out)
        _within(y.view(T, d_out), exp, bound)
        # rows in a sequence-first order
        y = C.cvmm_lora(x.view(3, -1, d_in).transpose(0, 1), ids.view(3, -1).t(), a, b, weight=w, scale=scale.cuda(),
                        base=bs.view(3, -1, d_out).transpose(0, 1))
        _within(y.transpose(0, 1).reshape(T, d_out), exp, bound)


@pytest.mark.parametrize("T", [4, 64, 700])
@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_infinities_stay_with_their_rows(T, dtype):
    """An adapter of NaN and infinities, a row of NaN: all other rows and adapters
    as without them, bit for bit; rows without an adapter never read one."""
    d_in, d_out, r, n = 256, 128, 16, 4
    t = _make(T, d_in, d_out, r, n, "own", dtype, True, False, 3)
    t["ids"][::4], t["ids"][1::4], t["ids"][2::4] = 0, 1, -1
    x, ids, a, b, w, grad = _dev(t, "x", "ids", "a", "b", "weight", "grad")
    bad_a, bad_b, bad_x, bad_g = a.clone(), b.clone(), x.clone(), grad.clone()
    bad_a[1, 3] = NAN
    bad_b[1, :, 5] = INF
    bad_b[1, 2] = -INF
    keep = ids.ne(1)
    bad_x[~keep] = NAN
    bad_g[~keep] = INF

    def run(g, *v):
        v = [q.detach().requires_grad_() for q in v]
        y = C.cvmm_lora(v[0], ids, v[1], v[2], weight=w)
        return (y, *torch.autograd.grad(y, v, g))

    y, gx, ga, gb = run(bad_g, bad_x, bad_a, bad_b)
    ye, gxe, gae, gbe = run(grad, x, a, b)
    assert torch.equal(y[keep], ye[keep]) and torch.equal(gx[keep], gxe[keep])
    others = torch.arange(n, device="cuda").ne(1)
    assert torch.equal(ga[others], gae[others]) and torch.equal(gb[others], gbe[others])
    assert bool(torch.isnan(y[~keep]).all())


def test_no_rows():
    t = _make(0, 64, 32, 8, 3, "one", BF)
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")
    leaves = [v.requires_grad_() for v in (x, a, b)]
    y = C.cvmm_lora(x, ids, a, b, weight=w)
    assert y.shape == (0, 32)
    gx, ga, gb = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert gx.shape == x.shape and not ga.any() and not gb.any()


def test_autocast_and_masters_in_32_bits():
    """float32 rows and adapters under autocast: rounded to the op type, gradients
    in their own types, the adapters' from unrounded sums."""
    t = _make(300, 256, 192, 16, 6, "runs", F32, True, True, 4)
    r = {k: (v.to(BF) if k in ("x", "a", "b", "weight", "grad") else v) for k, v in t.items()}
    x, ids, a, b, w, bs = _dev(t, "x", "ids", "a", "b", "weight", "base")
    leaves = [v.requires_grad_() for v in (x, a, b, bs)]
    with torch.autocast("cuda", dtype=BF):
        y = C.cvmm_lora(x, ids, a, b, weight=w, base=bs, scale=2.0)
    assert y.dtype == BF
    exp, bound, _, _ = O.lora(r["x"], t["ids"], r["a"], r["b"], r["weight"], t["base"], 2.0, BF)
    _within(y, exp, bound)
    got = torch.autograd.grad(y, leaves, r["grad"].cuda())
    assert all(v.dtype == F32 for v in got)
    grads = O.lora_grads(r["x"], t["ids"], r["a"], r["b"], r["grad"], r["weight"], 2.0, BF, F32, F32)
    for name, v in zip(("x", "a", "b"), got):
        _within(v, *grads[name])
    assert torch.equal(got[3], r["grad"].cuda().float())


def test_gradients_against_differences():
    T, d_in, d_out, r, n = 23, 12, 9, 3, 3
    t = _make(T, d_in, d_out, r, n, "own", F32, True, False, 5)
    x, ids, a, b, w, grad = _dev(t, "x", "ids", "a", "b", "weight", "grad")
    leaves = [v.requires_grad_() for v in (x, a, b)]
    got = torch.autograd.grad(C.cvmm_lora(x, ids, a, b, weight=w, scale=1.5), leaves, grad)
    base = {k: t[k].double() for k in ("x", "a", "b")}

    def f(**v):
        q = {**base, **v}
        return float((O.lora(q["x"], t["ids"], q["a"], q["b"], t["weight"], None, 1.5)[0] * t["grad"].double()).sum())

    for name, v in zip(("x", "a", "b"), got):
        flat = base[name].reshape(-1)
        num, step = torch.zeros_like(flat), 1e-6
        for i in range(flat.numel()):
            up, lo = flat.clone(), flat.clone()
            up[i] += step
            lo[i] -= step
            num[i] = (f(**{name: up.view_as(base[name])}) - f(**{name: lo.view_as(base[name])})) / (2 * step)
        # bilinear: differences are exact but for the 64-bit sums' rounding over the step
        # (|f| below 1e3: 1e3 * 1e-13 / 1e-6); 32-bit sums of at most 23 x 12 terms below 20
        assert float((v.cpu().double().view(-1) - num).abs().max()) <= 1e-4 + 300 * 2.0 ** -23 * 20


def test_selection_shared_with_the_products():
    """The router's selection as adapters beside the frozen 4-bit down projection."""
    T, k, E, d_in, d_out, r = 90, 4, 16, 64, 128, 8
    g = torch.Generator().manual_seed(6)
    logits = torch.randn(T, E, generator=g).cuda()
    _, sel, routed = C.cvmm_route_scored(logits, k)
    keys = C.cvmm_mx4_quantize((torch.randn(E, d_in, d_out, generator=g) / 8).cuda(), dim=1)
    t = _make(T * k, d_in, d_out, r, E, "one", BF, False, False, 6)
    x, a, b = _dev(t, "x", "a", "b")
    xr = x.view(T, k, d_in)
    down = C.cvmm_prepare_sel2(routed, route_input=True)
    base = C.cvmm_mx4(xr, down, keys)
    y = C.cvmm_lora(xr, down, a, b, base=base)
    assert y.shape == (T, k, d_out)
    exp, bound, _, _ = O.lora(t["x"], sel.cpu().reshape(-1), t["a"], t["b"], None, base.cpu().view(T * k, d_out), 1.0, BF)
    _within(y.view(T * k, d_out), exp, bound)
    # the token-input selection has the same routes
    assert torch.equal(y, C.cvmm_lora(xr, routed, a, b, base=base))


@pytest.mark.parametrize("T,dtype", [(4, BF), (300, BF), (90, F32)])
def test_other_stream_and_graph(T, dtype):
    t = _make(T, 256, 192, 16, 5, "own", dtype, True, False, 7)
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = C.cvmm_lora(x, ids, a, b, weight=w)
    torch.cuda.current_stream().wait_stream(side)
    exp, bound, _, _ = O.lora(t["x"], t["ids"], t["a"], t["b"], t["weight"], None, 1.0, dtype)
    _within(y, exp, bound)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            yg = C.cvmm_lora(x, ids, a, b, weight=w)
        with torch.cuda.graph(second):
            ys = C.cvmm_lora(x, ids, a, b, weight=w, scale=2.0)
        for seed in (8, 9, 10):
            new = _make(T, 256, 192, 16, 5, "own", dtype, True, False, seed)
            x.copy_(new["x"])
            ids.copy_(new["ids"])
            graph.replay()
            second.replay()
            e1 = C.cvmm_lora(x, ids, a, b, weight=w)
            e2 = C.cvmm_lora(x, ids, a, b, weight=w, scale=2.0)
            torch.cuda.synchronize()
            assert torch.equal(yg, e1) and torch.equal(ys, e2)


def test_backward_in_a_graph():
    t = _make(300, 128, 192, 16, 5, "runs", BF, True, False, 11)
    x, ids, a, b, w, grad = _dev(t, "x", "ids", "a", "b", "weight", "grad")
    leaves = [v.requires_grad_() for v in (x, a, b)]

    def step():
        return torch.autograd.grad(C.cvmm_lora(x, ids, a, b, weight=w), leaves, grad)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for seed in (12, 13, 14):
        new = _make(300, 128, 192, 16, 5, "runs", BF, True, False, seed)
        with torch.no_grad():
            x.copy_(new["x"])
            ids.copy_(new["ids"])
            grad.copy_(new["grad"])
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(c, e) for c, e in zip(captured, eager))


@pytest.mark.parametrize("weight,base,presorted", [(True, False, False), (False, True, True), (True, True, False)])
def test_compiled_with_gradients(weight, base, presorted):
    t = _make(77, 64, 72, 8, 4, "own", BF, weight, base, 15)
    x, ids, a, b, w, bs, grad = _dev(t, "x", "ids", "a", "b", "weight", "base", "grad")

    def f(x, a, b):
        sel = C.cvmm_prepare_sel2(ids, route_input=True) if presorted else ids
        return C.cvmm_lora(x, sel, a, b, weight=w, base=bs, scale=1.25)

    res = []
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        leaves = [v.detach().requires_grad_() for v in (x, a, b)]
        y = fn(*leaves)
        res.append((y, *torch.autograd.grad(y, leaves, grad)))
    for e, c in zip(*res):
        assert e.dtype == c.dtype and torch.equal(e, c)


@pytest.mark.parametrize("T", [20, 700])
def test_selection_built_by_hand(T):
    """Rows without an adapter sorted first (ids below 0), their infinities and NaN in
    no adapter's gradient."""
    t = _make(T, 128, 64, 16, 5, "own", BF, False, False, 8)
    t["ids"][::7] = -1
    none = t["ids"] < 0
    t["x"][none], t["grad"][none] = NAN, INF
    ids = t["ids"].cuda()
    key, at = torch.sort(ids, stable=True)
    outs = []
    for sel in (ids, C.CVMMSel(ids, key, at), C.cvmm_prepare_sel(ids, 5), C.cvmm_prepare_sel2(ids.view(T, 1))):
        x, a, b, g = _dev(t, "x", "a", "b", "grad")
        x, a, b = (v.requires_grad_() for v in (x, a, b))
        y = C.cvmm_lora(x, sel, a, b)
        outs.append((y, *torch.autograd.grad(y, [x, a, b], g)))
    assert all(bool(v.isfinite().all()) for v in outs[0])
    for out in outs[1:]:
        assert all(torch.equal(v, w) for v, w in zip(outs[0], out))


@pytest.mark.parametrize("n", [3, 8, 12])
def test_selection_sorted_for_another_count(n):
    T = 500
    t = _make(T, 128, 64, 16, n, "own", BF, False, False, 9)
    ids = torch.randint(-2, 12, (T, 1), generator=torch.Generator().manual_seed(9)).cuda()
    sel = C.cvmm_prepare_sel2(ids, route_input=True)
    C.cvmm(torch.zeros(T, 1, 64, device="cuda", dtype=BF), sel, torch.zeros(8, 64, 64, device="cuda", dtype=BF))
    outs = []
    for s in (ids.view(T), sel, C.cvmm_prepare_sel2(sel, route_input=True)):
        x, a, b, g = _dev(t, "x", "a", "b", "grad")
        x, a, b = (v.requires_grad_() for v in (x, a, b))
        y = C.cvmm_lora(x, s, a, b)
        outs.append((y, *torch.autograd.grad(y, [x, a, b], g)))
    for out in outs[1:]:
        assert all(torch.equal(v, w) for v, w in zip(outs[0], out))


def test_forward_mode_is_refused():
    t = _make(9, 16, 8, 4, 2, "own", F32)
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")
    y = C.cvmm_lora(x, ids, a, b, weight=w)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(Exception):
            C.cvmm_lora(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)), ids, a, b, weight=w)
        assert torch.equal(y, C.cvmm_lora(x, ids, a, b, weight=w))


def test_refusals_on_the_device():
    t = _make(6, 16, 8, 4, 3, "own", BF)
    x, ids, a, b, w = _dev(t, "x", "ids", "a", "b", "weight")
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids[:5], a, b)
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids, a, b[:2])
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids, a, b, weight=w.t())
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids, a, b, weight=w.requires_grad_())
    with torch.no_grad():
        C.cvmm_lora(x, ids, a, b, weight=w)
    w.requires_grad_(False)
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids, a, b, base=x)
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids, a, b, scale=torch.ones(2, device="cuda"))
    with pytest.raises(TypeError):
        C.cvmm_lora(x, ids.float(), a, b)
    with pytest.raises(TypeError):
        C.cvmm_lora(x.double(), ids, a, b)
    with pytest.raises(ValueError):
        C.cvmm_lora(x, C.cvmm_prepare_sel2(ids[:3], route_input=True), a, b)
    with pytest.raises(ValueError):
        C.cvmm_lora(x, ids, torch.zeros(3, 16, 300, device="cuda", dtype=BF), torch.zeros(3, 300, 8, device="cuda", dtype=BF))
    with pytest.raises(RuntimeError):
        C.cvmm_lora(x, ids.cpu(), a, b)
