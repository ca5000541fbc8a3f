"""Microscaled 4-bit values and the products with 4-bit expert weights against
the 64-bit oracle.

Tolerances: an output in a 16-bit type is off by half a step of it, eps / 2 of
its value; a sum of n products in 32 bits by at most n * 2^-23 of the sum of
their magnitudes (each addition rounds or truncates once); a weighted sum adds
half a step of each route's row.  Quantised values have to be equal."""
import pytest
import torch

import cvmm_codex_amd as C
from oracle import mx4_oracle as O

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(got, exp):
    got = got.cpu().double()
    assert got.shape == exp.shape
    nan = torch.isnan(exp)
    assert torch.equal(torch.isnan(got), nan)
    assert torch.equal(got[~nan], exp[~nan])


# ---------------------------------------------------------------------------
# quantisation
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 128), (4, 511), (3, 512), (2, 513),
                                    (9, 1000), (64, 2048)])
def test_rows(rows, d, dtype):
    g = _gen(rows * d)
    t = (torch.randn(rows, d, generator=g) * torch.exp(2 * torch.randn(d, generator=g))).to(dtype)
    q = C.cvmm_mx4_quantize(t.cuda())
    assert q.shape == t.shape and q.dim == 1
    exp = O.quantize(t)
    _same(q.dequantize(), exp)
    _same(q.dequantize(BF), exp)
    _same(q.dequantize(HF), exp.to(HF).double())


@pytest.mark.parametrize("dtype", [F32, BF, HF])
@pytest.mark.parametrize("E,K,N", [(1, 1, 1), (2, 32, 64), (3, 33, 65), (2, 127, 16), (1, 128, 63), (4, 129, 128),
                                   (2, 300, 100), (5, 512, 192)])
def test_keys(E, K, N, dtype):
    g = _gen(E * K * N)
    t = (torch.randn(E, K, N, generator=g) * torch.exp(2 * torch.randn(N, generator=g))).to(dtype)
    exp = O.quantize(t, 1)
    for src in (t.cuda(), t.cuda().transpose(1, 2).contiguous().transpose(1, 2),
                torch.cat([t, t], 2).cuda()[:, :, N:]):
        q = C.cvmm_mx4_quantize(src, dim=1)
        assert q.shape == t.shape and q.dim == 1
        _same(q.dequantize(), exp)
        _same(q.dequantize(BF), exp)


@pytest.mark.parametrize("dtype", [F32, BF, HF])
def test_keys_past_the_caches(dtype):
    """Over 256 MB of keys give what their experts give one by one."""
    E, K = 2, 8200
    N = 4100 if dtype == F32 else 8200
    t = torch.randn(E, K, N, device="cuda").to(dtype)
    assert t.numel() * t.element_size() >= 256 << 20
    got = C.cvmm_mx4_quantize(t, dim=1).dequantize()
    for e in range(E):
        assert torch.equal(got[e:e + 1], C.cvmm_mx4_quantize(t[e:e + 1], dim=1).dequantize())


def test_ties_extremes_and_non_finite_blocks():
    grid = torch.tensor([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 7, 7.999])
    near = torch.cat([grid, grid * (1 + 2.0 ** -23), grid * (1 - 2.0 ** -23)])
    blocks = []
    for e in (-149, -140, -129, -128, -127, -126, -125, -124, -60, 0, 60, 120, 124):
        v = torch.cat([near, -near]) if e > -120 else torch.cat([grid, -grid])
        v = torch.cat([v, torch.zeros(-v.numel() % 31)]).view(-1, 31)
        top = torch.full((v.shape[0], 1), 4.0)  # the block's scale is 2^e
        b = torch.cat([top, v], 1).double() * 2.0 ** e
        blocks.append(b.float().clamp(-torch.finfo(F32).max, torch.finfo(F32).max))
    t = torch.cat(blocks)
    t = torch.cat([t, torch.zeros(1, 32), -torch.zeros(1, 32)])
    bad = torch.randn(3, 32)
    bad[0, 5], bad[1, 7], bad[2, 31] = float("nan"), float("inf"), -float("inf")
    t = torch.cat([t, bad, torch.randn(1, 32)])
    q = C.cvmm_mx4_quantize(t.cuda())
    _same(q.dequantize(), O.quantize(t))
    keys = t.t().contiguous().unsqueeze(0)
    _same(C.cvmm_mx4_quantize(keys.cuda(), dim=1).dequantize(), O.quantize(keys, 1))


def test_leading_dims_strides_and_idempotence():
    g = _gen(4)
    t = torch.randn(3, 4, 200, generator=g)
    for src in (t.cuda(), t.cuda().double(), torch.cat([t, t], 2).cuda()[..., 77:277],
                t.cuda().permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        q = C.cvmm_mx4_quantize(src)
        assert q.shape == t.shape
        _same(q.dequantize(), O.quantize(src.float()))
    v = q.dequantize()
    _same(C.cvmm_mx4_quantize(v).dequantize(), v.cpu().double())
    empty = C.cvmm_mx4_quantize(t.cuda()[:0])
    assert empty.dequantize(BF).shape == (0, 4, 200)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
SIZES = [  # T, d_in, d_out, E, k
    (1, 32, 64, 4, 1),
    (3, 33, 65, 5, 2),
    (17, 129, 63, 8, 8),
    (64, 128, 128, 4, 2),
    (40, 520, 200, 3, 3),
    (300, 1000, 312, 7, 4),
    (130, 64, 513, 2, 1),
    (257, 384, 320, 16, 8),
    # each tile height and width of the products on either side of its rule
    (30, 256, 128, 8, 2),        # K split over waves
    (260, 640, 320, 64, 4),      # 16-row tiles, narrow and (next) wide
    (260, 320, 640, 64, 4),
    (400, 136, 320, 8, 1),       # 32-row
    (400, 320, 256, 8, 1),
    (900, 130, 72, 3, 2),        # 64-row
    (900, 264, 520, 3, 2),
    (2100, 1100, 96, 2, 2),      # more than one chunk of 4-bit rows
]
MODES = ["up", "down", "token_weighted"]


def _case(T, d_in, d_out, E, k, dtype, mode, seed=0, skew=False):
    g = _gen(seed + T * d_in + d_out)
    logits = torch.randn(T, E, generator=g) + (4 * torch.randn(E, generator=g) if skew else 0)
    gates, sel = torch.softmax(logits, -1).topk(k, -1)
    x = torch.randn(T, k, d_in, generator=g) if mode == "down" else torch.randn(T, d_in, generator=g)
    keys = O.quantize(torch.randn(E, d_in, d_out, generator=g) / d_in ** 0.5, 1).float()
    grad = torch.randn(*((T, k, d_out) if mode == "up" else (T, d_out)), generator=g).to(dtype)
    return x.to(dtype), sel, keys, (None if mode == "up" else gates), grad


def _tol(name, o, dtype, K, N, k, rounded_rows):
    eps, step = torch.finfo(dtype).eps / 2 * 1.01, 2.0 ** -23
    tiny = (k + 1) * 2.0 ** -25 if dtype == HF else 1e-37
    if name == "y":
        t = eps * o["y"].abs() + (K + k + 8) * step * o["y_abs"] + tiny
        return t + eps * o["y_rows"] if "y_rows" in o else t
    if name == "grad_x":
        t = eps * o["grad_x"].abs() + (N + k + 8) * step * o["grad_x_abs"] + tiny
        return t + eps * o["grad_x_rows"] if rounded_rows else t
    return (N + K + 8) * step * o["grad_gates_abs"] + 1e-37


def _within(got, exp, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == exp.shape, (what, got.shape, exp.shape)
    bad = ~((got - exp).abs() <= tol)
    assert not bool(bad.any()), (what, float(((got - exp).abs() / tol)[bad].max()), int(bad.sum()))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,d_in,d_out,E,k", SIZES)
def test_product_and_gradients(T, d_in, d_out, E, k, mode, dtype):
    x, sel, keys, gates, grad = _case(T, d_in, d_out, E, k, dtype, mode, skew=T % 2 == 1)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    xd = x.cuda().requires_grad_()
    gd = None if gates is None else gates.cuda().requires_grad_()
    s = C.cvmm_prepare_sel2(sel.cuda(), gd, route_input=mode == "down")
    with torch.autocast("cuda", dtype=dtype):
        y = C.cvmm_mx4(xd, s, packed)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, [xd] + ([] if gd is None else [gd]), grad.cuda())
    o = O.product(x, sel, keys, gates, grad)
    _within(y, o["y"], _tol("y", o, dtype, d_in, d_out, k, False), "y")
    assert grads[0].dtype == dtype
    _within(grads[0], o["grad_x"], _tol("grad_x", o, dtype, d_in, d_out, k, mode != "down"), "grad_x")
    if gd is not None:
        assert grads[1].dtype == torch.float32
        _within(grads[1], o["grad_gates"], _tol("grad_gates", o, dtype, d_in, d_out, k, False), "grad_gates")


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,d_in,d_out,E,k", SIZES)
def test_product_of_4_bit_rows(T, d_in, d_out, E, k, mode, dtype):
    x, sel, keys, gates, _ = _case(T, d_in, d_out, E, k, dtype, mode, seed=1)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    s = C.cvmm_prepare_sel2(sel.cuda(), None if gates is None else gates.cuda(), route_input=mode == "down")
    with torch.no_grad():
        y = C.cvmm_mx4(x.cuda(), s, packed, quantize_input=True)
    o = O.product(O.quantize(x), sel, keys, gates)
    assert y.dtype == dtype
    _within(y, o["y"], _tol("y", o, dtype, d_in, d_out, k, False), "y")


def test_gradient_against_differences():
    """The product is linear in the rows and the weights: differences over a
    whole step are exact but for the rounding of the two outputs."""
    T, d_in, d_out, E, k = 4, 64, 64, 3, 2
    x, sel, keys, gates, grad = _case(T, d_in, d_out, E, k, HF, "down", seed=2)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    xd, gd = x.cuda().requires_grad_(), gates.cuda().requires_grad_()

    def f(xx, gg):
        return C.cvmm_mx4(xx, C.cvmm_prepare_sel2(sel.cuda(), gg, route_input=True), packed)

    y = f(xd, gd)
    gx, gg = torch.autograd.grad(y, [xd, gd], grad.cuda())
    base = float((y.double() * grad.cuda().double()).sum())
    # half a step of each y (below 8 in size) and of each route's row, twice, against |grad| < 5
    noise = 2 * T * d_out * 5 * 8 * 2.0 ** -11 * 2
    with torch.no_grad():
        for t, j, i in ((0, 0, 0), (1, 1, 5), (3, 0, 63)):
            h = 256.0
            xx = xd.detach().clone()
            xx[t, j, i] += h
            num = (float((f(xx, gd).double() * grad.cuda().double()).sum()) - base) / h
            # the moved outputs are up to h times larger
            tol = (noise + h * d_out * 5 * 2.0 ** -11 * 2) / h + 2.0 ** -11 * abs(num)
            assert abs(num - float(gx[t, j, i])) <= tol
        for t, j in ((0, 0), (2, 1)):
            h = 4.0
            w = gd.detach().clone()
            w[t, j] += h
            num = (float((f(xd, w).double() * grad.cuda().double()).sum()) - base) / h
            assert abs(num - float(gg[t, j])) <= 5 * noise / h


def test_matches_the_16_bit_product():
    """Weights on the 4-bit grid: the same operands as cvmm in bf16, which rounds
    an unweighted product once as well."""
    T, d_in, d_out, E, k = 200, 512, 256, 8, 4
    x, sel, keys, _, _ = _case(T, d_in, d_out, E, k, BF, "up", seed=3)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF):
        a = C.cvmm(x.cuda(), C.cvmm_prepare_sel2(sel.cuda()), keys.cuda())
        b = C.cvmm_mx4(x.cuda(), C.cvmm_prepare_sel2(sel.cuda()), C.cvmm_mx4_quantize(keys.cuda(), dim=1))
    # each is off by half a step of the value and by the 32-bit sums
    tol = 2 * (2.0 ** -8 * b.double().abs() + d_in * 2.0 ** -23 * 6 * d_in ** 0.5)
    assert bool(((a.double() - b.double()).abs() <= tol).all())


@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("T", [5, 200])
def test_ids_outside_the_experts_and_idle_experts(T, quantize):
    d_in, d_out, E, k = 96, 72, 9, 3
    x, sel, keys, gates, grad = _case(T, d_in, d_out, E, k, BF, "down", seed=5)
    sel = sel % 4                      # experts 4.. idle
    sel[0, 1], sel[T - 1, 2], sel[T // 2, 0] = -1, E, 1000
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    xq = O.quantize(x) if quantize else x
    with torch.no_grad():
        y = C.cvmm_mx4(x.cuda(), C.cvmm_prepare_sel2(sel.cuda(), gates.cuda(), route_input=True), packed, quantize)
        u = C.cvmm_mx4(x.cuda(), C.cvmm_prepare_sel2(sel.cuda(), route_input=True), packed, quantize)
    o = O.product(xq, sel, keys, gates)
    _within(y, o["y"], _tol("y", o, BF, d_in, d_out, k, False), "y")
    o = O.product(xq, sel, keys)
    _within(u, o["y"], _tol("y", o, BF, d_in, d_out, k, False), "y")
    if not quantize:
        xd, gd = x.cuda().requires_grad_(), gates.cuda().requires_grad_()
        y = C.cvmm_mx4(xd, C.cvmm_prepare_sel2(sel.cuda(), gd, route_input=True), packed)
        gx, gg = torch.autograd.grad(y, [xd, gd], grad.cuda())
        o = O.product(x, sel, keys, gates, grad)
        _within(gx, o["grad_x"], _tol("grad_x", o, BF, d_in, d_out, k, False), "grad_x")
        _within(gg, o["grad_gates"], _tol("grad_gates", o, BF, d_in, d_out, k, False), "grad_gates")
        x2 = x[:, 0].cuda().requires_grad_()
        u = C.cvmm_mx4(x2, C.cvmm_prepare_sel2(sel.cuda()), packed)
        g2 = torch.randn(T, k, d_out, generator=_gen(9)).to(BF)
        gx, = torch.autograd.grad(u, [x2], g2.cuda())
        o = O.product(x[:, 0], sel, keys, None, g2)
        _within(gx, o["grad_x"], _tol("grad_x", o, BF, d_in, d_out, k, True), "grad_x")


def test_strided_rows_other_types_and_no_tokens():
    T, d_in, d_out, E, k = 30, 200, 136, 4, 2
    x, sel, keys, gates, grad = _case(T, d_in, d_out, E, k, BF, "up", seed=6)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    o = O.product(x, sel, keys, None, grad)
    wide = torch.cat([x, x, x], 1).cuda()
    s = C.cvmm_prepare_sel2(sel.cuda())
    for view in (wide[:, d_in:2 * d_in], torch.cat([x[:, :1], x], 1).cuda()[:, 1:],
                 x.t().contiguous().cuda().t(), x.float().cuda()):
        xd = view.detach().requires_grad_()
        with torch.autocast("cuda", dtype=BF):
            y = C.cvmm_mx4(xd, s, packed)
        _within(y, o["y"], _tol("y", o, BF, d_in, d_out, k, False), "y")
        gd = grad.cuda().transpose(0, 1).contiguous().transpose(0, 1)
        gx, = torch.autograd.grad(y, [xd], gd)
        assert gx.dtype == view.dtype
        _within(gx, o["grad_x"], _tol("grad_x", o, BF, d_in, d_out, k, True), "grad_x")
    with torch.no_grad():
        y = C.cvmm_mx4(x.cuda()[:0], C.cvmm_prepare_sel2(sel.cuda()[:0]), packed)
        assert y.shape == (0, k, d_out)
    xd = x.cuda()[:0].requires_grad_()
    g0, = torch.autograd.grad(C.cvmm_mx4(xd, C.cvmm_prepare_sel2(sel.cuda()[:0]), packed).sum(), [xd])
    assert g0.shape == (0, d_in)


def test_non_finite_rows_stay_in_their_rows():
    T, d_in, d_out, E, k = 40, 128, 64, 2, 1
    x, sel, keys, _, _ = _case(T, d_in, d_out, E, k, BF, "up", seed=7)
    clean = x.clone()
    x[3, 5], x[9, 100] = float("nan"), float("inf")
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    with torch.no_grad():
        for quantize in (False, True):
            a = C.cvmm_mx4(x.cuda(), C.cvmm_prepare_sel2(sel.cuda()), packed, quantize)
            b = C.cvmm_mx4(clean.cuda(), C.cvmm_prepare_sel2(sel.cuda()), packed, quantize)
            rows = [t for t in range(T) if t not in (3, 9)]
            assert torch.equal(a[rows], b[rows])
            assert bool(torch.isnan(a[3]).all()) and not bool(torch.isfinite(a[9]).all())


def test_on_another_stream_and_in_a_graph():
    T, d_in, d_out, E, k = 32, 256, 192, 16, 4
    x, sel, keys, gates, _ = _case(T, d_in, d_out, E, k, BF, "down", seed=8)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    xd, sd, gd = x.cuda(), sel.cuda(), gates.cuda()
    o = O.product(x, sel, keys, gates)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def call(quantize):
        return C.cvmm_mx4(xd, C.cvmm_prepare_sel2(sd, gd, route_input=True), packed, quantize)

    with torch.no_grad():
        with torch.cuda.stream(side):
            y = call(False)
        torch.cuda.current_stream().wait_stream(side)
        _within(y, o["y"], _tol("y", o, BF, d_in, d_out, k, False), "y")
        for quantize in (False, True):
            call(quantize)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = call(quantize)
            for seed in (11, 12, 13):
                x2, s2, _, g2, _ = _case(T, d_in, d_out, E, k, BF, "down", seed=seed)
                xd.copy_(x2)
                sd.copy_(s2)
                gd.copy_(g2)
                graph.replay()
                eager = call(quantize)
                torch.cuda.synchronize()
                assert torch.equal(out, eager)


def test_weights_past_32_bit_offsets():
    """130 experts of 8192 x 8192: 4.6 GB of codes; the last expert's alone hold
    values."""
    E, K, N, T = 130, 8192, 8192, 3
    g = _gen(1)
    keys = torch.zeros(E, K, N, dtype=BF, device="cuda")
    last = O.quantize(torch.randn(K, 64, generator=g) / 64, 0).to(BF)
    keys[-1, :, N - 64:] = last.cuda()
    packed = C.cvmm_mx4_quantize(keys, dim=1)
    del keys
    assert packed.codes.numel() > 2 ** 32
    x = torch.randn(T, K, generator=g).to(BF)
    sel = torch.tensor([[E - 1], [0], [E - 1]])
    exp = x.double() @ last.double()
    exp[1] = 0
    tol = 2.0 ** -8 * exp.abs() + K * 2.0 ** -23 * (x.double().abs() @ last.double().abs()) + 1e-37
    with torch.no_grad():
        y = C.cvmm_mx4(x.cuda(), C.cvmm_prepare_sel2(sel.cuda()), packed)[:, 0]
        _within(y[:, N - 64:], exp, tol, "y")
        assert not bool(y[:, :N - 64].any())
    del packed
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("quantize", [False, True])
@pytest.mark.parametrize("d_out", [1000, 2056])
def test_route_rows_past_the_caches(d_out, quantize, dtype):
    """Weighted sums over more than 256 MB of route rows: a token's row does not
    depend on where it lies."""
    k, few, E, d_in = 4, 61, 3, 64
    n = (256 << 20) // (few * k * d_out * 2) + 1
    assert n * few * k * d_out * 2 >= 256 << 20
    x, sel, keys, gates, _ = _case(few, d_in, d_out, E, min(k, E), dtype, "down", seed=2)
    x = torch.cat([x, x[:, :1]], 1)
    sel, gates = torch.cat([sel, sel[:, :1]], 1), torch.cat([gates, gates[:, 1:2]], 1)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    s = C.cvmm_prepare_sel2(sel.repeat(n, 1).cuda(), gates.repeat(n, 1).cuda(), route_input=True)
    with torch.no_grad():
        y = C.cvmm_mx4(x.repeat(n, 1, 1).cuda(), s, packed, quantize_input=quantize)
    o = O.product(O.quantize(x) if quantize else x, sel, keys, gates)
    _within(y[:few], o["y"], _tol("y", o, dtype, d_in, d_out, k, False), "y")
    assert torch.equal(y.view(n, few, d_out), y[:few].expand(n, few, d_out))


def test_compiled():
    T, d_in, d_out, E, k = 24, 128, 64, 4, 2
    x, sel, keys, gates, grad = _case(T, d_in, d_out, E, k, BF, "down", seed=4)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)

    def f(xx, gg):
        return C.cvmm_mx4(xx, C.cvmm_prepare_sel2(sel.cuda(), gg, route_input=True), packed)

    outs = []
    for fn in (f, torch.compile(f, backend="aot_eager")):
        xd, gd = x.cuda().requires_grad_(), gates.cuda().requires_grad_()
        y = fn(xd, gd)
        outs.append((y, *torch.autograd.grad(y, [xd, gd], grad.cuda())))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_block_of_router_and_both_projections():
    """The example's MoE block end to end against the same lines in 64 bits."""
    from examples import mx4_moe
    T, D, H, E, k = 48, 256, 96, 16, 4
    block = mx4_moe.MX4MoE(D, H, E, k, groups=4, topk_groups=2, seed=0).cuda()
    x = torch.randn(T, D, generator=_gen(3)).to(BF).cuda()
    with torch.no_grad():
        y, sel = block(x)
    logits = (x @ block.gate).cpu()
    w, se = O.route(logits, k, bias=block.bias.cpu(), scores="sigmoid", groups=4, topk_groups=2, scale=block.scale)
    assert torch.equal(sel.cpu(), se)
    up, down = block.up.dequantize().cpu(), block.down.dequantize().cpu()
    h = O.product(x.cpu(), se, up)["y"].to(BF)
    h = torch.nn.functional.gelu(h.float()).to(BF)
    o = O.product(h, se, down, w)
    # a step of h's rounding (2^-8, twice: product and GELU) reaches y as that part of its terms
    tol = _tol("y", o, BF, H, D, k, False) + 4 * 2.0 ** -8 * o["y_abs"]
    _within(y, o["y"], tol, "y")


def _selector(kind, mode, sel, gates, keys):
    """The same selection as a user may hold it: ids, a selector whose sort was
    read, one that cvmm() sorted, one built by hand."""
    if kind == "ids":
        return sel
    s = C.cvmm_prepare_sel2(sel, gates, route_input=mode == "down")
    if kind == "resolved":
        assert s.sel.numel() == sel.numel()
    elif kind == "shared":
        T, k = sel.shape
        x = torch.randn(*((T, k) if mode == "down" else (T,)), keys.shape[1], device="cuda")
        with torch.no_grad(), torch.autocast("cuda", dtype=BF):
            C.cvmm(x, s, keys)
    else:
        ids, perm = torch.sort(sel.reshape(-1), stable=True)
        up = mode != "down"
        s = C.CVMMSel(sel.int(), ids.int().view(sel.shape), perm // sel.shape[1] if up else perm, perm if up else None,
                      gates)
    return s


@pytest.mark.parametrize("kind,mode", [("ids", "down"), *((s, m) for s in ("resolved", "shared", "built")
                                                          for m in MODES)])
def test_gradients_of_every_kind_of_selection(kind, mode):
    T, d_in, d_out, E, k = 50, 136, 72, 5, 3
    x, sel, keys, gates, grad = _case(T, d_in, d_out, E, k, BF, mode, seed=21)
    if kind == "ids":  # one row per route, no routing weights
        gates, grad = None, torch.randn(T, k, d_out, generator=_gen(22)).to(BF)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    xd = x.cuda().requires_grad_()
    gd = None if gates is None else gates.cuda().requires_grad_()
    y = C.cvmm_mx4(xd, _selector(kind, mode, sel.cuda(), gd, keys.cuda()), packed)
    grads = torch.autograd.grad(y, [xd] + ([] if gd is None else [gd]), grad.cuda())
    o = O.product(x, sel, keys, gates, grad)
    _within(y, o["y"], _tol("y", o, BF, d_in, d_out, k, False), "y")
    _within(grads[0], o["grad_x"], _tol("grad_x", o, BF, d_in, d_out, k, mode != "down"), "grad_x")
    if gd is not None:
        _within(grads[1], o["grad_gates"], _tol("grad_gates", o, BF, d_in, d_out, k, False), "grad_gates")
    with torch.no_grad():
        plain = C.cvmm_mx4(xd, _selector(kind, mode, sel.cuda(), gd, keys.cuda()), packed)
        rows = C.cvmm_mx4(xd, _selector(kind, mode, sel.cuda(), gd, keys.cuda()), packed, quantize_input=True)
    assert torch.equal(plain, y)
    o = O.product(O.quantize(x), sel, keys, gates)
    _within(rows, o["y"], _tol("y", o, BF, d_in, d_out, k, False), "4-bit rows")


def test_forward_mode_is_refused():
    """A tangent has no rule here: an error, not an output without one.  Plain
    tensors inside a forward-mode level are multiplied as ever."""
    T, d_in, d_out, E, k = 6, 64, 64, 3, 2
    x, sel, keys, gates, _ = _case(T, d_in, d_out, E, k, BF, "down", seed=23)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    xd, gd = x.cuda(), gates.cuda()

    def call(xx, gg, quantize=False, pending=True):
        s = C.cvmm_prepare_sel2(sel.cuda(), gg, route_input=True)
        if not pending:
            assert s.sel.numel()
        return C.cvmm_mx4(xx, s, packed, quantize)

    y, yq = call(xd, gd), call(xd, gd, True)
    for mode in (torch.no_grad, torch.enable_grad):
        with mode(), torch.autograd.forward_ad.dual_level():
            for pending in (True, False):
                for quantize in (False, True):
                    with pytest.raises(Exception):
                        call(torch.autograd.forward_ad.make_dual(xd, torch.ones_like(xd)), gd, quantize, pending)
                    with pytest.raises(Exception):
                        call(xd, torch.autograd.forward_ad.make_dual(gd, torch.ones_like(gd)), quantize, pending)
                assert torch.equal(call(xd, gd, False, pending), y) and torch.equal(call(xd, gd, True, pending), yq)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("dtype", [BF, HF])
def test_gradients_equal_exact_differences(mode, dtype):
    """Rows of -1, 0 and 1, weights of the grid, powers of two as routing weights:
    no output rounds, so the linear product's differences are its gradients,
    to the last bit.  Every gradient of a routing weight and a spread of those
    of the rows."""
    T, d_in, d_out, E, k = 5, 40, 24, 3, 2
    g = _gen(31)
    levels = torch.tensor([-1.0, -0.5, 0.0, 0.5, 1.0])
    keys = levels[torch.randint(0, 5, (E, d_in, d_out), generator=g)]
    x = torch.randint(-1, 2, (T, k, d_in) if mode == "down" else (T, d_in), generator=g).to(dtype)
    sel = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    gates = None if mode == "up" else 2.0 ** torch.randint(-1, 2, (T, k), generator=g)
    grad = torch.randint(-1, 2, (T, k, d_out) if mode == "up" else (T, d_out), generator=g).to(dtype)
    packed = C.cvmm_mx4_quantize(keys.cuda(), dim=1)
    assert torch.equal(packed.dequantize().cpu(), keys)
    xd = x.cuda().requires_grad_()
    gd = None if gates is None else gates.cuda().requires_grad_()

    def f(xx, gg):
        return C.cvmm_mx4(xx, C.cvmm_prepare_sel2(sel.cuda(), gg, route_input=mode == "down"), packed)

    y = f(xd, gd)
    assert torch.equal(y.detach().cpu().double(), O.product(x, sel, keys, gates)["y"])   # nothing rounded
    got = torch.autograd.grad(y, [xd] + ([] if gd is None else [gd]), grad.cuda())
    weighed = lambda v: float((v.double() * grad.cuda().double()).sum())
    with torch.no_grad():
        base = weighed(y)

        def differences(t, at, call):
            out = []
            for i in at:
                moved = t.detach().clone()
                moved.view(-1)[i] += 1
                out.append(weighed(call(moved)) - base)
            return torch.tensor(out, dtype=torch.float64)

        at = list(range(0, x.numel(), 7))
        num = differences(xd, at, lambda t: f(t, gd))
        assert int((num != 0).sum()) > len(at) // 2
        assert torch.equal(got[0].reshape(-1)[at].cpu().double(), num)
        if gd is not None:
            num = differences(gd, range(T * k), lambda t: f(xd, t))
            assert int((num != 0).sum()) > T * k // 2
            assert torch.equal(got[1].reshape(-1).cpu().double(), num)


def test_compiled_quantisation_and_block():
    """Quantised rows and keys, and a router with both products traced as one graph,
    against the same lines in eager mode."""
    T, D, H, E, k = 24, 128, 96, 8, 2
    g = _gen(41)
    x, logits = torch.randn(T, D, generator=g).to(BF).cuda(), torch.randn(T, E, generator=g).cuda()
    w_up, w_down = torch.randn(E, D, H, generator=g).cuda(), torch.randn(E, H, D, generator=g).cuda()

    def values(t, w):
        return C.cvmm_mx4_quantize(t).dequantize(BF), C.cvmm_mx4_quantize(w, dim=1).dequantize()

    up, down = C.cvmm_mx4_quantize(w_up, dim=1), C.cvmm_mx4_quantize(w_down, dim=1)

    def block(xx, ll):
        gates, _, sel = C.cvmm_route_scored(ll, k, scores="sigmoid")
        h = torch.relu(C.cvmm_mx4(xx, sel, up))
        return C.cvmm_mx4(h, C.cvmm_prepare_sel2(sel, gates, route_input=True), down)

    for a, c in zip(values(x, w_up), torch.compile(values, backend="aot_eager", fullgraph=True)(x, w_up)):
        assert torch.equal(a, c)
    res = []
    for fn in (block, torch.compile(block, backend="aot_eager")):
        xx, ll = x.clone().requires_grad_(), logits.clone().requires_grad_()
        y = fn(xx, ll)
        res.append((y, *torch.autograd.grad(y, [xx, ll], torch.ones_like(y))))
    for a, c in zip(*res):
        assert torch.equal(a, c)
