"""The router of balanced models against the 64-bit oracle: the choice exactly,
the weights and gradients to their rounding."""
import pytest
import torch

import cvmm_codex_amd as C
from oracle import mx4_oracle as O

pytestmark = pytest.mark.gpu
INF = float("inf")

CASES = [  # T, E, k, scores, groups, kept, bias, renormalize, scale, dtype
    (1, 1, 1, "softmax", 1, 1, False, True, 1.0, torch.float32),
    (5, 4, 2, "sigmoid", 2, 1, True, True, 2.5, torch.bfloat16),
    (33, 12, 3, "sigmoid", 4, 2, True, True, 2.5, torch.float32),
    (32, 256, 8, "sigmoid", 8, 4, True, True, 2.5, torch.bfloat16),
    (17, 32, 32, "softmax", 1, 1, True, False, 1.0, torch.float16),
    (40, 64, 8, "sigmoid", 64, 9, True, True, 1.0, torch.float32),
    (300, 128, 8, "softmax", 1, 1, True, True, 1.0, torch.bfloat16),
    (300, 60, 5, "softmax", 5, 3, False, False, 0.5, torch.float16),
    (700, 129, 1, "sigmoid", 3, 2, False, True, 1.0, torch.float32),
    (50, 500, 16, "softmax", 4, 2, True, True, 1.0, torch.float32),
    (70, 1000, 64, "sigmoid", 8, 3, True, True, 1.5, torch.bfloat16),
    (9, 1024, 8, "softmax", 32, 5, True, True, 1.0, torch.float32),
    # either side of the chunk rule: 128 and 256 routes, chunks of 8, 32, 64 and more tokens
    (16, 64, 8, "sigmoid", 1, 1, True, True, 1.0, torch.bfloat16),
    (65, 64, 2, "softmax", 1, 1, True, True, 1.0, torch.float32),
    (256, 40, 1, "sigmoid", 4, 3, True, True, 1.0, torch.float16),
    (257, 200, 1, "softmax", 1, 1, False, True, 1.0, torch.float32),
    (3000, 256, 4, "sigmoid", 8, 3, True, True, 2.5, torch.bfloat16),
    (17000, 16, 2, "softmax", 1, 1, True, True, 1.0, torch.bfloat16),
    (5000, 1000, 3, "sigmoid", 1, 1, True, False, 1.0, torch.float32),
]


def _logits(T, E, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (1.5 * torch.randn(T, E, generator=g)).to(dtype), 0.1 * torch.randn(E, generator=g), g


def _check(w, sel, routed, logits, k, kw):
    we, se = O.route(logits, k, **kw)
    assert torch.equal(sel.cpu(), se)
    assert w.dtype == torch.float32
    # 64-bit scores rounded once; 1e-12 covers exp's own rounding
    fin = torch.isfinite(we)
    assert torch.equal(torch.isfinite(w.cpu()), fin)
    err = (w.cpu().double() - we).abs()[fin]
    assert bool((err <= we.abs()[fin] * (2.0 ** -24 + 1e-12) + 1e-45).all())
    ids, order = torch.sort(se.reshape(-1), stable=True)
    assert torch.equal(routed.sel.view(-1).cpu(), ids.int())
    assert torch.equal(routed.out_index.cpu(), order)
    assert torch.equal(routed.sel_index.cpu(), order // k)


@pytest.mark.parametrize("T,E,k,scores,groups,kept,bias,renorm,scale,dtype", CASES)
def test_choice_weights_and_order(T, E, k, scores, groups, kept, bias, renorm, scale, dtype):
    logits, b, _ = _logits(T, E, dtype)
    kw = dict(bias=b if bias else None, scores=scores, groups=groups, topk_groups=kept, renormalize=renorm, scale=scale)
    w, sel, routed = C.cvmm_route_scored(logits.cuda(), k, **{**kw, "bias": b.cuda() if bias else None})
    _check(w, sel, routed, logits, k, kw)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,kept", [(1, 1), (4, 2)])
def test_ties_and_values_past_the_ordinary(scores, groups, kept):
    """Equal logits (ties to the lower id), 32-bit neighbours, masks of -inf and
    of the type's lowest value, NaN, +inf under the sigmoid, a whole row of -inf."""
    T, E, k = 24, 32, 6
    logits, b, g = _logits(T, E, torch.float32)
    logits[0] = 0.25
    logits[1] = torch.randint(0, 3, (E,), generator=g).float()
    logits[2] = 1.0 + torch.randperm(E, generator=g).float() * 2.0 ** -23
    logits[3, ::2] = -INF
    logits[4, 5:] = torch.finfo(torch.float32).min
    logits[5, 3] = float("nan")
    logits[6] = -INF
    logits[7, :30] = -INF
    if scores == "sigmoid":
        logits[8, 7] = INF
        logits[9] = -200.0
    if scores == "softmax":  # the row's softmax is NaN throughout
        logits[10, 2] = INF
    kw = dict(scores=scores, groups=groups, topk_groups=kept, scale=2.0)
    w, sel, routed = C.cvmm_route_scored(logits.cuda(), k, **kw)
    _check(w, sel, routed, logits, k, kw)


def test_bias_of_infinities_leaves_experts_out():
    T, E, k = 16, 24, 4
    logits, b, _ = _logits(T, E, torch.float32)
    b[::3] = -INF
    kw = dict(scores="sigmoid", groups=3, topk_groups=2, bias=b)
    w, sel, routed = C.cvmm_route_scored(logits.cuda(), k, **{**kw, "bias": b.cuda()})
    _check(w, sel, routed, logits, k, kw)
    assert not bool((sel % 3 == 0).any())


def test_strided_logits_leading_dims_and_no_tokens():
    logits, b, _ = _logits(60, 80, torch.bfloat16)
    view = logits.cuda()[:, 3:67]
    w, sel, routed = C.cvmm_route_scored(view, 4, scores="sigmoid")
    _check(w, sel, routed, logits[:, 3:67], 4, dict(scores="sigmoid"))
    w3, sel3, _ = C.cvmm_route_scored(view.reshape(5, 12, 64), 4, scores="sigmoid")
    assert w3.shape == (5, 12, 4) and torch.equal(w3.view(60, 4), w) and torch.equal(sel3.view(60, 4), sel)
    t = logits.cuda().t().contiguous().t()   # column-major
    w, sel, routed = C.cvmm_route_scored(t, 4)
    _check(w, sel, routed, logits, 4, {})
    w, sel, routed = C.cvmm_route_scored(logits[:0].cuda(), 4)
    assert w.shape == (0, 4) and sel.shape == (0, 4) and routed.sel.numel() == 0


@pytest.mark.parametrize("T,E,k,scores,groups,kept,bias,renorm,scale,dtype", CASES)
def test_gradient(T, E, k, scores, groups, kept, bias, renorm, scale, dtype):
    logits, b, g = _logits(T, E, dtype, 1)
    l = logits.cuda().requires_grad_()
    bd = b.cuda().requires_grad_() if bias else None
    w, sel, _ = C.cvmm_route_scored(l, k, bias=bd, scores=scores, groups=groups, topk_groups=kept,
                                    renormalize=renorm, scale=scale)
    gw = torch.randn(T, k, generator=g)
    got = torch.autograd.grad(w, [l], gw.cuda())[0].cpu().double()
    l64 = logits.double().requires_grad_()
    exp = torch.autograd.grad(O.route_weights(l64, sel.cpu(), scores, renorm, scale), [l64], gw.double())[0]
    # one rounding to the logits' type, and the 32-bit softmax row: exp's and
    # the sum's error (2^-20 of the row's largest terms, E <= 1024 of them)
    s = O.scores_of(logits, scores)
    terms = scale * gw.double().abs().amax(-1, keepdim=True) * 2 * (s if scores == "softmax" else torch.ones_like(s))
    if renorm:
        terms = terms / s.gather(1, sel.cpu()).sum(-1, keepdim=True)
    tol = exp.abs() * torch.finfo(dtype).eps / 2 * 1.01 + 2.0 ** -20 * terms
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert bool(((got - exp).abs() <= tol).all())


def test_gradient_against_differences():
    T, E, k = 7, 20, 4
    logits, b, g = _logits(T, E, torch.float32, 3)
    for scores in ("softmax", "sigmoid"):
        for renorm in (False, True):
            l = logits.cuda().requires_grad_()
            w, sel, _ = C.cvmm_route_scored(l, k, scores=scores, renormalize=renorm, scale=1.5)
            gw = torch.randn(T, k, generator=g)
            got = torch.autograd.grad(w, [l], gw.cuda())[0].cpu().double()
            num, h = torch.zeros(T, E, dtype=torch.float64), 1e-5
            for e in range(E):
                d = torch.zeros(T, E, dtype=torch.float64)
                d[:, e] = h
                up = O.route_weights(logits.double() + d, sel.cpu(), scores, renorm, 1.5)
                lo = O.route_weights(logits.double() - d, sel.cpu(), scores, renorm, 1.5)
                num[:, e] = ((up - lo) * gw.double()).sum(-1) / (2 * h)
            # central differences: h^2 of third derivatives below 10; 32-bit gradients
            assert float((got - num).abs().max()) <= 10 * h * h + 2.0 ** -20 * 10


def test_on_another_stream_and_in_a_graph():
    T, E, k = 32, 256, 8
    logits, b, _ = _logits(T, E, torch.bfloat16)
    ld, bd = logits.cuda(), b.cuda()
    kw = dict(scores="sigmoid", groups=8, topk_groups=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.no_grad():
        w, sel, routed = C.cvmm_route_scored(ld, k, bias=bd, **kw)
    torch.cuda.current_stream().wait_stream(side)
    _check(w, sel, routed, logits, k, {**kw, "bias": b})
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        with torch.cuda.graph(graph):
            gw, gsel, _ = C.cvmm_route_scored(ld, k, bias=bd, **kw)
        for seed in (5, 6, 7):
            new, _, _ = _logits(T, E, torch.bfloat16, seed)
            ld.copy_(new)
            graph.replay()
            ew, esel, _ = C.cvmm_route_scored(ld, k, bias=bd, **kw)
            torch.cuda.synchronize()
            assert torch.equal(gsel, esel) and torch.equal(gw, ew)


def test_compiled():
    logits, b, _ = _logits(20, 64, torch.float32)
    f = lambda l: C.cvmm_route_scored(l, 4, scores="sigmoid", groups=4, topk_groups=2)[:2]
    w, sel = torch.compile(f, backend="eager", fullgraph=True)(logits.cuda())
    we, se = f(logits.cuda())
    assert torch.equal(w, we) and torch.equal(sel, se)


def test_forward_mode_is_refused():
    """A tangent has no rule here: an error, not weights without one.  Plain
    tensors inside a forward-mode level are routed as ever."""
    logits, b, _ = _logits(9, 16, torch.float32)
    l, bd = logits.cuda(), b.cuda()
    w, sel, _ = C.cvmm_route_scored(l, 3, bias=bd)
    for mode in (torch.no_grad, torch.enable_grad):
        with mode(), torch.autograd.forward_ad.dual_level():
            with pytest.raises(Exception):
                C.cvmm_route_scored(torch.autograd.forward_ad.make_dual(l, torch.ones_like(l)), 3, bias=bd)
            w2, sel2, _ = C.cvmm_route_scored(l, 3, bias=bd)
            assert torch.equal(w, w2) and torch.equal(sel, sel2)


@pytest.mark.parametrize("k", [63, 64])
@pytest.mark.parametrize("groups,kept", [(1, 1), (2, 1)])
def test_last_of_64_choices_goes_by_64_bit_scores(k, groups, kept):
    """The last chosen and the first left out differ by 2e-9 and are equal in 32
    bits: a sigmoid of 20 and of 21, moved by the bias."""
    n = k + 1
    logits = torch.zeros(3, n * groups)
    bias = torch.zeros(n * groups)
    bias[:k - 1] = 0.5 + 0.01 * torch.arange(k - 1)
    logits[:, k - 1], logits[:, k] = 20.0, 21.0
    bias[k - 1:n] = -0.75
    logits[:, n:] = -10.0
    kw = dict(scores="sigmoid", groups=groups, topk_groups=kept, bias=bias)
    w, sel, routed = C.cvmm_route_scored(logits.cuda(), k, **{**kw, "bias": bias.cuda()})
    assert not bool((sel == k - 1).any())
    _check(w, sel, routed, logits, k, kw)


@pytest.mark.parametrize("E,low", [(1024, -15.046297), (1024, -7.0), (1024, -5.0), (512, -15.046297), (512, -5.0),
                                   (256, -14.0), (100, -4.0)])
@pytest.mark.parametrize("groups,kept", [(1, 1), (2, 1)])
def test_sum_of_many_equal_scores(E, low, groups, kept):
    """One expert above E - 1 equal ones, whose 32-bit sum rounds the same way at
    every addition; a bias that nearly cancels the distance to one of them, on
    either side of the tie in steps of 2^-24."""
    logits = torch.full((1, E), low)
    logits[0, 0] = 0.0
    other = 1 if groups == 1 else E // 2
    s = O.scores_of(logits, "softmax")[0]
    tie = (s[0] - s[other]).float()
    for j in range(-24, 25):
        bias = torch.zeros(E)
        bias[other] = tie + j * 2.0 ** -24
        if groups > 1:  # the same second best in both groups: they compare as the two do
            bias[2], bias[other + 1] = 0.125, 0.125
        kw = dict(bias=bias, groups=groups, topk_groups=kept)
        w, sel, routed = C.cvmm_route_scored(logits.cuda(), 1, **{**kw, "bias": bias.cuda()})
        _check(w, sel, routed, logits, 1, kw)


@pytest.mark.parametrize("E,k", [(32, 5), (64, 64), (100, 63), (200, 8), (600, 3)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups", [1, 4])
def test_equal_scores_of_different_logits(scores, groups, E, k):
    """Logits whose 64-bit scores are the same number, with no bias or one of
    zeros: the lower id first, also next to a NaN."""
    T = 12
    g = torch.Generator().manual_seed(E + k)
    logits = torch.randn(T, E, generator=g)
    up = torch.randperm(E, generator=g).float()
    logits[0] = 40 + up                      # sigmoid 1
    logits[1, ::2] = 40 + up[::2]
    logits[2] = -800 - up                    # sigmoid 0
    logits[3] = -800 - up                    # softmax 0 but for one
    logits[3, E // 2] = 0
    logits[4] = up * 1e-20                   # the logits' difference vanishes in either
    logits[5, 1::3] = up[1::3] * 1e-22
    logits[6] = logits[0]
    logits[6, E - 1] = float("nan")
    logits[7] = -800 - up
    logits[7, :3] = torch.tensor([0.0, 1.0, -1.0])
    logits[8, ::3] = -INF
    logits[9, E // 3:] = torch.finfo(torch.float32).min
    logits[10] = 28 + up / 64                # sigmoid: 1 - s from 2^-40 down to where 1 takes it
    bias = torch.zeros(E)
    kw = dict(scores=scores, groups=groups, topk_groups=groups)
    w, sel, routed = C.cvmm_route_scored(logits.cuda(), k, **kw)
    _check(w, sel, routed, logits, k, kw)
    wb, selb, _ = C.cvmm_route_scored(logits.cuda(), k, bias=bias.cuda(), **kw)
    assert torch.equal(selb, sel)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_sum_below_the_clamp(scores):
    """Chosen scores that sum to less than 1e-20 are divided by that: weights and
    gradients of scale * s / 1e-20."""
    T, E, k, scale = 6, 24, 4, 1.5
    g = torch.Generator().manual_seed(8)
    logits = -52 - 3 * torch.rand(T, E, generator=g)
    logits[:, 5] = 0.0
    b = torch.zeros(E)
    b[5] = -2.0           # the one large score is not chosen
    l = logits.cuda().requires_grad_()
    w, sel, routed = C.cvmm_route_scored(l, k, bias=b.cuda(), scores=scores, scale=scale)
    kw = dict(bias=b, scores=scores, scale=scale)
    _check(w.detach(), sel, routed, logits, k, kw)
    l64 = logits.double().requires_grad_()
    s = O.scores_of(l64, scores).gather(1, sel.cpu())
    assert float(s.sum(-1).max()) < 1e-20 and float(w.sum(-1).max()) < scale
    gw = torch.randn(T, k, generator=g)
    got, = torch.autograd.grad(w, [l], gw.cuda())
    exp, = torch.autograd.grad(scale * s / 1e-20, [l64], gw.double())
    # one rounding to fp32; the softmax row in 32 bits: |x| < 56 roundings of the
    # exp's argument, a few more of exp, sum, quotient, difference and product
    tol = exp.abs() * 2.0 ** -24 * (1.01 if scores == "sigmoid" else 70)
    assert bool(((got.cpu().double() - exp).abs() <= tol + 1e-45).all())


@pytest.mark.parametrize("scores,groups,kept,renorm,bias", [("sigmoid", 4, 2, True, True), ("softmax", 1, 1, False, False),
                                                            ("softmax", 8, 3, True, True)])
def test_compiled_with_gradients(scores, groups, kept, renorm, bias):
    """Traced through the registered shapes and the registered backward: the eager
    call's weights, choice, sorted selection and gradients, bit for bit."""
    logits, b, g = _logits(21, 64, torch.bfloat16, 9)
    bd = b.cuda() if bias else None
    gw = torch.randn(21, 5, generator=g).cuda()

    def f(l):
        w, sel, routed = C.cvmm_route_scored(l, 5, bias=bd, scores=scores, groups=groups, topk_groups=kept,
                                             renormalize=renorm, scale=2.0)
        return w, sel, routed.sel, routed.sel_index, routed.out_index

    res = []
    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        l = logits.cuda().requires_grad_()
        out = fn(l)
        res.append((*out, *torch.autograd.grad(out[0], [l], gw)))
    for a, c in zip(*res):
        assert a.dtype == c.dtype and torch.equal(a, c)
