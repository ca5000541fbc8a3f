"""The balance loss: compiled calls, very many tokens."""
import math

import pytest
import torch

import cvmm_codex_amd as C

pytestmark = pytest.mark.gpu


def test_compiled_terms_have_no_gradient():
    g = torch.Generator().manual_seed(0)
    logits = torch.randn(3, 40, 16, generator=g).cuda()
    sel = torch.randint(0, 16, (3, 40, 2), generator=g).cuda()

    def f(l):
        return C.cvmm_balance_loss(l, sel, weight=0.5, z_weight=0.01)

    for fn in (f, torch.compile(f, backend="aot_eager", fullgraph=True)):
        leaf = logits.detach().requires_grad_()
        loss, terms, counts = fn(leaf)
        assert loss.requires_grad and not terms.requires_grad and not counts.requires_grad
        with pytest.raises(RuntimeError):
            torch.autograd.grad(terms.sum(), leaf)
        (grad,) = torch.autograd.grad(loss, leaf)
        assert bool(grad.any())


def test_sums_of_very_many_tokens():
    """Equal tokens, whose 32-bit sums lose most: each addition the same part of a step, the
    same way.  A lane adds at most 256 of them, the workgroup 64 such sums (the additions'
    errors, half a step each, add up at most); an exponential, its sum and quotient and the
    result's rounding are within 16 more halves of a step."""
    T = 1 << 27
    c = -1.15625
    logits = torch.tensor([c, 0.0], dtype=torch.bfloat16, device="cuda").repeat(T, 1)
    sel = torch.zeros(T, 1, dtype=torch.int32, device="cuda")
    loss, terms, counts = C.cvmm_balance_loss(logits, sel)
    assert counts.tolist() == [T, 0]
    exp = 2.0 / (1.0 + math.exp(-c))
    assert abs(float(terms[0]) - exp) <= (256 + 64 + 16) * 2.0 ** -24 * exp
    assert float(loss) == float(terms[0])
    # sum of the exponentials: 2^-23 of 1.3 off, so its logarithm 2^-23 + half a step of
    # 0.27, 10 half steps; twice that and a rounding in the square
    z = math.log(1.0 + math.exp(c)) ** 2
    assert abs(float(terms[1]) - z) <= (256 + 64 + 32) * 2.0 ** -24 * z


@pytest.mark.parametrize("kind", ["load", "entropy"])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_balance_of_weight_0_passes_no_nan_on(kind, scores):
    """With a weight of 0 the rows of finite logits have the gradient of z alone."""
    g = torch.Generator().manual_seed(1)
    logits = torch.randn(2, 30, 24, generator=g).cuda()
    sel = torch.randint(0, 24, (2, 30, 2), generator=g).cuda()
    logits[0, 7, 3] = float("nan")
    leaf = logits.requires_grad_()
    loss, terms, _ = C.cvmm_balance_loss(leaf, sel, kind=kind, scores=scores, per_sequence=True, weight=0.0, z_weight=0.5)
    (grad,) = torch.autograd.grad(loss, leaf)
    l = logits.detach().double().cpu()
    exp = torch.logsumexp(l, -1, keepdim=True) * torch.softmax(l, -1) / 60
    rows = torch.ones(2, 30, dtype=torch.bool)
    rows[0, 7] = False
    assert bool(grad[~rows].isnan().all())
    # a logarithm, an exponential and their quotient to a few steps each, 24 addends
    tol = 64 * 2.0 ** -24 * ((1 + torch.logsumexp(l, -1, keepdim=True).abs()) * torch.softmax(l, -1) / 60)
    assert bool(((grad.cpu().double() - exp).abs() <= tol)[rows].all())


@pytest.mark.parametrize("E", [8, 100, 300, 1024])
def test_infinite_logits(E):
    """logsumexp of a row is infinite where a logit is, NaN where one is NaN."""
    g = torch.Generator().manual_seed(2)
    for value, with_nan in ((math.inf, False), (-math.inf, False), (math.inf, True)):
        logits = torch.randn(1, 20, E, generator=g)
        logits[0, 5, E // 2] = value
        if with_nan:
            logits[0, 5, E - 1] = math.nan
        sel = torch.randint(0, E, (1, 20, 2), generator=g)
        _, terms, _ = C.cvmm_balance_loss(logits.cuda(), sel.cuda(), scores="sigmoid")
        z = (torch.logsumexp(logits.double(), -1) ** 2).mean()
        assert bool(terms[1].isnan()) == bool(z.isnan()) and bool(terms[1].isinf()) == bool(z.isinf())
        if z.isfinite():   # 20 rows of a logarithm and a square, each to 32 steps
            assert abs(float(terms[1]) - float(z)) <= 64 * 2.0 ** -24 * float(z)
