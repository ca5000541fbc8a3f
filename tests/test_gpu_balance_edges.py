"""The balance loss: compiled calls, very many tokens."""
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
