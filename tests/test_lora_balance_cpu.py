"""Adapters and balance loss without a GPU: the oracle against plain formulas, the
refusals that need no device, and the library's argument checks."""
import ctypes

import pytest
import torch

import cvmm_codex_amd as C
from cvmm_codex_amd import _native as N
from oracle import lora_oracle as O

FAKE = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    if not N.available():
        from cvmm_codex_amd import build
        build.build(verbose=False)
    return N.lib()


def _lora_case(seed=0, T=19, d_in=12, d_out=10, r=3, n=4):
    g = torch.Generator().manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    return (rnd(T, d_in), torch.randint(-1, n + 1, (T,), generator=g), rnd(n, d_in, r), rnd(n, r, d_out),
            rnd(d_in, d_out), rnd(T, d_out))


def test_oracle_of_adapters_is_the_formula():
    x, ids, a, b, w, base = _lora_case()
    y, bound, _, _ = O.lora(x, ids, a, b, w, base, 0.5)
    exp = base + x @ w
    for t in range(x.shape[0]):
        if 0 <= ids[t] < a.shape[0]:
            exp[t] += 0.5 * (x[t] @ a[ids[t]]) @ b[ids[t]]
    assert torch.allclose(y, exp, rtol=1e-12, atol=1e-12) and bool((bound > 0).all())


def test_oracle_gradients_are_autograd_s():
    x, ids, a, b, w, g = _lora_case(1)
    leaves = [v.requires_grad_() for v in (x, a, b)]
    y = x @ w
    rows = []
    for t in range(x.shape[0]):
        i = int(ids[t])
        rows.append(0.5 * (x[t] @ a[i]) @ b[i] if 0 <= i < a.shape[0] else torch.zeros_like(y[t]))
    exp = torch.autograd.grad(y + torch.stack(rows), leaves, g)
    got = O.lora_grads(x.detach(), ids, a.detach(), b.detach(), g, w, 0.5)
    for name, e in zip(("x", "a", "b"), exp):
        assert torch.allclose(got[name][0], e, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_hold_for_a_32_bit_emulation(dtype):
    """Sums in float32, inner rows and output rounded once: within the bounds."""
    x, ids, a, b, w, base = (v if v.dtype == torch.int64 else v.to(dtype) for v in _lora_case(2, 60, 40, 30, 8, 3))
    y, bound, _, _ = O.lora(x, ids, a, b, w, base, 1.5, dtype)
    out = base.float() + x.float() @ w.float()
    for t in range(x.shape[0]):
        if 0 <= ids[t] < 3:
            h = (1.5 * (x[t].float() @ a[ids[t]].float())).to(dtype).float()
            out[t] += h @ b[ids[t]].float()
    assert bool(((out.to(dtype).double() - y).abs() <= bound).all())
    # and they are no blanket: an adapter left out is seen
    assert bool(((x.double() @ w.double() + base.double() - y).abs() > bound).any())


def test_oracle_of_the_balance_loss():
    """Even loads and probabilities: load 1, entropy -log E; hand counts."""
    logits = torch.zeros(1, 4, 4, dtype=torch.float64)
    sel = torch.tensor([[[0, 1], [2, 3], [0, 1], [2, 3]]])
    loss, terms, counts = O.balance(logits, sel, weight=2.0)
    assert counts.tolist() == [2, 2, 2, 2]
    assert abs(float(loss) - 2.0) < 1e-12 and abs(float(terms[1]) - torch.log(torch.tensor(4.0)) ** 2) < 1e-6
    _, terms, _ = O.balance(logits, sel, kind="entropy")
    assert abs(float(terms[0]) + float(torch.log(torch.tensor(4.0)))) < 1e-6
    mask = torch.tensor([[True, False, True, False]])
    _, _, counts = O.balance(logits, sel, mask=mask)
    assert counts.tolist() == [2, 2, 0, 0]


def test_host_tensors_are_refused():
    x, ids, a, b, w, base = _lora_case()
    with pytest.raises(RuntimeError):
        C.cvmm_lora(x.float(), ids, a.float(), b.float(), weight=w.float())
    with pytest.raises(RuntimeError):
        C.cvmm_balance_loss(torch.zeros(2, 3, 4), torch.zeros(2, 3, 1, dtype=torch.int64))


def test_balance_arguments_fail_before_launch(lib):
    def call(dtype=0, tokens=16, ld=8, E=8, k=2, group=16, kind=0, scores=0, ws=FAKE, ws_bytes=1 << 20, loss=FAKE):
        return lib.cvmm_balance_loss(FAKE, dtype, tokens, ld, E, FAKE, 1, k, None, group, kind, scores, 1.0, 0.0, loss,
                                     FAKE, FAKE, FAKE, ws, ws_bytes, None)

    assert lib.cvmm_balance_loss_workspace_bytes(16, 16, 8) > 0
    assert lib.cvmm_balance_loss_workspace_bytes(0, 1, 8) == 0
    assert lib.cvmm_balance_loss_workspace_bytes(16, 16, 2000) == 0
    assert call(dtype=7) == 1 and call(ld=4) == 1 and call(group=5) == 1 and call(group=0) == 1
    assert call(kind=2) == 1 and call(scores=2) == 1 and call(k=0) == 1 and call(E=0) == 1
    assert call(E=1025, ld=1025) == 2 and call(tokens=2048, group=1) == 2 and call(tokens=1 << 31, group=1 << 31) == 2
    assert call(ws=None) == 3 and call(ws_bytes=8) == 3
    assert call(loss=None) == 1 and b"NULL" in lib.cvmm_last_error()
    back = lambda dtype=0, gld=8, coef=FAKE: lib.cvmm_balance_loss_backward(FAKE, dtype, 16, 8, 8, None, 16, 0, coef,
                                                                            FAKE, FAKE, gld, None)
    assert back(dtype=5) == 1 and back(gld=7) == 1 and back(coef=None) == 1


def test_lora_arguments_fail_before_launch(lib):
    def call(x=FAKE, op=N.BF16, rows=4, ld=16, n=3, d_in=16, d_out=8, rank=4, base=None, base_dtype=0, base_ld=8,
             out=FAKE, out_ld=8, inner=None, inner_ld=0, ws=FAKE, ws_bytes=1 << 20):
        return lib.cvmm_lora(x, op, rows, ld, None, 0, 0, FAKE, 64, 4, 1, FAKE, 32, 8, 1, n, d_in, d_out, rank, FAKE, 1,
                             None, None, 1.0, base, base_dtype, base_ld, out, out_ld, inner, inner_ld, ws, ws_bytes,
                             None)

    assert lib.cvmm_lora_workspace_bytes(1000, 4, 64, 64, 5, N.BF16, 1, 0) >= 1000 * 32 * 2
    assert lib.cvmm_lora_workspace_bytes(1000, 4, 64, 64, 5, N.BF16, 1, 1) >= 1000 * (32 + 64) * 2 + 2 * 4 * 64 * 8 * 2
    assert lib.cvmm_lora_workspace_bytes(100, 4, 64, 64, 300, N.BF16, 1, 0) == 0
    assert lib.cvmm_lora_workspace_bytes(0, 4, 64, 64, 8, N.BF16, 1, 1) == 0
    assert call(op=9) == 1 and call(rows=-1) == 1 and call(ld=8) == 1 and call(n=0) == 1 and call(rank=0) == 1
    assert call(rank=257) == 2 and call(rows=1 << 31) == 2
    assert call(out_ld=4) == 1 and call(base=FAKE, base_ld=4) == 1 and call(base=FAKE, base_dtype=N.F16) == 1
    assert call(inner=FAKE, inner_ld=3) == 1
    assert call(ws=None) == 3 and call(ws_bytes=16) == 3
    assert call(x=None) == 1 and call(out=None) == 1
    assert call(rows=0, x=None) == 0

    def grads(op=N.BF16, rows=4, grad_ld=8, inner_ld=4, dtype=0, order=FAKE, offsets=FAKE, ga=FAKE, gb=FAKE, ws=FAKE,
              ws_bytes=1 << 30):
        return lib.cvmm_lora_bwd_adapters(FAKE, op, rows, 16, FAKE, grad_ld, FAKE, FAKE, inner_ld, 3, 16, 8, 4, order,
                                          offsets, ga, gb, dtype, ws, ws_bytes, None)

    assert grads(op=9) == 1 and grads(grad_ld=4) == 1 and grads(inner_ld=3) == 1 and grads(dtype=4) == 1
    assert grads(order=None) == 1 and grads(offsets=None) == 1
    assert grads(ga=None, gb=None) == 0
