"""The operators of a fine-tuned and served mixture-of-experts block together: the
example's block against the same lines in 64 bits, captured steps against eager ones."""
import pytest
import torch

from examples import mx4_finetune

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
D, H, E, K, N, R = 128, 96, 16, 4, 5, 8
SCALE = 2.0


def _block():
    return mx4_finetune.AdaptedMoE(D, H, E, K, N, R, seed=1).cuda()


def _batch(S, T, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(S, T, D, generator=g).to(BF)
    grad = torch.randn(S, T, D, generator=g).to(BF)
    adapters = torch.randint(-1, N, (S,), generator=g)
    mask = torch.arange(T) < torch.randint(1, T + 1, (S, 1), generator=g)
    return x, grad, adapters, mask


def _plain(block, x, sel, adapters, mask):
    """(leaves, y, balance loss) in 64 bits, for the experts that the block chose."""
    p = {n: t.detach().cpu().double().requires_grad_() for n, t in block.named_parameters()}
    x = x.double().requires_grad_()
    up, down = block.up.dequantize().cpu().double(), block.down.dequantize().cpu().double()
    live = (adapters >= 0).double()[:, None, None]
    at = adapters.clamp(min=0)
    z = x @ block.proj.cpu().double() + live * SCALE * (x @ p["seq_a"][at]) @ p["seq_b"][at]
    logits = z @ p["gate"]
    s = torch.sigmoid(logits)
    w = s.gather(-1, sel)
    w = w / w.sum(-1, keepdim=True)
    rows = lambda v, m: (v.unsqueeze(-2) @ m[sel]).squeeze(-2)
    h = torch.nn.functional.gelu(rows(z.unsqueeze(-2).expand(*z.shape[:-1], K, D), up))
    d = rows(h, down) + SCALE * rows(rows(h, p["exp_a"]), p["exp_b"])
    y = z + (d * w.unsqueeze(-1)).sum(-2)
    n = mask.sum(1).double()
    P = (s / s.sum(-1, keepdim=True) * mask[..., None]).sum(1) / n[:, None]
    c = (torch.nn.functional.one_hot(sel, E).sum(-2) * mask[..., None]).sum(1).double()
    balance = (E * c / (K * n[:, None]) * P).sum(1).mean()
    zl = (torch.logsumexp(logits, -1) ** 2 * mask).sum() / mask.sum()
    return {"x": x, **p}, y, 0.01 * balance + 0.001 * zl, c.sum(0).long()


@pytest.mark.parametrize("S,T", [(1, 1), (3, 37), (2, 300)])
def test_training_step(S, T):
    block, (x, grad, adapters, mask) = _block(), _batch(S, T, seed=S + T)
    xd = x.cuda().requires_grad_()
    y, aux, terms, counts, sel = block(xd, adapters.cuda(), mask.cuda())
    params = dict(block.named_parameters())
    # (a masked token's y is no part of a loss; its row still routes)
    gd = (grad * mask[..., None]).cuda()
    got = torch.autograd.grad([y, aux], [xd, *params.values()], [gd, torch.ones_like(aux)])
    leaves, ye, auxe, ce = _plain(block, x, sel.cpu(), adapters, mask)
    exp = torch.autograd.grad([ye, auxe], [leaves["x"], *(leaves[n] for n in params)],
                              [gd.cpu().double(), torch.ones_like(auxe)], allow_unused=True)
    assert torch.equal(counts.cpu(), ce)
    # A value passes through at most 12 roundings to 8 bits of mantissa on its way through the
    # block (z, inner values, logits, up, GELU, down, inner values, sum, product, row sum, y: 11)
    # and as many again in its gradient, each off by at most 2^-8 of the norm of what it rounds;
    # the block's maps keep norms within a factor of 2 of each other.  Sums of such errors: 24
    # roundings of independent signs, of 2^-8 / sqrt(3) in the mean square, sqrt(24) of those,
    # times 2 for the factor and 2 for where a sum is smaller than its terms.
    tol = 4 * (24 / 3) ** 0.5 * 2.0 ** -8
    for name, a, b in zip(["y", "aux", "x", *params], [y, aux, *got], [ye, auxe, *exp]):
        if b is None:
            b = torch.zeros(a.shape, dtype=torch.float64)
        diff = float((a.detach().cpu().double() - b.detach()).norm())
        assert diff <= tol * float(b.detach().norm()), f"{name}: {diff} of {float(b.detach().norm())}"


def test_captured_step_and_decode():
    """A step with gradients and a decode step in graphs, replayed for new inputs."""
    block = _block()
    params = list(block.parameters())

    def step(x, grad, adapters, mask):
        y, aux, _, counts, _ = block(x, adapters, mask)
        return [y, aux, counts, *torch.autograd.grad([y, aux], params, [grad, torch.ones_like(aux)])]

    def decode(x, adapters):
        with torch.no_grad():
            y, *_, sel = block(x, adapters)
        return [y, sel]

    train = [t.cuda() for t in _batch(3, 50, 0)]
    dec = [t.cuda() for t in (_batch(6, 1, 1)[0], _batch(6, 1, 1)[2])]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(2):
            step(*train), decode(*dec)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for f, args in ((step, train), (decode, dec)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f(*args)
        graphs.append((g, f, args, out))
    for seed in (2, 3, 4):
        b, d = _batch(3, 50, seed), _batch(6, 1, seed + 10)
        for held, new in zip(train + dec, [*b, d[0], d[2]]):
            held.copy_(new.cuda())
        for g, f, args, out in graphs:
            g.replay()
            torch.cuda.synchronize()
            for got, exp in zip(out, f(*args)):
                assert torch.equal(got, exp)


def test_example_runs(capsys):
    mx4_finetune.main()
    assert "one token of each sequence" in capsys.readouterr().out
