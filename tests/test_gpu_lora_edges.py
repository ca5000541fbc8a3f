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
