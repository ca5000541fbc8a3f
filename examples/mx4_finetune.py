"""Fine-tuning a mixture-of-experts block whose weights stay frozen: 4-bit experts
with a low-rank adapter each beside their down projection, a projection shared by
several fine-tunings with an adapter per sequence, and the router's balance loss
over padded sequences.

    python examples/mx4_finetune.py   # a few steps, then decoded tokens, on one GPU
"""
from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from cvmm_codex_amd import (cvmm_balance_loss, cvmm_gate_logits, cvmm_lora, cvmm_mx4, cvmm_mx4_quantize,
                            cvmm_prepare_sel2, cvmm_route_scored)


class AdaptedMoE(torch.nn.Module):
    """x [sequences, tokens, d_model] and an adapter per sequence (-1: none) ->
    projection, then top-k of `experts` on its output, added to it."""

    def __init__(self, d_model: int, d_expert: int, experts: int, k: int, adapters: int, rank: int, seed: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g) / s[-2] ** 0.5
        par = lambda t: torch.nn.Parameter(t.bfloat16())
        self.k, self.scale = k, 2.0
        self.gate = par(rnd(d_model, experts))
        self.register_buffer("bias", torch.zeros(experts))
        self.register_buffer("proj", rnd(d_model, d_model).bfloat16())
        self.seq_a, self.seq_b = par(rnd(adapters, d_model, rank)), par(0.1 * rnd(adapters, rank, d_model))
        self.exp_a, self.exp_b = par(rnd(experts, d_expert, rank)), par(0.1 * rnd(experts, rank, d_model))
        self._weights = rnd(experts, d_model, d_expert), rnd(experts, d_expert, d_model)
        self.up = self.down = None

    def cuda(self, device=None):
        """Moves the block to the GPU and lays the expert weights out in 4 bits."""
        super().cuda(device)
        self.up, self.down = (cvmm_mx4_quantize(w.to(self.gate.device), dim=1) for w in self._weights)
        return self

    def forward(self, x: torch.Tensor, adapters: torch.Tensor, mask: torch.Tensor | None = None):
        """(y, balance loss, [balance, z], routes per expert, chosen experts)."""
        ids = adapters[:, None].expand(x.shape[:-1])
        z = cvmm_lora(x, ids, self.seq_a, self.seq_b, weight=self.proj, scale=self.scale)
        logits = cvmm_gate_logits(z, self.gate)
        weights, sel, routed = cvmm_route_scored(logits, self.k, bias=self.bias, scores="sigmoid")
        aux, terms, counts = cvmm_balance_loss(logits, sel, scores="sigmoid", mask=mask, per_sequence=True, weight=0.01,
                                               z_weight=0.001)
        h = F.gelu(cvmm_mx4(z, routed, self.up))
        rows = cvmm_prepare_sel2(routed, route_input=True)
        d = cvmm_lora(h, rows, self.exp_a, self.exp_b, base=cvmm_mx4(h, rows, self.down), scale=self.scale)
        y = z + (d * weights.unsqueeze(-1)).sum(-2).to(d.dtype)
        return y, aux, terms, counts, sel


def main():
    block = AdaptedMoE(512, 128, 32, 4, adapters=3, rank=16).cuda()
    opt = torch.optim.SGD(block.parameters(), lr=0.1)
    x, target = (torch.randn(4, 333, 512, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    adapters = torch.tensor([0, 2, -1, 1], device="cuda")
    mask = torch.arange(333, device="cuda") < torch.tensor([[333], [200], [77], [310]], device="cuda")
    for step in range(5):
        y, aux, terms, counts, _ = block(x, adapters, mask)
        loss = F.mse_loss(y[mask].float(), target[mask].float()) + aux
        opt.zero_grad()
        loss.backward()
        opt.step()
        block.bias += 0.01 * torch.sign(counts.float().mean() - counts)
        print(f"step {step}: loss {float(loss.detach()):.4f}, balance {float(terms[0]):.4f}, z {float(terms[1]):.3f}, "
              f"most and least loaded expert {int(counts.max())} and {int(counts.min())}")
    with torch.no_grad():
        y, *_, sel = block(torch.randn(4, 1, 512, device="cuda", dtype=torch.bfloat16), adapters)
        print("one token of each sequence", tuple(y.shape), "experts of the first", sel[0, 0].tolist())


if __name__ == "__main__":
    main()
