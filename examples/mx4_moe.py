"""A mixture-of-experts feed-forward block with 4-bit expert weights: the router
of balanced models, the up and the down projection, as served.

    python examples/mx4_moe.py        # a prompt, then decoded tokens, on one GPU

Fine-tuning runs the same lines with gradients: they reach the input, the gate
and the routing weights; the expert weights stay as they are.
"""
from __future__ import annotations

import os
import sys

import torch
import torch.nn.functional as F

if __name__ == "__main__":
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from cvmm_codex_amd import cvmm_gate_logits, cvmm_mx4, cvmm_mx4_quantize, cvmm_prepare_sel2, cvmm_route_scored


class MX4MoE(torch.nn.Module):
    """d_model -> experts of d_expert -> d_model, top-k of `experts`."""

    def __init__(self, d_model: int, d_expert: int, experts: int, k: int, groups: int = 1, topk_groups: int = 1,
                 scale: float = 2.5, seed: int = 0):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        self.k, self.groups, self.topk_groups, self.scale = k, groups, topk_groups, scale
        self.gate = torch.nn.Parameter((torch.randn(d_model, experts, generator=g) / d_model ** 0.5).bfloat16())
        # the balance bias: moved by the trainer towards even loads, no gradient
        self.register_buffer("bias", 0.01 * torch.randn(experts, generator=g))
        self._weights = (torch.randn(experts, d_model, d_expert, generator=g) / d_model ** 0.5,
                         torch.randn(experts, d_expert, d_model, generator=g) / d_expert ** 0.5)
        self.up = self.down = None

    def cuda(self, device=None):
        """Moves the block to the GPU and lays the expert weights out in 4 bits."""
        super().cuda(device)
        self.up, self.down = (cvmm_mx4_quantize(w.to(self.gate.device), dim=1) for w in self._weights)
        return self

    def forward(self, x: torch.Tensor, quantize_input: bool = False):
        """(y, chosen experts) of x [..., d_model] in bf16."""
        weights, sel, routed = cvmm_route_scored(cvmm_gate_logits(x, self.gate), self.k, bias=self.bias,
                                                 scores="sigmoid", groups=self.groups, topk_groups=self.topk_groups,
                                                 scale=self.scale)
        h = F.gelu(cvmm_mx4(x, routed, self.up, quantize_input))
        return cvmm_mx4(h, cvmm_prepare_sel2(routed, weights, route_input=True), self.down, quantize_input), sel


def main():
    block = MX4MoE(1024, 256, 64, 8, groups=8, topk_groups=4).cuda()
    nbytes = block.up.nbytes + block.down.nbytes
    print(f"expert weights: {nbytes / 2 ** 20:.1f} MiB in 4 bits")
    with torch.no_grad():
        prompt = torch.randn(1, 777, 1024, device="cuda", dtype=torch.bfloat16)
        y, sel = block(prompt)
        y4, _ = block(prompt, quantize_input=True)
        print("prompt", tuple(y.shape), "4-bit inputs differ by",
              f"{float((y4 - y).float().norm() / y.float().norm()):.3f} of the norm")
        for step in range(3):
            y, sel = block(torch.randn(4, 1024, device="cuda", dtype=torch.bfloat16))
            print("step", step, "experts of the first sequence", sel[0].tolist())


if __name__ == "__main__":
    main()
