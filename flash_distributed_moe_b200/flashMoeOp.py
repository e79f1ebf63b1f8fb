"""Drop-in module wrapper: runs a Qwen3 sparse-MoE block's forward through the launcher, in place.

Mirrors the reference's FlashMoeBlockWrapper (test/singleGPU/python/flashMoeOp.py:7-38) without
importing vLLM: any module exposing `gate.weight` [E,H], `experts.w13_weight` [E,2I,H] and
`experts.w2_weight` [E,H,I] works (vLLM's Qwen3MoeSparseMoeBlock has exactly these).
"""
from __future__ import annotations

import torch

from .flashFfn import gated_ffn, quantize_ffn_weights
from .flashMoeLauncher import MoeKernelLauncher


class FlashMoeBlockWrapper(torch.nn.Module):
    def __init__(self, qwen3MoeSparseMoeBlockModule: torch.nn.Module, maxTokens: int, topk: int = 8):
        super().__init__()
        self.qwen3MoeSparseMoeBlockModule = qwen3MoeSparseMoeBlockModule
        self.launcher = MoeKernelLauncher()
        gateWeights = qwen3MoeSparseMoeBlockModule.gate.weight
        ffn1ExpertWeights = qwen3MoeSparseMoeBlockModule.experts.w13_weight
        ffn2ExpertWeights = qwen3MoeSparseMoeBlockModule.experts.w2_weight
        uniqueid = self.launcher.getDistributedUniqueId(empty=True)
        self.launcher.create(gateWeights.detach(), ffn1ExpertWeights.detach(), ffn2ExpertWeights.detach(),
                             maxTokens, uniqueid, 0, 1, topk=topk)
        self.maxTokens = maxTokens

    def __del__(self):
        try:
            self.launcher.destroy()
        except Exception:
            pass

    def forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
        num_tokens, _ = hidden_states.shape
        if num_tokens <= self.maxTokens:
            # in-place: output memory = input memory
            self.launcher.launch(hidden_states, hidden_states)
            return hidden_states
        # larger batches go to the wrapped block (the reference calls a non-existent super().forward here)
        return self.qwen3MoeSparseMoeBlockModule(hidden_states)


class FlashFfnBlockWrapper(torch.nn.Module):
    """The same for a dense block: any module exposing `gate_up_proj.weight` [2I,H] (gate rows first) and
    `down_proj.weight` [H,I], without biases and with SiLU between them, e.g. the dense layers and shared experts of the same models.  With `fourBit` the
    weights are quantised once, here, and the forward pass reads them at half a byte per value."""

    def __init__(self, mlpModule: torch.nn.Module, fourBit: bool = False):
        super().__init__()
        for projection in (mlpModule.gate_up_proj, mlpModule.down_proj):
            if getattr(projection, "bias", None) is not None:
                raise RuntimeError("projections with a bias are not supported")
        self.mlpModule = mlpModule
        self.fourBitWeights = None
        if fourBit:
            self.fourBitWeights = quantize_ffn_weights(mlpModule.gate_up_proj.weight.detach(),
                                                       mlpModule.down_proj.weight.detach())

    def forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
        if self.fourBitWeights is not None:
            return gated_ffn(hidden_states, *self.fourBitWeights)
        return gated_ffn(hidden_states, self.mlpModule.gate_up_proj.weight, self.mlpModule.down_proj.weight)
