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


# A module of these (by name: several projects have one of their own) is SiLU, with or without the product by the other half.
_SILU = {"SiLU", "SiluAndMul", "SiLUActivation", "Swish", "silu", "swish", "silu_and_mul"}


def _refuse_what_is_more_than_the_block(mlp: torch.nn.Module) -> None:
    """The wrapper replaces the whole forward of `mlp`, so there may be nothing in it but the two products and SiLU."""
    projections = (mlp.gate_up_proj, mlp.down_proj)
    for projection in projections:
        if getattr(projection, "bias", None) is not None:
            raise RuntimeError("projections with a bias are not supported")
    for projection, flag, default in ((mlp.gate_up_proj, "gather_output", False), (mlp.down_proj, "reduce_results", True)):
        if int(getattr(projection, "tp_size", 1)) > 1 and getattr(projection, flag, default):
            raise RuntimeError("projections whose results are put together over ranks are not supported")
    for name, child in mlp.named_children():
        if child in projections or isinstance(child, torch.nn.Identity) or type(child).__name__ in _SILU:
            continue
        if isinstance(child, torch.nn.Dropout) and child.p == 0:
            continue
        raise RuntimeError(f"{name} ({type(child).__name__}) is no part of a block with SiLU between its projections")
    for name, _ in mlp.named_parameters(recurse=False):
        raise RuntimeError(f"{name} is no part of a block with SiLU between its projections")
    for name in ("act_fn", "activation_fn", "activation", "act", "hidden_act"):
        act = getattr(mlp, name, None)
        if act is None or isinstance(act, torch.nn.Module):  # modules: above
            continue
        if (act if isinstance(act, str) else getattr(act, "__name__", "")) not in _SILU:
            raise RuntimeError(f"{name} of the block is not SiLU")


class FlashFfnBlockWrapper(torch.nn.Module):
    """The same for a dense block: any module exposing `gate_up_proj.weight` [2I,H] (gate rows first) and
    `down_proj.weight` [H,I] that computes down_proj(silu(gate) * up) and nothing else, e.g. the dense layers and
    shared experts of the same models.  Refused are biases, a factor on the result (`expert_gate`), other activations
    than SiLU, and projections that sum or gather over ranks.  With `fourBit` the weights are quantised once, here, and
    the forward pass reads them at half a byte per value."""

    def __init__(self, mlpModule: torch.nn.Module, fourBit: bool = False):
        super().__init__()
        _refuse_what_is_more_than_the_block(mlpModule)
        self.mlpModule = mlpModule
        self.fourBitWeights = None
        if fourBit:
            self.fourBitWeights = quantize_ffn_weights(mlpModule.gate_up_proj.weight.detach(),
                                                       mlpModule.down_proj.weight.detach())

    def forward(self, hidden_states: torch.Tensor) -> torch.Tensor:
        if self.fourBitWeights is not None:
            return gated_ffn(hidden_states, *self.fourBitWeights)
        return gated_ffn(hidden_states, self.mlpModule.gate_up_proj.weight, self.mlpModule.down_proj.weight)
