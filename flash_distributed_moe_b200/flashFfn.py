"""The gated feed-forward block (SwiGLU) of a dense layer or of a shared expert, with its gradient.

    y = gated_ffn(x, w13, w2)       # (silu(x w13[:I]^T) * (x w13[I:]^T)) w2^T

`w13` and `w2` are laid out as one expert of the mixture-of-experts layer: [2I, H] with the gate projection's rows
first, and [H, I].  bf16 or fp16, or, without gradients, 4-bit weights (`quantize_ffn_weights`).
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Tuple, Union

import torch

from . import _lib
from .flashMx4 import Mx4Tensor, check_no_tangent, check_not_traced, mx4_quantize

_DTYPES = {torch.bfloat16: 0, torch.float16: 2}
Weight = Union[torch.Tensor, Mx4Tensor]


@functools.lru_cache(maxsize=1024)
def _config(hidden: int, inter: int, dtype: torch.dtype):
    return C.byref(_lib.FlashMoeFfnConfig(hidden, inter, _DTYPES[dtype], (C.c_int32 * 5)()))


def _check(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name} tensor is undefined")
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"{name} must be bfloat16 or float16")


def _check_weights(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor) -> None:
    dtype, device = x.dtype, x.get_device()
    for t, name in ((w13, "w13"), (w2, "w2")):
        _check(t, name)
        if t.dtype != dtype or t.get_device() != device:
            raise RuntimeError(f"{name} must have the dtype and device of x")
        if not t.is_contiguous() or t.data_ptr() % 16:
            raise RuntimeError(f"{name} must be contiguous and start on 16 bytes")
    shape = w2.shape
    if len(shape) != 2 or w13.shape != (2 * shape[1], shape[0]) or x.shape[-1] != shape[0]:
        raise RuntimeError("x, w13 and w2 must be [..., hidden], [2*inter, hidden] and [hidden, inter]")
    if shape[0] % 8 or shape[1] % 8 or shape[0] == 0 or shape[1] == 0:
        raise RuntimeError("hidden and inter must be multiples of 8")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[..., n] as contiguous rows on 16 bytes; a copy only where the tensor is neither."""
    if t.dim() != 2 or not t.is_contiguous():
        t = t.reshape(-1, t.shape[-1]).contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _aligned(nbytes: int) -> int:
    return (nbytes + 255) & -256


def _forward(x: torch.Tensor, w13: torch.Tensor, w2: torch.Tensor, save: bool):
    (hidden, inter), tokens = w2.shape, x.shape[0]
    part = tokens * inter
    # as FlashMoeFfnSavedBytes and FlashMoeFfnWorkspaceBytes give them
    nbytes = _aligned(4 * part) + 2 * _aligned(2 * part) if save else _aligned(2 * part)
    y = torch.empty_like(x)
    buf = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    to = buf.data_ptr()
    _lib.run(x.get_device(), "FlashMoeFfnForward", _config(hidden, inter, x.dtype), x.data_ptr(), w13.data_ptr(),
             w2.data_ptr(), y.data_ptr(), to if save else None, None if save else to, nbytes, tokens)
    return y, buf


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w13, w2):
        y, saved = _forward(x, w13, w2, save=True)
        ctx.save_for_backward(x, w13, w2, saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, w13, w2, saved = ctx.saved_tensors
        (hidden, inter), tokens = w2.shape, x.shape[0]
        dy = _rows(dy)
        need = ctx.needs_input_grad
        dx = torch.empty_like(x) if need[0] else None
        dw13 = torch.empty_like(w13) if need[1] else None
        dw2 = torch.empty_like(w2) if need[2] else None
        nbytes = _aligned(4 * tokens * inter)  # FlashMoeFfnWorkspaceBytes
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
        _lib.run(x.get_device(), "FlashMoeFfnBackward", _config(hidden, inter, x.dtype), dy.data_ptr(), x.data_ptr(),
                 w13.data_ptr(), w2.data_ptr(), saved.data_ptr(), dx.data_ptr() if need[0] else None,
                 dw13.data_ptr() if need[1] else None, dw2.data_ptr() if need[2] else None, ws.data_ptr(), nbytes, tokens)
        return dx, dw13, dw2


def gated_ffn(x: torch.Tensor, w13: Weight, w2: Weight) -> torch.Tensor:
    """x [..., H] -> [..., H].  Asynchronous on the current torch stream of x's device.  Differentiable in x, w13 and w2
    by torch's reverse mode, once: the gate and up projections of the tokens and silu(g) * u are kept for the backward
    pass, in 24 bits and in the dtype.  With Mx4Tensor weights (w13 [2, I, H], w2 [H, I]) x and the activations are
    quantised to 4 bits too, and there is no gradient.

    Operands of a product are rounded to the dtype: h = silu(g) * u, and in the backward pass the gradients of g and u.
    In fp16 all three are infinite beyond 65504 and vanish below 3e-8, as in a program of torch operators.

    The same call gives the same bits.  A call that keeps nothing for a backward pass may use another kernel than one
    that does, and another number of tokens another one again, whose sums have another order: results then differ by
    the rounding of the sums, e.g. those of a checkpointed block from its recomputation.

    Forward-mode derivatives and recorders of torch operators (torch.jit.trace, make_fx) are refused; torch.compile runs
    the call between its graphs.

    A training step may be captured into a CUDA graph while no eager graph of the same leaves is alive: torch keeps the
    gradient accumulators of such a graph on its stream, which a captured backward pass of any operator, this one
    included, cannot join, and raises an error."""
    _check(x, "x")
    if x.dim() < 1:
        raise RuntimeError("x must be [..., hidden]")
    check_not_traced()
    check_no_tangent(x, w13, w2)
    if isinstance(w13, Mx4Tensor) or isinstance(w2, Mx4Tensor):
        return _mx4_ffn(x, w13, w2)
    _check_weights(x, w13, w2)
    rows = _rows(x)
    if (x.requires_grad or w13.requires_grad or w2.requires_grad) and torch.is_grad_enabled():
        y = _GatedFfn.apply(rows, w13, w2)
    else:
        y, _ = _forward(rows, w13, w2, save=False)
    return y if x.dim() == 2 else y.reshape(x.shape)


def quantize_ffn_weights(w13: torch.Tensor, w2: torch.Tensor) -> Tuple[Mx4Tensor, Mx4Tensor]:
    """[2I, H] and [H, I] weights of a block as 4-bit matrices for gated_ffn; H and I multiples of 32."""
    if w13.dim() != 2 or w2.dim() != 2 or tuple(w13.shape) != (2 * w2.shape[1], w2.shape[0]):
        raise RuntimeError("w13 and w2 must be [2*inter, hidden] and [hidden, inter]")
    return mx4_quantize(w13.view(2, w2.shape[1], w2.shape[0])), mx4_quantize(w2)


def _mx4_ffn(x: torch.Tensor, w13: Mx4Tensor, w2: Mx4Tensor) -> torch.Tensor:
    if not isinstance(w13, Mx4Tensor) or not isinstance(w2, Mx4Tensor):
        raise RuntimeError("w13 and w2 must both be 4-bit weights or neither")
    if torch.is_grad_enabled() and x.requires_grad:
        raise RuntimeError("gated_ffn has no gradient with 4-bit weights")
    if w13.device != x.device or w2.device != x.device:
        raise RuntimeError("x, w13 and w2 must be on the same device")
    if len(w2.shape) != 2 or tuple(w13.shape) != (2, w2.shape[1], w2.shape[0]) or x.shape[-1] != w2.shape[0]:
        raise RuntimeError("x, w13 and w2 must be [..., hidden], [2, inter, hidden] and [hidden, inter]")
    if w2.shape[0] % 32:
        raise RuntimeError("hidden and inter must be multiples of 32")
    rows, (hidden, inter) = _rows(x.detach()), w2.shape
    cfg = _config(hidden, inter, x.dtype)
    y = torch.empty_like(rows)
    nbytes = _lib.lib().FlashMoeMx4FfnWorkspaceBytes(cfg, rows.shape[0])
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.run(x.get_device(), "FlashMoeMx4FfnForward", cfg, rows.data_ptr(), *w13._pointers, *w2._pointers,
             y.data_ptr(), ws.data_ptr(), nbytes, rows.shape[0])
    return y.reshape(x.shape)


def dense_status(reset: bool = False) -> int:
    """Code of the first device-side error of the dense operators in this process, 0 if none.  After one, calls are
    refused until reset."""
    code = C.c_uint32(0)
    _lib.check(_lib.lib().FlashMoeDenseStatus(C.byref(code), int(reset)), "DenseStatus")
    return int(code.value)
