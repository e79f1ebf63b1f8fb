"""4-bit microscaled matrices and products: half a byte per value and one power-of-two scale per 32 of them.

    w = mx4_quantize(weight)                 # [N, K] or [B, N, K], once
    y = mx4_matmul(mx4_quantize(x), w)       # x [M, K] -> [M, N]
    h = mx4_gated_matmul(mx4_quantize(x), w13)   # w13 [2, I, K] -> silu(x w13[0]^T) * (x w13[1]^T)

The values are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), the scales E8M0; a block's scale is
2^(floor(log2(largest magnitude)) - 2), elements are rounded to nearest even and saturate at 6, and a block that
holds a NaN or an infinity stands for NaN.  Products are exact in their operands and accumulated in fp32; the sigmoid of
a gate value g is off by at most 2^-21 + |g| 2^-23 of itself, which an fp32 result shows.
None of these functions has a gradient: 4-bit weights are constants, and a product refuses activations whose origin needs
one, where gradients are on.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import get_proxy_mode

from . import _lib

# what torch.jit.is_tracing and get_proxy_mode ask first, at a third of their time
_is_tracing, _dispatch_modes = torch._C._is_tracing, torch._C._len_torch_dispatch_stack
DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


def _check_dtype(dtype: torch.dtype) -> int:
    if dtype not in DTYPES:
        raise RuntimeError("dtype must be bfloat16, float16 or float32")
    return DTYPES[dtype]


def check_no_tangent(*tensors) -> None:
    """Forward-mode derivatives are refused: a result without a tangent would stand for a derivative of zero."""
    if forward_ad._current_level < 0:  # no dual tensors outside a level
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("forward-mode derivatives are not supported")


def check_not_traced() -> None:
    """A recorder of torch operators (torch.jit.trace, make_fx) sees the allocation of a result and not the call that fills
    it: its program would return memory as it is found.  torch.compile runs these calls between its graphs."""
    if _is_tracing() or (_dispatch_modes() > 0 and get_proxy_mode() is not None):
        raise RuntimeError("the dense operators cannot be recorded by torch.jit.trace or make_fx")


def _scale_bytes(batch: int, rows: int, cols: int) -> int:
    """The size of the scales, as FlashMoeMx4ScaleBytes gives it."""
    return batch * -(-rows // 128) * -(-cols // 256) * 1024


class Mx4Tensor:
    """A 4-bit matrix [rows, cols] or batch of them [batch, rows, cols].  `values` uint8 [..., rows, cols / 2] with the
    even element in the low half of a byte; `scales` uint8, in blocks of 512 for 128 rows and 128 columns, where those of
    columns that do not exist are not 255 (which stands for NaN; mx4_quantize writes 0)."""

    __slots__ = ("shape", "device", "_tensors", "_buffer", "_pointers", "_needs_gradient")

    def __init__(self, values: torch.Tensor, scales: torch.Tensor):
        for t, name in ((values, "values"), (scales, "scales")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or not t.is_contiguous() or t.data_ptr() % 16:
                raise RuntimeError(f"{name} must be a contiguous uint8 tensor that starts on 16 bytes")
        if values.dim() not in (2, 3) or values.shape[-1] == 0 or values.shape[-1] % 16 != 0:
            raise RuntimeError("values must be [rows, cols / 2] or [batch, rows, cols / 2] with cols a multiple of 32")
        batch = 1 if values.dim() == 2 else values.shape[0]
        if scales.numel() != _scale_bytes(batch, values.shape[-2], 2 * values.shape[-1]):
            raise RuntimeError("scales must have 512 bytes per 128 rows and 128 columns, an even number of blocks per row")
        if values.device != scales.device:
            raise RuntimeError("values and scales must be on the same device")
        self.shape = torch.Size((*values.shape[:-1], values.shape[-1] * 2))
        self.device = values.device
        self._tensors, self._buffer = (values, scales), None
        self._pointers = values.data_ptr(), scales.data_ptr()
        self._needs_gradient = False

    @classmethod
    def _of_buffer(cls, buffer: torch.Tensor, shape: torch.Size, pointers, needs_gradient: bool = False) -> "Mx4Tensor":
        """Values and scales one after the other in a buffer of the right size."""
        self = cls.__new__(cls)
        self.shape, self.device = shape, buffer.device
        self._tensors, self._buffer, self._pointers = None, buffer, pointers
        self._needs_gradient = needs_gradient
        return self

    def __reduce__(self):
        # copies and unpickled matrices have memory of their own, and with it addresses of their own
        return Mx4Tensor, (self.values, self.scales), (None, {"_needs_gradient": self._needs_gradient})

    def _split(self):
        if self._tensors is None:
            n = self.shape.numel() // 2
            self._tensors = self._buffer[:n].view(*self.shape[:-1], self.shape[-1] // 2), self._buffer[n:]
        return self._tensors

    @property
    def values(self) -> torch.Tensor:
        return self._split()[0]

    @property
    def scales(self) -> torch.Tensor:
        return self._split()[1]

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the matrix stands for, exact unless they leave the type's range."""
        check_not_traced()
        code, shape, device = _check_dtype(dtype), self.shape, self.device
        if device.type != "cuda":
            raise RuntimeError("values must be a CUDA tensor")
        out = torch.empty(shape, dtype=dtype, device=device)
        _lib.run(device.index, "FlashMoeMx4Dequantize", *self._pointers, shape[0] if len(shape) == 3 else 1, shape[-2],
                 shape[-1], code, out.data_ptr())
        return out


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """x [rows, cols] or [batch, rows, cols], bf16, fp16 or fp32, cols a multiple of 32; rows may be strided if they
    start on 16 bytes.  Asynchronous on the current torch stream of x's device.  What comes of the result is a constant to
    autograd."""
    if not isinstance(x, torch.Tensor):
        raise RuntimeError("x tensor is undefined")
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    check_not_traced()
    check_no_tangent(x)
    code, shape, device = _check_dtype(x.dtype), x.shape, x.device
    if len(shape) not in (2, 3) or shape[-1] == 0 or shape[-1] % 32 != 0:
        raise RuntimeError("x must be [rows, cols] or [batch, rows, cols] with cols a multiple of 32")
    batch, rows, cols = shape if len(shape) == 3 else (1, *shape)
    ptr = x.data_ptr()
    aligned = ptr % 16 == 0
    if x.is_contiguous():
        batch_stride, row_stride = rows * cols, cols  # multiples of 32 elements
    else:
        per16 = 16 // x.element_size()
        batch_stride, row_stride = x.stride(0) if batch > 1 else 0, x.stride(-2) if rows > 1 else 0
        aligned = aligned and x.stride(-1) == 1 and batch_stride % per16 == 0 and row_stride % per16 == 0
    if not aligned:
        raise RuntimeError("rows of x must be contiguous and start on 16 bytes")
    n = batch * rows * cols // 2
    buffer = torch.empty(n + _scale_bytes(batch, rows, cols), dtype=torch.uint8, device=device)
    to = buffer.data_ptr()
    _lib.run(device.index, "FlashMoeMx4Quantize", ptr, code, batch, rows, cols, batch_stride, row_stride, to, to + n)
    return Mx4Tensor._of_buffer(buffer, shape, (to, to + n), x.requires_grad and torch.is_grad_enabled())


def _product(a: Mx4Tensor, b: Mx4Tensor, out_dtype: torch.dtype, gated: bool) -> torch.Tensor:
    if not isinstance(a, Mx4Tensor) or not isinstance(b, Mx4Tensor):
        raise RuntimeError("operands must be Mx4Tensors")
    check_not_traced()
    if a._needs_gradient and torch.is_grad_enabled():
        raise RuntimeError("products of 4-bit matrices have no gradient; quantise x.detach() or run under torch.no_grad()")
    code = _check_dtype(out_dtype)
    device, sa, sb = a.device, a.shape, b.shape
    if device != b.device or device.type != "cuda":
        raise RuntimeError("operands must be on the same CUDA device")
    if len(sa) != 2 or len(sb) != (3 if gated else 2) or sa[-1] != sb[-1] or (gated and sb[0] != 2):
        raise RuntimeError("operands must be [M, K] and " + ("[2, N, K]" if gated else "[N, K]"))
    m, n = sa[0], sb[-2]
    out = torch.empty((m, n), dtype=out_dtype, device=device)
    _lib.run(device.index, "FlashMoeMx4Matmul", *a._pointers, *b._pointers, out.data_ptr(), code, m, n, sa[1], int(gated))
    return out


def mx4_matmul(a: Mx4Tensor, b: Mx4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K], b [N, K] -> a b^T [M, N]."""
    return _product(a, b, out_dtype, False)


def mx4_gated_matmul(a: Mx4Tensor, w13: Mx4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K], w13 [2, I, K] -> silu(a w13[0]^T) * (a w13[1]^T) [M, I], rounded once."""
    return _product(a, w13, out_dtype, True)
