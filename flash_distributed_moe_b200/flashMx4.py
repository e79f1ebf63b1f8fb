"""4-bit microscaled matrices and products: half a byte per value and one power-of-two scale per 32 of them.

    w = mx4_quantize(weight)                 # [N, K] or [B, N, K], once
    y = mx4_matmul(mx4_quantize(x), w)       # x [M, K] -> [M, N]
    h = mx4_gated_matmul(mx4_quantize(x), w13)   # w13 [2, I, K] -> silu(x w13[0]^T) * (x w13[1]^T)

The values are E2M1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign), the scales E8M0; a block's scale is
2^(floor(log2(largest magnitude)) - 2), elements are rounded to nearest even and saturate at 6, and a block that
holds a NaN or an infinity stands for NaN.  Products are exact in their operands and accumulated in fp32.
None of these functions has a gradient.
"""
from __future__ import annotations

import torch

from . import _lib

DTYPES = {torch.bfloat16: 0, torch.float32: 1, torch.float16: 2}


def _check_dtype(dtype: torch.dtype) -> int:
    if dtype not in DTYPES:
        raise RuntimeError("dtype must be bfloat16, float16 or float32")
    return DTYPES[dtype]


class Mx4Tensor:
    """A 4-bit matrix [rows, cols] or batch of them [batch, rows, cols].  `values` uint8 [..., rows, cols / 2] with the
    even element in the low half of a byte; `scales` uint8, in blocks of 512 for 128 rows and 128 columns."""

    __slots__ = ("values", "scales", "shape")

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
        self._set(values, scales)

    def _set(self, values, scales):
        self.values, self.scales = values, scales
        self.shape = torch.Size((*values.shape[:-1], values.shape[-1] * 2))
        return self

    @property
    def device(self) -> torch.device:
        return self.values.device

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values that the matrix stands for.  Exact in fp32; in bf16 and fp16 unless they leave the type's range."""
        code = _check_dtype(dtype)
        values, shape = self.values, self.shape
        if not values.is_cuda:
            raise RuntimeError("values must be a CUDA tensor")
        out = torch.empty(shape, dtype=dtype, device=values.device)
        _lib.run(values.get_device(), "FlashMoeMx4Dequantize", values.data_ptr(), self.scales.data_ptr(),
                 shape[0] if len(shape) == 3 else 1, shape[-2], shape[-1], code, out.data_ptr())
        return out


def _scale_bytes(batch: int, rows: int, cols: int) -> int:
    """The size of the scales, as FlashMoeMx4ScaleBytes gives it."""
    return batch * -(-rows // 128) * -(-cols // 256) * 1024


def mx4_quantize(x: torch.Tensor) -> Mx4Tensor:
    """x [rows, cols] or [batch, rows, cols], bf16, fp16 or fp32, cols a multiple of 32; rows may be strided if they
    start on 16 bytes.  Asynchronous on the current torch stream of x's device."""
    if not isinstance(x, torch.Tensor):
        raise RuntimeError("x tensor is undefined")
    if not x.is_cuda:
        raise RuntimeError("x must be a CUDA tensor")
    code = _check_dtype(x.dtype)
    shape = x.shape
    if len(shape) not in (2, 3) or shape[-1] == 0 or shape[-1] % 32 != 0:
        raise RuntimeError("x must be [rows, cols] or [batch, rows, cols] with cols a multiple of 32")
    batch, rows, cols = shape if len(shape) == 3 else (1, *shape)
    ptr = x.data_ptr()
    if x.is_contiguous():
        strides = (rows * cols, cols)  # multiples of 32 elements
        aligned = ptr % 16 == 0
    else:
        per16 = 16 // x.element_size()
        strides = (x.stride(0) if batch > 1 else 0, x.stride(-2) if rows > 1 else 0)
        aligned = ptr % 16 == 0 and x.stride(-1) == 1 and strides[0] % per16 == 0 and strides[1] % per16 == 0
    if not aligned:
        raise RuntimeError("rows of x must be contiguous and start on 16 bytes")
    values = torch.empty((*shape[:-1], cols // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty(_scale_bytes(batch, rows, cols), dtype=torch.uint8, device=x.device)
    _lib.run(x.get_device(), "FlashMoeMx4Quantize", ptr, code, batch, rows, cols, *strides, values.data_ptr(),
             scales.data_ptr())
    return Mx4Tensor.__new__(Mx4Tensor)._set(values, scales)


def _product(a: Mx4Tensor, b: Mx4Tensor, out_dtype: torch.dtype, gated: bool) -> torch.Tensor:
    if not isinstance(a, Mx4Tensor) or not isinstance(b, Mx4Tensor):
        raise RuntimeError("operands must be Mx4Tensors")
    code = _check_dtype(out_dtype)
    av, bv, sa, sb = a.values, b.values, a.shape, b.shape
    if av.device != bv.device or not av.is_cuda:
        raise RuntimeError("operands must be on the same CUDA device")
    if len(sa) != 2 or len(sb) != (3 if gated else 2) or sa[-1] != sb[-1] or (gated and sb[0] != 2):
        raise RuntimeError("operands must be [M, K] and " + ("[2, N, K]" if gated else "[N, K]"))
    m, n = sa[0], sb[-2]
    out = torch.empty((m, n), dtype=out_dtype, device=av.device)
    _lib.run(av.get_device(), "FlashMoeMx4Matmul", av.data_ptr(), a.scales.data_ptr(), bv.data_ptr(), b.scales.data_ptr(),
             out.data_ptr(), code, m, n, sa[1], int(gated))
    return out


def mx4_matmul(a: Mx4Tensor, b: Mx4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K], b [N, K] -> a b^T [M, N]."""
    return _product(a, b, out_dtype, False)


def mx4_gated_matmul(a: Mx4Tensor, w13: Mx4Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """a [M, K], w13 [2, I, K] -> silu(a w13[0]^T) * (a w13[1]^T) [M, I], rounded once."""
    return _product(a, w13, out_dtype, True)
