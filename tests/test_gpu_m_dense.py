"""GPU: the dense operators one behind another, where they are refused, and where their waits run out."""
import ctypes as C

import pytest
import torch

import dense_testlib as dl
from flash_distributed_moe_b200 import _lib, mx4_quantize

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def stream():
    return C.c_void_p(torch.cuda.current_stream().cuda_stream)


@pytest.mark.parametrize("m,n,k", [(16, 1024, 512), (300, 4096, 512), (2048, 4096, 512)])
def test_a_launch_reads_what_the_one_before_has_written(m, n, k):
    """Product, quantisation of its result and the inverse in the same memory again and again, none of them waited for."""
    lib, rounds = _lib.lib(), 12
    g = torch.Generator().manual_seed(1)
    xs = [mx4_quantize(torch.randn(m, k, generator=g).to(BF16).cuda()) for _ in range(rounds)]
    w = mx4_quantize(torch.randn(n, k, generator=g).to(BF16).cuda())
    h = torch.empty(m, n, dtype=BF16, device="cuda")
    values = torch.empty(m, n // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(lib.FlashMoeMx4ScaleBytes(1, m, n), dtype=torch.uint8, device="cuda")
    outs = [torch.empty(m, n, dtype=FP32, device="cuda") for _ in range(rounds)]
    kept = [torch.empty_like(h) for _ in range(rounds)]
    torch.cuda.synchronize()
    for wait in (False, True):
        got = []
        for x, out, keep in zip(xs, outs, kept):
            for step in (
                    lambda: lib.FlashMoeMx4Matmul(*x._pointers, *w._pointers, h.data_ptr(), 0, m, n, k, 0, stream()),
                    lambda: lib.FlashMoeMx4Quantize(h.data_ptr(), 0, 1, m, n, 0, n, values.data_ptr(), scales.data_ptr(), stream()),
                    lambda: lib.FlashMoeMx4Dequantize(values.data_ptr(), scales.data_ptr(), 1, m, n, 1, out.data_ptr(), stream())):
                assert step() == 0
                if wait:
                    torch.cuda.synchronize()
            if wait:
                keep.copy_(h)
                got.append(torch.equal(out, before[len(got)]))
        torch.cuda.synchronize()
        before = [out.clone() for out in outs]
    assert all(got)
    for out, h in zip(outs, kept):
        assert torch.equal(out, dl.mx4(h).float())
