"""GPU: the dense operators one behind another, where they are refused, and where their waits run out."""
import ctypes as C
import os
import subprocess
import sys
import threading

import pytest
import torch

import dense_testlib as dl
from flash_distributed_moe_b200 import _lib, dense_status, gated_ffn, mx4_matmul, mx4_quantize, quantize_ffn_weights

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
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


def config(hidden, inter, dtype=0):
    return C.byref(_lib.FlashMoeFfnConfig(hidden, inter, dtype, (C.c_int32 * 5)()))


def room(nbytes):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device="cuda")


def forward(tokens, hidden, inter):
    x, w13, w2, _ = dl.make(tokens, hidden, inter, BF16)
    lib, cfg, y = _lib.lib(), config(hidden, inter), torch.empty_like(x)
    ws = room(lib.FlashMoeFfnWorkspaceBytes(cfg, tokens, 0))
    return [y], (x, w13, w2, ws), lambda: lib.FlashMoeFfnForward(cfg, x.data_ptr(), w13.data_ptr(), w2.data_ptr(), y.data_ptr(), None,
                                                             ws.data_ptr(), ws.numel(), tokens, stream())


def training_forward(tokens, hidden, inter):
    x, w13, w2, _ = dl.make(tokens, hidden, inter, BF16)
    lib, cfg, y = _lib.lib(), config(hidden, inter), torch.empty_like(x)
    saved = room(lib.FlashMoeFfnSavedBytes(cfg, tokens))
    return [y], (x, w13, w2, saved), lambda: lib.FlashMoeFfnForward(cfg, x.data_ptr(), w13.data_ptr(), w2.data_ptr(), y.data_ptr(),
                                                                saved.data_ptr(), None, 0, tokens, stream())


def backward(tokens, hidden, inter):
    x, w13, w2, dy = dl.make(tokens, hidden, inter, BF16)
    lib, cfg = _lib.lib(), config(hidden, inter)
    saved, ws = room(lib.FlashMoeFfnSavedBytes(cfg, tokens)), room(lib.FlashMoeFfnWorkspaceBytes(cfg, tokens, 1))
    y, grads = torch.empty_like(x), [torch.empty_like(t) for t in (x, w13, w2)]
    assert lib.FlashMoeFfnForward(cfg, x.data_ptr(), w13.data_ptr(), w2.data_ptr(), y.data_ptr(), saved.data_ptr(), None, 0,
                                  tokens, stream()) == 0
    return grads, (x, w13, w2, dy, saved, ws), lambda: lib.FlashMoeFfnBackward(
        cfg, dy.data_ptr(), x.data_ptr(), w13.data_ptr(), w2.data_ptr(), saved.data_ptr(), *[t.data_ptr() for t in grads],
        ws.data_ptr(), ws.numel(), tokens, stream())


def product(m, n, k, gated=0, dtype=BF16):
    g = torch.Generator().manual_seed(3)
    a = mx4_quantize(torch.randn(m, k, generator=g).cuda())
    b = mx4_quantize(torch.randn(*((2, n, k) if gated else (n, k)), generator=g).cuda())
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    return [out], (a, b), lambda: _lib.lib().FlashMoeMx4Matmul(*a._pointers, *b._pointers, out.data_ptr(), {BF16: 0, FP32: 1}[dtype],
                                                              m, n, k, gated, stream())


def block_of_4_bits(tokens, hidden, inter):
    x, w13, w2, _ = dl.make(tokens, hidden, inter, BF16)
    q13, q2 = quantize_ffn_weights(w13, w2)
    lib, cfg, y = _lib.lib(), config(hidden, inter), torch.empty_like(x)
    ws = room(lib.FlashMoeMx4FfnWorkspaceBytes(cfg, tokens))
    return [y], (x, q13, q2, ws), lambda: lib.FlashMoeMx4FfnForward(cfg, x.data_ptr(), *q13._pointers, *q2._pointers, y.data_ptr(),
                                                                ws.data_ptr(), ws.numel(), tokens, stream())


# the streaming kernel with one CTA per tile (one k block) and with several, the pair kernel with one pair per tile and
# with several, every epilogue, several products in one launch
@pytest.mark.parametrize("make,size", [
    (forward, (4, 64, 64)), (forward, (4, 2048, 768)), (forward, (120, 4096, 1024)), (forward, (300, 256, 256)),
    (forward, (300, 2048, 128)), (training_forward, (40, 256, 256)), (training_forward, (300, 2048, 128)),
    (backward, (40, 256, 264)), (backward, (300, 2048, 128)), (backward, (1000, 1024, 1032)),
    (product, (3, 512, 256)), (product, (3, 512, 8192)), (product, (200, 133, 4096)), (product, (300, 264, 512)),
    (product, (300, 256, 16384)), (product, (5, 512, 4096, 1)), (product, (300, 512, 4096, 1)),
    (product, (5, 512, 4096, 1, FP32)), (product, (300, 512, 4096, 0, FP32)), (product, (300, 512, 4096, 1, FP32)),
    (block_of_4_bits, (20, 2048, 768)), (block_of_4_bits, (300, 320, 544))])
def test_every_wait_ends(monkeypatch, make, size):
    results, kept, call = make(*size)
    assert call() == 0
    torch.cuda.synchronize()
    want = [t.clone() for t in results]
    lib = _lib.lib()
    monkeypatch.setenv("FLASHMOE_TIMEOUT_MS", "30")
    lib.FlashMoeTestDenseStall(1)
    try:
        assert call() == 0
    finally:
        lib.FlashMoeTestDenseStall(0)
    torch.cuda.synchronize()  # the kernels returned, the context is alive
    assert dense_status() in (21, 22, 23, 24)
    assert call() != 0  # refused
    assert dense_status(reset=True) != 0 and dense_status() == 0
    monkeypatch.delenv("FLASHMOE_TIMEOUT_MS")
    for t in results:
        t.fill_(float("nan"))
    assert call() == 0
    torch.cuda.synchronize()
    assert dense_status() == 0 and all(torch.equal(a, b) for a, b in zip(results, want))


def test_quantisation_is_refused_after_an_error_too(monkeypatch):
    """It would take the result of the product that failed for numbers."""
    _, kept, call = product(3, 512, 256)
    x, q = torch.ones(4, 64, dtype=BF16, device="cuda"), kept[0]
    want = mx4_quantize(x).dequantize()
    monkeypatch.setenv("FLASHMOE_TIMEOUT_MS", "30")
    _lib.lib().FlashMoeTestDenseStall(1)
    try:
        assert call() == 0
    finally:
        _lib.lib().FlashMoeTestDenseStall(0)
    torch.cuda.synchronize()
    for refused in (lambda: mx4_quantize(x), q.dequantize, lambda: quantize_ffn_weights(x.repeat(32, 1), x.repeat(16, 1))):
        with pytest.raises(RuntimeError, match="999"):
            refused()
    assert dense_status(reset=True) != 0
    assert torch.equal(mx4_quantize(x).dequantize(), want)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_more_weight_rows_than_a_grid_has_blocks(dtype):
    n, k = 8388608, 32  # 65536 tiles of 128
    g = torch.Generator(device="cuda").manual_seed(7)
    a = mx4_quantize(torch.randn(3, k, generator=g, device="cuda"))
    b = mx4_quantize(torch.randn(n, k, generator=g, device="cuda"))
    y = mx4_matmul(a, b, dtype)
    want, e = dl.product(a.dequantize(FP32).double(), b.dequantize(FP32).double())
    dl.assert_within(y, want, dl.rounded(want, e, dtype))


def test_weight_gradients_beyond_32_bits():
    """[T, 2I] has 2.3e9 elements and only the last tokens have a gradient.  The products of the others are zeros, which a
    32-bit sum takes without an error, so the bound is that of the last tokens alone: one that grew with all of them would
    let zeros or a gradient of the other sign pass."""
    tokens, hidden, inter, last = 70000, 64, 16384, 300
    g = torch.Generator(device="cuda").manual_seed(13)
    r = lambda *s, std: torch.empty(*s, device="cuda").normal_(0, std, generator=g).to(BF16)  # noqa: E731
    x, w13, w2 = r(tokens, hidden, std=1.0), r(2 * inter, hidden, std=0.2), r(hidden, inter, std=inter ** -0.5)
    dy = torch.zeros(tokens, hidden, dtype=BF16, device="cuda")
    dy[-last:] = r(last, hidden, std=1.0)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    _, dw13, dw2 = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    want = dl.ffn_grads(x[-last:].detach(), w13.detach(), w2.detach(), dy[-last:])
    for name, got, (value, bound) in zip(("dw13", "dw2"), (dw13, dw2), want[1:]):
        dl.assert_within(got, value, bound, name)
        for wrong in (torch.zeros_like(got), -got, 3 * got):
            with pytest.raises(AssertionError):
                dl.assert_within(wrong, value, bound, name)


def test_gradient_of_tokens_that_are_one_row():
    # 50 equal rows of dx, added by torch in 32 bits and rounded once; zeros are far outside this bound
    x, w13, w2, _ = dl.make(1, 72, 136, FP16, seed=3)
    one = x.clone().requires_grad_()
    gated_ffn(one.expand(50, 72), w13, w2).backward(torch.ones(50, 72, dtype=FP16, device="cuda"))
    value, bound = dl.ffn_grads(x, w13, w2, torch.ones_like(x))[0]
    value, bound = 50 * value, dl.rounded(50 * value, 50 * bound + 50 * 2.0 ** -24 * 50 * value.abs(), FP16)
    dl.assert_within(one.grad, value, bound)
    with pytest.raises(AssertionError):
        dl.assert_within(torch.zeros_like(one.grad), value, bound)


@pytest.mark.parametrize("m", [16, 300])
@pytest.mark.parametrize("ea,eb", [(-120, 0), (-120, 118), (118, -120), (-60, -60), (60, 60), (118, 0)])
def test_products_of_far_apart_scales(m, ea, eb):
    g = torch.Generator().manual_seed(4)
    a = mx4_quantize((torch.randn(m, 512, generator=g) * 2.0 ** ea).cuda())
    b = mx4_quantize((torch.randn(264, 512, generator=g) * 2.0 ** eb).cuda())
    want, e = dl.product(a.dequantize(FP32).double(), b.dequantize(FP32).double())
    dl.assert_within(mx4_matmul(a, b, FP32), want, dl.rounded(want, e, FP32))


@pytest.mark.parametrize("tokens,hidden,inter", [(40, 256, 264), (300, 2048, 128), (777, 1000, 2744), (2000, 1024, 2048)])
def test_gradients_have_the_same_bits_each_time(tokens, hidden, inter):
    x, w13, w2, dy = dl.make(tokens, hidden, inter, BF16, seed=9)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    first = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(gated_ffn(*leaves), leaves, dy)))


def test_training_steps_of_several_threads():
    args = [dl.make(t, 512, 768, BF16, seed=t) for t in (4, 90, 200, 700)]

    def step(x, w13, w2, dy):
        leaves = [t.detach().requires_grad_() for t in (x, w13, w2)]
        y = gated_ffn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    want = [step(*a) for a in args]
    torch.cuda.synchronize()
    equal = []

    def work(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(15):
                got = step(*args[i])
                s.synchronize()
                equal.append(all(torch.equal(a, b) for a, b in zip(got, want[i])))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(args))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(equal) == 60 and all(equal) and dense_status() == 0


@pytest.mark.parametrize("tokens", [3, 300])
@pytest.mark.parametrize("what", ["forward", "training", "product"])
def test_the_first_call_of_a_process_inside_a_capture(what, tokens):
    program = f"""
import sys
sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}]
import torch, dense_testlib as dl, flash_distributed_moe_b200 as fm
x, w13, w2, dy = dl.make({tokens}, 256, 264, torch.bfloat16)
w = w13.float()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    if "{what}" == "forward":
        with torch.no_grad():
            y = fm.gated_ffn(x, w13, w2)
    elif "{what}" == "training":
        leaves = [t.requires_grad_() for t in (x, w13, w2)]
        y = fm.gated_ffn(*leaves)
        grads = torch.autograd.grad(y, leaves, dy)
    else:
        a, b = fm.mx4_quantize(x), fm.mx4_quantize(w)
        y = fm.mx4_matmul(a, b)
graph.replay()
torch.cuda.synchronize()
if "{what}" == "product":
    want, e = dl.product(dl.mx4(x), dl.mx4(w))
    dl.assert_within(y, want, dl.rounded(want, e, torch.bfloat16))
else:
    dl.assert_within(y.detach(), *dl.ffn(x.detach(), w13.detach(), w2.detach()))
if "{what}" == "training":
    for got, (value, bound) in zip(grads, dl.ffn_grads(x.detach(), w13.detach(), w2.detach(), dy)):
        dl.assert_within(got, value, bound)
assert fm.dense_status() == 0
"""
    out = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=120)
    assert out.returncode == 0, out.stderr[-2000:]
