"""GPU: 4-bit microscaled quantisation (exact) and products (within the bound of a 32-bit sum and one rounding)."""
import pytest
import torch

import dense_testlib as dl
from flash_distributed_moe_b200 import (Mx4Tensor, dense_status, gated_ffn, mx4_gated_matmul, mx4_matmul, mx4_quantize,
                                        quantize_ffn_weights)

pytestmark = pytest.mark.gpu
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = [BF16, FP16, FP32]


def values(*shape, dtype=BF16, seed=0):
    """Normal values whose rows differ in size by factors of up to a million (fp16: a thousand)."""
    g = torch.Generator().manual_seed(seed)
    spread = 3.5 if dtype == FP16 else 7.0
    size = torch.exp(spread * (2 * torch.rand(*shape[:-1], 1, generator=g) - 1))
    return (torch.randn(*shape, generator=g) * size).to(dtype).cuda()


def scale_of(q, row, block, batch=0):
    """The documented place of a scale."""
    rows, cols = q.shape[-2:]
    chunks = (cols + 255) // 256 * 2
    chunk = (batch * ((rows + 127) // 128) + row // 128) * chunks + block // 4
    return q.scales[chunk * 512 + row % 32 * 16 + row % 128 // 32 * 4 + block % 4].item()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 32), (1, 4096), (3, 96), (127, 256), (128, 288), (129, 512), (1000, 2080),
                                   (2, 40, 64), (3, 130, 320)])
def test_quantize(shape, dtype):
    x = values(*shape, dtype=dtype)
    q = mx4_quantize(x)
    assert q.shape == x.shape and q.values.shape == (*shape[:-1], shape[-1] // 2)
    want = dl.mx4(x)
    for out in TYPES:
        got = q.dequantize(out)
        assert got.dtype == out and torch.equal(got, want.to(out))


def test_the_grid_its_borders_and_the_layout():
    # a block with 6 in it has the scale 1: every half step of the grid, both signs, ties to the even code
    points = [0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6, 6.5, 7, 7.75, .2499, .2501, 2.4999, 2.5001, 4.999, 5.001]
    want = [0, 0, .5, 1, 1, 1, 1.5, 2, 2, 2, 3, 4, 4, 4, 6, 6, 6, 6, 0, .5, 2, 3, 4, 6]
    x = torch.tensor([points + [6.0] * 8, [-p for p in points] + [6.0] * 8], dtype=FP32, device="cuda")
    q = mx4_quantize(x)
    assert q.dequantize(FP32)[0, :24].tolist() == want and q.dequantize(FP32)[1, :24].tolist() == [-v for v in want]
    assert q.values[0, 1].item() == (1 | 2 << 4)  # 0.5 and 1: the even element in the low half
    rows = torch.arange(300)[:, None] % 90 - 45
    blocks = torch.arange(9).repeat_interleave(32)[None, :]
    big = torch.exp2((rows + blocks).double()).float().cuda()
    q = mx4_quantize(big)
    for r in (0, 1, 31, 32, 127, 128, 200, 299):
        for b in range(9):
            assert scale_of(q, r, b) == r % 90 - 45 + b - 2 + 127


def test_extremes():
    x = torch.zeros(8, 64, dtype=FP32, device="cuda")
    x[1, :32] = 3.4e38             # the largest scale
    x[2, 0] = 1e-45                # the smallest number there is
    x[3, 5] = 2.0 ** -126
    x[4, 40] = float("nan")
    x[5, 3] = float("-inf")
    x[6, 0], x[6, 1] = 1e30, 1e-30  # far below the block's scale
    x[7, 0], x[7, 1] = -0.0, 2.0 ** -127
    q = mx4_quantize(x)
    got, want = q.dequantize(FP32), dl.mx4(x).float()
    assert torch.equal(got.nan_to_num(nan=-1.0), want.nan_to_num(nan=-1.0))
    assert torch.isnan(got[4, 32:]).all() and torch.isnan(got[5, :32]).all()
    assert torch.isfinite(got[4, :32]).all() and torch.isfinite(got[5, 32:]).all()
    for dtype in (BF16, FP16):
        top = torch.full((1, 32), torch.finfo(dtype).max, dtype=dtype, device="cuda")
        low = torch.full((1, 32), torch.finfo(dtype).smallest_normal, dtype=dtype, device="cuda")
        for t in (top, low):
            assert torch.equal(mx4_quantize(t).dequantize(dtype), dl.mx4(t).to(dtype))


def test_strided_rows_and_padding():
    wide = values(50, 512)
    assert torch.equal(mx4_quantize(wide[::2, 64:320]).dequantize(), dl.mx4(wide[::2, 64:320]).to(BF16))
    batch = values(4, 33, 64)
    assert torch.equal(mx4_quantize(batch[1:, 1:]).dequantize(), dl.mx4(batch[1:, 1:]).to(BF16))
    q = mx4_quantize(values(5, 96))  # scales of rows and columns that do not exist are 0
    s = q.scales.view(2, 32, 4, 4).clone()
    s[0, :5, 0, :3] = 0
    assert q.scales.numel() == 1024 and not s.any()
    assert mx4_quantize(values(0, 64)).dequantize().shape == (0, 64)


# rows of the result around the tiles of 16, 128 and 256; columns ragged, fewer than a tile, of several; k of one
# block of 32, ragged in the stage of 256, of several stages
SIZES = [(1, 8, 32), (1, 4096, 12288), (3, 133, 96), (16, 128, 256), (17, 129, 288), (64, 1000, 2080), (100, 264, 512),
         (128, 512, 1024), (129, 128, 64), (256, 256, 256), (300, 520, 800), (513, 1544, 2080), (700, 77, 320), (1000, 8, 4096)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(m, n, k, dtype):
    a, b = mx4_quantize(values(m, k)), mx4_quantize(values(n, k, seed=1))
    y = mx4_matmul(a, b, dtype)
    want, e = dl.product(a.dequantize(FP32).double(), b.dequantize(FP32).double())
    if dtype == FP16:  # beyond fp16's range a result is infinite
        fits = want.abs() + e < 65000
        assert torch.isinf(y[want.abs() - e > 66000]).all()
        y, want, e = y[fits], want[fits], e[fits]
    dl.assert_within(y, want, dl.rounded(want, e, dtype))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_gated_product(m, n, k, dtype):
    x = torch.randn(m, k, generator=torch.Generator().manual_seed(2)).to(BF16).cuda()
    w = (torch.randn(2, n, k, generator=torch.Generator().manual_seed(3)) * 1.5 / k ** 0.5).to(BF16).cuda()
    a, b = mx4_quantize(x), mx4_quantize(w)
    h = mx4_gated_matmul(a, b, dtype)
    w64 = b.dequantize(FP32).double()
    want, e, _ = dl.gated(a.dequantize(FP32).double(), w64[0], w64[1])
    dl.assert_within(h, want, dl.rounded(want, e, dtype))
    assert torch.equal(h, mx4_gated_matmul(a, b, dtype))


@pytest.mark.parametrize("m", [20, 300])
def test_nan_blocks_reach_their_rows_only(m):
    x, w = values(m, 320), values(200, 320, seed=1)
    want = mx4_matmul(mx4_quantize(x), mx4_quantize(w))
    x[11, 33] = float("nan")
    w[150, 0] = float("inf")
    y = mx4_matmul(mx4_quantize(x), mx4_quantize(w))
    assert torch.isnan(y[11]).all() and torch.isnan(y[:, 150]).all()
    keep = torch.ones_like(y, dtype=torch.bool)
    keep[11], keep[:, 150] = False, False
    assert torch.equal(y[keep], want[keep])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,hidden,inter", [(1, 256, 96), (20, 2048, 768), (300, 320, 544)])
def test_block_with_4bit_weights(tokens, hidden, inter, dtype):
    # the operators as a serving program runs them together: the same bits as the calls one by one
    x, w13, w2, _ = dl.make(tokens, hidden, inter, dtype)
    q13, q2 = quantize_ffn_weights(w13, w2)
    y = gated_ffn(x.view(1, tokens, hidden), q13, q2)
    h = mx4_gated_matmul(mx4_quantize(x), q13, dtype)
    assert torch.equal(y[0], mx4_matmul(mx4_quantize(h), q2, dtype))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z = gated_ffn(x, q13, q2)
    x.copy_(x.flip(0))
    graph.replay()
    assert torch.equal(z, gated_ffn(x, q13, q2))


def test_another_stream():
    x, w = values(200, 512), mx4_quantize(values(256, 512, seed=1))
    want = mx4_matmul(mx4_quantize(x), w)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = mx4_matmul(mx4_quantize(x), w)
    s.synchronize()
    assert torch.equal(got, want)


def test_different_products_at_once():
    """On streams of their own: products that need from 32 columns of an SM's tensor memory to all of them."""
    calls = []
    for i, tokens in enumerate((1, 33, 64, 120, 300)):
        x = values(tokens, 512, seed=i)
        q, w, w13 = mx4_quantize(x), *(mx4_quantize(values(*s, 512, seed=9)) for s in ((520,), (2, 384)))
        dense = dl.make(tokens, 512, 768, BF16, seed=i)[:3]
        calls += [lambda q=q, w=w: mx4_matmul(q, w), lambda q=q, w13=w13: mx4_gated_matmul(q, w13), lambda d=dense: gated_ffn(*d)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in calls], [[] for _ in calls]
    for _ in range(8):
        for c, s, g in zip(calls, streams, got):
            with torch.cuda.stream(s):
                g.append(c())
    torch.cuda.synchronize()
    assert all(torch.equal(g, w) for gs, w in zip(got, want) for g in gs)
    assert dense_status() == 0


def test_refusals():
    x = values(4, 64)
    for bad in (x.double(), x[:, :40], x[0], x.cpu(), x.t().contiguous().t(), values(4, 65)[:, 1:], None, x.view(1, 1, 4, 64)):
        with pytest.raises(RuntimeError):
            mx4_quantize(bad)
    a = mx4_quantize(x)
    for args in ((a, mx4_quantize(values(4, 96))), (a, x), (x, a), (a, mx4_quantize(values(2, 4, 64))), (a, a, torch.int32)):
        with pytest.raises(RuntimeError):
            mx4_matmul(*args)
    for w in (a, mx4_quantize(values(3, 4, 64))):
        with pytest.raises(RuntimeError):
            mx4_gated_matmul(a, w)
    with pytest.raises(RuntimeError):
        a.dequantize(torch.float64)
    x, w13, w2, _ = dl.make(4, 64, 64, BF16)
    q13, q2 = quantize_ffn_weights(w13, w2)
    for args in ((x, q13, w2), (x, w13, q2), (x, q2, q13), (x.requires_grad_(), q13, q2), (x.detach()[:, :32], q13, q2)):
        with pytest.raises(RuntimeError):
            gated_ffn(*args)
    with pytest.raises(RuntimeError):
        quantize_ffn_weights(w13[:64], w2)
    assert isinstance(q13, Mx4Tensor)


def test_offsets_beyond_32_bits():
    rows, cols, last = 70000, 32768, 200  # 2.3e9 elements
    x = torch.empty(rows, cols, dtype=BF16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(5))
    q = mx4_quantize(x)
    small = mx4_quantize(x[-last:].clone())
    assert torch.equal(q.values[-last:], small.values)
    assert torch.equal(q.dequantize()[-last:], dl.mx4(x[-last:]).to(BF16))
    w = mx4_quantize(values(64, cols, seed=1))
    y, part = mx4_matmul(q, w), mx4_matmul(small, w)
    want, e = dl.product(small.dequantize(FP32).double(), w.dequantize(FP32).double())
    for got in (y[-last:], part):
        dl.assert_within(got, want, dl.rounded(want, e, BF16))
