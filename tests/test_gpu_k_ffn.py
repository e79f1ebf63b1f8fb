"""GPU: the gated feed-forward block and its gradient against the formulas in 64 bits, within bounds that count every
rounding (dense_testlib), at the sizes where tiles, k blocks, clusters and the split of the k axis begin and end."""
import ctypes as C

import pytest
import torch

import dense_testlib as dl
from flash_distributed_moe_b200 import FlashFfnBlockWrapper, _lib, dense_status, gated_ffn

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


# tokens around the tiles of 16, 128 and 256; hidden and inter smaller than a tile, ragged, and of several tiles
SIZES = [(1, 8, 8), (1, 2048, 768), (2, 72, 136), (15, 256, 264), (16, 64, 128), (17, 1000, 328), (64, 136, 2048),
         (65, 512, 520), (127, 520, 72), (128, 640, 640), (129, 128, 128), (255, 200, 392), (256, 256, 256),
         (257, 264, 520), (333, 2048, 768), (700, 72, 1288), (1030, 1032, 24)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
def test_forward(tokens, hidden, inter, dtype):
    x, w13, w2, _ = dl.make(tokens, hidden, inter, dtype)
    y = gated_ffn(x, w13, w2)
    assert y.dtype == dtype
    dl.assert_within(y, *dl.ffn(x, w13, w2))
    assert torch.equal(y, gated_ffn(x, w13, w2))  # the same call, the same bits


@pytest.mark.parametrize("tokens", [97, 130, 147, 160, 161, 183, 192, 193])
def test_more_tokens_of_large_weights(tokens):
    x, w13, w2, _ = dl.make(tokens, 4120, 5480, BF16, seed=10)  # 129 MB
    y = gated_ffn(x, w13, w2)
    dl.assert_within(y, *dl.ffn(x, w13, w2))
    assert torch.equal(y, gated_ffn(x, w13, w2))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tokens,hidden,inter", SIZES)
def test_training_step(tokens, hidden, inter, dtype):
    x, w13, w2, dy = dl.make(tokens, hidden, inter, dtype, seed=1)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    y = gated_ffn(*leaves)
    dl.assert_within(y.detach(), *dl.ffn(x.detach(), w13.detach(), w2.detach()), "y")
    grads = torch.autograd.grad(y, leaves, dy)
    for name, g, (want, bound) in zip(("dx", "dw13", "dw2"), grads, dl.ffn_grads(x.detach(), w13.detach(), w2.detach(), dy)):
        assert g.dtype == dtype
        dl.assert_within(g, want, bound, name)


def test_gradient_against_differences():
    # <dy, F(v + e d) - F(v - e d)> / 2e in 64 bits, for a random direction d of each input; the central difference
    # itself is off by e^2 times the third derivative, far below the bound of the 16-bit gradient
    x, w13, w2, dy = dl.make(40, 136, 264, BF16, seed=2)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    grads = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    bounds = dl.ffn_grads(x.detach(), w13.detach(), w2.detach(), dy)
    base = [t.detach().double() for t in leaves]

    def f(args):
        g, u = (args[0] @ args[1].t()).chunk(2, dim=1)
        return ((torch.nn.functional.silu(g) * u) @ args[2].t() * dy.double()).sum()

    for i in range(3):
        d = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)).cuda()
        e = 1e-5
        up, down = (f(base[:i] + [base[i] + k * d] + base[i + 1:]) for k in (e, -e))
        want = ((up - down) / (2 * e)).item()
        got = (grads[i].double() * d).sum().item()
        assert abs(got - want) <= (bounds[i][1] * d.abs()).sum().item()


def test_no_tokens():
    x, w13, w2, dy = dl.make(0, 64, 72, BF16)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    y = gated_ffn(*leaves)
    assert y.shape == (0, 64)
    dx, dw13, dw2 = torch.autograd.grad(y, leaves, dy)
    assert dx.shape == (0, 64) and not dw13.any() and not dw2.any()
    with torch.no_grad():
        assert gated_ffn(x, w13, w2).shape == (0, 64)


def test_leading_dimensions_strides_and_alignment():
    x, w13, w2, _ = dl.make(30, 128, 64, BF16)
    want = gated_ffn(x, w13, w2)
    assert torch.equal(gated_ffn(x.view(2, 3, 5, 128), w13, w2), want.view(2, 3, 5, 128))
    assert torch.equal(gated_ffn(x[0], w13, w2), gated_ffn(x[:1], w13, w2)[0])
    wide = torch.zeros(30, 200, dtype=BF16, device="cuda")
    wide[:, 3:131] = x  # rows that start on odd addresses
    assert torch.equal(gated_ffn(wide[:, 3:131], w13, w2), want)
    assert torch.equal(gated_ffn(x.t().contiguous().t(), w13, w2), want)
    flat = torch.zeros(30 * 128 + 1, dtype=BF16, device="cuda")
    flat[1:] = x.flatten()  # contiguous, but not on 16 bytes
    assert torch.equal(gated_ffn(flat[1:].view(30, 128), w13, w2), want)


def test_some_gradients_only_and_a_broadcast_gradient():
    x, w13, w2, _ = dl.make(50, 72, 136, FP16, seed=3)
    ones = torch.ones_like(x)
    full = [t.clone().requires_grad_() for t in (x, w13, w2)]
    want = torch.autograd.grad(gated_ffn(*full), full, ones)
    gated_ffn(*full).sum().backward()  # the gradient of y is one number, expanded
    for t, g in zip(full, want):
        assert torch.equal(t.grad, g)
    for i in range(3):
        args = [x, w13, w2]
        args[i] = args[i].clone().requires_grad_()
        assert torch.equal(torch.autograd.grad(gated_ffn(*args), args[i], ones)[0], want[i])
    shared = x.clone().requires_grad_()  # the same leaf twice
    (gated_ffn(shared, w13, w2) + gated_ffn(shared, w13, w2)).backward(ones)
    assert torch.equal(shared.grad, want[0] + want[0])
    expanded = x[:1].clone().requires_grad_()
    gated_ffn(expanded.expand(50, 72), w13, w2).backward(ones)
    dl.assert_within(expanded.grad[0], 50 * want_row(x, w13, w2), 51 * bound_row(x, w13, w2) + 50 * dl.U[FP16] * 50 *
                     want_row(x, w13, w2).abs())


def want_row(x, w13, w2):
    return dl.ffn_grads(x[:1], w13, w2, torch.ones_like(x[:1]))[0][0][0]


def bound_row(x, w13, w2):
    return dl.ffn_grads(x[:1], w13, w2, torch.ones_like(x[:1]))[0][1][0]


@pytest.mark.parametrize("tokens", [40, 300])
def test_rows_do_not_touch_each_other(tokens):
    # a NaN or an infinity in one token stays there; other tokens keep their bits
    x, w13, w2, _ = dl.make(tokens, 200, 264, BF16, seed=4)
    want = gated_ffn(x, w13, w2)
    bad = x.clone()
    bad[7, 3], bad[tokens - 1, 0] = float("nan"), float("inf")
    y = gated_ffn(bad, w13, w2)
    keep = torch.ones(tokens, dtype=torch.bool, device="cuda")
    keep[7] = keep[tokens - 1] = False
    assert torch.equal(y[keep], want[keep])
    assert torch.isnan(y[7]).all() and not torch.isfinite(y[tokens - 1]).all()


def test_large_gate_values():
    # gates of +-200: the sigmoid is 0 or 1 in 32 bits, nothing overflows
    x, w13, w2, dy = dl.make(33, 64, 64, BF16, seed=5)
    w13[:64] *= 100
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    y = gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    assert all(torch.isfinite(t).all() for t in (y, *grads))


@pytest.mark.parametrize("tokens", [5, 200])
def test_memory_around_the_results_is_left_alone(tokens):
    # through the C ABI, with the results inside larger buffers
    hidden, inter = 200, 136
    x, w13, w2, dy = dl.make(tokens, hidden, inter, BF16, seed=6)
    lib, cfg = _lib.lib(), C.byref(_lib.FlashMoeFfnConfig(hidden, inter, 0, (C.c_int32 * 5)()))
    pad = 4096
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)

    def framed(*shape):
        n = torch.Size(shape).numel()
        buf = torch.full((n + 2 * pad,), 7.0, dtype=BF16, device="cuda")
        return buf, buf[pad:pad + n].view(*shape)

    ybuf, y = framed(tokens, hidden)
    gbuf, gu = framed(lib.FlashMoeFfnSavedBytes(cfg, tokens) // 2)
    dbuf = [framed(*t.shape) for t in (x, w13, w2)]
    sizes = [lib.FlashMoeFfnWorkspaceBytes(cfg, tokens, b) for b in (0, 1)]
    wbuf = [framed(s // 2) for s in sizes]
    for keep in (None, gu.data_ptr()):
        assert lib.FlashMoeFfnForward(cfg, x.data_ptr(), w13.data_ptr(), w2.data_ptr(), y.data_ptr(), keep,
                                      wbuf[0][1].data_ptr(), sizes[0], tokens, stream) == 0
        dl.assert_within(y, *dl.ffn(x, w13, w2))
    assert lib.FlashMoeFfnBackward(cfg, dy.data_ptr(), x.data_ptr(), w13.data_ptr(), w2.data_ptr(), gu.data_ptr(),
                                   *[t.data_ptr() for _, t in dbuf], wbuf[1][1].data_ptr(), sizes[1], tokens, stream) == 0
    for (_, got), (want, bound) in zip(dbuf, dl.ffn_grads(x, w13, w2, dy)):
        dl.assert_within(got, want, bound)
    for buf in (ybuf, gbuf, *[b for b, _ in dbuf], *[b for b, _ in wbuf]):
        assert (buf[:pad] == 7).all() and (buf[-pad:] == 7).all()


def test_result_in_place_of_the_tokens():
    hidden, inter = 256, 136
    for tokens in (9, 300):
        x, w13, w2, _ = dl.make(tokens, hidden, inter, BF16, seed=7)
        want = gated_ffn(x, w13, w2)
        lib, cfg = _lib.lib(), C.byref(_lib.FlashMoeFfnConfig(hidden, inter, 0, (C.c_int32 * 5)()))
        ws = torch.empty(lib.FlashMoeFfnWorkspaceBytes(cfg, tokens, 0), dtype=torch.uint8, device="cuda")
        assert lib.FlashMoeFfnForward(cfg, x.data_ptr(), w13.data_ptr(), w2.data_ptr(), x.data_ptr(), None, ws.data_ptr(),
                                      ws.numel(), tokens, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
        assert torch.equal(x, want)


def test_two_streams_at_once():
    args = [dl.make(t, 512, 768, BF16, seed=t)[:3] for t in (4, 200)]
    want = [gated_ffn(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(gated_ffn(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.parametrize("tokens", [3, 200])
def test_captured_and_replayed(tokens):
    x, w13, w2, dy = dl.make(tokens, 256, 264, BF16, seed=8)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]

    def step():
        y = gated_ffn(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    outs = []
    for g in graphs:  # two graphs that are replayed one after the other and together
        with torch.cuda.graph(g):
            outs.append(step())
    with torch.cuda.graph(serving := torch.cuda.CUDAGraph()), torch.no_grad():
        served = gated_ffn(*leaves)
    for seed in (9, 10):
        with torch.no_grad():
            x.copy_(dl.make(tokens, 256, 264, BF16, seed=seed)[0])
        for g in (*graphs, serving):
            g.replay()
        want = step()
        with torch.no_grad():
            assert torch.equal(served, gated_ffn(*leaves))
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_wrapper_runs_a_dense_block():
    class Mlp(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.gate_up_proj = torch.nn.Linear(256, 2 * 96, bias=False, dtype=BF16, device="cuda")
            self.down_proj = torch.nn.Linear(96, 256, bias=False, dtype=BF16, device="cuda")

    m = Mlp()
    x = dl.make(20, 256, 96, BF16)[0]
    w13, w2 = m.gate_up_proj.weight.detach(), m.down_proj.weight.detach()
    y = FlashFfnBlockWrapper(m)(x)
    dl.assert_within(y.detach(), *dl.ffn(x, w13, w2))
    y.sum().backward()
    assert m.gate_up_proj.weight.grad is not None and m.down_proj.weight.grad is not None
    with torch.no_grad():
        assert FlashFfnBlockWrapper(m, fourBit=True)(x).shape == y.shape
    m.down_proj.bias = torch.nn.Parameter(torch.zeros(256, dtype=BF16, device="cuda"))
    with pytest.raises(RuntimeError):
        FlashFfnBlockWrapper(m)


@pytest.mark.parametrize("hidden,inter", [(256, 256), (2048, 128)])  # the second with a shared k axis
def test_a_wait_that_runs_out(monkeypatch, hidden, inter):
    x, w13, w2, _ = dl.make(300, hidden, inter, BF16)
    want = gated_ffn(x, w13, w2)
    torch.cuda.synchronize()
    monkeypatch.setenv("FLASHMOE_TIMEOUT_MS", "50")
    lib, cfg = _lib.lib(), C.byref(_lib.FlashMoeFfnConfig(hidden, inter, 0, (C.c_int32 * 5)()))
    ws = torch.empty(lib.FlashMoeFfnWorkspaceBytes(cfg, 300, 0), dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    assert lib.FlashMoeTestFfnStall(cfg, x.data_ptr(), w13.data_ptr(), w2.data_ptr(), y.data_ptr(), ws.data_ptr(), ws.numel(),
                                    300, C.c_void_p(torch.cuda.current_stream().cuda_stream)) == 0
    torch.cuda.synchronize()  # the kernel returned, the context is alive
    assert dense_status() in (22, 24)
    with pytest.raises(RuntimeError):
        gated_ffn(x, w13, w2)
    assert dense_status(reset=True) in (22, 24) and dense_status() == 0
    monkeypatch.delenv("FLASHMOE_TIMEOUT_MS")
    assert torch.equal(gated_ffn(x, w13, w2), want)


def test_refusals():
    x, w13, w2, _ = dl.make(4, 64, 64, BF16)
    bad = [(x.float(), w13, w2), (x, w13.half(), w2), (x, w13, w2.float()), (x.cpu(), w13, w2), (x, w13.cpu(), w2),
           (x[:, :32], w13, w2), (x, w13[:64], w2), (x, w13, w2[:, :32]), (x, w13.t().contiguous().t(), w2),
           (x, w13, None), (None, w13, w2), dl.make(4, 60, 64, BF16)[:3], dl.make(4, 64, 60, BF16)[:3]]
    for args in bad:
        with pytest.raises(RuntimeError):
            gated_ffn(*args)
    flat = torch.zeros(2 * 64 * 64 + 1, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError):
        gated_ffn(x, flat[1:].view(128, 64), w2)
    y = gated_ffn(x.requires_grad_(), w13, w2)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError):  # no second derivative
        dx.sum().backward()


def test_a_nan_token_reaches_the_gradients():
    x, w13, w2, dy = dl.make(20, 64, 72, BF16, seed=11)
    x[5, 7] = float("nan")
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    dx, dw13, dw2 = torch.autograd.grad(gated_ffn(*leaves), leaves, dy)
    keep = torch.arange(20, device="cuda") != 5
    assert torch.isnan(dx[5]).all() and torch.isfinite(dx[keep]).all()
    assert torch.isnan(dw13).all() and torch.isnan(dw2).all()


def test_offsets_beyond_32_bits():
    # [T, 2I] has 2.3e9 elements: the last tokens' results, and the weights' gradients from those tokens alone
    tokens, hidden, inter, last = 70000, 64, 16384, 300
    g = torch.Generator(device="cuda").manual_seed(12)
    r = lambda *s, std: torch.empty(*s, device="cuda").normal_(0, std, generator=g).to(BF16)  # noqa: E731
    x, w13, w2 = r(tokens, hidden, std=1.0), r(2 * inter, hidden, std=0.2), r(hidden, inter, std=inter ** -0.5)
    dy = torch.zeros(tokens, hidden, dtype=BF16, device="cuda")
    dy[-last:] = r(last, hidden, std=1.0)
    leaves = [t.requires_grad_() for t in (x, w13, w2)]
    y = gated_ffn(*leaves)
    grads = torch.autograd.grad(y, leaves, dy)
    tail = [t.detach() for t in (x[-last:], w13, w2)]
    dl.assert_within(y[-last:].detach(), *dl.ffn(*tail))
    want = dl.ffn_grads(*tail, dy[-last:])
    assert not grads[0][:-last].any()
    dl.assert_within(grads[0][-last:], *want[0])
    for got, (value, bound) in zip(grads[1:], want[1:]):
        # the zeros of the other tokens add nothing, but the sums have more terms
        dl.assert_within(got, value, bound * (tokens / last))
