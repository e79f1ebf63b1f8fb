"""The dense operators' Python and C entries without a GPU: what a call must not do silently."""
import copy
import ctypes as C
import io
import os
import pickle
import subprocess

import pytest
import torch

import moe_testlib as tl
from flash_distributed_moe_b200 import (FlashFfnBlockWrapper, Mx4Tensor, gated_ffn, mx4_gated_matmul, mx4_matmul,
                                        mx4_quantize, quantize_ffn_weights, _lib, build as build_mod)


def matrix(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    bytes_of = lambda *s: torch.randint(0, 254, s, dtype=torch.uint8, generator=g)  # noqa: E731
    batch, rows, cols = shape if len(shape) == 3 else (1, *shape)
    return Mx4Tensor(bytes_of(*shape[:-1], cols // 2), bytes_of(batch * -(-rows // 128) * -(-cols // 256) * 1024))


def split_matrix(*shape):
    """As mx4_quantize makes them: values and scales in one buffer."""
    q = matrix(*shape)
    buffer = torch.cat([q.values.flatten(), q.scales])
    return Mx4Tensor._of_buffer(buffer, q.shape, (buffer.data_ptr(), buffer.data_ptr() + q.values.numel()))


def through_torch_save(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


@pytest.mark.parametrize("make", [matrix, split_matrix])
@pytest.mark.parametrize("shape", [(4, 64), (2, 130, 288)])
@pytest.mark.parametrize("again", [copy.deepcopy, copy.copy, lambda q: pickle.loads(pickle.dumps(q)), through_torch_save,
                                   lambda q: copy.deepcopy({"w": [q]})["w"][0]])
def test_a_copied_or_stored_matrix_has_its_own_addresses(make, shape, again):
    """The kernels take addresses: those of a copy are not the original's, which may be gone, nor another process's."""
    q = make(*shape)
    values, scales = q.values.clone(), q.scales.clone()
    r = again(q)
    if again is not copy.copy:
        assert r.values.data_ptr() != q.values.data_ptr() and r.scales.data_ptr() != q.scales.data_ptr()
        q.values.zero_(), q.scales.zero_()
    assert r.shape == q.shape and r.device == q.device
    assert torch.equal(r.values, values) and torch.equal(r.scales, scales)
    assert r._pointers == (r.values.data_ptr(), r.scales.data_ptr()) and r._pointers[0] % 16 == r._pointers[1] % 16 == 0


class Calls(list):
    """The C entries that were called, in place of running them."""

    def run(self, device, name, *args):
        self.append(name)


class OnGpu(torch.Tensor):
    """A tensor of the CPU that says it lies on the GPU."""
    is_cuda = True


@pytest.fixture
def calls(monkeypatch):
    """The Python side with C entries that do nothing."""
    from flash_distributed_moe_b200 import _lib
    c = Calls()
    monkeypatch.setattr(_lib, "run", c.run)
    return c


def on_gpu(t):
    return t.as_subclass(OnGpu)


def block(tokens=4, hidden=64, inter=64):
    g = torch.Generator().manual_seed(1)
    return [on_gpu(torch.randn(*s, generator=g).to(torch.bfloat16)) for s in ((tokens, hidden), (2 * inter, hidden), (hidden, inter))]


def test_forward_mode_derivatives_are_refused(calls):
    """Without a tangent the result would stand for a derivative of zero."""
    fw = torch.autograd.forward_ad
    args = block()
    assert gated_ffn(*args).shape == (4, 64) and calls == ["FlashMoeFfnForward"]
    del calls[:]
    with fw.dual_level():
        gated_ffn(*args)  # no dual tensor among them
        for i in range(3):
            dual = list(args)
            dual[i] = fw.make_dual(args[i], torch.ones_like(args[i]))
            for call in (lambda: gated_ffn(*dual), lambda: mx4_quantize(dual[i])):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        with pytest.raises(RuntimeError, match="forward-mode"):
            gated_ffn(fw.make_dual(args[0], torch.ones_like(args[0])), matrix(2, 64, 64), matrix(64, 64))
        with pytest.raises(RuntimeError, match="forward-mode"):
            quantize_ffn_weights(args[1], fw.make_dual(args[2], torch.ones_like(args[2])))
    assert calls == ["FlashMoeFfnForward", "FlashMoeMx4Quantize"]  # the weights of the last call that are no dual tensor


def recorders():
    from torch.fx.experimental.proxy_tensor import make_fx
    return {"trace": lambda f, x: torch.jit.trace(f, x, check_trace=False), "make_fx": lambda f, x: make_fx(f)(x),
            "make_fx symbolic": lambda f, x: make_fx(f, tracing_mode="symbolic")(x), "export": lambda f, x: torch.export.export(Call(f), (x,))}


class Call(torch.nn.Module):
    def __init__(self, f):
        super().__init__()
        self.forward = f


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("recorder", sorted(recorders()))
def test_recorders_of_operators_are_refused(calls, monkeypatch, recorder):
    """They would record the allocation of the result and not the call that fills it."""
    from flash_distributed_moe_b200 import flashFfn
    monkeypatch.setattr(flashFfn, "_check", lambda t, name: None)  # recorders' own tensors are not OnGpu
    x, w13, w2 = (t.as_subclass(torch.Tensor) for t in block())
    q, q13 = matrix(64, 64), matrix(2, 64, 64)
    q.device = q13.device = torch.device("cuda", 0)

    def through(f):
        with pytest.raises(Exception, match="cannot be recorded|FakeTensor|Unsupported|data_ptr|data pointer|not supported"):
            recorders()[recorder](f, x)

    through(lambda a: gated_ffn(a, w13, w2))
    through(lambda a: gated_ffn(a.clone().requires_grad_(), w13, w2))
    if recorder in ("trace", "make_fx"):
        through(lambda a: mx4_quantize(on_gpu(a)).values)
        monkeypatch.setattr(torch, "empty", lambda *s, **k: torch.zeros(*s, dtype=k["dtype"]))
        through(lambda a: a + q.dequantize())
        through(lambda a: a + mx4_matmul(q, q))
        through(lambda a: a + mx4_gated_matmul(q, q13))
    assert not calls


@pytest.mark.filterwarnings("ignore")
def test_compiled_programs_make_the_call(calls, monkeypatch):
    from flash_distributed_moe_b200 import flashFfn
    monkeypatch.setattr(flashFfn, "_check", lambda t, name: None)
    x, w13, w2 = (t.as_subclass(torch.Tensor) for t in block())
    for grad in (False, True):
        f = torch.compile(lambda a: gated_ffn(2 * a, w13, w2) + 1, backend="eager")
        assert f(x.clone().requires_grad_(grad)).requires_grad == grad
    assert calls == ["FlashMoeFfnForward"] * 2


def test_products_do_not_drop_the_gradient_of_their_activations(calls, monkeypatch):
    """As gated_ffn does on 4-bit weights: what needs a gradient and has none is refused.  Weights are constants."""
    monkeypatch.setattr(torch, "empty", lambda *s, **k: torch.zeros(*s, dtype=k["dtype"]))
    x, w = (block()[i].clone() for i in (0, 2))

    def quantize(t):
        q = mx4_quantize(t)
        q.device = torch.device("cuda", 0)
        return q

    w13 = quantize(w.repeat(2, 1, 1))
    leaf, param = x.clone().requires_grad_(), w.clone().requires_grad_()
    for a, needs in ((x, False), (leaf, True), (2 * leaf, True), (leaf.detach(), False)):
        for call in (lambda q: mx4_matmul(q, quantize(w)), lambda q: mx4_matmul(q, quantize(param)), lambda q: mx4_gated_matmul(q, w13)):
            q = quantize(a)
            if needs:
                with pytest.raises(RuntimeError, match="no gradient"):
                    call(q)
            else:
                assert not call(q).requires_grad
            with torch.no_grad():
                assert not call(q).requires_grad and not call(quantize(a)).requires_grad
    with torch.no_grad():
        q = quantize(leaf)
    assert not mx4_matmul(q, quantize(w)).requires_grad  # cut off when it was quantised
    assert not quantize(leaf).dequantize().requires_grad  # a value like any other
    with pytest.raises(RuntimeError, match="no gradient"):
        mx4_matmul(copy.copy(quantize(leaf)), quantize(w))


class Mlp(torch.nn.Module):
    def __init__(self, act=None, **more):
        super().__init__()
        self.gate_up_proj = torch.nn.Linear(64, 2 * 32, bias=False)
        self.down_proj = torch.nn.Linear(32, 64, bias=False)
        if act is not None:
            self.act_fn = act
        for name, value in more.items():
            setattr(self, name, value)


class SiluAndMul(torch.nn.Module):
    pass


class GeluAndMul(torch.nn.Module):
    pass


def with_attributes(mlp, where, **attributes):
    for name, value in attributes.items():
        setattr(getattr(mlp, where), name, value)
    return mlp


def test_the_wrapper_takes_blocks_that_are_what_it_computes():
    for mlp in (Mlp(), Mlp(torch.nn.SiLU()), Mlp(SiluAndMul()), Mlp(torch.nn.functional.silu), Mlp(hidden_act="silu"),
                Mlp(dropout=torch.nn.Dropout(0.0)), Mlp(expert_gate=None), Mlp(torch.nn.Identity(), hidden_act="silu"),
                with_attributes(Mlp(), "down_proj", tp_size=1, reduce_results=True),
                with_attributes(Mlp(), "down_proj", tp_size=2, reduce_results=False)):
        assert FlashFfnBlockWrapper(mlp).mlpModule is mlp


def test_the_wrapper_refuses_blocks_that_compute_more():
    """Its forward replaces the module's: a sum over ranks, a factor or another activation would be left out."""
    for mlp in (Mlp(torch.nn.GELU()), Mlp(GeluAndMul()), Mlp(torch.nn.functional.gelu), Mlp(torch.tanh), Mlp(hidden_act="gelu"),
                Mlp(activation_fn=torch.nn.functional.gelu), Mlp(expert_gate=torch.nn.Linear(64, 1)),
                Mlp(scale=torch.nn.Parameter(torch.ones(64))), Mlp(norm=torch.nn.LayerNorm(64)), Mlp(dropout=torch.nn.Dropout(0.1)),
                with_attributes(Mlp(), "down_proj", tp_size=2, reduce_results=True), with_attributes(Mlp(), "down_proj", tp_size=4),
                with_attributes(Mlp(), "gate_up_proj", tp_size=2, gather_output=True),
                with_attributes(Mlp(), "down_proj", bias=torch.nn.Parameter(torch.zeros(64)))):
        for four_bit in (False, True):
            with pytest.raises(RuntimeError):
                FlashFfnBlockWrapper(mlp, fourBit=four_bit)


def test_every_accepted_product_has_a_grid_that_can_be_launched(tmp_path):
    exe = str(tmp_path / "dense_limits_test.bin")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", exe, os.path.join(tl.ROOT, "tests", "cpp", "dense_limits_test.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


@pytest.mark.parametrize("m,n,dtype", [(1, 8388484, 0), (1, 8388482, 1), (8388481, 12, 0), (1 << 30, 1, 2), (1 << 30, 2, 1)])
def test_products_without_a_grid_are_refused(m, n, dtype):
    build_mod.build()
    for gated in (0, 1):
        assert _lib.lib().FlashMoeMx4Matmul(*[i << 45 for i in range(1, 6)], dtype, m, n, 32, gated, None) == 1  # cudaErrorInvalidValue


def overlaps(read, written, sizes, but=()):
    """Addresses far apart, but for one written range that begins with, ends in or lies within another one."""
    base = {name: (i + 1) << 32 for i, name in enumerate([*read, *written])}
    for w in written:
        for other in base:
            if other == w or (w, other) in but or (other, w) in but:
                continue
            for at in {base[other], base[other] + sizes[other] - 16, max(base[other] - sizes[w] + 16, 16)}:
                yield {**base, w: at}


def test_results_on_other_memory_of_the_call_are_refused():
    """Launches of a call overlap: dx in the place of x would be read by the product for dw13 in parts."""
    build_mod.build()
    lib, T, H, I, invalid = _lib.lib(), 10, 64, 96, 1
    cfg = C.byref(_lib.FlashMoeFfnConfig(H, I, 0, (C.c_int32 * 5)()))
    part = -(-T * I * 2 // 256) * 256
    size = dict(x=T * H * 2, dy=T * H * 2, y=T * H * 2, dx=T * H * 2, w13=4 * I * H, dw13=4 * I * H, w2=2 * I * H, dw2=2 * I * H,
                saved=-(-T * I * 4 // 256) * 256 + 2 * part)
    for ws in ("saved", "workspace"):
        for a in overlaps(("x", "w13", "w2"), ("y", ws), {**size, "workspace": T * I * 2}, but={("y", "x")}):
            assert lib.FlashMoeFfnForward(cfg, a["x"], a["w13"], a["w2"], a["y"], a.get("saved"), a.get("workspace"), 1 << 20, T,
                                          None) == invalid, a
    for a in overlaps(("dy", "x", "w13", "w2", "saved"), ("dx", "dw13", "dw2", "workspace"), {**size, "workspace": T * I * 4}):
        assert lib.FlashMoeFfnBackward(cfg, *[a[n] for n in ("dy", "x", "w13", "w2", "saved", "dx", "dw13", "dw2", "workspace")],
                                       1 << 20, T, None) == invalid, a
    scales = lambda batch, rows, cols: lib.FlashMoeMx4ScaleBytes(batch, rows, cols)  # noqa: E731
    for a in overlaps(("x",), ("values", "scales"), dict(x=(T - 1) * 80 * 2 + H * 2, values=T * H // 2, scales=scales(1, T, H))):
        assert lib.FlashMoeMx4Quantize(a["x"], 0, 1, T, H, 0, 80, a["values"], a["scales"], None) == invalid, a
    for a in overlaps(("values", "scales"), ("out",), dict(out=T * H * 4, values=T * H // 2, scales=scales(1, T, H))):
        assert lib.FlashMoeMx4Dequantize(a["values"], a["scales"], 1, T, H, 1, a["out"], None) == invalid, a
    for gated in (0, 1):
        names, b = ("av", "as", "bv", "bs"), 1 + gated
        for a in overlaps(names, ("out",), dict(av=T * H // 2, bv=b * I * H // 2, out=T * I * 4, **{"as": scales(1, T, H)}, bs=scales(b, I, H))):
            assert lib.FlashMoeMx4Matmul(*[a[n] for n in names], a["out"], 1, T, I, H, gated, None) == invalid, a
    names = ("x", "v13", "s13", "v2", "s2")
    total = lib.FlashMoeMx4FfnWorkspaceBytes(cfg, T)
    for a in overlaps(names, ("y", "ws"), dict(x=T * H * 2, y=T * H * 2, v13=I * H, v2=I * H // 2, s13=scales(2, I, H), s2=scales(1, H, I),
                                               ws=total), but={("y", "x")}):
        assert lib.FlashMoeMx4FfnForward(cfg, *[a[n] for n in names], a["y"], a["ws"], total, T, None) == invalid, a
