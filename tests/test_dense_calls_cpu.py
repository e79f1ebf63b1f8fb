"""The dense operators' Python and C entries without a GPU: what a call must not do silently."""
import copy
import io
import pickle

import pytest
import torch

import moe_testlib  # noqa: F401  (sets sys.path)
from flash_distributed_moe_b200 import Mx4Tensor, gated_ffn, mx4_quantize, quantize_ffn_weights


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
