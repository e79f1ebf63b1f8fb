"""The dense operators' Python and C entries without a GPU: what a call must not do silently."""
import copy
import io
import pickle

import pytest
import torch

import moe_testlib  # noqa: F401  (sets sys.path)
from flash_distributed_moe_b200 import Mx4Tensor


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
