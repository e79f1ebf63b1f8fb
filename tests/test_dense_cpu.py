"""Host side of the dense operators without a GPU: launch plans, workspace sizes and what is refused before any CUDA
call."""
import ctypes as C
import os
import subprocess

import pytest
import torch

import moe_testlib as tl
from flash_distributed_moe_b200 import (Mx4Tensor, _lib, build as build_mod, gated_ffn, mx4_matmul, mx4_quantize,
                                        quantize_ffn_weights)

INVALID = 1  # cudaErrorInvalidValue


@pytest.fixture(scope="module")
def lib():
    build_mod.build()
    return _lib.lib()


def _cfg(hidden, inter, dtype=0):
    return C.byref(_lib.FlashMoeFfnConfig(hidden, inter, dtype, (C.c_int32 * 5)()))


def test_launch_plans(tmp_path):
    exe = str(tmp_path / "dense_plan_test.bin")
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", exe, os.path.join(tl.ROOT, "tests", "cpp", "dense_plan_test.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout


def test_workspace_sizes(lib):
    assert lib.FlashMoeFfnWorkspaceBytes(_cfg(64, 72), 100, 0) == (100 * 72 * 2 + 255) // 256 * 256
    assert lib.FlashMoeFfnWorkspaceBytes(_cfg(64, 72), 0, 0) == 0
    assert lib.FlashMoeFfnWorkspaceBytes(_cfg(4096, 12288), 1 << 20, 1) == 4 * (1 << 20) * 12288  # beyond 32 bits
    assert lib.FlashMoeFfnSavedBytes(_cfg(4096, 12288), 1 << 20) == 8 * (1 << 20) * 12288
    assert lib.FlashMoeMx4ScaleBytes(1, 129, 288) == 2 * 4 * 512
    assert lib.FlashMoeMx4FfnWorkspaceBytes(_cfg(64, 96), 10) > 0
    assert lib.FlashMoeMx4FfnWorkspaceBytes(_cfg(64, 72), 10) == 0


@pytest.mark.parametrize("cfg", [(60, 64, 0), (64, 60, 0), (0, 64, 0), (64, -8, 0), (64, 64, 1), (64, 64, 7), (1 << 21, 64, 0)])
def test_unsupported_blocks(lib, cfg):
    assert lib.FlashMoeFfnWorkspaceBytes(_cfg(*cfg), 10, 0) == 0
    assert lib.FlashMoeFfnForward(_cfg(*cfg), *[None] * 6, 0, 10, None) == INVALID
    assert lib.FlashMoeFfnBackward(_cfg(*cfg), *[None] * 9, 0, 10, None) == INVALID


def test_null_misaligned_and_short_arguments(lib):
    ok = 4096  # never dereferenced: every call below is refused first
    good = dict(x=ok, w13=ok, w2=ok, y=ok, gu=None, ws=ok, nbytes=1 << 20, tokens=10)

    def call(**change):
        a = {**good, **change}
        return lib.FlashMoeFfnForward(_cfg(64, 64), a["x"], a["w13"], a["w2"], a["y"], a["gu"], a["ws"], a["nbytes"], a["tokens"], None)

    for name in ("x", "w13", "w2", "y", "ws"):
        assert call(**{name: None}) == INVALID and call(**{name: ok + 2}) == INVALID
    assert call(gu=ok + 8) == INVALID and call(nbytes=100) == INVALID and call(tokens=-1) == INVALID
    assert lib.FlashMoeFfnForward(None, ok, ok, ok, ok, None, ok, 1 << 20, 10, None) == INVALID
    assert call(tokens=0) == 0
    assert lib.FlashMoeFfnBackward(_cfg(64, 64), ok, ok, ok, ok, None, ok, ok, ok, ok, 1 << 20, 10, None) == INVALID
    assert lib.FlashMoeFfnBackward(_cfg(64, 64), ok, ok, ok, ok, ok, ok + 2, ok, ok, ok, 1 << 20, 10, None) == INVALID
    assert lib.FlashMoeMx4Quantize(ok, 0, 1, 4, 64, 0, 60, ok, ok, None) == INVALID   # rows not on 16 bytes
    assert lib.FlashMoeMx4Quantize(ok, 3, 1, 4, 64, 0, 64, ok, ok, None) == INVALID   # no such dtype
    assert lib.FlashMoeMx4Quantize(ok, 0, 1, 4, 40, 0, 40, ok, ok, None) == INVALID   # columns not a multiple of 32
    assert lib.FlashMoeMx4Quantize(ok, 0, 70000, 4, 64, 256, 64, ok, ok, None) == INVALID
    assert lib.FlashMoeMx4Quantize(None, 0, 1, 0, 64, 0, 64, None, None, None) == 0   # nothing to do
    assert lib.FlashMoeMx4Dequantize(ok, ok, 1, 4, 64, 5, ok, None) == INVALID
    assert lib.FlashMoeMx4Matmul(ok, ok, ok, ok, ok, 0, 4, 4, 40, 0, None) == INVALID
    assert lib.FlashMoeMx4Matmul(ok, ok, ok, ok, None, 0, 4, 4, 64, 0, None) == INVALID
    assert lib.FlashMoeMx4Matmul(ok, ok, ok, ok, ok + 4, 0, 4, 4, 64, 0, None) == INVALID
    assert lib.FlashMoeMx4Matmul(None, None, None, None, None, 0, 0, 4, 64, 0, None) == 0
    assert lib.FlashMoeMx4FfnForward(_cfg(64, 72), *[ok] * 7, 1 << 20, 10, None) == INVALID
    code = C.c_uint32(9)
    assert lib.FlashMoeDenseStatus(C.byref(code), 1) == 0 and code.value == 0


def test_cpu_tensors_are_refused():
    x, w13, w2 = (torch.zeros(*s, dtype=torch.bfloat16) for s in ((4, 64), (128, 64), (64, 64)))
    with pytest.raises(RuntimeError, match="CUDA"):
        gated_ffn(x, w13, w2)
    with pytest.raises(RuntimeError, match="CUDA"):
        mx4_quantize(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_ffn_weights(w13, w2)
    with pytest.raises(RuntimeError, match="Mx4Tensor"):
        mx4_matmul(x, x)
    q = Mx4Tensor(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8))
    assert q.shape == (4, 64)
    with pytest.raises(RuntimeError):
        gated_ffn(x, q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        mx4_matmul(q, q)
    with pytest.raises(RuntimeError, match="CUDA"):
        q.dequantize()


def test_4bit_tensors_are_checked_when_they_are_made():
    v, s = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(1024, dtype=torch.uint8)
    for values, scales in ((v.char(), s), (v, s.char()), (v, s[:512]), (v[:, ::2], s), (v[0], s), (v[:, :8], s), (None, s),
                           (v, torch.zeros(2048, dtype=torch.uint8)[::2])):
        with pytest.raises(RuntimeError):
            Mx4Tensor(values, scales)
