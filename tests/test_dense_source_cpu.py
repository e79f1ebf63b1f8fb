"""What the kernels of the dense operators have to keep to and no run can show: read from their sources."""
import os
import re

import moe_testlib as tl

CSRC = os.path.join(tl.ROOT, "flash_distributed_moe_b200", "csrc")
KERNELS = ("dense_gemm.cuh", "dense_kernels.cu", "dense_launch.cuh", "mx4_kernels.cu", "ptx_cluster.cuh")


def source(name):
    """A source file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_no_read_only_loads_in_kernels_that_start_early():
    """Every launch may start while the launch before it still writes what it is going to read."""
    assert "programmaticStreamSerializationAllowed = 1" in source("dense_launch.cuh")
    for name in KERNELS:
        text = source(name)
        for word in ("__ldg", "ld.global.nc", "__restrict__", "__ldca", "__ldcs", "__ldlu"):
            assert word not in text, f"{name}: {word}"
    for load in re.findall(r'asm\s*(\w*)\("(ld\.global[^"]*)".*?;\n', source("ptx_cluster.cuh"), re.S):
        assert load[0] == "volatile", load


def test_lanes_that_issue_come_together_after_every_wait():
    """A lane left behind by a whole ring of stages would wait for a phase that is over; nothing but the source makes the
    lanes of a warp go on together.  So no role waits lane by lane, and no lane leaves a loop of waits before the others."""
    text = source("dense_gemm.cuh")
    waiter, kernels = text[:text.index("pack2(")], text[text.index("pack2("):]
    assert re.search(r"bool wait_together\([^)]*\) const \{\s*if \(__all_sync\([^;]*\)\) return true;\s*if \(ok\) ok = wait\([^)]*\);\s*__syncwarp\(\);\s*return ok;", waiter)
    assert re.search(r"bool wait_warp\([^)]*\) const \{\s*return __all_sync\(", waiter)
    calls = re.findall(r"wt\.(wait\w*|slow)\(", kernels)
    assert calls.count("wait_together") == 5 and set(calls) == {"wait_together", "wait_warp"}
    for call in re.finditer(r"(\S+) = wt\.wait_together\([^;]*, (\w+)\);", kernels):
        assert call.group(1) == call.group(2) == "ok"
    assert not re.search(r"for \([^;]*; *ok\b", kernels)


def test_a_ctas_shared_memory_outlives_the_stores_of_its_cluster():
    """A CTA whose wait ran out has not counted the partial sums that the others store into its shared memory.  It may not
    leave before they have; one that waited for all of them may."""
    text = source("dense_gemm.cuh")
    for kernel, until in (("stream_gemm(", r"if \(p\.split > 1 && abort_flag\) ptx::cluster_sync_relaxed\(\);\s*wt\.drain\(\);"),
                          ("pair_gemm(", r"wt\.drain\(\);\s*ptx::cluster_sync_relaxed\(\);")):
        body = text[text.index(kernel):]
        end = body[body.rindex("__syncthreads();", 0, re.search(r"ptx::tmem_dealloc\w*\(", body).start()):]
        assert re.match(r"__syncthreads\(\);\s*" + until, end), kernel
