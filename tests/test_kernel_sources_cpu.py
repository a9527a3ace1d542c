"""Rules of the kernels' sources that no run shows: breaking them is undefined behaviour that a compiler may let pass."""
import glob
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tritonblas_b200", "csrc")


def _statements(path):
    text = re.sub(r"//[^\n]*", "", open(path).read())
    return [" ".join(s.split()) for s in re.split(r"[;{}]", text) if s.strip()]


def test_cluster_barriers_are_reached_by_whole_warps():
    """barrier.cluster.arrive is .aligned: every lane of a warp executes it together. A warp or block barrier right before it says so."""
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        st = _statements(path)
        for i, s in enumerate(st):
            if s == "cluster_arrive()":
                found += 1
                before = [q for q in st[:i] if not q.startswith("if ")][-1]
                assert before in ("__syncwarp()", "__syncthreads()"), (os.path.basename(path), before)
    assert found >= 3


def test_the_next_kernel_starts_after_tensor_memory_is_taken():
    """Kernels of this library take tensor memory while they wait for the kernel before them. One that let the next kernel start
    ahead of its own request could find the columns it needs held by blocks that wait for it."""
    found = 0
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for body in text.split("__global__")[1:]:
            if "tmem_alloc<" in body and "griddep_launch_dependents()" in body:
                found += 1
                assert body.index("tmem_alloc<") < body.index("griddep_launch_dependents()"), os.path.basename(path)
    assert found >= 4
