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


def test_the_adapters_projection_takes_tensor_memory_between_wait_and_launch():
    """A block that holds tensor memory while it waits for another kernel could keep a block of that kernel from getting its own."""
    text = open(os.path.join(CSRC, "lora.cu")).read()
    body = text[text.index("lora_project_tc_kernel("):]
    assert body.index("griddep_wait()") < body.index("tmem_alloc<1>") < body.index("griddep_launch_dependents()")
