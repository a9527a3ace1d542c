"""More calls that the per-token operators refuse, all before any CUDA call."""
import pytest
import torch

import tritonblas_b200 as tb


def test_topk_is_a_whole_number():
    for bad in (2.5, 2.0, "2", None):
        with pytest.raises(TypeError):
            tb.moe_route(torch.randn(4, 8), bad)
