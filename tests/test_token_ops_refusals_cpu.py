"""More calls that the per-token operators refuse, all before any CUDA call."""
import pytest
import torch

import tritonblas_b200 as tb


def test_topk_is_a_whole_number():
    for bad in (2.5, 2.0, "2", None):
        with pytest.raises(TypeError):
            tb.moe_route(torch.randn(4, 8), bad)


def test_outputs_that_overlap_themselves():
    bf, z = torch.bfloat16, torch.zeros
    case = z(4, 64, dtype=bf), z(40, 64, dtype=bf).T, z(3, 8, 64, dtype=bf), z(3, 40, 8, dtype=bf), z(4, dtype=torch.int32)
    flat = z(1000, dtype=bf)
    for bad in (z(1, 40, dtype=bf).expand(4, 40), z(4, 1, dtype=bf).expand(4, 40), flat.as_strided((4, 40), (39, 1)), flat.as_strided((4, 40), (1, 3))):
        with pytest.raises(ValueError, match="overlap itself"):
            tb.lora_matmul(*case, out=bad)
    for good in (z(4, 40, dtype=bf), z(40, 4, dtype=bf).T, z(8, 80, dtype=bf)[::2, ::2], flat.as_strided((4, 40), (40, 1)), flat.as_strided((4, 40), (1, 4)), flat.as_strided((4, 40), (3, 7)),
                 z(1, 40, dtype=bf).expand(1, 40)):
        x, w, a, b, ids = case
        with pytest.raises(RuntimeError, match="CUDA"):         # nothing to say against it but where it is
            tb.lora_matmul(x[:good.shape[0]], w, a, b, ids[:good.shape[0]], out=good)
