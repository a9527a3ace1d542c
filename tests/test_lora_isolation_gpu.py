"""A request's adapter is its own affair: infinities and NaN in one adapter's lora_b, a server's other user's, say, change no row
without that adapter. Bounds as in test_lora_gpu; an element that is formed again sums k + rank terms in another order, which the
bound covers."""
import pytest
import torch

import tritonblas_b200 as tb
from tests.test_lora_gpu import make, reference

pytestmark = pytest.mark.gpu


def check_rows(got, rows, x, w, a, b, ids, scales=None, bias=None):
    clean = torch.nan_to_num(b, 0.0, 0.0, 0.0)
    ref, bound = reference(x, w, a, clean, ids, scales=scales, bias=bias)
    err = (got.double() - ref).abs()[rows]
    assert torch.isfinite(got[rows]).all()
    assert (err <= bound[rows]).all(), f"worst err / bound {float((err / bound[rows]).max()):.3g}"
    assert tb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout", ["T", "N"])
@pytest.mark.parametrize("T,K,N,R,L", [(2, 512, 264, 16, 3), (20, 1024, 1000, 24, 6), (64, 256, 520, 64, 64), (64, 192, 256, 128, 64), (5, 256, 40000, 8, 4),
                                       (33, 4096, 2048, 16, 9), (65, 512, 520, 16, 3), (130, 264, 200, 40, 200), (333, 2056, 1256, 24, 6), (600, 128, 640, 72, 2)])
def test_a_broken_adapter_stays_with_its_rows(T, K, N, R, L, layout, dtype):
    x, w, a, b, ids, s = make(T, K, N, R, L, dtype, layout=layout)
    ids[0], ids[-1] = 0, -1
    bias = torch.randn(N, device="cuda")
    want = tb.lora_matmul(x, w, a, b, ids, s, bias=bias)
    b[0, N // 2, R - 1] = float("nan")                  # one entry: one feature
    got = tb.lora_matmul(x, w, a, b, ids, s, bias=bias)
    others, features = ids != 0, torch.arange(N, device="cuda") != N // 2
    assert torch.equal(got[:, features], want[:, features]) and torch.isnan(got[~others][:, N // 2]).all()
    check_rows(got, others, x, w, a, b, ids, scales=s, bias=bias)
    b[0] = float("inf")                                 # all of it
    got = tb.lora_matmul(x, w, a, b, ids, s, bias=bias)
    assert not torch.isfinite(got[~others]).any()
    check_rows(got, others, x, w, a, b, ids, scales=s, bias=bias)
    b[1:][torch.arange(1, L, device="cuda") % 2 == 0] = float("nan")      # and others with it
    broken = (ids >= 0) & (ids % 2 == 0)
    got = tb.lora_matmul(x, w, a, b, ids, s, bias=bias)
    check_rows(got, ~broken, x, w, a, b, ids, scales=s, bias=bias)
    assert not torch.isfinite(got[broken]).any()


def test_strided_output_and_a_captured_graph():
    x, w, a, b, ids, s = make(300, 256, 328, 16, 4, torch.bfloat16)
    b[2] = float("nan")
    rows = ids != 2
    buf = torch.full((302, 333), 7.0, dtype=x.dtype, device="cuda")
    tb.lora_matmul(x, w, a, b, ids, s, out=buf[1:301, 2:330])
    check_rows(buf[1:301, 2:330], rows, x, w, a, b, ids, scales=s)
    buf[1:301, 2:330] = 7.0
    assert (buf == 7.0).all()
    wide = torch.full((328, 300), 7.0, dtype=x.dtype, device="cuda")
    check_rows(tb.lora_matmul(x, w, a, b, ids.long(), s, out=wide.T), rows, x, w, a, b, ids, scales=s)
    small = (x[:40].contiguous(), w, a, b, ids[:40].contiguous(), s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tb.lora_matmul(*small)
    for seed in (5, 6):
        small[0].copy_(make(40, 256, 328, 16, 4, torch.bfloat16, seed=seed)[0])
        graph.replay()
        check_rows(out, small[4] != 2, *small[:5], scales=s)


def test_rows_of_nan_with_several_adapters():
    """Nothing is finite by the formula: every element is looked at again, and the call still ends."""
    for T in (64, 700):
        x, w, a, b, ids, s = make(T, 512, 1024, 16, 5, torch.bfloat16)
        got = tb.lora_matmul(x * float("nan"), w, a, b, ids, s)
        assert torch.isnan(got).all() and tb.device_status() == 0


@pytest.mark.parametrize("T", [40, 300])
def test_what_is_not_finite_by_the_formula_stays_what_it_is(T):
    """Rows of x with a NaN or an infinity, infinite entries of an adapter that cancel or not, all beside a broken adapter: NaN where
    the formula in 64 bits has NaN, infinities of its sign where it has those."""
    x, w, a, b, ids, s = make(T, 128, 264, 16, 5, torch.bfloat16)
    s = s.abs() + 0.25
    ids[:6] = torch.tensor([0, 1, 2, 3, 4, -1], device="cuda")
    b[0] = float("nan")
    b[1, 7, 3], b[1, 9, 2], b[1, 9, 5] = float("inf"), float("inf"), float("-inf")
    x[T // 2, 5], x[T // 3, 9], x[T // 4, 0] = float("nan"), float("inf"), float("-inf")
    got = tb.lora_matmul(x, w, a, b, ids, s).double()
    want = x.double() @ w.double()
    for i in range(5):
        rows = ids == i
        want[rows] += float(s[i]) * (x[rows].double() @ a[i].double().T) @ b[i].double().T
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    sure = torch.isfinite(want) & (want.abs() < 1e30)
    assert torch.isfinite(got[sure]).all() and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
