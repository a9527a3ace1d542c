"""The rank-sized products of lora_matmul are kept to more bits than the result has, and stay in range where that is promised.

With few entries per row, powers of two mostly, sums in fp32 are exact or round once per term (u = 2^-24). A product v is kept in
two 16-bit halves: half a step of each, (eps / 2)^2 relative, in float16 2^-25 at least. The result rounds by half a step."""
import pytest
import torch

import tritonblas_b200 as tb

pytestmark = pytest.mark.gpu

SHAPES = [(1, 4096, 520, 16, 3), (20, 512, 200, 8, 5), (33, 1024, 264, 24, 40), (64, 512, 1000, 40, 64), (64, 256, 20000, 16, 9), (64, 4096, 520, 128, 30),
          (65, 512, 264, 16, 3), (130, 256, 200, 72, 7), (300, 2048, 520, 32, 300), (1000, 512, 1544, 64, 8), (700, 256, 640, 104, 1)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,N,R,L", SHAPES)
def test_both_halves_of_the_rank_sized_product_count(T, K, N, R, L, dtype):
    """No shared projection; two neighbouring ranks hold v and (1 + 2^-6) v, and the result is their difference, 2^-6 of v: smaller
    than half a step of either."""
    g = torch.Generator(device="cuda").manual_seed(T + R)
    x = torch.randn(T, K, device="cuda", generator=g).to(dtype)
    w = torch.zeros(N, K, dtype=dtype, device="cuda").T
    a, b = torch.zeros(L, R, K, dtype=dtype, device="cuda"), torch.zeros(L, N, R, dtype=dtype, device="cuda")
    big, small = (torch.randint(0, K // 2, (L, R // 2), device="cuda", generator=g) * 2 + i for i in (0, 1))
    i, even, small_entry = torch.arange(L, device="cuda").unsqueeze(1), torch.arange(0, R, 2, device="cuda"), 2.0 ** -9
    a[i, even, big], a[i, even, small] = 1.0, small_entry                     # bits that one 16-bit number cannot hold
    a[i, even + 1, big], a[i, even + 1, small] = 1.0 + 2.0 ** -6, small_entry
    pair = torch.randint(0, R // 2, (L, N), device="cuda", generator=g)
    n = torch.arange(N, device="cuda")
    b[i, n, 2 * pair], b[i, n, 2 * pair + 1] = -1.0, 1.0
    ids = torch.randint(-1, L, (T,), device="cuda", generator=g, dtype=torch.int32)
    scales = torch.rand(L, device="cuda", generator=g) + 0.5
    got = tb.lora_matmul(x, w, a, b, ids, scales)
    f = torch.finfo(dtype)
    ref, bound = torch.zeros(T, N, dtype=torch.float64, device="cuda"), torch.zeros(T, N, dtype=torch.float64, device="cuda")
    for t in range(T):
        l = int(ids[t])
        if l < 0:
            continue
        s, xt = scales[l].double(), x[t].double()
        v0 = s * (xt[big[l]] + xt[small[l]] * small_entry)
        v1 = s * (xt[big[l]] * (1 + 2.0 ** -6) + xt[small[l]] * small_entry)
        ref[t] = (v1 - v0)[pair[l]]
        m = (v0.abs() + v1.abs())[pair[l]]
        # sums of two terms and the scale: 3 u; the halves; their sum: 3 u
        bound[t] = m * (6 * 2.0 ** -24 + f.eps ** 2 / 4) + (2.0 ** -24 if dtype == torch.float16 else 0.0)
    bound += f.eps / 2 * ref.abs() + f.smallest_normal * f.eps / 2
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), f"worst err / bound {float((err / bound).max()):.3g}, {int((err > bound).sum())} off"
    assert tb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,N,R,L", [(1, 4096, 4096, 16, 8), (48, 4096, 8192, 64, 30), (64, 1024, 1024, 128, 64), (333, 2056, 5000, 24, 6), (2048, 4096, 4096, 64, 8)])
def test_an_update_is_as_good_as_its_rounding(T, K, N, R, L, dtype):
    """Random adapters without a shared projection: in the mean a row is off by its own rounding, uniform up to half a step of the
    power of two below a value (whose mean square is less than 1 / 1.5 of the values'), and 2^-14 for fp32 sums. A v rounded to 16
    bits would add as much again."""
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, K, device="cuda", generator=g).to(dtype)
    w = torch.zeros(N, K, dtype=dtype, device="cuda").T
    a = (torch.randn(L, R, K, device="cuda", generator=g) * K ** -0.5).to(dtype)
    b = (torch.randn(L, N, R, device="cuda", generator=g) * R ** -0.5).to(dtype)
    ids = torch.randint(0, L, (T,), device="cuda", generator=g)
    got = tb.lora_matmul(x, w, a, b, ids).double()
    ref = torch.empty(T, N, dtype=torch.float64, device="cuda")
    for l in torch.unique(ids).tolist():
        rows = ids == l
        ref[rows] = (x[rows].double() @ a[l].double().T) @ b[l].double().T
    rms = (got - ref).pow(2).mean().sqrt() / ref.pow(2).mean().sqrt()
    assert rms <= torch.finfo(dtype).eps / 2 * 3 ** -0.5 * 1.5 ** -0.5 + 2.0 ** -14, rms
    assert tb.device_status() == 0
