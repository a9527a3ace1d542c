"""Expert feed-forward of a few tokens at the ends of its range.

What a result may be off by: sums of n terms by n 2^-23 of their magnitudes; the activation h = silu(g) u by 2^-20 (an exponential
within 4 u, u = 2^-24, a sum, a quotient, a product) and what g and u were off; its two 16-bit halves by half a step of each
((eps / 2)^2 relative, in float16 2^-28 at least); a routing weight and a sum by 4 u; the output by its half step."""
import pytest
import torch

import tritonblas_b200 as tb

pytestmark = pytest.mark.gpu


def routed(T, E, K, g):
    ids = torch.rand(T, E, device="cuda", generator=g).argsort(1)[:, :K].to(torch.int32)
    return ids, torch.softmax(torch.randn(T, K, device="cuda", generator=g), 1)


def dense_reference(x, w1, w2, ids, w):
    """(value, bound) in 64 bits for any weights; sums of n terms are off by n u times their magnitudes."""
    f = torch.finfo(x.dtype)
    E, _, F = w2.shape
    u = 2.0 ** -23
    out = torch.zeros(x.shape, dtype=torch.float64, device="cuda")
    bound = out.clone()
    floor = 2.0 ** -28 if x.dtype == torch.float16 else 0.0
    for e in range(E):
        share = (w.double() * (ids == e)).sum(1, keepdim=True)
        a, b = w1[e].double(), w2[e].double()
        z, dz = x.double() @ a.T, (x.double().abs() @ a.abs().T) * ((a != 0).sum(1).max() * u)
        g, up, dg, du = z[:, :F], z[:, F:], dz[:, :F], dz[:, F:]
        silu = g * torch.sigmoid(g)
        h = silu * up
        dh = 1.1 * dg * up.abs() + silu.abs() * du + 1.1 * dg * du + (2.0 ** -20 + f.eps ** 2 / 4) * h.abs() + floor
        out += share * (h @ b.T)
        bound += share.abs() * (dh @ b.abs().T + ((b != 0).sum(1).max() + 6) * u * (h.abs() @ b.abs().T))
    return out, bound + f.eps / 2 * out.abs() + f.smallest_normal * f.eps / 2


def check(got, *case):
    ref, bound = dense_reference(*case)
    assert torch.isfinite(got).all()
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), f"worst err / bound {float((err / bound).max()):.3g}"
    assert tb.device_status() == 0


@pytest.mark.parametrize("T", [1, 5, 40, 128])
@pytest.mark.parametrize("x_scale,w2_scale", [(3e-3, 64.0), (1e-2, 8.0), (1e-2, 1.0), (1.0, 1.0), (1e2, 2.0 ** -7), (8e2, 2.0 ** -13)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_small_and_large_activations(dtype, x_scale, w2_scale, T):
    """silu(gate) * up from 1e-6 to 1e7: float16 numbers end at 65504 and lose their bits below 6e-5."""
    E, K, H, F = 6, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(T)
    x = (torch.randn(T, H, device="cuda", generator=g) * x_scale).to(dtype)
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) * H ** -0.5).to(dtype)
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) * w2_scale).to(dtype)
    ids, w = routed(T, E, K, g)
    check(tb.moe_mlp(x, w1, w2, ids, w), x, w1, w2, ids, w)
