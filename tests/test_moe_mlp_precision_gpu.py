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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,K,H,F", [(1, 64, 8, 4096, 1536), (16, 64, 8, 4096, 1536), (128, 64, 8, 4096, 1536), (5, 60, 4, 2048, 704), (40, 16, 4, 1024, 4096)])
def test_both_halves_count_at_model_size(T, E, K, H, F, dtype):
    """Model-sized weights with one entry per row of w1 and two per row of w2, so that no sum rounds: out = w (h_f - h_f'), where f'
    has f's gate and an up weight 2^-6 larger. The difference is 2^-6 of h, whose high half alone is off by up to eps / 2: a low
    half that went missing anywhere would be a wrong result."""
    g = torch.Generator(device="cuda").manual_seed(T + F)
    x = torch.randn(T, H, device="cuda", generator=g).to(dtype)
    w1, w2 = torch.zeros(E, 2 * F, H, dtype=dtype, device="cuda"), torch.zeros(E, H, F, dtype=dtype, device="cuda")
    e = torch.arange(E, device="cuda").unsqueeze(1)
    half = torch.arange(F // 2, device="cuda")
    gate_col = torch.randint(0, H, (E, F // 2), device="cuda", generator=g)
    up_col = torch.randint(0, H, (E, F // 2), device="cuda", generator=g)
    w1[e, 2 * half, gate_col] = w1[e, 2 * half + 1, gate_col] = 1.0
    w1[e, F + 2 * half, up_col] = 1.0
    w1[e, F + 2 * half + 1, up_col] = 1.0 + 2.0 ** -6
    pair = torch.randint(0, F // 2, (E, H), device="cuda", generator=g)
    row = torch.arange(H, device="cuda")
    w2[e, row, 2 * pair] = -1.0
    w2[e, row, 2 * pair + 1] = 1.0
    ids, w = routed(T, E, K, g)
    got = tb.moe_mlp(x, w1, w2, ids, w)
    # expectation by the structure: h of the pair's first feature times 2^-6
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    mag = ref.clone()
    for t in range(T):
        for j in range(K):
            i = int(ids[t, j])
            gate, up = x[t, gate_col[i]].double(), x[t, up_col[i]].double()
            h = gate * torch.sigmoid(gate) * up
            ref[t] += w[t, j].double() * h[pair[i]] * 2.0 ** -6
            mag[t] += w[t, j].double() * h[pair[i]].abs() * (2 + 2.0 ** -6)
    f = torch.finfo(dtype)
    floor = 2.0 ** -27 if dtype == torch.float16 else 0.0
    bound = mag * (2.0 ** -20 + f.eps ** 2 / 4 + (K + 6) * 2.0 ** -24) + floor + f.eps / 2 * ref.abs() + f.smallest_normal * f.eps / 2
    err = (got.double() - ref).abs()
    assert (err <= bound).all(), f"worst err / bound {float((err / bound).max()):.3g}"
    # with the high halves alone the expectation itself is far outside
    assert (mag * f.eps / 8 > bound).float().mean() > 0.5 and tb.device_status() == 0


@pytest.mark.parametrize("T", [1, 16, 128])
def test_the_layer_at_model_size(T):
    """64 experts of 4096 x 1536, top-8, random weights. In the mean over a row the result is off by its own rounding, uniform up to
    2^-8 of the power of two below a value (whose mean square is less than 1 / 1.5 of the values'), and by what fp32 sums of 4096
    terms leave: 2^-14 is ample for random signs. A low half that went missing adds as much as the rounding itself."""
    E, K, H, F = 64, 8, 4096, 1536
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) * H ** -0.5).bfloat16()
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) * F ** -0.5).bfloat16()
    ids, w = routed(T, E, K, g)
    got = tb.moe_mlp(x, w1, w2, ids, w).double()
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for i in torch.unique(ids).tolist():
        tok, slot = (ids == i).nonzero(as_tuple=True)
        z = x[tok].double() @ w1[i].double().T
        act = z[:, :F] * torch.sigmoid(z[:, :F]) * z[:, F:]
        ref.index_add_(0, tok, (act @ w2[i].double().T) * w[tok, slot].double().unsqueeze(1))
    rms = (got - ref).pow(2).mean(1).sqrt() / ref.pow(2).mean(1).sqrt()
    assert (rms <= 2.0 ** -8 * 3 ** -0.5 * 1.5 ** -0.5 + 2.0 ** -14).all(), rms.max()
    assert tb.device_status() == 0
