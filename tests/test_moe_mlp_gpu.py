"""Expert feed-forward of a few tokens (moe_mlp) against the formula in 64 bits, with a bound computed per element.

Bound. The products accumulate in fp32 with at most one unit in the last place (2^-23 of the running sum) per term, so a sum
of n products a b is off by at most n 2^-23 sum |a b|. With dg, du those bounds for gate and up, |silu'| <= 1.1 and the
exponential and the product good to 8 units: dh = 1.1 dg |u| + |silu(g)| du + 1.1 dg du + 2^-20 |h|. h is kept as two 16-bit
halves: another eps^2 / 4 |h| (and half the smallest subnormal). Then out is off by
sum_j w (sum_f |W2| dh + ffn 2^-22 sum_f |W2 h|) + topk 2^-23 sum |.| and one rounding eps / 2 |out|."""
import pytest
import torch

import tritonblas_b200 as tb

pytestmark = pytest.mark.gpu


def make(T, E, K, H, F, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + 7 * E + K)
    x = torch.randn(T, H, device="cuda", generator=g).to(dtype)
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) * H ** -0.5).to(dtype)
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) * F ** -0.5).to(dtype)
    ids = torch.rand(T, E, device="cuda", generator=g).argsort(1)[:, :K].to(torch.int32)
    w = torch.softmax(torch.randn(T, K, device="cuda", generator=g), 1)
    return x, w1, w2, ids, w


def reference(x, w1, w2, ids, w):
    """(value, bound) in 64 bits."""
    T, H = x.shape
    E, _, F = w2.shape
    u = torch.finfo(x.dtype)
    xd = x.double()
    out = torch.zeros(T, H, dtype=torch.float64, device=x.device)
    mag, bound = out.clone(), out.clone()
    for e in range(E):
        share = (w.double() * (ids == e)).sum(1, keepdim=True)
        tok = (ids == e).any(1).nonzero().squeeze(1)
        if tok.numel() == 0:
            continue
        a, s = w1[e].double(), share[tok]
        h = xd[tok] @ a.T
        dh = (xd[tok].abs() @ a.abs().T) * (H * 2.0 ** -23)
        gate, up, dg, du = h[:, :F], h[:, F:], dh[:, :F], dh[:, F:]
        silu = gate * torch.sigmoid(gate)
        act = silu * up
        dact = 1.1 * dg * up.abs() + silu.abs() * du + 1.1 * dg * du + (2.0 ** -20 + u.eps ** 2 / 4) * act.abs() + u.smallest_normal * u.eps
        b = w2[e].double()
        out[tok] += s * (act @ b.T)
        m = act.abs() @ b.abs().T
        mag[tok] += s.abs() * m
        bound[tok] += s.abs() * (dact @ b.abs().T + F * 2.0 ** -22 * m)
    return out, bound + ids.shape[1] * 2.0 ** -23 * mag + u.eps / 2 * out.abs() + u.smallest_normal * u.eps


def check(got, x, w1, w2, ids, w, what=""):
    ref, bound = reference(x, w1, w2, ids, w)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= bound).all(), f"{what}: worst err / bound {float((err / bound).max()):.3g} at {(err / bound).argmax().item()}"
    assert tb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,E,K,H,F", [(1, 1, 1, 64, 64), (1, 8, 2, 256, 128), (2, 5, 3, 200, 72), (16, 8, 4, 512, 384), (17, 8, 8, 1024, 96),
                                       (31, 60, 4, 264, 704), (64, 16, 8, 512, 256), (100, 7, 3, 328, 200), (128, 32, 8, 512, 136),
                                       (128, 2, 2, 256, 128), (3, 300, 10, 8, 8), (128, 1, 1, 16, 1000),
                                       (128, 1024, 32, 64, 32), (32, 16, 9, 64, 48), (1, 2, 2, 1024, 1160)])
def test_matches_formula(T, E, K, H, F, dtype):
    case = make(T, E, K, H, F, dtype)
    check(tb.moe_mlp(*case), *case, f"{T} {E} {K} {H} {F}")


def test_ids_of_both_widths_out_of_range_and_repeated():
    x, w1, w2, ids, w = make(24, 6, 4, 256, 128, torch.bfloat16)
    ids[3] = -1                                     # a token with no expert: zeros
    ids[5] = torch.tensor([6, 2, 1 << 20, -7])
    ids[7] = torch.tensor([4, 4, 1, 4])             # the same expert three times: its weights add up
    ids[9] = 0
    for t in (ids, ids.long(), ids.long() + torch.where(ids.long() == 6, 1 << 40, 0)):
        got = tb.moe_mlp(x, w1, w2, t, w)
        assert (got[3] == 0).all()
        check(got, x, w1, w2, ids, w)
    ids[:] = -1
    assert (tb.moe_mlp(x, w1, w2, ids, w) == 0).all()


def test_one_expert_for_everybody():
    """128 tokens on one expert: more rows than a group holds, so its second projection is read in several groups."""
    x, w1, w2, ids, w = make(128, 4, 2, 256, 192, torch.bfloat16)
    ids[:, 0] = 2
    ids[:, 1] = torch.where(torch.arange(128, device="cuda") % 5 == 0, 1, -1)
    check(tb.moe_mlp(x, w1, w2, ids, w), x, w1, w2, ids, w)


def test_strides_alignment_and_out():
    x, w1, w2, ids, w = make(20, 4, 2, 256, 128, torch.bfloat16)
    want = tb.moe_mlp(x, w1, w2, ids, w)
    wide_x = torch.full((20, 300), float("nan"), dtype=x.dtype, device="cuda")
    wide_x[:, 3:259] = x                            # rows that are not 16-byte aligned
    assert torch.equal(tb.moe_mlp(wide_x[:, 3:259], w1, w2, ids, w), want)
    wide_x[:, 8:264] = x
    assert torch.equal(tb.moe_mlp(wide_x[:, 8:264], w1, w2, ids, w), want)
    wide_w1 = torch.full((4, 300, 264), float("nan"), dtype=x.dtype, device="cuda")
    wide_w1[:, :256, :256] = w1
    wide_w2 = torch.full((4, 256, 136), float("nan"), dtype=x.dtype, device="cuda")
    wide_w2[:, :, :128] = w2
    assert torch.equal(tb.moe_mlp(x, wide_w1[:, :256, :256], wide_w2[:, :, :128], ids, w), want)
    assert torch.equal(tb.moe_mlp(x.T.contiguous().T, w1, w2.transpose(1, 2).contiguous().transpose(1, 2), ids.T.contiguous().T, w.double()), want)
    for cols, first in ((300, 0), (259, 1)):        # rows of `out` on 8-byte boundaries, and not
        buf = torch.full((22, cols), 7.0, dtype=x.dtype, device="cuda")
        got = tb.moe_mlp(x, w1, w2, ids, w, out=buf[1:21, first:first + 256])
        assert got.data_ptr() == buf[1:21, first:first + 256].data_ptr() and torch.equal(got, want)
        buf[1:21, first:first + 256] = 7.0
        assert (buf == 7.0).all()                   # nothing outside the view was written
    # out may be the input: every token has been read before the first result is written
    y = x.clone()
    assert torch.equal(tb.moe_mlp(y, w1, w2, ids, w, out=y), want)
    assert tb.device_status() == 0


def test_extreme_values_stay_in_their_token():
    x, w1, w2, ids, w = make(40, 8, 2, 256, 128, torch.bfloat16)
    want = tb.moe_mlp(x, w1, w2, ids, w)
    bad = x.clone()
    bad[11, 5] = float("nan")
    bad[30, 0] = float("inf")
    got = tb.moe_mlp(bad, w1, w2, ids, w)
    keep = [t for t in range(40) if t not in (11, 30)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[11]).all()
    # weights of experts nobody chose are not part of any result
    used = set(ids.flatten().tolist())
    x1, ids1, wt1 = x[:1], ids[:1], w[:1]
    w1n, w2n = w1.clone(), w2.clone()
    for e in set(range(8)) - set(ids1.flatten().tolist()):
        w1n[e], w2n[e] = float("nan"), float("nan")
    assert torch.equal(tb.moe_mlp(x1, w1n, w2n, ids1, wt1), tb.moe_mlp(x1, w1, w2, ids1, wt1)) and used
    assert tb.device_status() == 0


def test_zero_tokens():
    x, w1, w2, ids, w = make(4, 4, 2, 64, 64, torch.bfloat16)
    assert tb.moe_mlp(x[:0], w1, w2, ids[:0], w[:0]).shape == (0, 64)


def test_repeats_are_bit_identical_and_streams_do_not_share_state():
    cases = [make(T, 16, 4, 512, 256, torch.bfloat16, seed=T) for T in (1, 9, 33, 128)]
    want = [tb.moe_mlp(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(20):         # four streams at once, each with its own problem
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                got[i].append(tb.moe_mlp(*c))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(g, w) for g in got[i])
    assert tb.device_status() == 0


def test_captured_graphs_replay_with_new_inputs():
    a, b = make(8, 16, 4, 512, 256, torch.bfloat16), make(40, 16, 4, 512, 256, torch.bfloat16)
    tb.moe_mlp(*a), tb.moe_mlp(*b)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tb.moe_mlp(*c))
        graphs.append(graph)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for c in (a, b):
        n = make(c[0].shape[0], 16, 4, 512, 256, torch.bfloat16, seed=77)
        for old, new in zip(c, n):
            old.copy_(new)
    torch.cuda.synchronize()
    for _ in range(5):          # two graphs, two streams, at once
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
    torch.cuda.synchronize()
    check(outs[0], *a)
    check(outs[1], *b)


def test_routed_layer_end_to_end():
    """Router product, router and experts as a decode step calls them, against the same chain in 64 bits at the chosen ids."""
    T, E, K, H, F = 12, 32, 6, 512, 256
    x, w1, w2, _, _ = make(T, E, K, H, F, torch.bfloat16)
    wr = (torch.randn(E, H, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3)) * H ** -0.5).bfloat16()
    logits = tb.matmul(x, wr.T)
    weights, ids = tb.moe_route(logits, K)
    out = tb.moe_mlp(x, w1, w2, ids, weights)
    check(out, x, w1, w2, ids, weights)
    ref = torch.softmax(torch.topk(logits.double(), K, dim=1).values, 1)
    assert torch.allclose(weights.double(), ref, rtol=1e-5)
