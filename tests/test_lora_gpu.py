"""A shared projection with one low-rank adapter per row (lora_matmul) against the formula in 64 bits, bound per element.

Bound. fp32 accumulation is off by at most one unit in the last place per term, n 2^-23 sum |a b| for n products. The
rank-sized product v is such a sum over k, scaled (one rounding) and rounded to the operands' type (finfo.eps / 2, or half the
smallest subnormal), so dv = s k 2^-23 sum |x a| + (2^-23 + eps / 2) |v| + tiny eps / 2. The output sums k + rank + 1 terms:
(k + rank + 1) 2^-23 (sum |x w| + sum |v b| + |bias|) + sum dv |b| + eps / 2 |out|."""
import pytest
import torch

import tritonblas_b200 as tb

pytestmark = pytest.mark.gpu


def make(T, K, N, R, L, dtype, seed=0, layout="T"):
    g = torch.Generator(device="cuda").manual_seed(seed + T + 3 * N + R)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)
    x = rnd(T, K).to(dtype)
    w = (rnd(N, K) * K ** -0.5).to(dtype).T
    w = w if layout == "T" else w.contiguous()
    a = (rnd(L, R, K) * K ** -0.5).to(dtype)
    b = (rnd(L, N, R) * R ** -0.5).to(dtype)
    ids = torch.randint(-1, L, (T,), device="cuda", generator=g, dtype=torch.int32)
    scales = torch.rand(L, device="cuda", generator=g) * 2 - 0.5
    return x, w, a, b, ids, scales


def reference(x, w, a, b, ids, scales=None, bias=None):
    f = torch.finfo(x.dtype)
    K, R = x.shape[1], a.shape[1]
    xd, wd = x.double(), w.double()
    out = xd @ wd
    mag = xd.abs() @ wd.abs()
    if bias is not None:
        out, mag = out + bias.double(), mag + bias.double().abs()
    extra = torch.zeros_like(out)
    for i in range(a.shape[0]):
        rows = (ids == i).nonzero().squeeze(1)
        if rows.numel() == 0:
            continue
        s = 1.0 if scales is None else float(scales[i])
        ad, bd = a[i].double(), b[i].double()
        v = s * (xd[rows] @ ad.T)
        dv = abs(s) * K * 2.0 ** -23 * (xd[rows].abs() @ ad.abs().T) + (2.0 ** -23 + f.eps / 2) * v.abs() + f.smallest_normal * f.eps / 2
        out[rows] += v @ bd.T
        mag[rows] += v.abs() @ bd.abs().T
        extra[rows] += dv @ bd.abs().T
    return out, (K + R + 1) * 2.0 ** -23 * mag + extra + f.eps / 2 * out.abs() + f.smallest_normal * f.eps


def check(got, *case, what="", **kw):
    ref, bound = reference(*case, **kw)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= bound).all(), f"{what}: worst err / bound {float((err / bound).max()):.3g}, {int((err > bound).sum())} off, first {(err > bound).nonzero()[0].tolist()}"
    assert tb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,K,N,R,L", [(1, 64, 256, 8, 1), (1, 1024, 2048, 16, 8), (2, 72, 40, 8, 3), (5, 2056, 1000, 24, 6), (16, 512, 777, 64, 4),
                                       (33, 1024, 4096, 16, 40), (48, 520, 300, 128, 5), (64, 256, 512, 16, 64), (64, 4096, 8192, 32, 9),
                                       (65, 512, 512, 72, 3), (130, 264, 200, 40, 200), (333, 2056, 1250, 24, 6), (700, 128, 640, 16, 2), (1, 128, 64, 8, 1), (90, 192, 136, 16, 1),
                                       (1000, 512, 1536, 128, 10)])
def test_matches_formula(T, K, N, R, L, dtype):
    case = make(T, K, N, R, L, dtype)
    check(tb.lora_matmul(*case), *case, what=f"{T} {K} {N} {R} {L}")


@pytest.mark.parametrize("T", [3, 40, 200])
@pytest.mark.parametrize("layout", ["T", "N"])
def test_weight_layouts_bias_and_default_scale(T, layout):
    x, w, a, b, ids, s = make(T, 512, 768, 16, 4, torch.bfloat16, layout=layout)
    for bias in (None, torch.randn(768, device="cuda"), torch.randn(1536, device="cuda").bfloat16()[::2]):
        for scales in (None, s, s.double()):
            check(tb.lora_matmul(x, w, a, b, ids, scales=scales, bias=bias), x, w, a, b, ids, what=f"{T} {layout}",
                  scales=None if scales is None else s, bias=bias)


@pytest.mark.parametrize("T", [7, 64, 300])
def test_rows_without_an_adapter_are_the_shared_projection(T):
    x, w, a, b, ids, s = make(T, 512, 768, 16, 4, torch.bfloat16)
    a, b = torch.full_like(a, float("nan")), torch.full_like(b, float("nan"))     # nothing of an unused adapter may be read into a row
    ids[:] = -1
    ids[::3] = 4
    check(tb.lora_matmul(x, w, a, b, ids, s), x, w, a, b, torch.full_like(ids, -1))
    wide = ids.long()
    wide[1::3] = 1 << 40
    wide[2::3] = -(1 << 40)
    check(tb.lora_matmul(x, w, a, b, wide, s), x, w, a, b, torch.full_like(ids, -1))


@pytest.mark.parametrize("T", [16, 64, 256, 513])
@pytest.mark.parametrize("order", ["one", "each", "segments", "last"])
def test_orders_of_adapters(T, order):
    L = T if order == "each" else 5
    x, w, a, b, _, s = make(T, 256, 384, 8, L, torch.float16)
    t = torch.arange(T, device="cuda")
    ids = {"one": t * 0 + 3, "each": (t * 7) % L, "segments": t * 5 // T, "last": torch.where(t == T - 1, 4, -1)}[order].int()
    check(tb.lora_matmul(x, w, a, b, ids, s), x, w, a, b, ids, scales=s, what=order)


def test_strides_alignment_and_out():
    x, w, a, b, ids, s = make(50, 256, 328, 16, 4, torch.bfloat16)
    want = tb.lora_matmul(x, w, a, b, ids, s)
    buf = torch.full((50, 300), float("nan"), dtype=x.dtype, device="cuda")
    for first in (3, 8):
        buf[:, first:first + 256] = x
        assert torch.equal(tb.lora_matmul(buf[:, first:first + 256], w, a, b, ids, s), want)
        buf.fill_(float("nan"))
    wide_a = torch.full((4, 20, 264), float("nan"), dtype=x.dtype, device="cuda")
    wide_a[:, :16, :256] = a
    wide_b = torch.full((4, 330, 24), float("nan"), dtype=x.dtype, device="cuda")
    wide_b[:, :328, :16] = b
    assert torch.equal(tb.lora_matmul(x, w, wide_a[:, :16, :256], wide_b[:, :328, :16], ids.repeat_interleave(2)[::2], s), want)
    odd_w = torch.empty(328, 259, dtype=x.dtype, device="cuda")[:, 2:258].copy_(w.T).T          # pitch TMA cannot address
    assert torch.equal(tb.lora_matmul(x, odd_w, a, b, ids, s), want)
    for shape, pick in (((52, 333), lambda t: t[1:51, 2:330]), ((52, 336), lambda t: t[1:51, 8:336]), ((330, 50), lambda t: t[1:329].T)):
        t = torch.full(shape, 7.0, dtype=x.dtype, device="cuda")
        got = tb.lora_matmul(x, w, a, b, ids, s, out=pick(t))
        assert got.data_ptr() == pick(t).data_ptr() and torch.equal(got, want)
        pick(t).fill_(7.0)
        assert (t == 7.0).all()
    square = torch.zeros(50, 256, dtype=x.dtype, device="cuda")
    with pytest.raises(ValueError, match="out must not be x"):
        tb.lora_matmul(square, w[:, :256], a, b[:, :256], ids, s, out=square)
    one = tb.lora_matmul(x[:1].expand(50, 256), w, a, b, ids * 0, s)                             # one row, stride 0
    assert torch.equal(one, one[:1].expand(50, 328))
    assert tb.lora_matmul(x[:0], w, a, b, ids[:0], s).shape == (0, 328)
    assert tb.lora_matmul(x, w[:, :0], a, b[:, :0], ids, s).shape == (50, 0)
    assert tb.device_status() == 0


def test_extreme_values_stay_in_their_row():
    x, w, a, b, ids, s = make(60, 256, 512, 16, 4, torch.bfloat16)
    want = tb.lora_matmul(x, w, a, b, ids, s)
    bad = x.clone()
    bad[7, 3] = float("nan")
    bad[20, 9] = float("inf")
    got = tb.lora_matmul(bad, w, a, b, ids, s)
    keep = [t for t in range(60) if t not in (7, 20)]
    # inside one tile a row's projection stands beside zeros of the other rows; only the row itself meets its values
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[7]).all()
    assert tb.device_status() == 0


@pytest.mark.parametrize("T,K,N", [(5, 4096, 40000), (20, 8, 19200), (64, 64, 37888)])
def test_decode_with_whole_and_dealt_tiles(T, K, N):
    """More feature tiles than SMs: whole tiles, dealt ones and the update of either (the last case deals none)."""
    case = make(T, K, N, 16, 7, torch.bfloat16)
    check(tb.lora_matmul(*case), *case)
    bias = torch.randn(N, device="cuda")
    check(tb.lora_matmul(*case, bias=bias), *case[:5], scales=case[5], bias=bias)


@pytest.mark.parametrize("T,K,N,R,L", [(1, 64, 8, 8, 1), (1, 4096, 4096, 16, 8), (2, 72, 40, 8, 3), (17, 200, 136, 72, 5), (48, 520, 1000, 128, 40),
                                       (5, 1024, 19200, 24, 6), (64, 64, 37888, 16, 64), (65, 512, 520, 16, 3), (333, 2056, 1256, 24, 6)])
def test_weights_with_contiguous_outputs(T, K, N, R, L):
    """The (k, n) layout as stored, down to one column of tiles that ends inside its first half."""
    x, w, a, b, ids, s = make(T, K, N, R, L, torch.float16, layout="N")
    assert w.stride() == (N, 1)
    got = tb.lora_matmul(x, w, a, b, ids, s)
    check(got, x, w, a, b, ids, scales=s)
    wide = torch.full((K, N + 16), float("nan"), dtype=w.dtype, device="cuda")
    wide[:, 8:N + 8] = w
    assert torch.equal(tb.lora_matmul(x, wide[:, 8:N + 8], a, b, ids, s), got)
    row = w[:1].expand(K, N)                                                                     # one row of weights, stride 0
    check(tb.lora_matmul(x, row, a, b, ids, s), x, row, a, b, ids, scales=s)
    column = w[:, :1].expand(K, N)
    check(tb.lora_matmul(x, column, a, b, ids, s), x, column, a, b, ids, scales=s)


def test_many_streams_at_once():
    """Long batches on eight streams: more blocks than fit the device at once, none of which may hold up another's."""
    cases = [make(T, 2056, 1000, 16, 6, torch.bfloat16, seed=T) for T in (65, 128, 200, 333, 400, 64, 500, 1)]
    want = [tb.lora_matmul(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(40):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(tb.lora_matmul(*c))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i % len(cases)]) for i, g in enumerate(got)) and tb.device_status() == 0


@pytest.mark.parametrize("T,N,R", [(33, 37888, 16), (64, 37888, 16), (64, 20480, 72), (50, 56832, 32)])
def test_more_than_32_adapters_in_every_tile_of_a_block(T, N, R):
    """One adapter per row, and blocks that work on several tiles: each walks the whole list again."""
    x, w, a, b, _, s = make(T, 64, N, R, T, torch.bfloat16)
    ids = torch.randperm(T, device="cuda").int()
    check(tb.lora_matmul(x, w, a, b, ids, s), x, w, a, b, ids, scales=s)


@pytest.mark.parametrize("T,N,R", [(64, 256, 128), (64, 1000, 64), (40, 8192, 72), (64, 4096, 16), (17, 136, 40), (8, 640, 128), (48, 28672, 32)])
def test_long_updates_in_pieces(T, N, R):
    """Lists that are as long as the batch, shorter than the pieces they could have, a single entry, or empty."""
    x, w, a, b, _, s = make(T, 192, N, R, T, torch.bfloat16)
    t = torch.arange(T, device="cuda")
    bias = torch.randn(N, device="cuda")
    for ids in ((t * 7) % T, t % 9 - 1, t * 0 + T - 1, t * 0 - 1, torch.where(t == T - 1, 3, -1), t // 2):
        ids = ids.int()
        got = tb.lora_matmul(x, w, a, b, ids, s, bias=bias)
        check(got, x, w, a, b, ids, scales=s, bias=bias, what=str(ids.unique().numel()))
        assert torch.equal(got, tb.lora_matmul(x, w, a, b, ids, s, bias=bias))


def test_grad_is_refused():
    x, w, a, b, ids, s = make(4, 64, 64, 8, 2, torch.bfloat16)
    with pytest.raises(RuntimeError, match="inference only"):
        tb.lora_matmul(x, w, a.requires_grad_(True), b, ids, s)
    with torch.no_grad():
        check(tb.lora_matmul(x, w, a, b, ids, s), x, w, a.detach(), b, ids, scales=s)


def test_large_batch_is_cut_into_pieces(monkeypatch):
    from tritonblas_b200 import lora
    x, w, a, b, ids, s = make(1500, 128, 256, 8, 30, torch.bfloat16)
    want = tb.lora_matmul(x, w, a, b, ids, s)
    check(want, x, w, a, b, ids, scales=s)
    monkeypatch.setattr(lora, "_MAX_WORKSPACE", 1 << 20)
    got = tb.lora_matmul(x, w, a, b, ids, s)
    check(got, x, w, a, b, ids, scales=s)


def test_streams_and_captured_graphs():
    cases = [make(T, 512, 1024, 16, 6, torch.bfloat16, seed=T) for T in (1, 24, 100, 600)]
    want = [tb.lora_matmul(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[] for _ in cases]
    for _ in range(20):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                got[i].append(tb.lora_matmul(*c))
    torch.cuda.synchronize()
    for i, w in enumerate(want):
        assert all(torch.equal(g, w) for g in got[i])
    graphs, outs = [], []
    for c in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tb.lora_matmul(*c))
        graphs.append(graph)
    for c in cases:
        n = make(c[0].shape[0], 512, 1024, 16, 6, torch.bfloat16, seed=99)
        for old, new in zip(c, n):
            old.copy_(new)
    torch.cuda.synchronize()
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for o, c in zip(outs, cases):
        check(o, *c[:5], scales=c[5])


def test_back_to_back_calls_depend_on_each_other():
    """The second product reads what the first one wrote, launched while the first still drains."""
    x, w, a, b, ids, s = make(40, 512, 512, 16, 6, torch.bfloat16)
    y = x
    for _ in range(6):
        y = tb.lora_matmul(y, w, a, b, ids, s)
    z = x
    for _ in range(6):
        z = tb.lora_matmul(z, w, a, b, ids, s)
        torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_decode_step_chain():
    """Projection with adapters, router product, router and experts, as one decode step runs them."""
    T, H, F, E, K = 20, 512, 256, 16, 4
    x, w, a, b, ids, s = make(T, H, H, 16, 5, torch.bfloat16)
    g = torch.Generator(device="cuda").manual_seed(1)
    wr = (torch.randn(E, H, device="cuda", generator=g) * H ** -0.5).bfloat16()
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) * H ** -0.5).bfloat16()
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) * F ** -0.5).bfloat16()

    def step(x):
        h = tb.lora_matmul(x, w, a, b, ids, s)
        weights, chosen = tb.moe_route(tb.matmul(h, wr.T), K)
        return h, weights, chosen, tb.moe_mlp(h, w1, w2, chosen, weights)

    h, weights, chosen, out = step(x)
    check(h, x, w, a, b, ids, scales=s)
    from tests.test_moe_mlp_gpu import check as check_experts
    check_experts(out, h, w1, w2, chosen, weights)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(captured, (h, weights, chosen, out)))
