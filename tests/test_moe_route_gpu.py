"""Expert router (moe_route) against a 64-bit restatement: ids exactly, weights and gradients within derived bounds.

Bounds. A weight is a quotient of fp32 exponentials: the argument l - max rounds once (relative error |l - max| 2^-24 of the
exponential), expf is within 2 units in the last place, the sum of n terms within n 2^-24 (far less in the tree order used),
and a division and a product round once each: (|l - max| + n + 8) 2^-23 relative covers all of it. A gradient is a few such
weights times the given gradient plus one rounding to the logits' type (finfo.eps / 2)."""
import pytest
import torch

import tritonblas_b200 as tb

pytestmark = pytest.mark.gpu


def reference(logits, topk, scoring, renormalize, grad=None):
    """Ids, weights and logit gradient in 64 bits, from a stable descending sort."""
    l = logits.double().cpu()
    l = torch.where(torch.isnan(l), torch.full_like(l, float("-inf")), l)
    order = torch.argsort(-l, dim=1, stable=True)[:, :topk]
    chosen = torch.gather(l, 1, order)
    dead = chosen == float("-inf")
    if scoring == "softmax":
        top = l.max(1, keepdim=True).values
        ex = torch.exp(l - torch.where(top > float("-inf"), top, torch.zeros_like(top)))
        p = ex / ex.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        p = torch.sigmoid(l)
    s = torch.gather(p, 1, order).masked_fill(dead, 0.0)
    total = s.sum(1, keepdim=True)
    safe = torch.where(total > 0, total, torch.ones_like(total))
    w = s / safe if renormalize else s
    ids = order.masked_fill(dead, -1).to(torch.int32)
    if grad is None:
        return w, ids, None
    g = grad.double().cpu().masked_fill(dead, 0.0)
    if renormalize:
        g = ((g - (g * w).sum(1, keepdim=True)) / safe).masked_fill(dead, 0.0)
    dense = torch.zeros_like(l).scatter_(1, order, g)
    d = p * (dense - (dense * p).sum(1, keepdim=True)) if scoring == "softmax" else dense * p * (1 - p)
    return w, ids, d


def spread(logits):
    l = logits.double().cpu()
    l = l[torch.isfinite(l)]
    return float(l.max() - l.min()) if l.numel() else 0.0


def make(tokens, experts, dtype, seed=0, mask=True):
    g = torch.Generator().manual_seed(seed + 31 * tokens + experts)
    l = torch.randn(tokens, experts, generator=g) * 2
    if mask:
        l[torch.rand(tokens, experts, generator=g) < 0.1] = float("-inf")
        l[tokens // 2] = float("-inf")                  # a row with nothing to choose
        l[tokens // 3, : experts // 2] = float("nan")
        l[-1] = 0.25                                    # a row of ties
        l[0, -1] = torch.finfo(dtype).min               # the type's lowest value is an ordinary logit
    return l.to(dtype).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("tokens,experts,topk", [(1, 1, 1), (7, 8, 8), (33, 64, 8), (5, 60, 4), (130, 129, 32), (9, 256, 6), (3, 1000, 10), (2, 1024, 32)])
def test_forward_and_gradient(dtype, scoring, renormalize, tokens, experts, topk):
    logits = make(tokens, experts, dtype, mask=tokens > 1).requires_grad_(True)
    g = torch.Generator().manual_seed(5)
    grad = torch.randn(tokens, topk, generator=g).cuda()
    w, ids = tb.moe_route(logits, topk, scoring=scoring, renormalize=renormalize)
    (dl,) = torch.autograd.grad(w, logits, grad)
    rw, rids, rd = reference(logits.detach(), topk, scoring, renormalize, grad)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and dl.dtype == dtype
    assert torch.equal(ids.cpu(), rids)
    top = 30.0 if experts > 1 else 0.0      # exponentials of arguments below -30 are far under the bound's absolute part
    rel = (min(spread(logits.detach()), top) + experts + 8) * 2.0 ** -23
    assert ((w.detach().cpu().double() - rw).abs() <= rel * rw + 1e-12).all()
    # |d| <= few products of weights (at most 1 each, their errors `rel`) with the gradients of the row
    scale = grad.abs().double().cpu().sum(1, keepdim=True) * (1.0 if not (renormalize and scoring == "sigmoid") else 2.0)
    bound = torch.finfo(dtype).eps / 2 * rd.abs() + 8 * rel * scale + torch.finfo(dtype).tiny
    assert ((dl.cpu().double() - rd).abs() <= bound).all(), float(((dl.cpu().double() - rd).abs() - bound).max())
    # the path without autograd gives the same bits
    with torch.no_grad():
        w2, ids2 = tb.moe_route(logits, topk, scoring=scoring, renormalize=renormalize)
    assert torch.equal(w2, w.detach()) and torch.equal(ids2, ids)


@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(scoring, renormalize):
    """Central differences of the 64-bit formula at fixed choices: step 1e-4, truncation error about 1e-8 of the third derivative."""
    logits = make(6, 20, torch.float32, mask=False)
    grad = torch.randn(6, 5, generator=torch.Generator().manual_seed(1)).cuda()
    x = logits.clone().requires_grad_(True)
    w, ids = tb.moe_route(x, 5, scoring=scoring, renormalize=renormalize)
    (dl,) = torch.autograd.grad(w, x, grad)

    def value(l):
        p = torch.softmax(l, 1) if scoring == "softmax" else torch.sigmoid(l)
        s = torch.gather(p, 1, ids.long())
        if renormalize:
            s = s / s.sum(1, keepdim=True)
        return (s * grad.double()).sum(1)

    l, h = logits.double(), 1e-4
    for e in range(20):
        up, down = l.clone(), l.clone()
        up[:, e] += h
        down[:, e] -= h
        d = (value(up) - value(down)) / (2 * h)
        assert ((dl[:, e].double() - d).abs() <= 1e-5 * grad.abs().sum(1).double()).all()


def test_layouts_strides_and_empty():
    base = make(40, 96, torch.bfloat16, mask=False)
    want = tb.moe_route(base[:, :61].contiguous(), 7)
    for view in (base[:, :61], base[:, :61].T.contiguous().T):
        got = tb.moe_route(view, 7)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.empty(40 * 61 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(40, 61).copy_(base[:, :61])     # 2-byte aligned
    assert torch.equal(tb.moe_route(odd, 7)[1], want[1])
    row = base[:1, :61].expand(9, 61)                                                           # one row for all
    w, ids = tb.moe_route(row, 7)
    assert torch.equal(w, want[0][:1].expand(9, 7)) and torch.equal(ids, want[1][:1].expand(9, 7))
    w, ids = tb.moe_route(base[:0], 7)
    assert w.shape == (0, 7) and ids.shape == (0, 7)
    x = base[:0].detach().requires_grad_(True)
    (d,) = torch.autograd.grad(tb.moe_route(x, 7)[0].sum(), x)
    assert d.shape == (0, 96)
    # a broadcast gradient (stride 0) and a strided input
    x = base[:, ::2].detach().float().requires_grad_(True)
    (d,) = torch.autograd.grad(tb.moe_route(x, 4, renormalize=False)[0].sum(), x)
    _, _, rd = reference(x.detach(), 4, "softmax", False, torch.ones(40, 4))
    assert ((d.cpu().double() - rd).abs() <= 1e-5).all()


def test_second_derivative_is_refused():
    x = make(4, 16, torch.float32, mask=False).requires_grad_(True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(tb.moe_route(x, 2, renormalize=False)[0].sum(), x, create_graph=True)


def test_signed_zeros_tie_and_large_values():
    l = torch.tensor([[-0.0, 0.0, -1.0, 0.0], [3e38, -3e38, 1.0, 3e38]], device="cuda")
    w, ids = tb.moe_route(l, 3)
    assert ids.tolist() == [[0, 1, 3], [0, 3, 2]]
    assert torch.isfinite(w).all() and torch.allclose(w.sum(1), torch.ones(2, device="cuda"))


def test_an_infinite_logit_stays_in_its_row():
    """+inf: the softmax of its row is NaN by the formula, its sigmoid is 1; other rows of the same warp know nothing of it."""
    for experts in (16, 60, 200, 600):
        l = make(40, experts, torch.float32, mask=False)
        l[7, 3] = float("inf")
        keep = [t for t in range(40) if t != 7]
        clean = l.clone()
        clean[7, 3] = 100.0
        for renormalize in (True, False):
            w, ids = tb.moe_route(l, 4, renormalize=renormalize)
            ref_w, ref_ids = tb.moe_route(clean, 4, renormalize=renormalize)
            assert torch.isnan(w[7]).all() and torch.equal(w[keep], ref_w[keep]) and torch.equal(ids, ref_ids)
        w, ids = tb.moe_route(l, 4, scoring="sigmoid", renormalize=False)
        assert w[7, 0] == 1 and ids[7, 0] == 3 and torch.isfinite(w).all()


def test_capture_and_replay_and_compile():
    logits = make(64, 64, torch.bfloat16, mask=False)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        tb.moe_route(logits, 8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = tb.moe_route(logits, 8)
    logits.copy_(make(64, 64, torch.bfloat16, seed=9, mask=False))
    graph.replay()
    rw, rids, _ = reference(logits, 8, "softmax", True)
    assert torch.equal(ids.cpu(), rids)

    # forward and backward in one graph
    leaf = logits.detach().clone().requires_grad_(True)
    grad = torch.randn(64, 8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w, ids = tb.moe_route(leaf, 8, scoring="sigmoid")
        (d,) = torch.autograd.grad(w, leaf, grad)
    with torch.no_grad():
        leaf.copy_(make(64, 64, torch.bfloat16, seed=4, mask=False))
    graph.replay()
    _, rids2, rd = reference(leaf.detach(), 8, "sigmoid", True, grad)
    assert torch.equal(ids.cpu(), rids2)
    assert ((d.cpu().double() - rd).abs() <= 2.0 ** -8 * rd.abs() + 1e-5 * grad.abs().sum(1, keepdim=True).cpu()).all()
    del w, d, leaf

    def f(x):
        w, ids = tb.moe_route(x, 8, renormalize=False)
        return (w * 2).sum(), ids

    x = logits.detach().requires_grad_(True)
    value, ids = torch.compile(f, fullgraph=True)(x)
    value.backward()
    y = logits.detach().requires_grad_(True)
    f(y)[0].backward()
    assert torch.equal(x.grad, y.grad) and torch.equal(ids.cpu(), rids)


def test_ids_feed_the_dispatch_plan():
    """The ids go straight into the package's other expert path; a place without an expert (-1) is skipped there."""
    from tritonblas_b200.distributed import PeerMemoryMoE
    E, H, F, T = 8, 256, 128, 200
    g = torch.Generator(device="cuda").manual_seed(2)
    w1 = (torch.randn(E, 2 * F, H, device="cuda", generator=g) * H ** -0.5).bfloat16()
    w2 = (torch.randn(E, H, F, device="cuda", generator=g) * F ** -0.5).bfloat16()
    x = torch.randn(T, H, device="cuda", generator=g).bfloat16()
    logits = torch.randn(T, E, device="cuda", generator=g)
    logits[:50, 1:] = float("-inf")             # one live expert, topk 2
    w, ids = tb.moe_route(logits, 2)
    assert (ids[:50, 1] == -1).all() and (w[:50, 0] == 1).all() and (w[:50, 1] == 0).all()
    out, _ = PeerMemoryMoE(w1, w2, E, T * 2).forward(x, ids, w)
    h = x[:50].float() @ w1[0].float().T
    ref = (torch.nn.functional.silu(h[:, :F]) * h[:, F:]) @ w2[0].float().T
    # two chained bf16 products: activation and expert output are each rounded to bf16
    assert (out[:50].float() - ref).abs().max() <= 2e-2 * ref.abs().max()
    assert tb.device_status() == 0
