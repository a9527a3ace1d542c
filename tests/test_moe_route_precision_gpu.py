"""Router weights and gradients element by element, relative to what each element is made of.

Bounds, in half units u = 2^-24 of fp32 arithmetic. An exponential exp(l - m) is off by its argument's rounding (computed exactly
below: zero where both are short) and 4 u; a row's sum by the mean of those and a half unit per addition (as many as a lane holds
logits, 8 to 32, and five exchanges), a quotient by u and a product by u: argument + (11 + additions) u covers a softmax score. A sigmoid 1 / (1 + exp(-l)) or its complement
is off by 8 u, a sum of topk of them by topk u more. A gradient term g w - p dot or w (g - dot) is off by what its factors are,
dot by the sum of what |g w| are off and (topk + 2) u, and the result by half a step of its type."""
import pytest
import torch

import tritonblas_b200 as tb

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
MODES = [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)]


def expected(logits, topk, scoring, renormalize, grad):
    """(ids, weights, their bound, gradient, its bound) in 64 bits."""
    l32 = logits.detach().float().cpu()
    l32 = torch.where(torch.isnan(l32), torch.full_like(l32, float("-inf")), l32)
    l = l32.double()
    order = torch.argsort(-l, dim=1, stable=True)[:, :topk]
    dead = torch.gather(l, 1, order) == float("-inf")
    g = grad.double().cpu().masked_fill(dead, 0.0)
    pick = lambda t: torch.gather(t, 1, order).masked_fill(dead, 0.0)
    if scoring == "softmax":
        top = l32.max(1, keepdim=True).values
        top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
        off = torch.nan_to_num(((l32 - top).double() - (l - top.double())).abs())        # the argument's rounding
        p = torch.exp(l - top.double())
        if renormalize:
            s, so = pick(p), pick(off)
            w = s / s.sum(1, keepdim=True).clamp(min=1e-300)
            rel = so + so.max(1, keepdim=True).values + (topk + 32) * U
        else:
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            adds = (8 if logits.shape[1] <= 256 else 16 if logits.shape[1] <= 512 else 32) + 5
            rel_p = off + (p * off).sum(1, keepdim=True) + (11 + adds) * U
            w, rel = pick(p), pick(rel_p)
    else:
        s = torch.sigmoid(l)
        comp = pick(torch.sigmoid(-l))
        w, rel = pick(s), torch.full_like(g, 8 * U)
        if renormalize:
            # the scores' common factor cancels: the quotient stays good where the scores themselves are too small for fp32
            t = pick(torch.nn.functional.logsigmoid(l))
            t = torch.exp(t - t.masked_fill(dead, float("-inf")).max(1, keepdim=True).values.nan_to_num(neginf=0.0)).masked_fill(dead, 0.0)
            w = t / t.sum(1, keepdim=True).clamp(min=1e-300)
            m32 = torch.gather(l32, 1, order[:, :1])
            args = ((m32 - torch.gather(l32, 1, order)).double() - (m32.double() - torch.gather(l, 1, order))).abs().nan_to_num(0.0, 0.0, 0.0)
            rel = torch.where(m32 < 0, args + args.max(1, keepdim=True).values, torch.zeros_like(args)) + (topk + 40) * U
    dot = (g * w).sum(1, keepdim=True)
    ddot = (g * w).abs().mul(rel + (topk + 2) * U).sum(1, keepdim=True)
    if scoring == "softmax" and not renormalize:
        term, dterm = g * w, (g * w).abs() * (rel + 2 * U)
        d = (torch.zeros_like(l).scatter_(1, order, term) - p * dot)
        b = torch.zeros_like(l).scatter_(1, order, dterm) + p * ((rel_p + 3 * U) * dot.abs() + ddot)
    else:
        c = comp if scoring == "sigmoid" else torch.ones_like(w)
        inner, dinner = (g - dot, ddot + 2 * U * (g.abs() + dot.abs())) if renormalize else (g, torch.zeros_like(g))
        term = w * c * inner
        d = torch.zeros_like(l).scatter_(1, order, term.masked_fill(dead, 0.0))
        b = torch.zeros_like(l).scatter_(1, order, (w * c * dinner + term.abs() * (rel + 12 * U)).masked_fill(dead, 0.0))
    f = torch.finfo(logits.dtype)
    small = 2.0 ** -125         # exponentials below fp32's normal numbers
    b = b + f.eps / 2 * d.abs() + f.smallest_normal * f.eps / 2 + small * g.abs().sum(1, keepdim=True)
    return order.masked_fill(dead, -1).to(torch.int32), w, rel * w + small, d, b


def check(logits, topk, scoring, renormalize, seed=0):
    grad = torch.randn(logits.shape[0], topk, generator=torch.Generator().manual_seed(seed)).cuda()
    x = logits.detach().requires_grad_(True)
    w, ids = tb.moe_route(x, topk, scoring=scoring, renormalize=renormalize)
    (dl,) = torch.autograd.grad(w, x, grad)
    rids, rw, bw, rd, bd = expected(x, topk, scoring, renormalize, grad)
    assert torch.equal(ids.cpu(), rids)
    err = (w.detach().cpu().double() - rw).abs()
    assert (err <= bw).all(), f"weights: worst err / bound {float((err / bw).max()):.3g}"
    err = (dl.cpu().double() - rd).abs()
    assert (err <= bd).all(), f"gradient: worst err / bound {float((err / bd).max()):.3g} at {divmod(int((err / bd).argmax()), rd.shape[1])}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renormalize", [True, False])
def test_saturated_sigmoid_scores_keep_their_gradient(dtype, renormalize):
    """1 - s of a score next to 1 is exp(-l): it has no bits left in a rounded s."""
    g = torch.Generator().manual_seed(3)
    logits = (torch.rand(50, 40, generator=g) * 10 + 10).to(dtype).cuda()
    logits[:, ::2] -= 16
    check(logits, 6, "sigmoid", renormalize)
    x = torch.full((1, 4), 18.0, device="cuda", requires_grad=True)
    (d,) = torch.autograd.grad(tb.moe_route(x, 1, scoring="sigmoid", renormalize=False)[0].sum(), x)
    assert 1.4e-8 < float(d[0, 0]) < 1.6e-8         # e^-18


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("low", [-60.0, -95.0, -3e4])
def test_renormalised_sigmoid_of_very_negative_logits(dtype, low):
    """The scores of such a row are too small for fp32, their quotients are exponentials of differences."""
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(30, 24, generator=g) * 3 + low
    logits[::3, 5] = 2.0                                    # rows with one large score among them
    logits[4] = float("-inf")
    logits[6, 3:] = float("-inf")
    logits[8] = torch.finfo(dtype).min                      # a row of the type's lowest value: all alike
    logits = logits.to(dtype).cuda()
    check(logits, 6, "sigmoid", True)
    w, ids = tb.moe_route(logits, 6, scoring="sigmoid")
    live = (ids >= 0).any(1)
    # six quotients, each within (topk + 40) u plus its arguments' roundings, at most 2^-8 where logits are near 3e4 and fp32
    assert ((w.sum(1) - 1).abs()[live] <= 1e-2).all() and torch.allclose(w[8], torch.full((6,), 1 / 6, device="cuda"))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("experts", [24, 64, 200])
def test_small_softmax_scores(dtype, experts):
    """Scores down to exp(-80) of the largest: the error of an exponential does not grow with its distance from the maximum. The
    logits are multiples of 1/4, so their differences are exact."""
    g = torch.Generator().manual_seed(experts)
    logits = (torch.rand(40, experts, generator=g) * 320).round() / 4 - 40
    check(logits.to(dtype).cuda(), 7, "softmax", False)


def test_the_error_of_a_small_score_does_not_grow_with_its_distance():
    """One score of 1 and a tail that vanishes beside it: weight and sum are exactly 1, and d_i = -exp(l_i - l_0) is an exponential
    of an exact argument, good to 4 u, times two factors of 1."""
    logits = (-torch.arange(0, 84 * 64, 1).double() / 64).view(84, 64)[25:80].float().cuda()        # 25 to 80, in steps of 1/64
    logits[:, 0] = 0.0
    x = logits.requires_grad_(True)
    w, ids = tb.moe_route(x, 1, renormalize=False)
    assert (w == 1).all() and (ids == 0).all()
    (d,) = torch.autograd.grad(w.sum(), x)
    want = -torch.exp(logits.detach().double())[:, 1:]
    assert ((d.double()[:, 1:] - want).abs() <= 4 * U * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scoring,renormalize", MODES)
@pytest.mark.parametrize("tokens,experts,topk,offset", [(5, 24, 3, 0), (70, 100, 8, 1), (9, 256, 32, 0), (3, 257, 8, 0), (40, 300, 10, 0), (7, 304, 32, 0),
                                                        (33, 304, 4, 1), (6, 512, 8, 0), (4, 512, 1, 3), (5, 520, 9, 0), (3, 1000, 10, 0), (2, 1024, 32, 0),
                                                        (9, 1024, 2, 1)])
def test_every_width(tokens, experts, topk, offset, dtype, scoring, renormalize):
    """All lane counts, 8, 16 and 32 logits a lane, runs of eight and single elements (odd sizes, or a base that is `offset`
    elements behind a 16-byte boundary)."""
    g = torch.Generator().manual_seed(experts + topk)
    logits = torch.randn(tokens, experts, generator=g) * 2
    logits[torch.rand(tokens, experts, generator=g) < 0.05] = float("-inf")
    logits[-1] = 0.5
    logits[tokens // 2, 1:] = float("nan")
    buf = torch.empty(tokens * experts + offset, dtype=dtype, device="cuda")
    view = buf[offset:].view(tokens, experts)
    view.copy_(logits.to(dtype))
    check(view, topk, scoring, renormalize, seed=experts)
    if scoring == "softmax" and not renormalize:
        # the bound sees the gradient of the experts that were not chosen: without it the expectation itself is outside
        _, _, _, d, b = expected(view, topk, scoring, renormalize, torch.randn(tokens, topk, generator=torch.Generator().manual_seed(experts)))
        ids = tb.moe_route(view, topk)[1].cpu().long()
        kept = torch.zeros_like(d).scatter_(1, ids.clamp(min=0), 1.0)
        missing = (d.abs() > b) & (kept == 0)
        assert missing.sum() > 0.5 * ((kept == 0) & (view.cpu().float() > float("-inf"))).sum()


@pytest.mark.parametrize("scoring,renormalize", MODES)
@pytest.mark.parametrize("experts", [300, 1000])
def test_wide_rows_against_differences(experts, scoring, renormalize):
    """Central differences in 64 bits at fixed choices. Step 1e-4: truncation h^2 / 6 times a third derivative of at most 1, and
    cancellation 2^-53 / h; the kernel's own error is a few hundred u of sums of |g| times weights."""
    g = torch.Generator().manual_seed(experts)
    x = (torch.randn(2, experts, generator=g) * 1.5).cuda().requires_grad_(True)
    grad = torch.randn(2, 6, generator=g).cuda()
    w, ids = tb.moe_route(x, 6, scoring=scoring, renormalize=renormalize)
    (dl,) = torch.autograd.grad(w, x, grad)

    def value(l):
        p = torch.softmax(l, -1) if scoring == "softmax" else torch.sigmoid(l)
        s = torch.gather(p, -1, ids.long().expand(l.shape[0], 2, 6))
        if renormalize:
            s = s / s.sum(-1, keepdim=True)
        return (s * grad.double()).sum(-1)

    h = 1e-4
    step = torch.eye(experts, dtype=torch.float64, device="cuda").unsqueeze(1) * h
    l = x.detach().double().unsqueeze(0)
    d = ((value(l + step) - value(l - step)) / (2 * h)).T
    scale = (grad.double() * w.detach().double()).abs().sum(1, keepdim=True)
    assert ((dl.double() - d).abs() <= 3e-8 + 300 * U * scale).all()
    assert (d.abs() > 3e-8 + 300 * U * scale).sum() > (experts if scoring == "softmax" and not renormalize else 8)
