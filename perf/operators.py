"""Cases of the per-token serving operators: the expert router, the expert feed-forward of a few tokens, and the shared
projection with one low-rank adapter per request.

Every case is a dict of plain values. ``prepare`` makes its inputs on the GPU from a seed, ``run`` makes one pass, either in
plain torch operations (``own = False``) or through ``tritonblas_b200`` (``own = True``), ``work`` gives the bytes and
operations a pass cannot do without and ``exact`` the same result in 64 bits.

Operators (``kind``):

``route``  weights, ids = moe_route(logits, topk, scoring, renormalize). The k largest logits of every row, ties to the
           lowest index; their softmax (or sigmoid) scores, optionally divided by their sum. With ``grad`` also the
           gradient of the logits for a given gradient of the weights.
``experts`` out[t] = sum_j weights[t, j] * down_e(silu(gate_e(x_t)) * up_e(x_t)), e = ids[t, j], for a few tokens.
``lora``   out[t] = x[t] @ w + scales[a] * (x[t] @ lora_a[a].T) @ lora_b[a].T (+ bias), a = adapter_ids[t], -1 = none.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # router of one decode step of a small batch: three rows of 64 experts, nothing but latency
        dict(name="route_decode", kind="route", tokens=3, experts=64, topk=8, scoring="softmax", renormalize=True,
             dtype="fp32", grad=False),
        # router of a prefill of 16384 tokens over 64 experts, top-8, renormalised weights
        dict(name="route_prefill", kind="route", tokens=16384, experts=64, topk=8, scoring="softmax", renormalize=True,
             dtype="bf16", grad=False),
        # router of a training step, many experts, softmax without renormalisation: every logit has a gradient
        dict(name="route_train", kind="route", tokens=32771, experts=256, topk=8, scoring="softmax", renormalize=False,
             dtype="bf16", grad=True),
        # one token through 8 of 64 experts: a single user's decode step
        dict(name="experts_1", kind="experts", tokens=1, experts=64, topk=8, hidden=4096, ffn=1536, dtype="bf16"),
        # small experts, a few users: the shortest layer, where launches and waits count most
        dict(name="experts_small", kind="experts", tokens=5, experts=60, topk=4, hidden=2048, ffn=704, dtype="fp16"),
        # a batch of decoding users: most experts are read for one to four tokens each
        dict(name="experts_16", kind="experts", tokens=16, experts=64, topk=8, hidden=4096, ffn=1536, dtype="bf16"),
        # the largest batch of the few-token form: every expert is read
        dict(name="experts_128", kind="experts", tokens=128, experts=64, topk=8, hidden=4096, ffn=1536, dtype="bf16"),
        # one decoding user with an adapter beside a square projection
        dict(name="lora_1", kind="lora", tokens=1, k=4096, n=4096, rank=16, adapters=8, requests=1, bias=False, dtype="bf16"),
        # a decode batch, every user with an adapter of their own, beside a wide projection
        dict(name="lora_48", kind="lora", tokens=48, k=8192, n=28672, rank=16, adapters=32, requests=48, bias=False,
             dtype="bf16"),
        # odd sizes: a ragged mix of short prompts and single tokens, a bias, half precision
        dict(name="lora_ragged", kind="lora", tokens=333, k=2056, n=5000, rank=24, adapters=6, requests=21, bias=True,
             dtype="fp16"),
        # a prefill of eleven prompts with eight adapters
        dict(name="lora_prefill", kind="lora", tokens=4096, k=4096, n=8192, rank=64, adapters=8, requests=11, bias=False,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "lora", "lora"])
    if kind == "route":
        experts = _log_int(rng, 4, 512)
        return dict(kind="route", tokens=_log_int(rng, 1, 32768), experts=experts, topk=rng.randint(1, min(16, experts)),
                    scoring=rng.choice(["softmax", "softmax", "sigmoid"]), renormalize=rng.random() < 0.5,
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), grad=rng.random() < 0.5)
    if kind == "experts":
        while True:
            experts = _log_int(rng, 4, 256)
            hidden, ffn = 8 * _log_int(rng, 32, 1024), 8 * _log_int(rng, 16, 512)
            if experts * hidden * ffn <= 64 * 4096 * 1536:
                break
        return dict(kind="experts", tokens=_log_int(rng, 1, 128), experts=experts, topk=rng.randint(1, min(10, experts)),
                    hidden=hidden, ffn=ffn, dtype=rng.choice(["bf16", "bf16", "fp16"]))
    while True:
        tokens, k, n = _log_int(rng, 1, 8192), 8 * _log_int(rng, 32, 1024), 8 * _log_int(rng, 32, 3584)
        if tokens * k * n <= 4096 * 4096 * 8192:
            break
    return dict(kind="lora", tokens=tokens, k=k, n=n, rank=8 * rng.randint(1, 16), adapters=_log_int(rng, 1, 64),
                requests=min(tokens, _log_int(rng, 1, 96)), bias=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16"]))


# ------------------------------------------------------------------------------------------------------------ the inputs
def _used_experts(case):
    """Experts that at least one token is routed to: the expected number for even routing, which the inputs meet exactly."""
    e, k, t = case["experts"], case["topk"], case["tokens"]
    return max(k, min(e, t * k, round(e * (1.0 - (1.0 - k / e) ** t))))


def _request_adapters(case):
    """Slot in a permutation of the adapters of every request; every seventh request uses the bare projection."""
    return [(-1 if i % 7 == 6 else i % case["adapters"]) for i in range(case["requests"])]


def _used_adapters(case):
    return len({a for a in _request_adapters(case) if a >= 0})


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def prepare(case, seed):
    g = _gen(seed)
    dt = _DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g).mul_(scale).to(dt)

    def weights(*shape, scale):     # large weights are filled matrix by matrix, in their own type
        w = torch.empty(*shape, device="cuda", dtype=dt)
        for part in w:
            part.copy_(torch.randn(part.shape, device="cuda", dtype=torch.float32, generator=g).mul_(scale))
        return w

    st = {"case": dict(case)}
    if case["kind"] == "route":
        # expert popularity plus per-token preference; every 50th row masks half of its experts (-inf), one expert is a tie
        logits = torch.randn(case["tokens"], case["experts"], device="cuda", generator=g) * 1.5
        logits += torch.randn(case["experts"], device="cuda", generator=g)
        rows = torch.arange(case["tokens"], device="cuda").unsqueeze(1)
        cols = torch.arange(case["experts"], device="cuda").unsqueeze(0)
        logits.masked_fill_((rows % 50 == 49) & (cols % 2 == 1), float("-inf"))
        st["logits"] = logits.to(dt)
        st["logits"][:, -1] = st["logits"][:, 0]
        if case["grad"]:
            st["grad"] = torch.randn(case["tokens"], case["topk"], device="cuda", generator=g)
    elif case["kind"] == "experts":
        t, e, k, h, f = (case[n] for n in ("tokens", "experts", "topk", "hidden", "ffn"))
        st["x"] = randn(t, h)
        st["w1"] = weights(e, 2 * f, h, scale=h ** -0.5)
        st["w2"] = weights(e, h, f, scale=f ** -0.5)
        used = _used_experts(case)
        subset = torch.randperm(e, device="cuda", generator=g)[:used]
        score = torch.rand(t, used, device="cuda", generator=g)
        a = torch.arange(used, device="cuda")
        score[a % t, a] += 2.0          # every used expert is some token's choice
        st["ids"] = subset[score.topk(k, dim=1).indices].to(torch.int32)
        st["weights"] = torch.softmax(torch.randn(t, k, device="cuda", generator=g), dim=1)
    else:
        t, k, n, r, l = (case[q] for q in ("tokens", "k", "n", "rank", "adapters"))
        st["x"] = randn(t, k)
        st["w"] = randn(n, k, scale=k ** -0.5).T        # K contiguous, the layout weights are stored in
        st["lora_a"] = weights(l, r, k, scale=k ** -0.5)
        st["lora_b"] = weights(l, n, r, scale=0.3 * r ** -0.5)
        st["scales"] = torch.rand(l, device="cuda", generator=g) + 0.5
        st["bias"] = randn(n, scale=0.1) if case["bias"] else None
        perm = torch.randperm(l, device="cuda", generator=g)
        req = torch.tensor(_request_adapters(case), device="cuda")
        req = torch.where(req >= 0, perm[req.clamp(min=0)], req)
        # ragged requests: every one has a row, the other rows go to random requests; a request's rows stand together
        extra = torch.randint(0, case["requests"], (t - case["requests"],), device="cuda", generator=g)
        owner = torch.sort(torch.cat([torch.arange(case["requests"], device="cuda"), extra])).values
        st["adapter_ids"] = req[owner].to(torch.int32)
    return st


# ------------------------------------------------------------------------------------------------------- the plain forms
def _route_plain(logits, topk, scoring, renormalize, grad):
    l = logits.to(torch.float32)
    live = l > float("-inf")
    l = torch.where(live, l, torch.full_like(l, float("-inf")))
    order = torch.sort(l, dim=1, descending=True, stable=True).indices[:, :topk]
    sel_live = torch.gather(live, 1, order)
    ids = torch.where(sel_live, order, torch.full_like(order, -1)).to(torch.int32)
    if scoring == "softmax":
        top = l.max(dim=1, keepdim=True).values
        top = torch.where(top > float("-inf"), top, torch.zeros_like(top))
        ex = torch.exp(l - top)
        p = ex / ex.sum(dim=1, keepdim=True).clamp(min=1e-30)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    s = torch.gather(p, 1, order) * sel_live
    total = s.sum(dim=1, keepdim=True)
    w = s / torch.where(total > 0, total, torch.ones_like(total)) if renormalize else s
    if grad is None:
        return {"weights": w, "ids": ids}
    gs = grad * sel_live
    if renormalize:             # gradient of the scores of the chosen experts
        gs = (gs - (gs * w).sum(dim=1, keepdim=True)) / torch.where(total > 0, total, torch.ones_like(total)) * sel_live
    full = torch.zeros_like(l).scatter_(1, order, gs)
    if scoring == "softmax":
        dl = p * (full - (full * p).sum(dim=1, keepdim=True))
    else:
        dl = full * p * (1.0 - p)
    return {"weights": w, "ids": ids, "dlogits": dl.to(logits.dtype)}


def _experts_plain(x, w1, w2, ids, weights):
    t, k = ids.shape
    ffn = w2.shape[2]
    xf = x.to(torch.float32)
    out = torch.zeros(t, w2.shape[1], device=x.device, dtype=torch.float32)
    if t * k < w1.shape[0]:     # fewer choices than experts: one after the other
        for i in range(t):
            for j in range(k):
                e = ids[i, j].long().unsqueeze(0)
                h = w1.index_select(0, e)[0].to(torch.float32) @ xf[i]
                act = h[:ffn] / (1.0 + torch.exp(-h[:ffn])) * h[ffn:]
                out[i] += weights[i, j] * (w2.index_select(0, e)[0].to(torch.float32) @ act)
    else:
        for e in range(w1.shape[0]):
            h = xf @ w1[e].to(torch.float32).T
            act = h[:, :ffn] / (1.0 + torch.exp(-h[:, :ffn])) * h[:, ffn:]
            share = (weights * (ids == e)).sum(dim=1, keepdim=True)
            out += share * (act @ w2[e].to(torch.float32).T)
    return out.to(x.dtype)


def _lora_plain(x, w, lora_a, lora_b, ids, scales, bias):
    xf = x.to(torch.float32)
    y = xf @ w.to(torch.float32)
    for a in range(lora_a.shape[0]):
        low = (xf * (ids == a).unsqueeze(1)) @ lora_a[a].to(torch.float32).T
        y += (low * scales[a]) @ lora_b[a].to(torch.float32).T
    if bias is not None:
        y += bias.to(torch.float32)
    return y.to(x.dtype)


def run(state):
    case = state["case"]
    if case["kind"] == "route":
        grad = state.get("grad")
        if not own:
            return _route_plain(state["logits"], case["topk"], case["scoring"], case["renormalize"], grad)
        import tritonblas_b200 as tb
        if grad is None:
            w, ids = tb.moe_route(state["logits"], case["topk"], scoring=case["scoring"], renormalize=case["renormalize"])
            return {"weights": w, "ids": ids}
        logits = state["logits"].detach().requires_grad_(True)
        w, ids = tb.moe_route(logits, case["topk"], scoring=case["scoring"], renormalize=case["renormalize"])
        (dl,) = torch.autograd.grad(w, logits, grad)
        return {"weights": w.detach(), "ids": ids, "dlogits": dl}
    if case["kind"] == "experts":
        if not own:
            return _experts_plain(state["x"], state["w1"], state["w2"], state["ids"], state["weights"])
        import tritonblas_b200 as tb
        return tb.moe_mlp(state["x"], state["w1"], state["w2"], state["ids"], state["weights"])
    if not own:
        return _lora_plain(state["x"], state["w"], state["lora_a"], state["lora_b"], state["adapter_ids"], state["scales"],
                           state["bias"])
    import tritonblas_b200 as tb
    return tb.lora_matmul(state["x"], state["w"], state["lora_a"], state["lora_b"], state["adapter_ids"],
                          scales=state["scales"], bias=state["bias"])


# -------------------------------------------------------------------------------------------------------------- the work
def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    t = case["tokens"]
    if case["kind"] == "route":
        e, k = case["experts"], case["topk"]
        nbytes, flops = t * e * es + t * k * 8, t * e * 5
        if case["grad"]:
            nbytes += t * k * 4 + t * e * es        # the weights' gradient in, the logits' gradient out
            flops += t * e * 4
        return {"bytes": nbytes, "flops": flops}
    if case["kind"] == "experts":
        k, h, f = case["topk"], case["hidden"], case["ffn"]
        return {"bytes": _used_experts(case) * 3 * f * h * es + 2 * t * h * es + t * k * 8, "flops": t * k * 6 * f * h}
    k, n, r = case["k"], case["n"], case["rank"]
    with_adapter = sum(1 for a in _request_adapters(case) if a >= 0) / case["requests"]
    return {"bytes": (k * n + _used_adapters(case) * r * (k + n) + t * (k + n) + (n if case["bias"] else 0)) * es + t * 4,
            "flops": 2 * t * k * n + 2 * int(t * with_adapter) * r * (k + n)}


# --------------------------------------------------------------------------------------------------- the 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["kind"] == "route":
        l = st["logits"].to(f64)
        t, e = l.shape
        k = case["topk"]
        ninf = float("-inf")
        # rank of every entry: how many entries stand before it (larger, or equal with a lower index), by an index-broken sort
        key, idx = torch.sort(-l, dim=1, stable=True)
        top_l, ids = -key[:, :k], idx[:, :k]
        dead = top_l == ninf
        if case["scoring"] == "softmax":
            lse = torch.logsumexp(l, dim=1, keepdim=True)
            score, p = torch.exp(top_l - lse), torch.exp(l - lse)
        else:
            score, p = torch.sigmoid(top_l), torch.sigmoid(l)
        score = score.masked_fill(dead, 0.0)
        tot = score.sum(1, keepdim=True)
        w = score / tot if case["renormalize"] else score
        res = {"weights": w, "ids": ids.masked_fill(dead, -1)}
        if case["grad"]:
            g = st["grad"].to(f64).masked_fill(dead, 0.0)
            dense = torch.zeros(t, e, dtype=f64, device=l.device)
            if case["scoring"] == "softmax" and case["renormalize"]:
                # softmax over the chosen logits alone
                dense.scatter_(1, ids, w * (g - (g * w).sum(1, keepdim=True)))
            elif case["scoring"] == "softmax":
                dense.scatter_(1, ids, g * score)
                dense -= p * (g * score).sum(1, keepdim=True)
            else:
                if case["renormalize"]:
                    g = (g - (g * w).sum(1, keepdim=True)) / tot
                dense.scatter_(1, ids, g * score * (1.0 - score))
            res["dlogits"] = dense
        return res
    if case["kind"] == "experts":
        x, w1, w2, ids, wt = (st[n] for n in ("x", "w1", "w2", "ids", "weights"))
        f = w2.shape[2]
        out = torch.zeros(x.shape, dtype=f64, device=x.device)
        for e in torch.unique(ids).tolist():
            tok, slot = (ids == e).nonzero(as_tuple=True)
            h = torch.einsum("th,fh->tf", x[tok].to(f64), w1[e].to(f64))
            act = h[:, :f] * torch.sigmoid(h[:, :f]) * h[:, f:]
            out.index_add_(0, tok, torch.einsum("tf,hf->th", act, w2[e].to(f64)) * wt[tok, slot].to(f64).unsqueeze(1))
        return out
    y = torch.einsum("tk,kn->tn", st["x"].to(f64), st["w"].to(f64))
    for a in torch.unique(st["adapter_ids"]).tolist():
        if a < 0:
            continue
        rows = (st["adapter_ids"] == a).nonzero().squeeze(1)
        low = torch.einsum("tk,rk->tr", st["x"][rows].to(f64), st["lora_a"][a].to(f64)) * st["scales"][a].to(f64)
        y[rows] += torch.einsum("tr,nr->tn", low, st["lora_b"][a].to(f64))
    if st["bias"] is not None:
        y += st["bias"].to(f64)
    return y
