"""The per-token operators through torch.compile, torch.export, torch.func and forward-mode differentiation on the GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad

import tritonblas_b200 as tb
from tests.test_lora_gpu import make as make_lora
from tests.test_moe_mlp_gpu import make as make_experts

pytestmark = pytest.mark.gpu


class Step(torch.nn.Module):
    """A decode step: projection with adapters, router product, router, experts."""

    def __init__(self, T=12, H=256, F=128, E=16):
        super().__init__()
        self.x, w, a, b, ids, s = make_lora(T, H, H, 16, 5, torch.bfloat16)
        _, w1, w2, _, _ = make_experts(T, E, 4, H, F, torch.bfloat16)
        g = torch.Generator(device="cuda").manual_seed(1)
        router = (torch.randn(E, H, device="cuda", generator=g) * H ** -0.5).bfloat16()
        for name, t in dict(w=w, a=a, b=b, ids=ids, s=s, w1=w1, w2=w2, router=router).items():
            self.register_buffer(name, t)

    def forward(self, x):
        h = tb.lora_matmul(x, self.w, self.a, self.b, self.ids, scales=self.s)
        weights, chosen = tb.moe_route(tb.matmul(h, self.router.T), 4)
        return h, chosen, tb.moe_mlp(h, self.w1, self.w2, chosen, weights)


def test_compiled_and_exported_decode_step():
    step = Step()
    want = step(step.x)
    got = torch.compile(step, fullgraph=True)(step.x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    program = torch.export.export(step, (step.x,))
    assert all(torch.equal(a, b) for a, b in zip(program.module()(step.x), want))
    names = {str(n.target) for n in program.graph.nodes}
    assert {"tritonblas._lora_matmul.default", "tritonblas._moe_route.default", "tritonblas._moe_mlp.default"} <= names
    assert tb.device_status() == 0


def test_compiled_calls_with_out():
    x, w, a, b, ids, s = make_lora(20, 256, 256, 16, 5, torch.bfloat16)
    _, w1, w2, eids, ew = make_experts(20, 8, 2, 256, 128, torch.bfloat16)
    want = tb.lora_matmul(x, w, a, b, ids, s)
    want2 = tb.moe_mlp(want, w1, w2, eids, ew)

    def f(x, out, y):
        tb.lora_matmul(x, w, a, b, ids, s, out=out)
        tb.moe_mlp(out, w1, w2, eids, ew, out=y)
        return out + 0

    out, y = torch.zeros(256, 20, dtype=x.dtype, device="cuda").T, torch.zeros_like(x)
    assert torch.equal(torch.compile(f, fullgraph=True)(x, out, y), want) and torch.equal(out, want) and torch.equal(y, want2)


def test_registrations():
    check = torch.library.opcheck
    check(torch.ops.tritonblas._moe_mlp.default, make_experts(6, 8, 2, 64, 64, torch.bfloat16))
    x, w, a, b, ids, s = make_lora(6, 64, 40, 8, 3, torch.bfloat16)
    check(torch.ops.tritonblas._lora_matmul.default, (x, w, a, b, ids, s, torch.randn(40, device="cuda")))
    check(torch.ops.tritonblas._lora_matmul.default, (x, w, a, b, ids))
    check(torch.ops.tritonblas._lora_matmul_out.default, (x, w, a, b, ids, torch.empty(6, 40, dtype=x.dtype, device="cuda"), s))
    e = make_experts(6, 8, 2, 64, 64, torch.bfloat16)
    check(torch.ops.tritonblas._moe_mlp_out.default, (*e, torch.empty_like(e[0])))
    check(torch.ops.tritonblas._moe_route.default, (torch.randn(6, 16, device="cuda", requires_grad=True), 4, False, True))


def test_transforms_and_tangents():
    l = torch.randn(6, 16, device="cuda")
    with FakeTensorMode() as mode:
        fake = mode.from_tensor(l).requires_grad_(True)
        (d,) = torch.autograd.grad(tb.moe_route(fake, 4)[0].sum(), fake)
        assert d.shape == l.shape
    with pytest.raises(RuntimeError):           # registered operators have no torch.func rule (matmul's neither): said, not dropped
        torch.func.grad(lambda t: tb.moe_route(t, 4)[0][:, 0].sum())(l)
    case, experts = make_lora(6, 64, 40, 8, 3, torch.bfloat16), make_experts(6, 8, 2, 64, 64, torch.bfloat16)
    calls = (lambda t: tb.moe_route(t.float(), 4)[0], lambda t: tb.lora_matmul(t, *case[1:]), lambda t: tb.moe_mlp(t, *experts[1:]))
    for f in calls:
        t = torch.randn(6, 64, device="cuda").bfloat16()
        with forward_ad.dual_level():
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(forward_ad.make_dual(t, torch.ones_like(t)))
        with pytest.raises((RuntimeError, NotImplementedError)):
            torch.func.jvp(f, (t,), (torch.ones_like(t),))
        f(t)
