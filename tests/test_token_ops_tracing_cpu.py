"""The per-token operators under fake tensors and tracers: they are registered operators there, as matmul and addmm are, and no
address is asked for. Fake CUDA tensors need no GPU."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx

import tritonblas_b200 as tb
from tritonblas_b200._checks import traced

bf = torch.bfloat16


def cuda(*shape, dtype=bf):
    return torch.empty(*shape, dtype=dtype, device="cuda")


def route_args():
    return cuda(6, 16, dtype=torch.float32), 4


def mlp_args(T=6):
    return cuda(T, 64), cuda(8, 64, 64), cuda(8, 64, 32), cuda(T, 4, dtype=torch.int32), cuda(T, 4, dtype=torch.float32)


def lora_args(T=6):
    return cuda(T, 64), cuda(40, 64).T, cuda(3, 8, 64), cuda(3, 40, 8), cuda(T, dtype=torch.int64), cuda(3, dtype=torch.float32), cuda(40)


def test_plain_tensors_are_not_traced():
    assert not traced(torch.zeros(2)) and not traced(torch.nn.Parameter(torch.zeros(2)))
    with FakeTensorMode():
        assert traced(torch.zeros(2))
    assert torch.func.vmap(lambda t: torch.full_like(t, float(traced(t))))(torch.zeros(2)).all()


def test_fake_tensors():
    with FakeTensorMode():
        w, ids = tb.moe_route(*route_args())
        assert w.shape == ids.shape == (6, 4) and w.dtype == torch.float32 and ids.dtype == torch.int32 and w.is_cuda
        y = tb.moe_mlp(*mlp_args())
        assert y.shape == (6, 64) and y.dtype == bf and y.is_contiguous()
        z = tb.lora_matmul(*lora_args())
        assert z.shape == (6, 40) and z.dtype == bf and z.is_contiguous()
        out = cuda(40, 6).T
        assert tb.lora_matmul(*lora_args(), out=out) is out
        out = cuda(6, 64)
        assert tb.moe_mlp(*mlp_args(), out=out) is out
        logits = cuda(6, 16)
        w, ids = tb.moe_route(logits.requires_grad_(True), 4)
        d = torch.ops.tritonblas._moe_route_backward(logits.detach(), w.detach(), ids, w.detach(), False, True)
        assert w.requires_grad and d.shape == logits.shape and d.dtype == bf


def test_refusals_come_before_the_trace():
    with FakeTensorMode():
        with pytest.raises(ValueError):
            tb.moe_mlp(*mlp_args(T=129))
        x, *rest = lora_args()
        with pytest.raises(ValueError):
            tb.lora_matmul(x[:, :60], *rest)
        with pytest.raises(RuntimeError, match="inference only"):
            tb.lora_matmul(x.requires_grad_(True), *rest)
        with pytest.raises(ValueError):
            tb.moe_route(route_args()[0], 17)


def test_a_traced_decode_step_holds_the_operators():
    def step(x, w, a, b, ids, w1, w2, router):
        h = tb.lora_matmul(x, w, a, b, ids)
        weights, chosen = tb.moe_route(h @ router, 4)
        return tb.moe_mlp(h, w1, w2, chosen, weights)

    with FakeTensorMode():
        args = (cuda(6, 64), cuda(64, 64).T, cuda(3, 8, 64), cuda(3, 64, 8), cuda(6, dtype=torch.int32), cuda(8, 64, 64), cuda(8, 64, 32),
                cuda(64, 8))
        graph = make_fx(step)(*args)
    targets = [str(n.target) for n in graph.graph.nodes]
    assert [t for t in targets if t.startswith("tritonblas")] == ["tritonblas._lora_matmul.default", "tritonblas._moe_route.default",
                                                                  "tritonblas._moe_mlp.default"]


def test_tangents_are_refused():
    """Forward-mode differentiation: none of the operators has a rule, and a result without its tangent would be a wrong one. The
    refusal comes before any call into the library, so fake device checks suffice."""
    from torch.autograd import forward_ad
    from tritonblas_b200._checks import refuse_tangents
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.zeros(3), torch.ones(3))
        refuse_tangents("f", torch.zeros(3), None, torch.zeros(2, dtype=torch.int32))
        with pytest.raises(RuntimeError, match="forward-mode"):
            refuse_tangents("f", None, dual)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda t: refuse_tangents("f", t) or t, (torch.zeros(3),), (torch.ones(3),))


def test_operators_check_what_the_functions_check():
    """Called by name, with host tensors."""
    z = torch.zeros
    with pytest.raises(RuntimeError, match="CUDA"):
        torch.ops.tritonblas._moe_mlp(z(2, 64, dtype=bf), z(4, 64, 64, dtype=bf), z(4, 64, 32, dtype=bf), z(2, 2, dtype=torch.int32), z(2, 2))
    with pytest.raises(ValueError):
        torch.ops.tritonblas._moe_mlp(z(2, 60, dtype=bf), z(4, 64, 64, dtype=bf), z(4, 64, 32, dtype=bf), z(2, 2, dtype=torch.int32), z(2, 2))
    lora = (z(2, 64, dtype=bf), z(40, 64, dtype=bf).T, z(3, 8, 64, dtype=bf), z(3, 40, 8, dtype=bf), z(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        torch.ops.tritonblas._lora_matmul(*lora)
    with pytest.raises(ValueError):
        torch.ops.tritonblas._lora_matmul_out(*lora, z(2, 41, dtype=bf))
