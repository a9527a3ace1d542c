"""Host side of the per-token operators: which device their library calls are made on, and how long batches are cut."""
import contextlib

import pytest
import torch

import tritonblas_b200 as tb
from tritonblas_b200 import _lib, lora, moe
from tests.test_lora_gpu import check, make
from tests.test_moe_mlp_gpu import make as make_experts

pytestmark = pytest.mark.gpu


class Spy:
    """The library with every call of the operators recorded: its name, whether the tensors' device had been made current, and the
    rows and workspace of a tb_lora_args."""

    def __init__(self, monkeypatch):
        self.calls, self.inside, self.real = [], 0, _lib.lib
        for module in (lora, moe):
            monkeypatch.setattr(module, "on_device", self.on_device)
        monkeypatch.setattr(_lib, "lib", self)

    @contextlib.contextmanager
    def on_device(self, device):
        self.inside += 1
        yield
        self.inside -= 1

    def __getattr__(self, name):
        f = getattr(self.real, name)

        def call(*args):
            a = getattr(args[0], "_obj", None)
            self.calls.append((name, self.inside > 0, getattr(a, "m", None), getattr(a, "workspace_bytes", None)))
            return f(*args)
        return call


def test_every_call_that_goes_by_the_device_is_made_on_it(monkeypatch):
    """With one GPU the order of the calls is what can be seen: nothing asks for a plan before the tensors' device is current."""
    cases = [make(T, 128, 256, 8, 3, torch.bfloat16) for T in (5, 300)]
    experts = make_experts(4, 4, 2, 64, 64, torch.bfloat16)
    spy = Spy(monkeypatch)
    for c in cases:
        tb.lora_matmul(*c)
    tb.moe_mlp(*experts)
    logits = torch.randn(4, 8, device="cuda", requires_grad=True)
    tb.moe_route(logits, 2)[0].sum().backward()
    names = {c[0] for c in spy.calls}
    assert {"tb_lora_workspace_bytes", "tb_lora_gemm", "tb_moe_mlp", "tb_moe_route", "tb_moe_route_backward"} <= names
    free = {"tb_moe_mlp_workspace_bytes"}           # sizes alone decide it
    assert all(inside for name, inside, _, _ in spy.calls if name not in free)


def test_a_cut_batch_ends_in_the_decode_form_with_a_larger_workspace(monkeypatch):
    case = make(1044, 128, 2048, 8, 30, torch.bfloat16)
    bias = torch.randn(2048, device="cuda")
    spy = Spy(monkeypatch)
    tb.lora_matmul(*case, bias=bias)
    assert [c[2] for c in spy.calls if c[0] == "tb_lora_gemm"] == [1044]
    tb.lora_matmul(case[0][:512], *case[1:4], case[4][:512], case[5])
    half = [c[3] for c in spy.calls if c[0] == "tb_lora_gemm"][-1]
    del spy.calls[:]
    monkeypatch.setattr(lora, "_MAX_WORKSPACE", half)
    out = torch.full((1044, 2056), 7.0, dtype=torch.bfloat16, device="cuda")
    for layout in (out[:, 4:2052], out[:, 8:2056].T.contiguous().T):
        got = tb.lora_matmul(*case, bias=bias, out=layout)
        check(got, *case[:5], scales=case[5], bias=bias)
    assert (out[:, :4] == 7.0).all() and (out[:, 2052:] == 7.0).all()
    runs = [c for c in spy.calls if c[0] == "tb_lora_gemm"]
    assert [c[2] for c in runs] == [512, 512, 20] * 2 and runs[2][3] > runs[0][3] == half
