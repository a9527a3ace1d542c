"""Argument checks of the per-token operators, which come before any CUDA call, so they are tested without a GPU."""
import ctypes

import pytest
import torch

import tritonblas_b200 as tb
from tritonblas_b200 import _lib

bf = torch.bfloat16


def test_router_refusals():
    l = torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        tb.moe_route(l, 2)
    for bad in (lambda: tb.moe_route(l[0], 2), lambda: tb.moe_route(l, 0), lambda: tb.moe_route(l, 9),
                lambda: tb.moe_route(l, 2, scoring="max"), lambda: tb.moe_route(l.double(), 2), lambda: tb.moe_route(l.long(), 2),
                lambda: tb.moe_route(torch.randn(4, 1025), 2), lambda: tb.moe_route(torch.randn(4, 64), 33),
                lambda: tb.moe_route(torch.randn(4, 0), 1)):
        with pytest.raises(ValueError):
            bad()


def test_router_operators_refuse_host_tensors_and_shapes():
    """Traced code reaches the router through custom operators, which check what the plain function checks."""
    l = torch.randn(4, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        torch.ops.tritonblas._moe_route(l, 2, False, True)
    w, i = torch.zeros(4, 2), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        torch.ops.tritonblas._moe_route_backward(l, w, i, w, False, True)


def mlp_case(T=4, E=4, K=2, H=64, F=32, dtype=bf):
    return [torch.zeros(T, H, dtype=dtype), torch.zeros(E, 2 * F, H, dtype=dtype), torch.zeros(E, H, F, dtype=dtype),
            torch.zeros(T, K, dtype=torch.int32), torch.zeros(T, K)]


def test_expert_layer_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        tb.moe_mlp(*mlp_case())
    with pytest.raises(ValueError, match="PeerMemoryMoE"):
        tb.moe_mlp(*mlp_case(T=129))
    for kw in (dict(H=60), dict(F=20), dict(K=33), dict(dtype=torch.float32), dict(E=0)):
        with pytest.raises(ValueError):
            tb.moe_mlp(*mlp_case(**kw))
    for i, t in ((0, torch.zeros(4, 72, dtype=bf)), (1, torch.zeros(4, 32, 64, dtype=bf)), (2, torch.zeros(3, 64, 32, dtype=bf)),
                 (2, torch.zeros(4, 64, 32, dtype=torch.float16)), (3, torch.zeros(4, 2)), (3, torch.zeros(3, 2, dtype=torch.int32)),
                 (4, torch.zeros(4, 1)), (4, torch.zeros(4, 2, dtype=torch.int32))):
        case = mlp_case()
        case[i] = t
        with pytest.raises(ValueError):
            tb.moe_mlp(*case)


def lora_case(T=4, K=64, N=40, R=8, L=3, dtype=bf):
    return [torch.zeros(T, K, dtype=dtype), torch.zeros(N, K, dtype=dtype).T, torch.zeros(L, R, K, dtype=dtype),
            torch.zeros(L, N, R, dtype=dtype), torch.zeros(T, dtype=torch.int32)]


def test_adapter_projection_refusals():
    with pytest.raises(RuntimeError, match="CUDA"):
        tb.lora_matmul(*lora_case())
    for kw in (dict(K=60), dict(R=4), dict(R=136), dict(R=20), dict(L=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            tb.lora_matmul(*lora_case(**kw))
    for i, t in ((0, torch.zeros(4, 72, dtype=bf)), (1, torch.zeros(64, 41, dtype=bf)), (1, torch.zeros(64, 40, dtype=torch.float16)),
                 (2, torch.zeros(2, 8, 64, dtype=bf)), (3, torch.zeros(3, 40, 16, dtype=bf)), (4, torch.zeros(4)),
                 (4, torch.zeros(5, dtype=torch.int32)), (4, torch.zeros(4, 1, dtype=torch.int32))):
        case = lora_case()
        case[i] = t
        with pytest.raises(ValueError):
            tb.lora_matmul(*case)
    for kw in (dict(scales=torch.ones(4)), dict(scales=torch.ones(3, dtype=torch.int32)), dict(bias=torch.ones(41)),
               dict(bias=torch.ones(40, dtype=torch.float64)), dict(out=torch.zeros(4, 41, dtype=bf)), dict(out=torch.zeros(4, 40))):
        with pytest.raises(ValueError):
            tb.lora_matmul(*lora_case(), **kw)


def test_adapter_projection_c_entry_refusals():
    lib = _lib.lib

    def call(**kw):
        a = _lib.LoraArgs(4, 40, 64, 8, 3, _lib.BF16, 256, 64, 256, 1, 64, 256, 512, 64, 256, 320, 8, 256, 0, 0, 0, 256, 40, 1, 256,
                          1 << 30, 0, 0, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.tb_lora_gemm(ctypes.byref(a), None)

    assert call(m=0) == 0 and call(n=0) == 0
    for kw in (dict(m=-1), dict(k=60), dict(k=0), dict(rank=4), dict(rank=136), dict(num_adapters=0), dict(x=None), dict(w=None),
               dict(lora_a=None), dict(lora_b=None), dict(adapter_ids=None), dict(out=None), dict(x_row_stride=56),
               dict(lora_a_row_stride=56), dict(lora_b_row_stride=0), dict(w_stride_k=2, w_stride_n=2)):
        assert call(**kw) == 1, kw
    assert call(dtype=_lib.F32) == 2
    assert call(x=264) == 3 and call(lora_a=258) == 3 and call(x_row_stride=68) == 3 and call(adapter_ids=258) == 3 and call(scales=257) == 3
    assert call(workspace=None, x=256) in (3, 4) and call(workspace_bytes=100) == 4 and call(workspace=272) == 3
    assert lib.tb_lora_gemm(None, None) == 1 and lib.tb_lora_workspace_bytes(None) == 0
    assert call(out=257) == 3 and call(bias=257, bias_dtype=_lib.F32) == 3 and call(bias=256, bias_dtype=_lib.E4M3) == 2

    # weight rows (or columns) that overlap, and sizes whose tile or stage numbers would pass 32 bits
    assert call(w_stride_n=56) == 1 and call(w_stride_n=0) == 1 and call(w_stride_k=32, w_stride_n=1) == 1 and call(w_stride_k=0, w_stride_n=1) == 1
    wide = dict(x_row_stride=1 << 30, w_stride_n=1 << 30, lora_a_row_stride=1 << 30)
    assert call(k=1 << 29, **wide) == 1 and call(m=(1 << 30) + 1) == 1 and call(n=(1 << 30) + 1) == 1

    def need(**kw):
        a = _lib.LoraArgs(4, 40, 64, 8, 3, _lib.BF16, 256, 64, 256, 1, 64, 256, 512, 64, 256, 320, 8, 256, 0, 0, 0, 256, 40, 1, 256, 0, 0, 0, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.tb_lora_workspace_bytes(ctypes.byref(a))

    assert need() > 0 and need(m=5000) > need(m=500) > 0
    assert need(m=1 << 26, num_adapters=1000) == 0          # more block rows than a copy's coordinate can number
    assert need(rank=12) == 0 and need(m=0) == 0


def test_c_entry_points_refuse_bad_arguments():
    lib = _lib.lib
    one = ctypes.c_void_p(256)      # never dereferenced: every call below is refused before a launch
    route = lambda tokens, experts, topk, dtype=_lib.BF16, logits=one, stride=64, weights=one: lib.tb_moe_route(
        logits, dtype, stride, tokens, experts, topk, 0, 1, weights, one, None)
    assert route(0, 64, 8) == 0
    assert route(4, 64, 0) == 1 and route(4, 64, 33) == 1 and route(4, 8, 9) == 1 and route(4, 1025, 8, stride=1025) == 1
    assert route(-1, 64, 8) == 1 and route(4, 64, 8, stride=63) == 1 and route(4, 64, 8, logits=None) == 1 and route(4, 64, 8, weights=None) == 1
    assert route(4, 64, 8, dtype=_lib.E4M3) == 2 and route(4, 64, 8, logits=ctypes.c_void_p(257)) == 3
    assert lib.tb_moe_route_backward(one, _lib.F32, 64, 4, 64, 8, 0, 1, one, one, None, one, None) == 1
    assert lib.tb_moe_route_backward(one, _lib.F32, 64, 4, 64, 8, 0, 1, one, one, one, None, None) == 1

    def mlp(**kw):
        a = _lib.MoeMlpArgs(4, 2, 4, 64, 32, _lib.BF16, 256, 64, 256, 64 * 64, 64, 256, 64 * 32, 32, 256, 256, 256, 64, 256, 1 << 30, 0, 0)
        for k, v in kw.items():
            setattr(a, k, v)
        return lib.tb_moe_mlp(ctypes.byref(a), None)

    assert mlp(tokens=0) == 0
    for kw in (dict(tokens=129), dict(tokens=-1), dict(topk=0), dict(topk=33), dict(num_experts=0), dict(num_experts=1025), dict(hidden=60),
               dict(ffn=4), dict(x=None), dict(w1=None), dict(w2=None), dict(topk_ids=None), dict(topk_weights=None), dict(out=None),
               dict(x_row_stride=63), dict(w1_row_stride=63), dict(w2_row_stride=31), dict(out_row_stride=60)):
        assert mlp(**kw) == 1, kw
    assert mlp(dtype=_lib.F32) == 2
    assert mlp(workspace=None) == 4 and mlp(workspace_bytes=100) == 4
    assert mlp(workspace=300) == 3 and mlp(out=257) == 3 and mlp(topk_ids=258) == 3 and mlp(topk_weights=257) == 3
    assert lib.tb_moe_mlp(None, None) == 1
    assert lib.tb_moe_mlp_workspace_bytes(129, 2, 4, 64, 32) == 0 and lib.tb_moe_mlp_workspace_bytes(4, 2, 4, 64, 32) > 0


def test_expert_layer_structure_matches_the_header(tmp_path):
    import os
    import re
    import shutil
    import subprocess
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no host C compiler")
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "tritonblas_b200.h")
    for cname, mirror in (("tb_moe_mlp_args", _lib.MoeMlpArgs), ("tb_lora_args", _lib.LoraArgs)):
        names = [f[0] for f in mirror._fields_]
        lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{header}"', "int main(void) {",
                 f'printf("%zu\\n", sizeof({cname}));'] + [f'printf("%zu\\n", offsetof({cname}, {n}));' for n in names] + ["return 0; }"]
        (tmp_path / "l.c").write_text("\n".join(lines))
        subprocess.run([cc, "-std=c11", "-o", str(tmp_path / "l"), str(tmp_path / "l.c")], check=True)
        out = [int(v) for v in subprocess.run([str(tmp_path / "l")], check=True, capture_output=True, text=True).stdout.split()]
        assert out == [ctypes.sizeof(mirror)] + [getattr(mirror, n).offset for n in names], cname
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), open(header).read(), re.S).group(1)
        assert len(re.findall(r"[,;]", body)) == len(names)
