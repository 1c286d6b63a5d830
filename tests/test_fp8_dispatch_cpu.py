"""Calls of the fp8 operators that something records, fakes or transforms reach the registered operators.  No GPU call is made here."""
import os
import subprocess
import sys

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from composable_kernel_amd import torch_ops

F8 = torch.float8_e4m3fn
OPS = ["rmsnorm_fp8", "quantize_fp8", "gated_fp8", "fp8_linear"]


def layer(x, norm, wt, ws):
    q, s, h = torch_ops.rmsnorm_fp8(x, norm, x)
    q2, s2 = torch_ops.quantize_fp8(h)
    q3, s3 = torch_ops.gated_fp8(x, h, "fastgelu")
    y = [torch_ops.fp8_linear(a, b, wt, ws) for a, b in ((q, s), (q2, s2), (q3, s3))]
    return y[0] + y[1] + y[2]


def operands(device="cuda"):
    return (torch.empty(2, 3, 1000, dtype=torch.bfloat16, device=device), torch.empty(1000, dtype=torch.bfloat16, device=device),
            torch.empty(50, 1000, dtype=F8, device=device), torch.empty(1, 8, device=device))


def recorded(graph):
    """Names of the framework's operators in an fx graph, in order of their first use."""
    names = []
    for n in graph.nodes:
        if n.op == "call_function" and "wqgemm" in str(n.target):
            name = str(n.target).split("wqgemm.")[1].split(".")[0]
            if name not in names:
                names.append(name)
    return names


def test_the_public_functions_answer_under_fake_tensors():
    with FakeTensorMode():
        x, norm, wt, ws = operands()
        q, s, h = torch_ops.rmsnorm_fp8(x, norm, x)
        assert q.shape == x.shape and q.dtype == F8 and s.shape == (2, 3, 8) and h.shape == x.shape
        assert torch_ops.rmsnorm_fp8(x, norm)[2] is None
        assert torch_ops.gated_fp8(x, x, group_k=0)[1].shape == (2, 3, 1)
        assert torch_ops.quantize_fp8(x)[1].shape == (2, 3, 8)
        y = layer(x, norm, wt, ws)
        assert y.shape == (2, 3, 50) and y.dtype == torch.bfloat16 and y.device.type == "cuda"


def test_meta_tensors_have_shapes():
    y = layer(*operands("meta"))
    assert y.shape == (2, 3, 50) and y.dtype == torch.bfloat16


def test_a_traced_function_holds_the_operators():
    with FakeTensorMode():
        gm = make_fx(layer)(*operands())
    assert sorted(recorded(gm.graph)) == sorted(OPS)
    gm = make_fx(layer, tracing_mode="symbolic")(*operands("meta"))
    assert sorted(recorded(gm.graph)) == sorted(OPS)


def test_a_compiled_function_holds_the_operators():
    graphs = []

    def backend(gm, inputs):
        graphs.append(gm.graph)
        return lambda *a: (torch.zeros(2, 3, 50),)

    torch._dynamo.reset()
    torch.compile(layer, backend=backend, fullgraph=True)(*operands("cpu"))
    assert len(graphs) == 1 and sorted(recorded(graphs[0])) == sorted(OPS)


def test_tangents_are_refused():
    """A forward-mode derivative would be lost: the operators have none."""
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: torch_ops.quantize_fp8(d), lambda: torch_ops.gated_fp8(x, d), lambda: torch_ops.rmsnorm_fp8(d, w),
                     lambda: torch_ops.rmsnorm_fp8(x, forward_ad.make_dual(w, w)), lambda: torch_ops.rmsnorm_fp8(x, w, d)):
            with pytest.raises(RuntimeError, match="inference-only"):
                call()
    with pytest.raises(RuntimeError, match="inference-only"):
        torch.func.jvp(lambda v: torch_ops.quantize_fp8(v)[1], (x,), (x,))
    with pytest.raises(RuntimeError, match="inference-only"):
        torch.func.grad(lambda v: torch_ops.quantize_fp8(v)[1].sum())(x)


def test_what_is_intercepted():
    from composable_kernel_amd import _torch_front as front

    x = torch.zeros(4, 256)
    assert front.direct(x, None, x)
    with FakeTensorMode():
        assert not front.direct(x) and not front.direct(torch.zeros(3))
    assert not front.direct(x, FakeTensorMode().from_tensor(x)) and front.direct(torch.nn.Parameter(x))
    seen = []
    torch.func.vmap(lambda v: seen.append(front.direct(v)) or v)(x)
    make_fx(lambda v: seen.append(front.direct(v)) or v)(x)
    torch.jit.trace(lambda v: seen.append(front.direct(v)) or v, x, check_trace=False)
    assert seen and not any(seen)
    with torch.no_grad(), torch.inference_mode(), torch.autocast("cpu"):
        assert front.direct(x)
    assert front.direct(x)


ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("built", [False, True])
def test_the_module_does_without_its_short_way(built):
    """Not built, or built for another torch: the operators, and those for int4 / int8 weights, are there all the same."""
    code = f"""
import os, sys, warnings
import composable_kernel_amd
sys.modules["composable_kernel_amd._torch_front"] = None  # (an import of it fails)
exists = os.path.exists
os.path.exists = lambda p: {built} if str(p).endswith("_torch_front.so") else exists(p)
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    from composable_kernel_amd import torch_ops
assert ["_torch_front" in str(w.message) for w in seen if w.category is RuntimeWarning] == [True] * {built}, seen
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
x = torch.zeros(4, 256, dtype=torch.bfloat16)
with FakeTensorMode():
    f = torch.empty(4, 256, dtype=torch.bfloat16, device="cuda")
    q, s, h = torch_ops.rmsnorm_fp8(f, f[0], f)
    assert s.shape == (4, 2) and torch_ops.fp8_linear(q, s, q, s[:1]).shape == (4, 4)
for call in (lambda: torch_ops.quantize_fp8(x), lambda: torch_ops.fpaintb_linear(x, x, x[0], 4, "none", None)):
    try:
        call()
    except RuntimeError as e:
        assert "GPU only" in str(e), e
print("served")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "served" in r.stdout, r.stdout + r.stderr


def test_the_build_leaves_the_short_way_out_without_torch():
    front = os.path.join(ROOT, "composable_kernel_amd", "_torch_front.so")
    before = os.stat(front).st_mtime_ns
    r = subprocess.run(["make", "-C", os.path.join(ROOT, "composable_kernel_amd", "csrc"), "PYTHON=/bin/false", "-W",
                        os.path.join(ROOT, "composable_kernel_amd", "csrc") + "/torch_front.cpp", front], capture_output=True, text=True)
    assert r.returncode == 0 and "left out" in r.stdout, r.stdout + r.stderr
    assert os.stat(front).st_mtime_ns == before


def test_a_short_way_of_an_earlier_build_is_left_alone():
    code = """
import sys, types, warnings
import composable_kernel_amd
old = types.ModuleType("composable_kernel_amd._torch_front")
old.bind = old.linear = old.quantized = lambda *a: None
sys.modules[old.__name__] = old
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    from composable_kernel_amd import torch_ops
assert torch_ops._torch_front is torch_ops._NoFront and any("earlier source" in str(w.message) for w in seen)
print("served")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=200)
    assert r.returncode == 0 and "served" in r.stdout, r.stdout + r.stderr
