"""What the library accepts and refuses of the fp8 operators at the edges of their sizes.  No GPU call is made here."""
import copy

import numpy as np
import pytest
import torch

from composable_kernel_amd import capi, torch_ops, weights
from test_fp8_cpu import f8

LONG = 2 ** 31 - 1


@pytest.mark.parametrize("k,k_batch", [(LONG, 2), (2 ** 31 - 64, 2), (2 ** 31 - 4096, 65535), (LONG, 3)])
def test_slices_past_32_bits_are_refused(k, k_batch):
    """The last slice's end has to be a 32-bit number too."""
    for p in (f8(M=1, N=4, K=k, k_batch=k_batch), f8(M=1, N=4, K=k, k_batch=k_batch, flags=capi.FLAG_GENERIC),
              capi.fpAintB_problem(0x10000, 0x10000, 0x10000, 0x10000, 1, 4, k // 64 * 64, b_dtype=capi.I8, k_batch=k_batch)):
        assert not capi.is_supported(p)
        assert "2^31" in capi.lib.wqgemm_last_error().decode()


def test_the_longest_rows_run_on_the_general_kernel():
    """The matrix-core kernels step K by 128 in 32 bits: rows that end within a step of 2^31 go one by one."""
    for k in (LONG, 2 ** 31 - 255):
        assert capi.kernel_name(f8(M=1, N=4, K=k)) == "wq_gemm_generic"
    assert capi.kernel_name(f8(M=1, N=4, K=2 ** 31 - 256)) == "wq_gemm_f8f8_any"
    assert capi.is_supported(f8(M=1, N=4, K=2 ** 30, k_batch=2))


# ---- the layer as a part of a model ----

CASTS = {"half": lambda m: m.half(), "bfloat16": lambda m: m.bfloat16(), "double": lambda m: m.double(), "to": lambda m: m.to(torch.bfloat16),
         "type": lambda m: m.type(torch.float16), "to_device_and_dtype": lambda m: m.to("cpu", torch.float16), "float": lambda m: m.float()}


@pytest.mark.parametrize("cast", CASTS)
@pytest.mark.parametrize("bias", [False, True])
def test_casts_of_a_model_leave_the_weights_alone(cast, bias):
    bw = weights.quantize_fp8_blocks(np.random.default_rng(0).normal(0, 1, (130, 200)).astype(np.float32))
    layer = torch_ops.Fp8Linear(bw, torch.arange(130.0) if bias else None, device="cpu")
    model = torch.nn.Sequential(torch.nn.LayerNorm(200), layer)
    CASTS[cast](model)
    assert layer.weight.dtype == torch.float8_e4m3fn and layer.weight_scale.dtype == torch.float32
    assert layer.weight.shape == (130, 200) and np.array_equal(layer.weight.view(torch.uint8).numpy(), bw.weight)
    assert np.array_equal(layer.weight_scale.numpy(), bw.scale)
    assert "weight" in dict(layer.named_buffers()) and (not bias or layer.bias.dtype == model[0].weight.dtype)
    other = torch_ops.Fp8Linear(weights.quantize_fp8_blocks(np.ones((130, 200), np.float32)), torch.zeros(130) if bias else None, device="cpu")
    other.load_state_dict(copy.deepcopy(layer).state_dict())
    assert torch.equal(other.weight.view(torch.uint8), layer.weight.view(torch.uint8)) and torch.equal(other.weight_scale, layer.weight_scale)


def test_a_layer_moves_between_devices():
    bw = weights.quantize_fp8_blocks(np.ones((130, 200), np.float32))
    layer = torch_ops.Fp8Linear(bw, device="cpu").to("meta")
    assert layer.weight.device.type == layer.weight_scale.device.type == "meta" and layer.weight.dtype == torch.float8_e4m3fn
    layer = layer.to_empty(device="cpu")
    assert layer.weight.shape == (130, 200) and layer.weight_scale.shape == (2, 2) and layer.weight_scale.dtype == torch.float32


@pytest.mark.parametrize("dtype,kept", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float64, torch.float32)])
def test_a_bias_keeps_its_type(dtype, kept):
    bw = weights.quantize_fp8_blocks(np.ones((130, 200), np.float32))
    assert torch_ops.Fp8Linear(bw, torch.zeros(130, dtype=dtype), device="cpu").bias.dtype == kept
