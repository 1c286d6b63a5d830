"""PyTorch-ROCm front end of the weight-quantized GEMM: a linear layer whose weights live on the GPU in the
engine's packed formats, and a ``torch.library`` custom operator around the C ABI launch.

PyTorch supplies device memory and the stream; the arithmetic is the HIP kernels behind ``wqgemm_launch``
(there is no eager fallback: without the library or a GPU the operator raises).
"""
from __future__ import annotations

import ctypes
import os
import warnings

import torch
from torch.autograd import forward_ad

from . import capi
from .weights import BlockF8Weights, PackedWeights

_DT = {torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_EPILOGUES = {"none": capi.EPI_PASSTHROUGH, "fastgelu": capi.EPI_FASTGELU, "add": capi.EPI_ADD,
              "add_fastgelu": capi.EPI_ADD_FASTGELU}


@torch.library.custom_op("wqgemm::fpaintb_linear", mutates_args=())
def fpaintb_linear(x: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, bits: int, epilogue: str,
                   bias: torch.Tensor | None, layout: str = "packed") -> torch.Tensor:
    """y[m, n] = epilogue( sum_k x[m, k] * dequant(weight[n, k], scale[n]) [, bias[n]] ).

    layout = "preshuffled": the weight bytes are in the order of wqgemm_preshuffle_int4 / _int8; needs N a multiple of 32
    and K of 64, and raises where no matrix-core kernel can take the problem.

    x (M, K) fp16 / bf16, row-major; weight uint8 (N, K/2) packed int4 (bits = 4) or int8 (N, K) (bits = 8);
    scale and bias (N,) of x's dtype; epilogue in {"none", "fastgelu", "add", "add_fastgelu"}.
    Group-wise scales: scale of shape (G, N), one row per group of K / G consecutive k."""
    if not x.is_cuda:
        raise RuntimeError("wqgemm::fpaintb_linear runs on the GPU only")
    if x.dtype not in _DT or scale.dtype != x.dtype:
        raise TypeError("x and scale must both be float16 or both bfloat16")
    if epilogue not in _EPILOGUES:
        raise ValueError(f"unknown epilogue {epilogue!r}")
    if (bias is None) != (epilogue in ("none", "fastgelu")):
        raise ValueError("bias goes with the add / add_fastgelu epilogues only")
    if bits not in (4, 8):
        raise ValueError(f"bits must be 4 (packed int4) or 8 (int8), got {bits}")
    if layout not in ("packed", "preshuffled"):
        raise ValueError(f"layout must be 'packed' or 'preshuffled', got {layout!r}")
    if x.dim() != 2 or scale.dim() not in (1, 2):
        raise ValueError("x must be (M, K) and scale (N,) or (groups, N)")
    M, K = x.shape
    N = scale.shape[-1]
    group_k = 0
    if scale.dim() == 2:
        if scale.shape[0] == 0 or K % scale.shape[0] != 0:
            raise ValueError(f"K = {K} is not a whole number of the {scale.shape[0]} scale groups")
        group_k = K // scale.shape[0]
    # the kernels read weight / scale / bias through raw pointers: shapes, dtypes, devices and contiguity are checked here
    want = (N, K // 2) if bits == 4 else (N, K)
    if bits == 4 and K % 8 != 0:
        raise ValueError("packed int4 weights need K to be a multiple of 8")
    if tuple(weight.shape) != want or weight.dtype not in (torch.uint8, torch.int8):
        raise ValueError(f"weight must be an 8-bit tensor of shape {want} for bits = {bits}, got {tuple(weight.shape)} {weight.dtype}")
    for name, t in (("weight", weight), ("scale", scale), ("bias", bias)):
        if t is None:
            continue
        if t.device != x.device:
            raise ValueError(f"{name} is on {t.device}, x on {x.device}")
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if bias is not None and (tuple(bias.shape) != (N,) or bias.dtype != x.dtype):
        raise ValueError(f"bias must have shape ({N},) and x's dtype {x.dtype}, got {tuple(bias.shape)} {bias.dtype}")
    x = x.contiguous()
    # any M runs as it is: small-M kernel up to 64 rows, the tile kernels with a partial last row tile beyond
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    p = capi.fpAintB_problem(x.data_ptr(), weight.data_ptr(), scale.data_ptr(), y.data_ptr(), M, N, K,
                             a_dtype=_DT[x.dtype],
                             b_dtype=((capi.I4_PRESHUFFLED, capi.I8_PRESHUFFLED) if layout == "preshuffled"
                                      else (capi.I4_PACKED, capi.I8))[bits == 8],
                             epilogue=_EPILOGUES[epilogue], d0=bias.data_ptr() if bias is not None else None,
                             scale_group_k=group_k)
    if not capi.is_supported(p):
        raise RuntimeError("wqgemm::fpaintb_linear: " + capi.lib.wqgemm_last_error().decode())
    nbytes = capi.workspace_bytes(p)  # optional scratch (the planner's split-K partials)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    with torch.cuda.device(x.device):
        capi.launch(p, ws.data_ptr() if ws is not None else None, torch.cuda.current_stream().cuda_stream)
    return y


@fpaintb_linear.register_fake
def _(x, weight, scale, bits, epilogue, bias, layout="packed"):
    return x.new_empty((x.shape[0], scale.shape[-1]))


class WqLinear(torch.nn.Module):
    """Inference-only linear layer over packed weights (see ``weights.pack`` / ``weights.load_packed``)."""

    def __init__(self, pw: PackedWeights, bias: torch.Tensor | None = None, epilogue: str = "none", device="cuda"):
        super().__init__()
        dt = torch.float16 if pw.scale_dtype == "f16" else torch.bfloat16
        self.bits, self.in_features, self.out_features, self.layout = pw.bits, pw.K, pw.N, pw.layout
        self.register_buffer("weight", torch.from_numpy(pw.weight.copy()).to(device))
        self.register_buffer("scale", torch.from_numpy(pw.scale.view("int16").copy()).view(dt).to(device))
        self.register_buffer("bias", None if bias is None else bias.to(device=device, dtype=dt))
        self.epilogue = ("add" if epilogue == "none" else "add_fastgelu") if bias is not None else epilogue

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        lead = x.shape[:-1]
        y = fpaintb_linear(x.reshape(-1, self.in_features), self.weight, self.scale, self.bits, self.epilogue, self.bias,
                           self.layout)
        return y.reshape(*lead, self.out_features)


# ---- fp8 activations and weights with block-wise scales ----------------------------------------------------------------
#
# The operators of an 8-bit layer: rmsnorm_fp8, gated_fp8 and quantize_fp8 make e4m3fn activations with fp32 scales (one per
# 128 consecutive values, or one per row), fp8_linear multiplies them with e4m3fn weights that carry one scale per 128 x 128
# block.  All are inference-only, run on the current stream of the operands' device, allocate through torch's caching
# allocator only, and can be captured into a graph.  Called plainly they go straight to the C ABI; where something records,
# fakes or transforms the call (torch.compile, torch.jit.trace, make_fx, fake tensors, functorch, tensor subclasses), and as
# torch.ops.wqgemm.*, they are the custom operators registered below.

_F8 = torch.float8_e4m3fn
_ACTIVATIONS = {"silu": capi.ACT_SILU, "fastgelu": capi.ACT_FASTGELU}
_INT_MAX = 2 ** 31 - 1


# (small calls are bound by the host: what follows asks each tensor as little as it can.  The raw stream handle takes 0.07 us
# where torch.cuda.current_stream(...).cuda_stream takes 1.8)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class _NoFront:
    """In place of the short way where it was not built: every call goes through the registered operators."""
    linear = quantized = staticmethod(lambda *args: None)
    direct = staticmethod(lambda *tensors: False)


# (a call with nothing to copy, convert or refuse goes the short way, in C++: csrc/torch_front.cpp.  It answers None to the others)
try:
    from . import _torch_front
    if not hasattr(_torch_front, "direct"):
        raise ImportError("built from an earlier source")
except ImportError as e:
    if os.path.exists(os.path.join(os.path.dirname(__file__), "_torch_front.so")):
        warnings.warn(f"composable_kernel_amd/_torch_front.so cannot be loaded ({e}); calls of the fp8 operators take longer on the host "
                      "without it: build it again with `make -C composable_kernel_amd/csrc`", RuntimeWarning)
    _torch_front = _NoFront
else:
    _torch_front.bind(*(ctypes.cast(f, ctypes.c_void_p).value for f in (capi.lib.wqgemm_quantize, capi.lib.wqgemm_launch,
                                                                       capi.lib.wqgemm_workspace_bytes, capi.lib.wqgemm_last_error)), capi.WqError)


def _no_gradients(name, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{name} is inference-only: call it under torch.no_grad() or with tensors that need no gradient")
    if not torch.compiler.is_compiling() and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} is inference-only: its operands must carry no forward-mode tangent")


def _direct(*tensors):
    """Whether a call goes to the device as it stands, rather than to the registered operator."""
    return not torch.compiler.is_compiling() and tensors[0].is_cuda and _torch_front.direct(*tensors)


def _same_device(name, x, **others):
    if not x.is_cuda:
        raise RuntimeError(f"{name} runs on the GPU only")
    for k, t in others.items():
        if t is not None and t.device != x.device:
            raise ValueError(f"{name}: {k} is on {t.device}, the first operand on {x.device}")


def _rows(t, cols):
    """(tensor, rows, row stride): t as rows of `cols` contiguous elements, copied only if its layout cannot be read as such."""
    if t.dim() != 2:
        t = t.reshape(-1, cols)
    m = t.shape[0]
    if t.is_contiguous():
        ld = cols
    else:
        ld = t.stride(0) if m > 1 else cols
        if (t.stride(1) != 1 and cols > 1) or ld < cols:
            t, ld = t.contiguous(), cols
    if m > _INT_MAX or ld > _INT_MAX:
        raise ValueError("at most 2^31 - 1 rows, columns and elements between rows")
    return t, m, ld


def _launch_on(x, call, *args):
    """call(*args, stream) with x's device current: the library launches on the current device."""
    index = x.get_device()
    if torch.cuda.current_device() == index:
        call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            call(*args, _raw_stream(index))


def _fp8_linear(x, x_scale, weight, weight_scale, bias, epilogue, out_dtype):
    index = x.get_device()
    if (index < 0 or x_scale.get_device() != index or weight.get_device() != index or weight_scale.get_device() != index or
            (bias is not None and bias.get_device() != index)):
        _same_device("fp8_linear", x, x_scale=x_scale, weight=weight, weight_scale=weight_scale, bias=bias)
    if x.dtype != _F8 or weight.dtype != _F8:
        raise TypeError(f"x and weight must be float8_e4m3fn, got {x.dtype} and {weight.dtype}")
    if x_scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
        raise TypeError("x_scale and weight_scale must be float32")
    if out_dtype not in _DT:
        raise TypeError(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    if epilogue not in _EPILOGUES:
        raise ValueError(f"unknown epilogue {epilogue!r}")
    if (bias is None) != (epilogue in ("none", "fastgelu")):
        raise ValueError("bias goes with the add / add_fastgelu epilogues only")
    shape, w_shape = x.shape, weight.shape
    if not shape or len(w_shape) != 2:
        raise ValueError("x must be (..., K) and weight (N, K)")
    N, K = w_shape
    lead = shape[:-1]
    if shape[-1] != K or K == 0 or N == 0:
        raise ValueError(f"x {tuple(shape)} does not go with a weight of shape {(N, K)}")
    kb = (K + 127) >> 7
    if x_scale.shape != (*lead, kb):
        raise ValueError(f"x_scale must have shape {(*lead, kb)}, got {tuple(x_scale.shape)}")
    if weight_scale.shape != ((N + 127) >> 7, kb):
        raise ValueError(f"weight_scale must have shape {((N + 127) >> 7, kb)}, got {tuple(weight_scale.shape)}")
    if bias is not None:
        if bias.shape != (N,) or bias.dtype != out_dtype:
            raise ValueError(f"bias must have shape {(N,)} and the output's dtype {out_dtype}, got {tuple(bias.shape)} {bias.dtype}")
        bias = bias.contiguous()
    y = x.new_empty((*lead, N), dtype=out_dtype)
    x, M, lda = _rows(x, K)
    if M == 0:
        return y
    x_scale, _, ld_a_scale = _rows(x_scale, kb)
    weight, _, ldb = _rows(weight, K)
    weight_scale, _, ld_b_scale = _rows(weight_scale, kb)
    p = capi.f8_problem(x.data_ptr(), x_scale.data_ptr(), weight.data_ptr(), weight_scale.data_ptr(), y.data_ptr(), M, N, K,
                        c_dtype=_DT[out_dtype], lda=lda, ldb=ldb, ldc=N, ld_a_scale=ld_a_scale, ld_b_scale=ld_b_scale,
                        epilogue=_EPILOGUES[epilogue], d0=bias.data_ptr() if bias is not None else None,
                        flags=capi.FLAG_BF16_RTN)
    nbytes = capi.workspace_bytes(p)
    ws = x.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    _launch_on(x, capi.launch, p, ws.data_ptr() if nbytes else None)
    return y


def _quantized_rows(name, op, x, x2, weight, activation, eps, group_k, keep):
    """The common part of the quantisers, their operands' shapes and dtypes checked but for x's; keep: h is stored too."""
    dtype = _DT.get(x.dtype)
    if dtype is None:
        raise TypeError(f"{name}: inputs must be float16 or bfloat16, got {x.dtype}")
    shape = x.shape
    if not shape or shape[-1] == 0:
        raise ValueError(f"{name}: inputs must be (..., K) with K > 0")
    if group_k != 128 and group_k != 0:
        raise ValueError(f"group_k must be 128, or 0 for one scale per row, got {group_k}")
    K = shape[-1]
    groups = (K + 127) >> 7 if group_k else 1
    if x.is_contiguous():
        q, out = torch.empty_like(x, dtype=_F8), torch.empty_like(x) if keep else None
    else:
        q, out = x.new_empty(shape, dtype=_F8), x.new_empty(shape) if keep else None
    scale = x.new_empty((*shape[:-1], groups), dtype=torch.float32)
    x, M, ldx = _rows(x, K)
    if M == 0:
        return q, scale, out
    d = capi.Quant()
    d.op, d.dtype, d.M, d.K, d.group_k, d.ldx, d.ldq, d.ld_scale = op, dtype, M, K, group_k, ldx, K, groups
    d.x, d.q, d.scale = x.data_ptr(), q.data_ptr(), scale.data_ptr()
    if x2 is not None:
        x2, _, d.ldx2 = _rows(x2, K)
        d.x2 = x2.data_ptr()
    if weight is not None:
        weight = weight.contiguous()
        d.weight, d.eps, d.weight_dtype = weight.data_ptr(), eps, capi.F32 if weight.dtype == torch.float32 else dtype
        if keep:
            d.residual_out, d.ld_residual_out = out.data_ptr(), K
    d.activation = activation
    _launch_on(x, capi.quantize, d)
    return q, scale, out


def _quantize_fp8(x, group_k):
    if not x.is_cuda:
        _same_device("quantize_fp8", x)
    return _quantized_rows("quantize_fp8", capi.QUANT_ROWS, x, None, None, 0, 0.0, group_k, False)[:2]


def _gated_fp8(gate, up, activation, group_k):
    _same_device("gated_fp8", gate, up=up)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}")
    if up.shape != gate.shape or up.dtype != gate.dtype:
        raise ValueError(f"gate and up must have one shape and dtype, got {tuple(gate.shape)} {gate.dtype} and {tuple(up.shape)} {up.dtype}")
    return _quantized_rows("gated_fp8", capi.QUANT_GATED, gate, up, None, _ACTIVATIONS[activation], 0.0, group_k, False)[:2]


def _rmsnorm_fp8(x, weight, residual, eps, group_k):
    _same_device("rmsnorm_fp8", x, weight=weight, residual=residual)
    if weight.shape != x.shape[-1:] or weight.dim() != 1 or weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"weight must have shape {tuple(x.shape[-1:])} and dtype {x.dtype} or float32, got {tuple(weight.shape)} {weight.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have x's shape and dtype, got {tuple(residual.shape)} {residual.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _quantized_rows("rmsnorm_fp8", capi.QUANT_RMSNORM, x, residual, weight, 0, eps, group_k, residual is not None)


@torch.library.custom_op("wqgemm::fp8_linear", mutates_args=())
def _fp8_linear_op(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                   bias: torch.Tensor | None, epilogue: str, out_dtype: torch.dtype) -> torch.Tensor:
    return _fp8_linear(x, x_scale, weight, weight_scale, bias, epilogue, out_dtype)


@_fp8_linear_op.register_fake
def _(x, x_scale, weight, weight_scale, bias, epilogue, out_dtype):
    return x.new_empty((*x.shape[:-1], weight.shape[0]), dtype=out_dtype)


@torch.library.custom_op("wqgemm::quantize_fp8", mutates_args=())
def _quantize_fp8_op(x: torch.Tensor, group_k: int) -> tuple[torch.Tensor, torch.Tensor]:
    return _quantize_fp8(x, group_k)


@torch.library.custom_op("wqgemm::gated_fp8", mutates_args=())
def _gated_fp8_op(gate: torch.Tensor, up: torch.Tensor, activation: str, group_k: int) -> tuple[torch.Tensor, torch.Tensor]:
    return _gated_fp8(gate, up, activation, group_k)


@torch.library.custom_op("wqgemm::rmsnorm_fp8", mutates_args=())
def _rmsnorm_fp8_op(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None, eps: float,
                    group_k: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    q, scale, out = _rmsnorm_fp8(x, weight, residual, eps, group_k)
    return q, scale, out if out is not None else x.new_empty(0)  # (an operator's results are all tensors)


def _fake_quantized(x, group_k):
    return x.new_empty(x.shape, dtype=_F8), x.new_empty((*x.shape[:-1], (x.shape[-1] + 127) // 128 if group_k else 1), dtype=torch.float32)


@_quantize_fp8_op.register_fake
def _(x, group_k):
    return _fake_quantized(x, group_k)


@_gated_fp8_op.register_fake
def _(gate, up, activation, group_k):
    return _fake_quantized(gate, group_k)


@_rmsnorm_fp8_op.register_fake
def _(x, weight, residual, eps, group_k):
    return (*_fake_quantized(x, group_k), x.new_empty(x.shape if residual is not None else 0))


def fp8_linear(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
               bias: torch.Tensor | None = None, epilogue: str = "none",
               out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """y[..., n] = epilogue( sum_k x[..., k] x_scale[..., k // 128] weight[n, k] weight_scale[n // 128, k // 128] [, bias[n]] ).

    x (..., K) and weight (N, K) float8_e4m3fn; x_scale (..., ceil(K / 128)) and weight_scale (ceil(N / 128), ceil(K / 128))
    float32; bias (N,) of out_dtype, with the "add" / "add_fastgelu" epilogues ("none" and "fastgelu" go without).

    The fp8 matrix core adds 8 consecutive products in a window of 13 bits below the largest of them; all sums beyond those 8, the
    scales and the epilogue are fp32: an error of less than 7 * 2^-13 of sum_k |x weight| (scales included), on normally distributed
    operands 1.5e-5 of the outputs' root mean square.  One rounding to nearest even into out_dtype (float16 or bfloat16).  Any N and
    K; fastest where K is a multiple of 16 and the rows are 16-byte aligned."""
    if not torch.compiler.is_compiling() and x.is_cuda and epilogue in _EPILOGUES:
        y = _torch_front.linear(x, x_scale, weight, weight_scale, bias, _EPILOGUES[epilogue], out_dtype, _raw_stream)
        if y is not None:
            return y
    _no_gradients("fp8_linear", x, x_scale, weight, weight_scale, bias)
    call = _fp8_linear if _direct(x, x_scale, weight, weight_scale, bias) else _fp8_linear_op
    return call(x, x_scale, weight, weight_scale, bias, epilogue, out_dtype)


def quantize_fp8(x: torch.Tensor, group_k: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """x (..., K) float16 / bfloat16 -> (q, scale) with x ~ q * scale: q float8_e4m3fn of x's shape, scale float32 of shape
    (..., ceil(K / 128)), one per 128 consecutive values, or (..., 1) for group_k = 0 (what the C ABI's fp8 x int4
    MultiplyMultiply problems take as d1; fp8_linear takes scales by 128).  scale = max|x| / 448 of its group (groups below
    1e-12: as if the maximum were that); a NaN makes its whole group NaN."""
    if not torch.compiler.is_compiling() and x.is_cuda:
        r = _torch_front.quantized(capi.QUANT_ROWS, x, None, None, 0, 0.0, group_k, _raw_stream)
        if r is not None:
            return r[:2]
    _no_gradients("quantize_fp8", x)
    return (_quantize_fp8 if _direct(x) else _quantize_fp8_op)(x, group_k)


def gated_fp8(gate: torch.Tensor, up: torch.Tensor, activation: str = "silu",
              group_k: int = 128) -> tuple[torch.Tensor, torch.Tensor]:
    """quantize_fp8 of activation(gate) * up, evaluated in fp32 (activation "silu" or "fastgelu").  gate and up may be the
    two halves of one projection's output (row-strided views are read in place)."""
    if not torch.compiler.is_compiling() and gate.is_cuda and activation in _ACTIVATIONS:
        r = _torch_front.quantized(capi.QUANT_GATED, gate, up, None, _ACTIVATIONS[activation], 0.0, group_k, _raw_stream)
        if r is not None:
            return r[:2]
    _no_gradients("gated_fp8", gate, up)
    return (_gated_fp8 if _direct(gate, up) else _gated_fp8_op)(gate, up, activation, group_k)


def rmsnorm_fp8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None, eps: float = 1e-6,
                group_k: int = 128) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """h = x + residual; returns (q, scale) = quantize_fp8 of h / sqrt(mean(h^2) + eps) * weight, and h rounded to x's dtype
    (None without a residual).  The norm sees h unrounded; weight (K,) has x's dtype or float32."""
    if not torch.compiler.is_compiling() and x.is_cuda:
        r = _torch_front.quantized(capi.QUANT_RMSNORM, x, residual, weight, 0, eps, group_k, _raw_stream)
        if r is not None:
            return r
    _no_gradients("rmsnorm_fp8", x, weight, residual)
    if _direct(x, weight, residual):
        return _rmsnorm_fp8(x, weight, residual, eps, group_k)
    q, scale, out = _rmsnorm_fp8_op(x, weight, residual, eps, group_k)
    return q, scale, out if residual is not None else None


class Fp8Linear(torch.nn.Module):
    """Inference-only linear layer over e4m3fn weights with 128 x 128 block scales (see ``weights.quantize_fp8_blocks`` /
    ``weights.load_fp8_blocks``).

    forward takes float16 / bfloat16 activations, which it quantises by 128 itself and answers in their dtype, or an already
    quantised pair (q, scale) -- what rmsnorm_fp8, gated_fp8 and quantize_fp8 return first -- answered in ``out_dtype``.

    .half(), .bfloat16() and the like leave the weight's bytes and scales as they are.  The bias keeps the type it comes in
    (float16, bfloat16 or float32) and is rounded to the output's: one of that type already costs no launch of its own."""

    def __init__(self, bw: BlockF8Weights, bias: torch.Tensor | None = None, epilogue: str = "none", device="cuda",
                 out_dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        if epilogue not in ("none", "fastgelu"):
            raise ValueError(f"epilogue must be 'none' or 'fastgelu' (a bias is added in front of it), got {epilogue!r}")
        self.in_features, self.out_features, self.out_dtype = bw.K, bw.N, out_dtype
        self.register_buffer("weight", torch.from_numpy(bw.weight.copy()).view(_F8).to(device))
        self.register_buffer("weight_scale", torch.from_numpy(bw.scale.copy()).to(device))
        self.register_buffer("bias", None if bias is None else bias.to(device=device, dtype=bias.dtype if bias.dtype in _DT else torch.float32))
        self.epilogue = epilogue if bias is None else {"none": "add", "fastgelu": "add_fastgelu"}[epilogue]

    def _apply(self, fn, recurse=True):
        # (casts of a model take whatever is floating point: the weight and its scales pass through them as bytes)
        exact = (self.weight, self.weight_scale)

        def apply(t):
            if not any(t is e for e in exact):
                return fn(t)
            as_bytes = t.contiguous().view(torch.uint8)
            out = fn(as_bytes)
            return (out if out.dtype == torch.uint8 else as_bytes.to(out.device)).view(t.dtype)

        return super()._apply(apply, recurse)

    def forward(self, x):
        if isinstance(x, (tuple, list)):
            q, scale, out_dtype = x[0], x[1], self.out_dtype
        else:
            (q, scale), out_dtype = quantize_fp8(x), x.dtype
        bias = None if self.bias is None else self.bias.to(out_dtype)
        return fp8_linear(q, scale, self.weight, self.weight_scale, bias, self.epilogue, out_dtype)
