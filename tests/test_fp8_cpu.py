"""fp8 operators without a GPU: what the library accepts and refuses, the weights' quantiser and container, the torch
front end's argument checks.  No GPU call is made here."""
import numpy as np
import pytest
import torch

from composable_kernel_amd import capi, torch_ops, weights
import fp8_ref

FAKE = 0x10000  # never dereferenced by validation


def f8(**kw):
    d = dict(a=FAKE, sa=FAKE, b=FAKE, sb=FAKE, c=FAKE, M=256, N=512, K=1024)
    d.update(kw)
    args = [d.pop(k) for k in ("a", "sa", "b", "sb", "c", "M", "N", "K")]
    return capi.f8_problem(*args, **d)


@pytest.mark.parametrize("m", [1, 7, 16, 17, 64, 300, 4096])
@pytest.mark.parametrize("n,k", [(1, 1), (64, 128), (100, 1001), (4096, 4096), (5000, 4112)])
def test_every_size_has_a_matrix_core_kernel(m, n, k):
    p = f8(M=m, N=n, K=k)
    assert capi.is_supported(p), capi.lib.wqgemm_last_error()
    assert capi.kernel_name(p).startswith("wq_gemm_f8f8_")
    assert "DeviceGemmMultiD_ABScale" in capi.type_string(p)


@pytest.mark.parametrize("kw", [
    dict(a_dtype=capi.F8_FNUZ), dict(b_dtype=capi.F8_FNUZ), dict(flags=capi.FLAG_GENERIC), dict(a_layout=capi.COL_MAJOR),
    dict(b_layout=capi.ROW_MAJOR), dict(scale_block=(1, 100, 128)), dict(scale_block=(1, 128, 64)), dict(scale_block=(128, 128, 1024)),
])
def test_the_rest_runs_on_the_general_kernel(kw):
    p = f8(**kw)
    assert capi.is_supported(p) and capi.kernel_name(p) == "wq_gemm_generic"


def test_fnuz_with_the_promise_runs_on_the_matrix_core():
    p = f8(a_dtype=capi.F8_FNUZ, b_dtype=capi.F8_FNUZ, flags=capi.FLAG_F8_NO_SPECIALS)
    assert capi.kernel_name(p).startswith("wq_gemm_f8f8_")


@pytest.mark.parametrize("kw,word", [
    (dict(sa=None), "pairs"), (dict(sb=None), "pairs"), (dict(sa=None, sb=None), "block-wise"),
    (dict(a_dtype=capi.F16, c_dtype=capi.F16), "fp8 activations"), (dict(a_dtype=capi.I8), "fp8 activations"),
    (dict(c_dtype=capi.F32), "fp16 or bf16"), (dict(c_dtype=capi.I8), "fp16 or bf16"),
    (dict(scale_block=(0, 128, 128)), "positive"), (dict(scale_block=(1, 128, -1)), "positive"),
    (dict(ld_a_scale=7), "ld_a_scale"), (dict(ld_b_scale=7), "ld_a_scale / ld_b_scale"), (dict(sa=FAKE + 2), "aligned"),
    (dict(c=FAKE + 1), "aligned"), (dict(epilogue=capi.EPI_ACT_MUL_CLAMP), "epilogue"), (dict(epilogue=capi.EPI_ADD), "d0"),
    (dict(scale_group_k=128), "scale must be NULL"), (dict(flags=capi.FLAG_MFMA_32X32), "flags"), (dict(flags=capi.FLAG_TILE_256, lda=1032), "TILE"), (dict(flags=capi.FLAG_PINGPONG), "flags"),
    (dict(epilogue=capi.EPI_MULTIPLY_ADD, d0=FAKE, d1=FAKE, flags=capi.FLAG_BF16_RTN), "rounding"),
    (dict(M=0), "positive"), (dict(K=0), "positive"), (dict(lda=0), "positive"), (dict(ldc=100), "ldc"), (dict(a=None), "non-null"),
    (dict(k_begin=0, k_end=128), "fp32 partials"), (dict(k_batch=2, N=510), "multiples of 4"),
])
def test_refusals(kw, word):
    p = f8(**kw)
    assert not capi.is_supported(p)
    assert word in capi.lib.wqgemm_last_error().decode()
    with pytest.raises(capi.WqError):
        capi.launch(p)


def test_the_rounding_flag_is_for_fp8_weights():
    p = capi.fpAintB_problem(FAKE, FAKE, FAKE, FAKE, 256, 256, 256, a_dtype=capi.BF16, flags=capi.FLAG_BF16_RTN)
    assert not capi.is_supported(p)


def test_workspace_of_a_k_batch_covers_ragged_columns():
    p = f8(k_batch=4)
    assert capi.workspace_bytes(p) == 4 * 256 * 512 * 4
    with pytest.raises(capi.WqError) as e:
        capi.launch(p)  # no workspace: refused before anything is launched
    assert e.value.status == capi.ERR_WORKSPACE


def quant(**kw):
    d = capi.Quant()
    d.op, d.dtype, d.weight_dtype, d.M, d.K, d.group_k = capi.QUANT_ROWS, capi.BF16, capi.BF16, 4, 512, 128
    d.ldx = d.ldx2 = d.ld_residual_out = d.ldq = 512
    d.ld_scale, d.x, d.q, d.scale = 4, FAKE, FAKE, FAKE
    for k, v in kw.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize("kw", [
    dict(op=7), dict(M=0), dict(K=-1), dict(dtype=capi.F32), dict(dtype=capi.F8_E4M3FN), dict(group_k=64), dict(group_k=-128),
    dict(x=None), dict(q=None), dict(scale=None), dict(ldx=511), dict(ldq=511), dict(ld_scale=3), dict(K=513),
    dict(x=FAKE + 1), dict(scale=FAKE + 2), dict(x2=FAKE), dict(weight=FAKE), dict(residual_out=FAKE),
    dict(op=capi.QUANT_RMSNORM), dict(op=capi.QUANT_RMSNORM, weight=FAKE, eps=-1.0), dict(op=capi.QUANT_RMSNORM, weight=FAKE, eps=float("nan")),
    dict(op=capi.QUANT_RMSNORM, weight=FAKE, weight_dtype=capi.F16), dict(op=capi.QUANT_RMSNORM, weight=FAKE, x2=FAKE, ldx2=100),
    dict(op=capi.QUANT_RMSNORM, weight=FAKE, residual_out=FAKE, ld_residual_out=100),
    dict(op=capi.QUANT_RMSNORM, weight=FAKE + 2, weight_dtype=capi.F32),
    dict(op=capi.QUANT_GATED), dict(op=capi.QUANT_GATED, x2=FAKE, activation=2), dict(op=capi.QUANT_GATED, x2=FAKE, residual_out=FAKE),
])
def test_quantize_refusals(kw):
    with pytest.raises(capi.WqError) as e:
        capi.quantize(quant(**kw))
    assert e.value.status in (capi.ERR_INVALID, capi.ERR_UNSUPPORTED)
    assert "quantize" in str(e.value)


@pytest.mark.parametrize("kw", [dict(K=2 ** 30 + 1), dict(K=2 ** 31 - 1), dict(op=capi.QUANT_RMSNORM, weight=FAKE, K=2 ** 30 + 1),
                                dict(group_k=0, K=2 ** 31 - 1)])
def test_rows_too_long_for_32_bit_positions_are_refused(kw):
    d = quant(ldx=2 ** 31 - 1, ldq=2 ** 31 - 1, ld_scale=2 ** 31 - 1, **kw)
    with pytest.raises(capi.WqError) as e:
        capi.quantize(d)
    assert e.value.status == capi.ERR_UNSUPPORTED and "2^30" in str(e.value)


@pytest.mark.parametrize("kw", [
    dict(M=2 ** 19, N=2 ** 19), dict(M=2 ** 31 - 1), dict(N=2 ** 31 - 1, ldc=2 ** 31 - 1), dict(k_batch=65536),
    dict(M=2 ** 15, N=2 ** 13, k_batch=1024),
])
def test_more_tiles_than_a_launch_holds_are_refused(kw):
    # a launch holds fewer than 2^32 work items along x (a tile takes 256 per 128 x 128 outputs) and 65535 slices
    kw.setdefault("ldc", kw.get("N", 512))
    p = f8(**kw)
    assert not capi.is_supported(p)
    assert "too many tiles" in capi.lib.wqgemm_last_error().decode()


def test_strips_of_columns_stay_within_a_launch():
    # 16 columns take 1024 work items in the kernel for few rows: 2^32 are reached at 2^26 columns, where tiles take over
    assert capi.kernel_name(f8(M=1, N=2 ** 25, ldc=2 ** 25)) == "wq_gemm_f8f8_skinny_direct"
    assert "skinny" not in capi.kernel_name(f8(M=1, N=2 ** 26, ldc=2 ** 26))


def test_null_descriptor():
    assert capi.lib.wqgemm_quantize(None, None) == capi.ERR_INVALID


# ---- the weights' quantiser and container ----

@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (130, 257), (300, 1001)])
def test_quantize_fp8_blocks(n, k):
    rng = np.random.default_rng(n * k)
    w = rng.normal(0, 1, (n, k)).astype(np.float32)
    w[: n // 2] *= 1e-3
    w[0, 0] = 0
    bw = weights.quantize_fp8_blocks(w)
    assert bw.weight.shape == (n, k) and bw.scale.shape == (-(-n // 128), -(-k // 128))
    got = weights.dequantize_fp8_blocks(bw)
    s = np.repeat(np.repeat(bw.scale, 128, 0)[:n], 128, 1)[:, :k]
    # half a step of the value, or of the subnormals, and the fp32 roundings of the quotient and the product
    assert (np.abs(got - w) <= 2.0 ** -4 * np.abs(w) * (1 + 2.0 ** -4) + 2.0 ** -10 * s + 2.0 ** -21 * np.abs(w)).all()
    values = fp8_ref.f8_values(torch.from_numpy(bw.weight)).numpy()
    assert np.isfinite(values).all() and np.abs(values).max() <= 448


def test_blocks_of_zeros_and_refused_weights():
    bw = weights.quantize_fp8_blocks(np.zeros((130, 130), np.float32))
    assert (weights.dequantize_fp8_blocks(bw) == 0).all() and np.isfinite(bw.scale).all() and (bw.scale > 0).all()
    for bad in (np.full((4, 4), np.nan), np.full((4, 4), np.inf), np.zeros((0, 4)), np.zeros(4)):
        with pytest.raises(ValueError):
            weights.quantize_fp8_blocks(bad)


def test_container_round_trip(tmp_path):
    bw = weights.quantize_fp8_blocks(np.random.default_rng(0).normal(0, 1, (70, 200)).astype(np.float32))
    path = str(tmp_path / "w.npz")
    weights.save_fp8_blocks(path, bw)
    got = weights.load_fp8_blocks(path)
    assert (got.weight == bw.weight).all() and (got.scale == bw.scale).all() and (got.N, got.K) == (70, 200)
    with pytest.raises(ValueError):
        weights.load_packed(path)
    q, s = weights.quantize_per_channel(np.ones((8, 64), np.float32))
    weights.save_packed(path, weights.pack(q, s))
    with pytest.raises(ValueError):
        weights.load_fp8_blocks(path)
    with pytest.raises(ValueError):
        weights.BlockF8Weights(bw.weight, bw.scale[:, :1], 70, 200)


# ---- the torch front end ----

def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 256, dtype=torch.float8_e4m3fn), torch.zeros(4, 2)
    for call in (lambda: torch_ops.quantize_fp8(x), lambda: torch_ops.gated_fp8(x, x), lambda: torch_ops.rmsnorm_fp8(x, x[0]),
                 lambda: torch_ops.fp8_linear(q, s, q, s[:1])):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_tensors_that_need_gradients_are_refused():
    x = torch.zeros(4, 256, dtype=torch.bfloat16, requires_grad=True)
    for call in (lambda: torch_ops.quantize_fp8(x), lambda: torch_ops.gated_fp8(x, x), lambda: torch_ops.rmsnorm_fp8(x, x[0].detach()),
                 lambda: torch_ops.rmsnorm_fp8(x.detach(), x[0])):
        with pytest.raises(RuntimeError, match="inference-only"):
            call()


def test_the_short_way_leaves_the_rest_to_the_long_one():
    from composable_kernel_amd import _torch_front as front

    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(256)
    assert front.quantized(capi.QUANT_ROWS, x, None, None, 0, 0.0, 128, 0) is None          # not on a GPU
    assert front.quantized(capi.QUANT_RMSNORM, "x", x, w, 0, 1e-6, 128, 0) is None          # not a tensor
    assert front.quantized("op", x, None, None, 0, 0.0, 128, 0) is None
    assert front.linear(x, w, x, w, None, 0, torch.bfloat16, 0) is None
    assert front.linear(x, w, x, w, None, "none", "bf16", 0) is None
    for call in (front.quantized, front.linear, front.bind):
        with pytest.raises(TypeError):
            call(x)


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(2, 3, 1000, dtype=torch.float16, device="cuda")
        w = torch.empty(1000, dtype=torch.float16, device="cuda")
        q, s, r = torch.ops.wqgemm.rmsnorm_fp8(x, w, x, 1e-6, 128)
        assert q.shape == x.shape and q.dtype == torch.float8_e4m3fn and s.shape == (2, 3, 8) and r.shape == x.shape
        q, s = torch.ops.wqgemm.gated_fp8(x, x, "silu", 0)
        assert s.shape == (2, 3, 1)
        q, s = torch.ops.wqgemm.quantize_fp8(x, 128)
        wt = torch.empty(50, 1000, dtype=torch.float8_e4m3fn, device="cuda")
        y = torch.ops.wqgemm.fp8_linear(q, s, wt, torch.empty(1, 8, device="cuda"), None, "none", torch.bfloat16)
        assert y.shape == (2, 3, 50) and y.dtype == torch.bfloat16
