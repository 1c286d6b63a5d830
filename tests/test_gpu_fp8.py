"""The fp8 x fp8 product with block-wise scales and the quantisers of its activations on the GPU, against 64-bit references."""
import math
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

from composable_kernel_amd import capi, torch_ops, weights
import fp8_ref
from fp8_ref import BLOCK, U32

pytestmark = pytest.mark.gpu

EPI = {"none": capi.EPI_PASSTHROUGH, "fastgelu": capi.EPI_FASTGELU, "add": capi.EPI_ADD, "add_fastgelu": capi.EPI_ADD_FASTGELU}
DT = {torch.float16: capi.F16, torch.bfloat16: capi.BF16}


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def random_bits(rows, cols, g, fnuz_safe=False):
    """Every finite e4m3fn encoding, uniformly: the widest spread of values the format has (fnuz_safe: without the bytes of
    WQ_FLAG_F8_NO_SPECIALS)."""
    b = torch.randint(0, 256, (rows, cols), device="cuda", generator=g, dtype=torch.int32).to(torch.uint8)
    b[(b & 0x7F) == 0x7F] = 0x35
    if fnuz_safe:
        b[b == 0x80] = 0x35
    return b


INTEGERS = torch.tensor([0x00, 0x38, 0x40, 0x44, 0x48, 0x4A, 0x4C, 0x4E, 0x50], dtype=torch.uint8)  # 0 .. 8 in e4m3fn


def integer_bits(rows, cols, g):
    """Integers -8 .. 8.  Products are whole and at most 64, inside the matrix core's window of 13 bits, so that with scales of
    1 and 1/2 every sum up to K = 2^15 is a multiple of 1/4 below 2^22: exact in fp32 in any order."""
    v = INTEGERS.cuda()[torch.randint(0, 9, (rows, cols), device="cuda", generator=g)]
    return torch.where(torch.rand(rows, cols, device="cuda", generator=g) < 0.5, v | 0x80, v)


def problem(m, n, k, seed, *, bm=1, bn=128, bk=128, lda=None, ldb=None, offset=0, fnuz_safe=False, exact=False):
    """Operands in poisoned surroundings: bytes between and around the rows are NaN, scales around the tables are NaN."""
    g = gen(seed)
    lda, ldb = lda or k, ldb or k
    kb = -(-k // bk)
    out = {"m": m, "n": n, "k": k, "lda": lda, "ldb": ldb, "block": (bm, bn, bk)}
    for name, rows, ld in (("a", m, lda), ("b", n, ldb)):
        buf = torch.full((offset + rows * ld + 512,), 0x7F, dtype=torch.uint8, device="cuda")
        bits = integer_bits(rows, k, g) if exact else random_bits(rows, k, g, fnuz_safe)
        view = buf[offset:offset + rows * ld].view(rows, ld)
        view[:, :k] = bits
        out[name], out[name + "_bits"], out[name + "_ptr"] = buf, bits, view.data_ptr()
    for name, rows in (("sa", -(-m // bm)), ("sb", -(-n // bn))):
        t = torch.full((rows + 2, kb), float("nan"), device="cuda")
        r = torch.rand(rows, kb, device="cuda", generator=g)
        t[1:-1] = torch.where(r < 0.5, 0.5, 1.0) if exact else torch.exp2(r * 8 - 12)
        out[name] = t[1:-1]
    return out


def reference(P, bias=None, act="none", fnuz=(False, False)):
    bm, bn, bk = P["block"]
    a = fp8_ref.f8_values(P["a_bits"], fnuz[0]) * fp8_ref.expand(P["sa"], P["m"], P["k"], bm, bk)
    b = fp8_ref.f8_values(P["b_bits"], fnuz[1]) * fp8_ref.expand(P["sb"], P["n"], P["k"], bn, bk)
    return fp8_ref.linear(a, b, bias, act)


def launch(P, dtype, *, bias=None, act="none", ldc=None, k_batch=1, flags=capi.FLAG_BF16_RTN, workspace=True, a_dtype=capi.F8_E4M3FN,
           b_dtype=capi.F8_E4M3FN, noalloc=False, **kw):
    """Runs P; C lies in a guarded buffer whose surroundings have to stay as they were."""
    m, n = P["m"], P["n"]
    ldc = ldc or n
    buf = torch.full((m + 2, ldc), -77.0, dtype=dtype, device="cuda")
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), buf[1].data_ptr(), m, n, P["k"], c_dtype=DT[dtype],
                        a_dtype=a_dtype, b_dtype=b_dtype, lda=P["lda"], ldb=P["ldb"], ldc=ldc, epilogue=EPI[act],
                        d0=bias.data_ptr() if bias is not None else None, k_batch=k_batch, flags=flags, scale_block=P["block"], **kw)
    nbytes = capi.workspace_bytes(p) if workspace else 0
    ws = torch.full((nbytes + 256,), 0xFF, dtype=torch.uint8, device="cuda")
    print(f"{m}x{n}x{P['k']} {capi.type_string(p)}", flush=True)
    stream = torch.cuda.current_stream().cuda_stream
    if noalloc:
        capi.launch_noalloc(p, stream)
    else:
        capi.launch(p, ws.data_ptr() if nbytes else None, stream)
    torch.cuda.synchronize()
    guard = torch.full((), -77.0, dtype=dtype, device="cuda")
    assert bool((buf[0] == guard).all()) and bool((buf[-1] == guard).all()) and bool((buf[:, n:] == guard).all())
    assert bool((ws[nbytes:] == 0xFF).all())
    return buf[1:-1, :n]


def check(got, P, dtype, bias=None, act="none", **kw):
    y, size = reference(P, bias, act, **kw)
    bound = fp8_ref.linear_bound(y, size, P["k"], dtype, act)
    over = (got.double() - y).abs() - bound
    assert bool(torch.isfinite(got).all())
    assert float(over.max()) <= 0, f"over its bound by {float(over.max())} at {int(over.argmax())}"


def check_exact(got, P):
    """Data whose sums are exact: the output is the rounded sum, bit for bit."""
    y, _ = reference(P)
    want = y.to(torch.float32)
    assert bool((want.double() == y).all())
    assert torch.equal(got, want.to(got.dtype)), f"{int((got != want.to(got.dtype)).sum())} of {got.numel()} outputs differ"


SIZES = [(1, 128, 128), (1, 4096, 4096), (2, 1, 1), (5, 33, 17), (1, 257, 1001), (15, 64, 2048), (16, 256, 4112), (17, 300, 640), (33, 100, 384),
         (64, 1024, 1024), (65, 130, 272), (96, 512, 2816), (127, 129, 1100), (128, 128, 128), (129, 256, 256), (200, 1000, 528), (256, 256, 144),
         (300, 700, 1040), (513, 384, 512), (777, 520, 400), (1024, 1024, 384), (2048, 2304, 256),
         (4352, 4608, 512), (4300, 4616, 656)]  # (the last two: more tiles than resident workgroups)


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_sizes(m, n, k, dtype):
    P = problem(m, n, k, m * 7 + n * 3 + k)
    check(launch(P, dtype), P, dtype)
    P = problem(m, n, k, m * 5 + n * 2 + k, exact=True)
    check_exact(launch(P, torch.bfloat16 if k > 4000 else dtype), P)  # (sums up to 64 * K would leave fp16's range)


@pytest.mark.parametrize("m,n,k", [(1, 4096, 400), (4, 4000, 3968), (3, 8200, 272), (2, 8321, 1040), (5, 4090, 2048), (16, 4104, 640), (9, 8192, 8192),
                                   (12, 5001, 144), (16, 8208, 1936), (17, 4096, 2064), (32, 4100, 640), (25, 8190, 1168), (32, 8192, 4096)])
def test_few_rows(m, n, k):
    """Every kernel for few rows, with columns and rows past the edge and K tiles that do not fill the waves' turns."""
    P = problem(m, n, k, m + n + k, exact=True)
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), P["a_ptr"], m, n, k, scale_block=P["block"])
    assert "skinny" in capi.kernel_name(p)
    check_exact(launch(P, torch.bfloat16), P)
    P = problem(m, n, k, m + n)
    check(launch(P, torch.float16, k_batch=3 if n % 4 == 0 else 1), P, torch.float16)


@pytest.mark.parametrize("kernel,m,n,k", [
    ("64x64", 40, 520, 2048), ("64x64", 100, 1040, 656), ("64x64", 257, 514, 1040), ("64", 300, 11008, 656), ("64", 300, 11003, 1040),
    ("128_w8", 640, 5000, 1024), ("128_w8", 600, 4999, 1040), ("128", 1536, 11008, 656), ("128", 1530, 11003, 656), ("128x256", 512, 11008, 656),
    ("128x256", 500, 11003, 656), ("256", 768, 11008, 656), ("256", 760, 11001, 1040)])
def test_every_tile_kernel(kernel, m, n, k):
    P = problem(m, n, k, m + n + k, exact=True)
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), P["a_ptr"], m, n, k, scale_block=P["block"])
    assert capi.kernel_name(p) == "wq_gemm_f8f8_" + kernel
    check_exact(launch(P, torch.bfloat16), P)
    P = problem(m, n, k, m + n)
    check(launch(P, torch.float16), P, torch.float16)


@pytest.mark.parametrize("flags", [capi.FLAG_TILE_128, capi.FLAG_TILE_256, capi.FLAG_TILE_128 | capi.FLAG_TILE_256])
@pytest.mark.parametrize("m,n,k", [(5, 8, 400), (300, 700, 1040), (513, 1030, 528), (4300, 4616, 656)])
@pytest.mark.parametrize("act", ["none", "add_fastgelu"])
def test_chosen_tile_sizes(flags, m, n, k, act):
    """The tile size fixed by the caller; the largest is more tiles than resident workgroups of every kernel."""
    P = problem(m, n, k, m + k)
    P["sa"] *= 0.05
    bias = torch.randn(n, device="cuda", generator=gen(5)).bfloat16() if act != "none" else None
    check(launch(P, torch.bfloat16, bias=bias, act=act, flags=flags | capi.FLAG_BF16_RTN), P, torch.bfloat16, bias, act)


@pytest.mark.parametrize("m,n,k,lda,ldb,offset", [
    (1, 4096, 4095, None, None, 0), (4, 300, 117, 119, 130, 1), (16, 9000, 1000, 1004, None, 3), (30, 5000, 2047, None, 2049, 0), (64, 500, 1001, None, None, 5),
    (300, 700, 1040, 1041, 1040, 0), (257, 1030, 4096, None, None, 8), (700, 3000, 130, None, 133, 0), (100, 1024, 8191, None, None, 1)])
def test_rows_of_any_alignment(m, n, k, lda, ldb, offset):
    """Operands that are copied to aligned rows first, and the kernel that needs no copy (and no workspace) on the same ones."""
    P = problem(m, n, k, m + n, lda=lda, ldb=ldb, offset=offset, exact=True)
    kw = dict(lda=P["lda"], ldb=P["ldb"], scale_block=P["block"])
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), P["sa"].data_ptr(), m, n, k, **kw)
    assert "PaddedRows" in capi.type_string(p) and capi.workspace_bytes(p) >= (m + n) * (-(-k // 16) * 16)
    check_exact(launch(P, torch.bfloat16), P)
    check_exact(launch(P, torch.bfloat16, workspace=False), P)
    if capi.workspace_bytes(p) < capi.NOALLOC_SCRATCH_BYTES:
        check_exact(launch(P, torch.bfloat16, noalloc=True), P)
    Q = problem(m, n, k, m, lda=lda, ldb=ldb, offset=offset)
    check(launch(Q, torch.float16), Q, torch.float16)


@pytest.mark.parametrize("m,n,k,off", [(70, 300, 1001, 4), (40, 520, 2049, 12), (300, 515, 700, 8)])
def test_workspace_of_any_alignment(m, n, k, off):
    P = problem(m, n, k, m, exact=True)
    c = torch.full((m, n), -77.0, dtype=torch.bfloat16, device="cuda")
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), c.data_ptr(), m, n, k, scale_block=P["block"], flags=capi.FLAG_BF16_RTN)
    nbytes = capi.workspace_bytes(p)
    assert "PaddedRows" in capi.type_string(p)
    ws = torch.full((nbytes + 64,), 0xFF, dtype=torch.uint8, device="cuda")
    capi.launch(p, ws.data_ptr() + off, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check_exact(c, P)
    assert bool((ws[:off] == 0xFF).all()) and bool((ws[off + nbytes:] == 0xFF).all())


@pytest.mark.parametrize("flags", [0, capi.FLAG_TILE_128, capi.FLAG_TILE_256, capi.FLAG_TILE_128 | capi.FLAG_TILE_256])
@pytest.mark.parametrize("k", [16, 128, 144, 256, 368, 384])
@pytest.mark.parametrize("m,n,bm,bn", [(40, 200, 1, 128), (300, 700, 1, 32), (513, 1030, 128, 128), (4300, 4616, 3, 96)])
def test_short_rows(flags, k, m, n, bm, bn):
    """K of at most three scale blocks in the tile kernels, the largest with more tiles than resident workgroups."""
    P = problem(m, n, k, m + k, exact=True, bm=bm, bn=bn)
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), P["a_ptr"], m, n, k, scale_block=P["block"], flags=flags)
    assert capi.kernel_name(p) not in ("wq_gemm_f8f8_any", "wq_gemm_generic")
    check_exact(launch(P, torch.bfloat16, flags=flags | capi.FLAG_BF16_RTN), P)
    if k == 384:
        Q = problem(m, n, k, m, bm=bm, bn=bn)
        check(launch(Q, torch.float16, flags=flags, k_batch=2 if n % 4 == 0 else 1), Q, torch.float16)


@pytest.mark.parametrize("m,n,k", [(3, 257, 384), (40, 512, 640), (150, 384, 272), (300, 515, 1024)])
@pytest.mark.parametrize("act", ["fastgelu", "add", "add_fastgelu"])
def test_epilogues(m, n, k, act):
    for dtype in (torch.float16, torch.bfloat16):
        P = problem(m, n, k, m + n + k)
        P["sa"] *= 0.05  # (arguments of the activation around one)
        bias = torch.randn(n, device="cuda", generator=gen(5)).to(dtype) if act.startswith("add") else None
        check(launch(P, dtype, bias=bias, act=act), P, dtype, bias, act)


@pytest.mark.parametrize("m,n,k,lda,ldb,offset,ldc", [
    (5, 96, 256, 272, 320, 0, 104), (70, 200, 384, 400, 400, 16, 203), (300, 256, 512, 528, 640, 48, 264),   # padded, aligned rows
    (5, 96, 256, 259, 257, 0, 97), (70, 130, 384, 385, 391, 3, 131), (300, 200, 130, 131, 133, 5, 201),      # unaligned rows and base
    (20, 64, 1000, 1008, 1008, 0, 64), (260, 512, 1000, 1024, 1008, 0, 512),                                 # aligned rows, ragged K
])
def test_strides_and_alignment(m, n, k, lda, ldb, offset, ldc):
    P = problem(m, n, k, m + k, lda=lda, ldb=ldb, offset=offset)
    check(launch(P, torch.bfloat16, ldc=ldc), P, torch.bfloat16)
    P = problem(m, n, k, m + k, lda=lda, ldb=ldb, offset=offset, exact=True)
    check_exact(launch(P, torch.bfloat16, ldc=ldc), P)


@pytest.mark.parametrize("m", [4, 60, 300])
@pytest.mark.parametrize("block", [(128, 128, 128), (1, 32, 128), (7, 256, 128), (64, 96, 128), (3, 40, 128), (5, 17, 50), (1000, 1000, 4096)])
def test_block_shapes(m, block):
    bm, bn, bk = block
    P = problem(m, 320, 768, m + bm, bm=bm, bn=bn, bk=bk)
    got = launch(P, torch.float16)
    y, size = reference(P)
    # (the general kernel sums the K products one by one: K additions in place of 128 and the blocks')
    bound = fp8_ref.linear_bound(y, size, P["k"], torch.float16) + 3 * P["k"] * U32 * size
    assert bool(((got.double() - y).abs() <= bound).all())


def test_padded_scale_tables():
    P = problem(40, 384, 640, 3)
    for name in ("sa", "sb"):
        wide = torch.full((P[name].shape[0], 9), float("nan"), device="cuda")
        wide[:, :5] = P[name]
        P[name] = wide
    got = launch(P, torch.bfloat16, ld_a_scale=9, ld_b_scale=9)
    P["sa"], P["sb"] = P["sa"][:, :5], P["sb"][:, :5]
    check(got, P, torch.bfloat16)


@pytest.mark.parametrize("m", [1, 24, 200, 600])
@pytest.mark.parametrize("fnuz", [(True, True), (True, False), (False, True)])
def test_fnuz(m, fnuz):
    P = problem(m, 256, 512, m, fnuz_safe=True)
    a, b = (capi.F8_FNUZ if f else capi.F8_E4M3FN for f in fnuz)
    got = launch(P, torch.float16, a_dtype=a, b_dtype=b, flags=capi.FLAG_F8_NO_SPECIALS)
    check(got, P, torch.float16, fnuz=fnuz)
    general = launch(P, torch.float16, a_dtype=a, b_dtype=b, flags=capi.FLAG_GENERIC)
    y, size = reference(P, fnuz=fnuz)
    assert bool(((general.double() - y).abs() <= fp8_ref.linear_bound(y, size, 512, torch.float16) + 3 * 512 * U32 * size).all())


@pytest.mark.parametrize("m,n,k", [(1, 4096, 2048), (16, 512, 4096), (100, 300, 4096), (300, 512, 1152), (257, 4096, 2048)])
def test_split_k(m, n, k):
    """The caller's k_batch, the planner's split with and without a workspace, and the built-in scratch: one result up to the
    order of fp32 sums."""
    P = problem(m, n, k, k + m)
    check(launch(P, torch.bfloat16), P, torch.bfloat16)
    check(launch(P, torch.bfloat16, workspace=False), P, torch.bfloat16)
    check(launch(P, torch.bfloat16, noalloc=True), P, torch.bfloat16)
    for kb in (2, 3, 8, 32):
        check(launch(P, torch.bfloat16, k_batch=kb), P, torch.bfloat16)
    P = problem(m, n, k, k + m, exact=True)
    for kb in (1, 2, 3, 8, 32):
        check_exact(launch(P, torch.bfloat16, k_batch=kb), P)


@pytest.mark.parametrize("m", [3, 70, 300])
def test_k_slices_and_reduce(m):
    """The per-rank step of multi-GPU split-K: fp32 partials of K slices, then the reduction with the epilogue."""
    n, k = 256, 1000
    P = problem(m, n, k, m, lda=1008, ldb=1008)
    bias = torch.randn(n, device="cuda", generator=gen(1)).to(torch.bfloat16)
    slabs = torch.full((3, m, n), float("nan"), device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    for z, (k0, k1) in enumerate([(0, 384), (384, 896), (896, 1000)]):
        p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), slabs[z].data_ptr(), m, n, k, lda=1008, ldb=1008,
                            c_dtype=capi.F32, k_begin=k0, k_end=k1)
        capi.launch(p, None, stream)
    out = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), out.data_ptr(), m, n, k, c_dtype=capi.BF16,
                        lda=1008, ldb=1008, epilogue=capi.EPI_ADD, d0=bias.data_ptr(), flags=capi.FLAG_BF16_RTN)
    capi.reduce_finalize(p, slabs.data_ptr(), 3, stream)
    check(out, P, torch.bfloat16, bias, "add")


def test_bf16_rounding_is_chosen():
    """Truncation, as everywhere in the engine, or round to nearest even: exact sums that lie between two bf16 values."""
    m, n, k = 20, 64, 128
    P = problem(m, n, k, 1)
    P["a"].fill_(0), P["b"].fill_(0)
    one, eps = 0x38, 0x08  # 1 and 2^-6
    a, b = P["a"][:m * k].view(m, k), P["b"][:n * k].view(n, k)
    a[:, 0], a[:, 1], a[:, 2] = one, eps, eps
    b[:, 0], b[:, 1], b[:, 2] = one, 0x10, 0x08  # 1, 2^-5, 2^-6: 1 + 2^-11 + 2^-12
    P["sa"].fill_(1), P["sb"].fill_(1)
    assert bool((launch(P, torch.bfloat16, flags=0) == 1).all()) and bool((launch(P, torch.bfloat16) == 1).all())
    a[:, 1], b[:, 1] = 0x18, 0x20  # 2^-4 * 2^-3 = 2^-7: one step of bf16 above 1
    a[:, 2], b[:, 2] = 0x18, 0x1C  # 2^-4 * 1.5 * 2^-4: three quarters of a step
    assert bool((launch(P, torch.bfloat16, flags=0).float() == 1 + 2 ** -7).all())
    assert bool((launch(P, torch.bfloat16).float() == 1 + 2 ** -6).all())


@pytest.mark.parametrize("m", [2, 40, 130, 300])
def test_nan_and_infinity_stay_in_their_rows(m):
    n, k = 256, 640
    P = problem(m, n, k, m)
    P["a"][:m * k].view(m, k)[1, 300] = 0x7F
    P["sa"][0, 2] = float("inf")
    P["b"][:n * k].view(n, k)[130, 639] = 0xFF
    got = launch(P, torch.float16)
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[:, 130]).all()) and not bool(torch.isfinite(got[0]).any())
    rest = torch.ones(m, n, dtype=torch.bool, device="cuda")
    rest[:2] = False
    rest[:, 130] = False
    assert bool(torch.isfinite(got[rest]).all())


def test_rows_do_not_depend_on_their_neighbours():
    """The same rows alone and in a batch of the same kernel give the same bits; and twice the same call."""
    P = problem(512, 512, 1024, 9)
    whole = launch(P, torch.bfloat16)
    assert torch.equal(whole, launch(P, torch.bfloat16))
    P["b_bits"][:] = P["b_bits"].flip(0)
    P["b"][:512 * 1024].view(512, 1024)[:] = P["b_bits"]
    P["sb"][:] = P["sb"].flip(0)
    assert torch.equal(whole.flip(1), launch(P, torch.bfloat16))


def test_operands_beyond_32_bits():
    """Weights of more than 4 GiB between the first and the last row: a row pitch far larger than K."""
    n, k, ldb = 600, 256, 8_000_000
    P = problem(3, n, k, 2)
    b = torch.empty(n * ldb, dtype=torch.uint8, device="cuda")
    view = b.as_strided((n, k), (ldb, 1))
    view.copy_(P["b_bits"])
    P["b_ptr"], P["ldb"], P["keep"] = b.data_ptr(), ldb, b
    check(launch(P, torch.float16), P, torch.float16)
    a = torch.empty(300 * ldb * 2, dtype=torch.uint8, device="cuda")
    Q = problem(300, n, k, 3)
    a.as_strided((300, k), (2 * ldb, 1)).copy_(Q["a_bits"])
    Q["a_ptr"], Q["lda"], Q["b_ptr"], Q["ldb"], Q["keep"] = a.data_ptr(), 2 * ldb, b.data_ptr(), ldb, (a, b)
    Q["b_bits"] = P["b_bits"]
    Q["sb"] = P["sb"]
    check(launch(Q, torch.float16), Q, torch.float16)


def test_outputs_beyond_32_bits():
    """C and the weights past 4 GiB in the tile kernels: the last rows, and the last columns, of both."""
    m, n, k = 40000, 65536, 512
    P = problem(m, n, k, 5)
    got = launch(P, torch.bfloat16)
    tail = dict(P, m=200, a_bits=P["a_bits"][-200:], sa=P["sa"][-200:])
    check(got[-200:], tail, torch.bfloat16)
    del got
    ldb = 1 << 22
    b = torch.empty(1300 * ldb, dtype=torch.uint8, device="cuda")
    Q = problem(300, 1300, k, 6)
    b.as_strided((1300, k), (ldb, 1)).copy_(Q["b_bits"])
    Q["b_ptr"], Q["ldb"], Q["keep"] = b.data_ptr(), ldb, b
    check(launch(Q, torch.float16), Q, torch.float16)
    R = dict(Q, m=16, a_bits=Q["a_bits"][:16], sa=Q["sa"][:16])
    check(launch(R, torch.float16), R, torch.float16)


@pytest.mark.parametrize("m", [1, 10, 137])
@pytest.mark.parametrize("flags", [0, capi.FLAG_TILE_128, capi.FLAG_TILE_256, capi.FLAG_TILE_128 | capi.FLAG_TILE_256])
def test_nothing_behind_the_last_row(m, flags):
    """A C of many more rows than the product: all of a tile's rows past M, and those of the tile behind it, stay as they were."""
    n, k = 264, 640
    P = problem(m, n, k, m)
    c = torch.full((m + 600, n), -77.0, dtype=torch.float16, device="cuda")
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), c.data_ptr(), m, n, k, c_dtype=capi.F16,
                        scale_block=P["block"], flags=flags)
    capi.launch(p, None, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    check(c[:m], P, torch.float16)
    assert bool((c[m:] == -77).all())


# ---- quantisers ----

def rows(m, k, seed, dtype):
    g = gen(seed)
    v = torch.randn(m, k, device="cuda", generator=g) * torch.exp2(torch.rand(m, 1, device="cuda", generator=g) * 12 - 6)
    v *= 1 + 30 * (torch.rand(k, device="cuda", generator=g) < 0.02)
    if m > 2:
        v[m // 2] = 0
    return v.to(dtype)


QSIZES = [(1, 1), (1, 4096), (2, 128), (3, 127), (3, 129), (7, 512), (5, 513), (4, 1001), (9, 2048), (64, 640), (33, 5000), (600, 640), (520, 8192),
          (3, 16384), (515, 9001), (2, 40000), (1, 70001)]


@pytest.mark.parametrize("m,k", QSIZES)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize(m, k, group, dtype):
    x = rows(m, k, m + k, dtype)
    q, s = torch_ops.quantize_fp8(x, group)
    fp8_ref.check_quantized(q, s, x.double(), group, 0.0)


@pytest.mark.parametrize("m,k", QSIZES)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("dtype,act", [(torch.float16, "fastgelu"), (torch.bfloat16, "silu"), (torch.float16, "silu")])
def test_gated(m, k, group, dtype, act):
    both = torch.cat([rows(m, k, m + k, dtype).clamp(-30, 30), rows(m, k, m * 3 + k, dtype)], 1)
    gate, up = both[:, :k], both[:, k:]
    q, s = torch_ops.gated_fp8(gate, up, act, group)
    g = gate.double()
    y = (g * torch.special.expit(g) if act == "silu" else fp8_ref.fastgelu(g)) * up.double()
    # the exponent's argument is off by two roundings of its size (at most 30 for silu; for gelu up to 2 * (0.8 * 30 + 0.036 * 30^3)
    # = 2000, but past 90 the result is 0 or the argument itself: below 2^-126 it counts as absolute), the exponential, the sum, the
    # reciprocal and the products by a step each
    fp8_ref.check_quantized(q, s, y, group, (2 * 128 + 16) * U32, up.double().abs() * 2.0 ** -100)


@pytest.mark.parametrize("m,k", QSIZES)
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("dtype,residual,w32", [(torch.float16, False, False), (torch.bfloat16, True, False), (torch.float16, True, True)])
def test_rmsnorm(m, k, group, dtype, residual, w32):
    x = rows(m, k, m + k, dtype)
    r = rows(m, k, m * 5 + k, dtype) if residual else None
    w = (1 + 0.3 * torch.randn(k, device="cuda", generator=gen(3))).to(torch.float32 if w32 else dtype)
    q, s, out = torch_ops.rmsnorm_fp8(x, w, r, 1e-5, group)
    h = x.double() + (r.double() if residual else 0)
    y = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5) * w.double()
    # h is rounded once (relative U of itself; with cancellation still of h), the sum of squares is a chain of at most 8 * 8 + 16 additions per
    # thread at these widths (70001: 72) and a tree; half of that reaches the root; the mean, the root, the quotient and two products: 6 more
    fp8_ref.check_quantized(q, s, y, group, (1 + 50 + 8) * U32)
    if residual:
        assert out.dtype == dtype and bool(((out.double() - h).abs() <= fp8_ref.HALF_STEP[dtype] * h.abs() * (1 + 4 * U32) + fp8_ref.SMALLEST_HALF_STEP[dtype]).all())
        assert torch.equal(out, (x.float() + r.float()).to(dtype))
    else:
        assert out is None


def test_nan_and_infinity_poison_their_group_only():
    x = torch.ones(4, 512, dtype=torch.bfloat16, device="cuda")
    x[1, 130] = float("nan")
    x[2, 5] = float("inf")
    q, s = torch_ops.quantize_fp8(x)
    assert torch.isnan(s).nonzero().tolist() == [[1, 1]] and torch.isinf(s).nonzero().tolist() == [[2, 0]]
    v = q.float() * s.repeat_interleave(128, 1)
    assert bool(torch.isnan(v[1, 128:256]).all()) and bool(torch.isnan(v[2, 5])) and bool((v[0] == 1).all())
    assert int((~torch.isfinite(v)).sum()) == 256 and bool((v[torch.isfinite(v)] == 1).all())
    q, s = torch_ops.quantize_fp8(x, 0)
    assert torch.isnan(s[:, 0]).tolist() == [False, True, False, False] and torch.isinf(s[:, 0]).tolist() == [False, False, True, False]


def test_smallest_groups():
    """Zeros, values below the floor of the scale, and 16-bit subnormals."""
    x = torch.zeros(3, 256, dtype=torch.float16, device="cuda")
    x[1, 3] = 2.0 ** -24
    x[2, 200] = -65504.0
    q, s = torch_ops.quantize_fp8(x)
    fp8_ref.check_quantized(q, s, x.double(), 128, 0.0)
    assert bool((q[0].float() == 0).all()) and bool((s > 0).all()) and float(q[1, 3].float()) == 448 and float(q[2, 200].float()) == -448
    b = torch.zeros(1, 128, dtype=torch.bfloat16, device="cuda")
    b[0, 0] = 1e-20
    q, s = torch_ops.quantize_fp8(b)
    assert float(s[0, 0]) == float(torch.tensor(1e-12) / 448) and bool((q.float() == 0).all())


@pytest.mark.parametrize("op", ["rows", "norm", "gated"])
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("k,ld", [(300, 301), (256, 384), (1000, 1003), (20000, 20001)])
def test_strided_rows_in_place_and_guards(op, group, k, ld):
    """Odd pitches on every tensor, unaligned bases, the residual updated in place, and nothing written outside the rows."""
    m, dtype = 5, torch.bfloat16
    groups = -(-k // 128) if group else 1
    mk = lambda seed: torch.cat([torch.full((3,), float("nan"), device="cuda", dtype=dtype), torch.full((m * ld,), float("nan"), device="cuda", dtype=dtype)])  # noqa: E731
    x, x2 = mk(1), mk(2)
    xv, x2v = (t[3:].view(m, ld)[:, :k] for t in (x, x2))
    xv.copy_(rows(m, k, 1, dtype)), x2v.copy_(rows(m, k, 2, dtype))
    x0, r0 = xv.clone(), x2v.clone()
    w = torch.randn(k + 1, device="cuda", generator=gen(1)).to(dtype)[1:]
    q = torch.full((m, ld + 2), 0x55, dtype=torch.uint8, device="cuda")
    s = torch.full((m, groups + 1), -5.0, device="cuda")
    d = capi.Quant()
    d.op = {"rows": capi.QUANT_ROWS, "norm": capi.QUANT_RMSNORM, "gated": capi.QUANT_GATED}[op]
    d.dtype = d.weight_dtype = capi.BF16
    d.M, d.K, d.group_k, d.ldx, d.ldx2, d.ld_residual_out, d.ldq, d.ld_scale = m, k, group, ld, ld, ld, ld + 2, groups + 1
    d.x, d.q, d.scale, d.eps = xv.data_ptr(), q.data_ptr() + 1, s.data_ptr(), 1e-6
    if op != "rows":
        d.x2 = x2v.data_ptr()
    if op == "norm":
        d.weight, d.residual_out = w.data_ptr(), x2v.data_ptr()  # in place
    capi.quantize(d, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    got = q.view(-1)[1:1 + (m - 1) * (ld + 2) + k].as_strided((m, k), (ld + 2, 1)).view(torch.float8_e4m3fn)
    if op == "rows":
        y, rel = x0.double(), 0.0
    elif op == "norm":
        h = x0.double() + r0.double()
        y, rel = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-6) * w.double(), 60 * U32
        assert torch.equal(x2v, (x0.float() + r0.float()).to(dtype))
    else:
        g = x0.double()
        y, rel = g * torch.special.expit(g) * r0.double(), (2 * 128 + 16) * U32
    fp8_ref.check_quantized(got, s[:, :groups], y, group, rel, r0.double().abs() * 2.0 ** -100)
    assert bool((s[:, groups:] == -5).all()) and torch.equal(xv, x0)
    flat = q.view(-1).clone()
    flat[1:].as_strided((m, k), (ld + 2, 1)).fill_(0x55)
    assert bool((flat == 0x55).all())
    for t in (x, x2):
        outside = t[3:].view(m, ld)[:, k:]
        assert bool(torch.isnan(outside).all()) and bool(torch.isnan(t[:3]).all())


@pytest.mark.parametrize("op", ["rows", "norm", "gated"])
@pytest.mark.parametrize("group", [128, 0])
def test_quantisers_beyond_32_bits(op, group):
    """More than 2^31 elements: the rows at the end are those of a small call."""
    m, k, last, dtype = 70000, 40000, 5, torch.bfloat16
    x = torch.empty(m, k, dtype=dtype, device="cuda")
    x.view(-1, 8 * k)[:] = rows(8, k, 3, dtype).view(-1)
    x[-last:] = rows(last, k, 4, dtype)
    w = torch.randn(k, device="cuda", generator=gen(2)).to(dtype)
    call = {"rows": lambda v: torch_ops.quantize_fp8(v, group), "norm": lambda v: torch_ops.rmsnorm_fp8(v, w, v, 1e-6, group),
            "gated": lambda v: torch_ops.gated_fp8(v, v, "silu", group)}[op]
    for big, small in zip(call(x), call(x[-last:].clone())):
        if small is not None:
            assert torch.equal(big[-last:].view(torch.uint8), small.view(torch.uint8))


@pytest.mark.parametrize("op", ["rows", "norm"])
def test_more_rows_than_a_launch_holds(op):
    """One workgroup per row: 2^26 rows of 64 threads are 2^32 work items, more than one launch takes."""
    m, k, dtype = 2 ** 26 + 5, 3, torch.float16
    part = rows(1021, k, 8, dtype)
    x = part.repeat(m // 1021 + 1, 1)[:m]
    w = torch.ones(k, device="cuda", dtype=dtype)
    call = (lambda v: torch_ops.quantize_fp8(v, 0)) if op == "rows" else (lambda v: torch_ops.rmsnorm_fp8(v, w, v, 1e-6, 0))
    small = call(part)
    at = torch.arange(m, device="cuda") % 1021
    for got, want in zip(call(x), small):
        if want is not None:
            got, want = got.view(torch.uint8), want.view(torch.uint8)
            assert all(torch.equal(got[i:i + 2 ** 24], want[at[i:i + 2 ** 24]]) for i in range(0, m, 2 ** 24))


# ---- the torch front end, and the operators together ----

def test_linear_module_and_leading_dimensions():
    rng = np.random.default_rng(0)
    w = rng.normal(0, 0.05, (300, 400)).astype(np.float32)
    bw = weights.quantize_fp8_blocks(w)
    bias = torch.randn(300)
    layer = torch_ops.Fp8Linear(bw, bias=bias, epilogue="fastgelu")
    x = torch.randn(2, 5, 400, device="cuda", generator=gen(0)).half()
    y = layer(x)
    assert y.shape == (2, 5, 300) and y.dtype == torch.float16
    q, s = torch_ops.quantize_fp8(x)
    assert torch.equal(y, torch_ops.fp8_linear(q, s, layer.weight, layer.weight_scale, bias.cuda().half(), "add_fastgelu", torch.float16))
    pair = layer((q, s))
    assert pair.dtype == torch.bfloat16
    a = q.reshape(10, 400).float().double() * s.reshape(10, 4).double().repeat_interleave(128, 1)[:, :400]
    b = torch.from_numpy(weights.dequantize_fp8_blocks(bw)).cuda().double()
    ref, size = fp8_ref.linear(a, b, bias.cuda().half(), "add_fastgelu")
    bound = fp8_ref.linear_bound(ref, size, 400, torch.float16, "add_fastgelu") + 2 * U32 * size  # (dequantised in fp32: one more rounding)
    assert bool(((y.reshape(10, 300).double() - ref).abs() <= bound).all())


def test_empty_batches_and_column_views():
    w = torch.randn(64, 256, device="cuda", generator=gen(0))
    bw = weights.quantize_fp8_blocks(w.cpu().numpy())
    layer = torch_ops.Fp8Linear(bw)
    x = torch.randn(0, 256, device="cuda").bfloat16()
    assert layer(x).shape == (0, 64)
    q, s, r = torch_ops.rmsnorm_fp8(x, x.new_ones(256), x)
    assert q.shape == (0, 256) and s.shape == (0, 2) and r.shape == (0, 256)
    x = torch.randn(256, 40, device="cuda", generator=gen(1)).bfloat16()
    assert torch.equal(layer(x.t()), layer(x.t().contiguous()))       # (columns: copied)
    one = torch.randn(1, 256, device="cuda", generator=gen(2)).bfloat16()
    assert torch.equal(layer(one.expand(9, 256)), layer(one.repeat(9, 1)))  # (stride 0: copied)
    wt = layer.weight.t().contiguous().t()
    q, s = torch_ops.quantize_fp8(one)
    assert torch.equal(torch_ops.fp8_linear(q, s, wt, layer.weight_scale), layer((q, s)))


@pytest.mark.parametrize("shape", [(1, 4096), (5, 300), (2, 3, 640), (700,)])
@pytest.mark.parametrize("group", [128, 0])
def test_both_ways_into_the_library(shape, group):
    """What plain calls return (they go through C++) is what the long way returns, bit for bit; its dtypes, shapes and strides too."""
    k = shape[-1]
    x, r = (torch.randn(shape, device="cuda", generator=gen(s)).bfloat16() for s in (1, 2))
    w = torch.rand(k, device="cuda", generator=gen(3))
    wide = torch.cat([x, r], -1)
    f8 = torch.float8_e4m3fn
    for short, long in [(torch_ops.quantize_fp8(x, group), torch_ops._quantize_fp8(x, group)),
                        (torch_ops.gated_fp8(x, r, "fastgelu", group), torch_ops._gated_fp8(x, r, "fastgelu", group)),
                        (torch_ops.gated_fp8(wide[..., :k], wide[..., k:], "silu", group), torch_ops._gated_fp8(x, r, "silu", group)),
                        (torch_ops.rmsnorm_fp8(x, w, r, 1e-5, group), torch_ops._rmsnorm_fp8(x, w, r, 1e-5, group)),
                        (torch_ops.rmsnorm_fp8(x, w.bfloat16(), None, 0, group), torch_ops._rmsnorm_fp8(x, w.bfloat16(), None, 0, group))]:
        assert len(short) == len(long)
        for a, b in zip(short, long):
            assert (a is None) == (b is None)
            if a is not None:
                assert a.dtype == b.dtype and a.shape == b.shape and a.stride() == b.stride() and torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    q, s = torch_ops.quantize_fp8(x)
    weight = torch.randn(200, k, device="cuda", generator=gen(4)).to(f8)
    ws, bias = torch.rand(2, -(-k // 128), device="cuda", generator=gen(5)), torch.randn(200, device="cuda", generator=gen(6)).half()
    for args in [(None, "none", torch.bfloat16), (None, "fastgelu", torch.float16), (bias, "add", torch.float16)]:
        a, b = torch_ops.fp8_linear(q, s, weight, ws, *args), torch_ops._fp8_linear(q, s, weight, ws, *args)
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_gradients_are_refused():
    x = torch.randn(4, 256, device="cuda").bfloat16().requires_grad_()
    w = torch.ones(256, device="cuda", requires_grad=True)
    y = x.detach()
    calls = [lambda: torch_ops.quantize_fp8(x), lambda: torch_ops.gated_fp8(y, x), lambda: torch_ops.rmsnorm_fp8(y, w), lambda: torch_ops.rmsnorm_fp8(y, w.detach(), x)]
    for call in calls:
        with pytest.raises(RuntimeError, match="inference-only"):
            call()
        with torch.no_grad():
            assert not any(t.requires_grad for t in call() if t is not None)


def test_two_threads():
    """Each on its own stream, with its own errors."""
    x = torch.randn(300, 1024, device="cuda").bfloat16()
    want = [t.clone() for t in torch_ops.quantize_fp8(x)]
    bad = []
    torch.cuda.synchronize()

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(100):
                q, s = torch_ops.quantize_fp8(x)
                try:
                    torch_ops.quantize_fp8(x, 64 + i)
                    bad.append("accepted")
                except ValueError as e:
                    if str(64 + i) not in str(e):
                        bad.append(str(e))
            torch.cuda.current_stream().synchronize()
            if not (torch.equal(q.view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(s, want[1])):
                bad.append("differs")

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad[:3]


def test_refusals_of_the_front_end():
    x = torch.randn(4, 256, device="cuda", generator=gen(0)).bfloat16()
    q, s = torch_ops.quantize_fp8(x)
    w, ws = torch_ops.quantize_fp8(torch.randn(64, 256, device="cuda").bfloat16())[0], torch.ones(1, 2, device="cuda")
    ok = dict(x=q, x_scale=s, weight=w, weight_scale=ws)
    torch_ops.fp8_linear(**ok)
    for bad in (dict(x=x), dict(weight=w.float()), dict(x_scale=s.half()), dict(x_scale=s[:, :1]), dict(weight_scale=ws.t()), dict(weight=w[:, :128]),
                dict(out_dtype=torch.float32), dict(epilogue="relu"), dict(epilogue="add"), dict(bias=torch.zeros(64, device="cuda")),
                dict(bias=torch.zeros(63, device="cuda", dtype=torch.bfloat16), epilogue="add"), dict(x_scale=s.cpu()), dict(weight=w.cpu())):
        with pytest.raises((TypeError, ValueError)):
            torch_ops.fp8_linear(**{**ok, **bad})
    for call in (lambda: torch_ops.quantize_fp8(x, 64), lambda: torch_ops.quantize_fp8(x.float()), lambda: torch_ops.gated_fp8(x, x[:, :128]),
                 lambda: torch_ops.gated_fp8(x, x.half()), lambda: torch_ops.gated_fp8(x, x, "tanh"), lambda: torch_ops.rmsnorm_fp8(x, x[0, :5]),
                 lambda: torch_ops.rmsnorm_fp8(x, x[0].half()), lambda: torch_ops.rmsnorm_fp8(x, x[0], x[:2]), lambda: torch_ops.rmsnorm_fp8(x, x[0], eps=-1.0),
                 lambda: torch_ops.rmsnorm_fp8(x, x[0].cpu())):
        with pytest.raises((TypeError, ValueError)):
            call()


class Block(torch.nn.Module):
    """A gated MLP in 8 bits: norm with the residual -> gate/up projection -> gated activation -> down projection."""

    def __init__(self, d, f, seed):
        super().__init__()
        rng = np.random.default_rng(seed)
        self.norm = torch.nn.Parameter(torch.from_numpy(1 + 0.1 * rng.normal(0, 1, d)).bfloat16().cuda(), requires_grad=False)
        self.up = torch_ops.Fp8Linear(weights.quantize_fp8_blocks(rng.normal(0, d ** -0.5, (2 * f, d)).astype(np.float32)))
        self.down = torch_ops.Fp8Linear(weights.quantize_fp8_blocks(rng.normal(0, f ** -0.5, (d, f)).astype(np.float32)))
        self.f = f

    def forward(self, x, residual):
        q, s, residual = torch_ops.rmsnorm_fp8(x, self.norm, residual)
        y = self.up((q, s))
        return self.down(torch_ops.gated_fp8(y[..., :self.f], y[..., self.f:])), residual

    def reference(self, x, residual):
        h = x.double() + residual.double()
        y = h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * self.norm.double()
        deq = lambda l: l.weight.float().double() * fp8_ref.expand(l.weight_scale, *l.weight.shape, BLOCK, BLOCK)  # noqa: E731
        z = y @ deq(self.up).t()
        return (z[:, :self.f] * torch.special.expit(z[:, :self.f]) * z[:, self.f:]) @ deq(self.down).t(), h


@pytest.mark.parametrize("m", [1, 9, 130, 700])
@pytest.mark.parametrize("d,f", [(512, 1408), (400, 1000)])
def test_block_together(m, d, f):
    block = Block(d, f, m)
    x, r = (torch.randn(m, d, device="cuda", generator=gen(s)).bfloat16() for s in (1, 2))
    with torch.no_grad():
        y, res = block(x, r)
    ref, h = block.reference(x, r)
    assert torch.equal(res, (x.float() + r.float()).bfloat16())
    # two quantisations of a relative 2^-4 at most, whose errors are independent over the K summands of a product: their
    # root mean square (2^-4 / sqrt(3) at worst each, sqrt(2) for gate and up) bounds the relative error in the 2-norm
    rel = float((y.double() - ref).norm() / ref.norm())
    assert rel <= 2.0 ** -4 / math.sqrt(3) * (math.sqrt(2) + 1), rel


@pytest.mark.parametrize("m", [1, 20, 300])
def test_block_captured_and_replayed(m):
    """One graph, several replays with new inputs, eager work of the same modules between them."""
    block = Block(512, 1408, 0)
    x, r = (torch.randn(m, 512, device="cuda", generator=gen(s)).bfloat16() for s in (1, 2))
    with torch.no_grad():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x, r)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, res = block(x, r)
        for seed in range(5):
            x.copy_(torch.randn(m, 512, device="cuda", generator=gen(10 + seed)))
            r.copy_(torch.randn(m, 512, device="cuda", generator=gen(20 + seed)))
            graph.replay()
            torch.cuda.synchronize()
            want, want_res = block(x.clone(), r.clone())
            assert torch.equal(y, want) and torch.equal(res, want_res)


def test_first_call_of_a_process_is_captured():
    """Nothing that a first call sets up (code objects, shared memory above 64 KiB) disturbs a capture."""
    code = """
import torch
from composable_kernel_amd import torch_ops
x, g = torch.randn(600, 1024, device="cuda").bfloat16(), torch.cuda.CUDAGraph()
w, ws = torch.randn(512, 1024, device="cuda").to(torch.float8_e4m3fn), torch.rand(4, 8, device="cuda")
torch.cuda.synchronize()
with torch.cuda.graph(g):
    y = [torch_ops.fp8_linear(*torch_ops.quantize_fp8(x[:m]), w, ws) for m in (1, 12, 20, 300, 600)]
g.replay(), torch.cuda.synchronize()
for m, v in zip((1, 12, 20, 300, 600), y):
    assert torch.equal(v, torch_ops.fp8_linear(*torch_ops.quantize_fp8(x[:m]), w, ws)), m
print("same")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True,
                       text=True, timeout=100)
    assert r.returncode == 0 and "same" in r.stdout, r.stdout + r.stderr


def test_two_streams_at_once():
    """Calls that overlap on two streams have workspaces of their own."""
    block = Block(512, 1408, 1)
    xs = [torch.randn(100, 512, device="cuda", generator=gen(s)).bfloat16() for s in range(2)]
    with torch.no_grad():
        want = [block(x, x)[0] for x in xs]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in xs]
        got = [[], []]
        for _ in range(20):
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got[i].append(block(xs[i], xs[i])[0])
        torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_compiled_graph_sees_operators():
    """The registered operators answer what the plain functions do."""
    x = torch.randn(6, 512, device="cuda", generator=gen(0)).bfloat16()
    w = torch.ones(512, device="cuda")
    a, b = torch.ops.wqgemm.rmsnorm_fp8(x, w, x, 1e-6, 128), torch_ops.rmsnorm_fp8(x, w, x)
    assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))
    a, b = torch.ops.wqgemm.gated_fp8(x, x, "silu", 0), torch_ops.gated_fp8(x, x, group_k=0)
    assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(a, b))
    q, s = torch.ops.wqgemm.quantize_fp8(x, 128)
    wt = q[:3].contiguous()
    assert torch.equal(torch.ops.wqgemm.fp8_linear(q, s, wt, s[:1], None, "none", torch.float16), torch_ops.fp8_linear(q, s, wt, s[:1], out_dtype=torch.float16))


def test_per_token_scales_feed_the_int4_path():
    """group_k = 0 is the activation operand and the d1 of the fp8 x int4 MultiplyMultiply problem."""
    m, n, k = 40, 256, 512
    x = rows(m, k, 1, torch.float16)
    q, s = torch_ops.quantize_fp8(x, 0)
    w = torch.randint(-8, 8, (n, k), device="cuda", generator=gen(4)).to(torch.int8)
    packed = torch.empty(n, k // 2, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    capi.pack_int4(w.data_ptr(), k, k, n, packed.data_ptr(), k // 2, stream)
    ws = torch.rand(n, device="cuda", generator=gen(5)) + 0.5
    y = torch.empty(m, n, dtype=torch.float16, device="cuda")
    p = capi.fpAintB_problem(q.data_ptr(), packed.data_ptr(), None, y.data_ptr(), m, n, k, a_dtype=capi.F8_E4M3FN, c_dtype=capi.F16,
                             epilogue=capi.EPI_MULTIPLY_MULTIPLY, d0=ws.data_ptr(), d1=s.data_ptr())
    capi.launch(p, None, stream)
    a, b = q.float().double() * s.double(), w.double() * ws.double()[:, None]
    ref, size = fp8_ref.linear(a, b)
    bound = (2 * k + 8) * U32 * size + fp8_ref.HALF_STEP[torch.float16] * ref.abs() * (1 + 2.0 ** -8) + fp8_ref.SMALLEST_HALF_STEP[torch.float16]
    assert bool(((y.double() - ref).abs() <= bound)[torch.isfinite(y)].all()) and bool((torch.isfinite(y) | (ref.abs() > 65000)).all())


@pytest.mark.parametrize("args", [
    ("gemm_ab_scale", 12, 1, 0, 1, 1, 0, 1, 256, 256, 384, -1, -1, -1),
    ("gemm_ab_scale", 13, 1, 0, 1, 2, 0, 1, 300, 520, 1024, -1, -1, -1),
    ("gemm_ab_scale", 13, 1, 0, 1, 2, 0, 1, 64, 256, 4096, -1, -1, -1),
    ("gemm_ab_scale", 14, 1, 0, 1, 2, 0, 1, 16, 512, 640, 656, 672, 530),
    ("gemm_ab_scale", 12, 1, 0, 1, 2, 0, 1, 40, 100, 333, -1, -1, -1, 2, 7, 16),
])
def test_profiler_command_with_fp8_weights(args):
    """The command line's block-scaled operation with fp8 weights, through the C++ operator, verified on the host."""
    exe = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "example_wq_profiler")
    r = subprocess.run([exe, *map(str, args)], capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "verification: PASS" in r.stdout and "Best Perf for datatype" in r.stdout
    assert "16x16x128_f8f6f4" in r.stdout and "DeviceGemmMultiD_ABScale_Mfma_gfx950" in r.stdout
    if len(args) == 17:
        assert "rotating count: 7" in r.stdout
