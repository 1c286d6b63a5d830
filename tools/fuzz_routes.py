#!/usr/bin/env python3
"""Time-bounded random sweep over the fp16 / bf16 x int4 / int8 problem space of the C ABI.

Every case runs whatever kernel the dispatcher picks (tile kernels, small-M kernels, split-K with or without a
workspace, plain or pre-shuffled weights, per-channel or group-wise scales, every 16-bit epilogue, padded leading
dimensions) and the general kernel on the plain weight layout; on integer-valued inputs, whose fp32 sums are exact in
any order, the two outputs must be the same bits, and bytes of C outside the M x N block must stay untouched.

    python tools/fuzz_routes.py --seconds 300 --seed 1 --out gpurun_out/fuzz.json
"""
from __future__ import annotations

import argparse
import json
import os
import sys
import time

import numpy as np
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
sys.path.insert(0, os.path.join(ROOT, "tests"))

from composable_kernel_amd import capi  # noqa: E402
from gpu_util import bf16_bits, dev, f16_bits, pack_on_device, run_fpaintb  # noqa: E402

EPILOGUES = [("passthrough", capi.EPI_PASSTHROUGH, 0), ("fastgelu", capi.EPI_FASTGELU, 0), ("add", capi.EPI_ADD, 1),
             ("add_fastgelu", capi.EPI_ADD_FASTGELU, 1), ("multiply", capi.EPI_MULTIPLY, 1),
             ("multiply_fastgelu", capi.EPI_MULTIPLY_FASTGELU, 1), ("multiply_add_fastgelu", capi.EPI_MULTIPLY_ADD_FASTGELU, 2),
             ("convert_bf16_rtn", capi.EPI_CONVERT_BF16_RTN, 0), ("multiply_add_bits", capi.EPI_MULTIPLY_ADD, 2)]
VARIANTS = [capi.FLAG_LOCKSTEP, capi.FLAG_WAVES_2X4, capi.FLAG_DEQUANT_IN_L, capi.FLAG_DIRECT_STORE, capi.FLAG_GROUP8,
            capi.FLAG_MFMA_32X32]


def preshuffle(b, bits4: bool, K: int, N: int) -> torch.Tensor:
    stream = torch.cuda.current_stream().cuda_stream
    if bits4:
        out = torch.zeros(N * K // 2, dtype=torch.uint8, device="cuda")
        capi.preshuffle_int4(b.data_ptr(), K // 2, K, N, out.data_ptr(), K, stream)
    else:
        src = dev(b)
        out = torch.zeros(N * K, dtype=torch.int8, device="cuda")
        capi.preshuffle_int8(src.data_ptr(), K, K, N, out.data_ptr(), K, stream)
    torch.cuda.synchronize()
    return out


def one_case(rng) -> dict:
    a_dtype = (capi.F16, capi.BF16)[int(rng.integers(0, 2))]
    fmt = ("i4", "i8", "u8", "i4pre", "i8pre")[int(rng.integers(0, 5))]
    M = int(rng.choice([1, 2, 5, 8, 16, 17, 32, 48, 64, 65, 100, 128, 200, 256, 257, 300, 512, 700, 1024, 1500, 2048]))
    N = int(rng.choice([32, 64, 96, 128, 192, 256, 320, 512, 768, 1024, 1536, 2048, 4096]))
    K = int(rng.choice([64, 128, 192, 256, 384, 512, 640, 1024, 1536, 2048, 4096]))
    if fmt in ("i4", "i8", "u8") and rng.integers(0, 6) == 0:   # shapes off the tile grid: N % 4, K % 8 only
        N += int(rng.choice([4, 20, 100]))
        K += int(rng.choice([8, 40]))
    bits4 = fmt.startswith("i4")
    lo, hi = (-8, 8) if bits4 else (-128, 128)
    q = rng.integers(lo, hi, (N, K)).astype(np.int8)
    plain = pack_on_device(q, K, N) if bits4 else q
    plain_dtype = capi.I4_PACKED if bits4 else capi.I8
    bkw = {}   # leading dimension / layout of the weights under test
    if fmt == "u8":
        b, b_dtype = (q.astype(np.int16) + 128).astype(np.uint8), capi.U8_OFFSET
    elif fmt.endswith("pre"):
        b, b_dtype = preshuffle(plain, bits4, K, N), (capi.I4_PRESHUFFLED if bits4 else capi.I8_PRESHUFFLED)
    else:
        b, b_dtype = plain, plain_dtype
    if fmt in ("i8", "u8") and rng.integers(0, 5) == 0:      # row-major (K, N) weights
        ldb = N + int(rng.choice([0, 16]))
        bt = np.zeros((K, ldb), dtype=b.dtype)
        bt[:, :N] = b.T
        b, bkw = bt, dict(b_layout=capi.ROW_MAJOR, ldb=ldb)
    elif fmt in ("i8", "u8") and rng.integers(0, 3) == 0:    # padded columns
        ldb = K + int(rng.choice([16, 64]))
        bp = np.zeros((N, ldb), dtype=b.dtype)
        bp[:, :K] = b
        b, bkw = bp, dict(ldb=ldb)
    elif fmt == "i4" and rng.integers(0, 3) == 0:
        ldb = K + int(rng.choice([32, 64]))
        bp = torch.zeros((N, ldb // 2), dtype=torch.uint8, device="cuda")
        bp[:, :K // 2] = plain
        b, bkw = bp, dict(ldb=ldb)
    cvt = f16_bits if a_dtype == capi.F16 else bf16_bits
    lda = K + int(rng.choice([0, 0, 8, 64]))
    a = np.zeros((M, lda), dtype=np.uint16)
    a[:, :K] = cvt(np.round(rng.uniform(-2, 2, (M, K))))
    kw = dict(a_dtype=a_dtype, lda=lda)
    group = int(rng.choice([0, 0, 64, 128, 256]))
    if group and K % group == 0 and fmt != "u8":
        ld_scale = N + int(rng.choice([0, 0, 8]))
        s = np.zeros((K // group, ld_scale), dtype=np.uint16)
        s[:, :N] = cvt(rng.integers(1, 3, (K // group, N)).astype(np.float32))
        kw.update(scale_group_k=group, ld_scale=ld_scale)
    else:
        group = 0
        s = cvt(rng.integers(1, 3, N).astype(np.float32))
    name, epi, nd = EPILOGUES[int(rng.integers(0, len(EPILOGUES)))]
    if epi in (capi.EPI_CONVERT_BF16_RTN, capi.EPI_MULTIPLY_ADD) and a_dtype != capi.BF16:
        name, epi, nd = EPILOGUES[0]
    kw["epilogue"] = epi
    full_d = nd >= 1 and rng.integers(0, 4) == 0   # full (M, N) D tensors instead of per-column vectors
    ldd = N + int(rng.choice([0, 8])) if full_d else 0

    def d_operand():
        if not full_d:
            return cvt(rng.integers(-3, 4, N).astype(np.float32))
        d = np.zeros((M, ldd), dtype=np.uint16)
        d[:, :N] = cvt(rng.integers(-3, 4, (M, N)).astype(np.float32))
        return d

    if nd >= 1:
        kw.update(d0=d_operand(), ldd0=ldd)
    if nd >= 2:
        kw.update(d1=d_operand(), ldd1=ldd)
    if rng.integers(0, 2):
        kw["ldc"] = N + 8
    ref = run_fpaintb(a, plain, s, M, N, K, b_dtype=plain_dtype, flags=capi.FLAG_GENERIC, expect_kernel="wq_gemm_generic", **kw)
    flags = 0
    r = int(rng.integers(0, 6))
    if r == 0:
        flags = capi.FLAG_TILE_128
    elif r == 1:
        flags = capi.FLAG_TILE_256
        if rng.integers(0, 2):
            flags |= VARIANTS[int(rng.integers(0, len(VARIANTS)))]
    if rng.integers(0, 4) == 0 and K >= 512:
        kw["k_batch"] = int(rng.integers(2, 6))
    elif rng.integers(0, 3) == 0:   # the planner's own split-K is optional: without a workspace it runs one slice
        kw["use_workspace"] = False
    # a flag or a split the planner refuses for this shape is dropped, not an error of the sweep
    probe = capi.fpAintB_problem(1 << 20, 1 << 20, 1 << 20, 1 << 20, M, N, K, a_dtype=a_dtype, b_dtype=b_dtype, lda=lda,
                                 ldc=kw.get("ldc"), epilogue=epi, d0=(1 << 20) if nd >= 1 else None,
                                 d1=(1 << 20) if nd >= 2 else None, k_batch=kw.get("k_batch", 1), flags=flags,
                                 scale_group_k=group, ld_scale=kw.get("ld_scale", 0), ldd0=kw.get("ldd0", 0), ldd1=kw.get("ldd1", 0),
                                 **bkw)
    if not capi.is_supported(probe):
        flags = 0
        kw.pop("k_batch", None)
        probe.flags, probe.k_batch = 0, 1
        if not capi.is_supported(probe):
            return dict(skipped=capi.lib.wqgemm_last_error().decode(), fmt=fmt, M=M, N=N, K=K)
    kernel = capi.kernel_name(probe)
    got = run_fpaintb(a, b, s, M, N, K, b_dtype=b_dtype, flags=flags, **bkw, **kw)
    desc = dict(weights=bkw, full_d=bool(full_d), fmt=fmt, a="f16" if a_dtype == capi.F16 else "bf16", M=M, N=N, K=K, lda=lda, ldc=kw.get("ldc", N), group=group,
                epilogue=name, k_batch=kw.get("k_batch", 1), workspace=kw.get("use_workspace", True), flags=flags, kernel=kernel)
    # (an output still holding the poison pattern everywhere would compare equal: that is a failure too)
    desc["equal"] = bool(np.array_equal(got[:, :N], ref[:, :N]) and (got[:, :N] != 0x7BFF).any())
    desc["padding_untouched"] = bool((got[:, N:] == 0x7BFF).all())
    if not desc["equal"]:
        bad = got[:, :N] != ref[:, :N]
        desc["mismatches"] = int(bad.sum())
        if bad.any():
            i, j = np.argwhere(bad)[0]
            desc["first"] = [int(i), int(j), int(got[i, j]), int(ref[i, j])]
    return desc


def _run_i8(a, b, M, N, K, requant, flags, lda, ldb, ldc, bias, relu, use_workspace=True):
    a_t, b_t = dev(a), dev(b)
    e_t = torch.full((M + 16, ldc), 77, dtype=torch.int8, device="cuda")   # 16 guard rows
    bias_t = dev(np.ascontiguousarray(bias, np.int32)) if bias is not None else None
    epi = ((capi.EPI_ADD_RELU_MUL_CLAMP if relu else capi.EPI_ADD_ACT_MUL_CLAMP) if bias is not None
           else (capi.EPI_RELU_MUL_CLAMP if relu else capi.EPI_ACT_MUL_CLAMP))
    p = capi.fpAintB_problem(a_t.data_ptr(), b_t.data_ptr(), None, e_t.data_ptr(), M, N, K, a_dtype=capi.I8, b_dtype=capi.I8,
                             c_dtype=capi.I8, epilogue=epi, requant=requant, d0=bias_t.data_ptr() if bias_t is not None else None,
                             flags=flags, lda=lda, ldb=ldb, ldc=ldc)
    if not capi.is_supported(p):
        return None, None
    nbytes = capi.workspace_bytes(p)   # the planner's own split-K of a short grid: optional
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda") if nbytes and use_workspace else None
    capi.launch(p, ws.data_ptr() if ws is not None else None, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return e_t.cpu().numpy(), capi.kernel_name(p) + ("+splitk" if ws is not None else "")


def one_case_i8(rng) -> dict:
    """int8 x int8 -> int8 behind the requantisation epilogues: integer accumulation, so random data is exact."""
    M = int(rng.choice([1, 2, 5, 9, 12, 16, 64, 100, 128, 200, 256, 300, 513, 1024, 2048]))
    N = int(rng.choice([16, 48, 100, 128, 256, 384, 512, 1024, 2048, 4096, 8192]))
    K = int(rng.choice([128, 256, 384, 640, 1024, 2048, 2304, 4096, 5120, 8192]))
    lda, ldb, ldc = K + int(rng.choice([0, 0, 16, 128])), K + int(rng.choice([0, 0, 16, 128])), N + int(rng.choice([0, 0, 16]))
    a = rng.integers(-128, 128, (M, lda)).astype(np.int8)
    b = rng.integers(-128, 128, (N, ldb)).astype(np.int8)
    bias = rng.integers(-50000, 50001, N).astype(np.int32) if rng.integers(0, 2) else None
    relu = bool(rng.integers(0, 2))
    rq = float(rng.choice([1e-4, 1e-3, 0.03]))
    flags = (0, capi.FLAG_TILE_128, capi.FLAG_TILE_256)[int(rng.integers(0, 3))]
    use_ws = bool(rng.integers(0, 4))
    got, kernel = _run_i8(a, b, M, N, K, rq, flags, lda, ldb, ldc, bias, relu, use_ws)
    if got is None:
        got, kernel = _run_i8(a, b, M, N, K, rq, 0, lda, ldb, ldc, bias, relu, use_ws)
    ref, _ = _run_i8(a, b, M, N, K, rq, capi.FLAG_GENERIC, lda, ldb, ldc, bias, relu)
    desc = dict(fmt="i8xi8", M=M, N=N, K=K, lda=lda, ldb=ldb, ldc=ldc, bias=bias is not None, relu=relu, requant=rq, k_batch=1,
                kernel=kernel)
    desc["equal"] = bool(np.array_equal(got[:M, :N], ref[:M, :N]) and (got[:M, :N] != 77).any())
    desc["padding_untouched"] = bool((got[M:] == 77).all() and (got[:, N:] == 77).all())
    return desc


E4M3FNUZ = {0: 0x00, 1: 0x40, 2: 0x48, 3: 0x4C, 4: 0x50, -1: 0xC0, -2: 0xC8, -3: 0xCC, -4: 0xD0}   # bias 8
E4M3FN = {0: 0x00, 1: 0x38, 2: 0x40, 3: 0x44, 4: 0x48, -1: 0xB8, -2: 0xC0, -3: 0xC4, -4: 0xC8}     # bias 7


def one_case_f8(rng) -> dict:
    """fp8 x int4 + MultiplyMultiply[+FastGelu] on the fp8 matrix core, both byte formats, plain and pre-shuffled
    weights: small integers as activations and power-of-two factors keep every sum exact."""
    M = int(rng.choice([1, 7, 16, 64, 65, 100, 128, 256, 300, 512, 700, 1024, 2048]))
    N = int(rng.choice([256, 512, 1024, 2048, 4096, 8192]))
    K = int(rng.choice([128, 256, 384, 640, 1024, 2048, 4096]))
    fn = bool(rng.integers(0, 2))
    pre = bool(rng.integers(0, 2))
    q = rng.integers(-8, 8, (N, K)).astype(np.int8)
    plain = pack_on_device(q, K, N)
    b = preshuffle(plain, True, K, N) if pre else plain
    lda = K + int(rng.choice([0, 0, 16, 128]))
    lut = np.zeros(9, dtype=np.uint8)
    for v, code in (E4M3FN if fn else E4M3FNUZ).items():
        lut[v + 4] = code
    a = np.zeros((M, lda), dtype=np.uint8)
    a[:, :K] = lut[rng.integers(-4, 5, (M, K)) + 4]
    d0 = (2.0 ** rng.integers(-6, -2, N)).astype(np.float32)
    d1 = (2.0 ** rng.integers(-3, 1, M)).astype(np.float32)
    gelu = bool(rng.integers(0, 2))
    kw = dict(a_dtype=capi.F8_E4M3FN if fn else capi.F8_FNUZ, lda=lda, d0=d0, d1=d1,
              epilogue=capi.EPI_MULTIPLY_MULTIPLY_FASTGELU if gelu else capi.EPI_MULTIPLY_MULTIPLY)
    if rng.integers(0, 2):
        kw["ldc"] = N + 8
    kb = int(rng.integers(2, 6)) if (rng.integers(0, 4) == 0 and K >= 512) else 1
    flags = 0 if fn else capi.FLAG_F8_NO_SPECIALS
    if not pre and rng.integers(0, 4) == 0:
        flags |= capi.FLAG_PINGPONG
    ref = run_fpaintb(a, plain, None, M, N, K, flags=capi.FLAG_GENERIC, expect_kernel="wq_gemm_generic", **kw)
    b_dtype = capi.I4_PRESHUFFLED if pre else capi.I4_PACKED
    probe = capi.fpAintB_problem(1 << 20, 1 << 20, None, 1 << 20, M, N, K, a_dtype=kw["a_dtype"], c_dtype=capi.F16, b_dtype=b_dtype,
                                 lda=lda, ldc=kw.get("ldc"), epilogue=kw["epilogue"], d0=1 << 20, d1=1 << 20, k_batch=kb, flags=flags)
    kernel = capi.kernel_name(probe)   # the fp8 tile kernel, or (M <= 16) the fp16 image + streaming kernel
    assert kernel in ("wq_gemm_f8_mfma_256", "wq_gemm_skinny_ws", "wq_f8_fnuz_to_f16+wq_gemm_skinny_wsc"), kernel
    got = run_fpaintb(a, b, None, M, N, K, b_dtype=b_dtype, flags=flags, k_batch=kb,
                      use_workspace=bool(kb > 1 or rng.integers(0, 3)), **kw)
    desc = dict(fmt="f8xi4" + ("pre" if pre else ""), e4m3fn=fn, M=M, N=N, K=K, lda=lda, ldc=kw.get("ldc", N), gelu=gelu, k_batch=kb,
                flags=flags, kernel=kernel)
    # (an output still holding the poison pattern everywhere would compare equal: that is a failure too)
    desc["equal"] = bool(np.array_equal(got[:, :N], ref[:, :N]) and (got[:, :N] != 0x7BFF).any())
    desc["padding_untouched"] = bool((got[:, N:] == 0x7BFF).all())
    if not desc["equal"]:
        bad = got[:, :N] != ref[:, :N]
        desc["mismatches"] = int(bad.sum())
        if bad.any():
            i, j = np.argwhere(bad)[0]
            desc["first"] = [int(i), int(j), int(got[i, j]), int(ref[i, j])]
    return desc


def one_case_ab(rng) -> dict:
    """fp8 x int4 / int8 with block-wise scales of both operands: the dispatcher's kernel (the block-scaled fp8 matrix-core
    kernel where the block shape allows it) against the general kernel.  Small integers and power-of-two scales keep every
    block sum, every scaled partial and the running sum exact, so both must give the same bits."""
    M = int(rng.choice([1, 7, 64, 100, 128, 256, 300, 512, 700, 1024]))
    N = int(rng.choice([256, 512, 1024, 2048]))
    K = int(rng.choice([128, 256, 384, 640, 1024, 2048]))
    fn = bool(rng.integers(0, 2))
    bf = bool(rng.integers(0, 2))
    kind = int(rng.integers(0, 3))   # packed int4, pre-shuffled int4, int8
    bm = int(rng.choice([128, 128, 256, 64, 1, 1, 48]))
    bn = int(rng.choice([128, 128, 32, 64, 256, 16]))
    bk = int(rng.choice([128, 128, 128, 64, 256]))
    q = rng.integers(-8, 8, (N, K)).astype(np.int8)
    if kind == 2:
        b, b_dtype = dev(q), capi.I8
    else:
        b = pack_on_device(q, K, N)
        b_dtype = capi.I4_PACKED
        if kind == 1:
            b, b_dtype = preshuffle(b, True, K, N), capi.I4_PRESHUFFLED
    lda = K + int(rng.choice([0, 0, 16, 128]))
    lut = np.zeros(9, dtype=np.uint8)
    for v, code in (E4M3FN if fn else E4M3FNUZ).items():
        lut[v + 4] = code
    a = np.zeros((M, lda), dtype=np.uint8)
    a[:, :K] = lut[rng.integers(-4, 5, (M, K)) + 4]
    kblocks = (K + bk - 1) // bk
    ld_sa = kblocks + int(rng.choice([0, 0, 3]))
    ld_sb = kblocks + int(rng.choice([0, 0, 5]))
    sa = (2.0 ** rng.integers(-6, -2, ((M + bm - 1) // bm, ld_sa))).astype(np.float32)
    sb = (2.0 ** rng.integers(-5, 0, ((N + bn - 1) // bn, ld_sb))).astype(np.float32)
    kw = dict(a_dtype=capi.F8_E4M3FN if fn else capi.F8_FNUZ, lda=lda, a_block_scale=sa, b_block_scale=sb, scale_block=(bm, bn, bk),
              ld_a_scale=ld_sa, ld_b_scale=ld_sb, c_dtype=capi.BF16 if bf else capi.F16, b_dtype=b_dtype)
    if rng.integers(0, 2):
        kw["ldc"] = N + 8
    flags = 0 if fn else capi.FLAG_F8_NO_SPECIALS
    kb = int(rng.integers(2, 5)) if (rng.integers(0, 3) == 0 and K >= 512) else 1
    ref = run_fpaintb(a, b, None, M, N, K, flags=capi.FLAG_GENERIC, expect_kernel="wq_gemm_generic", **kw)
    probe = capi.fpAintB_problem(1 << 20, 1 << 20, None, 1 << 20, M, N, K, a_dtype=kw["a_dtype"], c_dtype=kw["c_dtype"], b_dtype=b_dtype,
                                 lda=lda, ldc=kw.get("ldc"), flags=flags, a_block_scale=1 << 20, b_block_scale=1 << 20,
                                 scale_block=(bm, bn, bk), ld_a_scale=ld_sa, ld_b_scale=ld_sb, k_batch=kb)
    if not capi.is_supported(probe):   # (pre-shuffled weights with a block shape only the general kernel takes: refused by design)
        return {"skipped": capi.lib.wqgemm_last_error().decode()}
    kernel = capi.kernel_name(probe).split("+")[0]   # (a planner's or caller's split appends the reduce stage)
    want = "wq_gemm_generic" if (kind == 2 or bk != 128 or bn % 32) else \
        "wq_gemm_f8_mfma_256_abscale" if bm % 128 == 0 else "wq_gemm_f8_mfma_256_abscale_rows"
    assert kernel == want, (kernel, want, bm, bn, bk, kind, kb)
    got = run_fpaintb(a, b, None, M, N, K, flags=flags, k_batch=kb, use_workspace=bool(kb > 1 or rng.integers(0, 3)), **kw)
    desc = dict(fmt=("i4", "i4pre", "i8")[kind], e4m3fn=fn, bf16=bf, M=M, N=N, K=K, lda=lda, ldc=kw.get("ldc", N), block=[bm, bn, bk],
                ld_scales=[ld_sa, ld_sb], k_batch=kb, kernel=kernel)
    desc["equal"] = bool(np.array_equal(got[:, :N], ref[:, :N]) and (got[:, :N] != 0x7BFF).any())
    desc["padding_untouched"] = bool((got[:, N:] == 0x7BFF).all())
    if not desc["equal"]:
        bad = got[:, :N] != ref[:, :N]
        desc["mismatches"] = int(bad.sum())
        if bad.any():
            i, j = np.argwhere(bad)[0]
            desc["first"] = [int(i), int(j), int(got[i, j]), int(ref[i, j])]
    return desc


def one_case_f8f8(rng) -> dict:
    """fp8 x fp8 with block-wise scales: any M, N, K, strides, alignment, block shape, epilogue, tile size and K split, whatever kernel
    the dispatcher picks against the general kernel.  Small integers and power-of-two scales keep every sum exact."""
    pick = lambda *v: int(rng.choice(v))  # noqa: E731
    M = pick(1, 3, 4, 5, 16, 17, 32, 33, 64, 65, 100, 128, 200, 256, 257, 400, 600, 1024, 2048) if rng.integers(0, 3) else int(rng.integers(1, 1500))
    N = pick(128, 256, 512, 1024, 2048, 4096) if rng.integers(0, 2) else int(rng.integers(1, 5000))
    K = pick(128, 256, 384, 400, 512, 640, 1024, 2048, 4096) if rng.integers(0, 2) else int(rng.integers(1, 4200))
    if rng.integers(0, 2):
        K = -(-K // 16) * 16
    fnuz = [bool(v) for v in rng.integers(0, 5, 2) == 0]
    bf, rtn = bool(rng.integers(0, 2)), bool(rng.integers(0, 2))
    bm, bn, bk = pick(1, 1, 128, 7, 64), pick(128, 128, 32, 96, 48), pick(128, 128, 128, 128, 64)
    off = [pick(0, 0, 0, 1, 16), pick(0, 0, 0, 3, 32)]
    lda, ldb, ldc = K + pick(0, 0, 16, 128, 5), K + pick(0, 0, 16, 64, 3), N + pick(0, 0, 8, 3)
    epi = pick(capi.EPI_PASSTHROUGH, capi.EPI_PASSTHROUGH, capi.EPI_FASTGELU, capi.EPI_ADD, capi.EPI_ADD_FASTGELU)
    k_batch = pick(2, 3, 5, 40) if rng.integers(0, 5) == 0 and N % 4 == 0 and ldc % 4 == 0 else 1  # (40: mostly more than K has blocks)
    pin = pick(0, 0, 0, capi.FLAG_TILE_128, capi.FLAG_TILE_256, capi.FLAG_TILE_128 | capi.FLAG_TILE_256)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(rng.integers(0, 1 << 30)))
    ptr = []
    keep = []
    for rows, ld, o, z in ((M, lda, off[0], fnuz[0]), (N, ldb, off[1], fnuz[1])):
        lut = torch.zeros(9, dtype=torch.uint8)
        for v, code in (E4M3FNUZ if z else E4M3FN).items():
            lut[v + 4] = code
        t = torch.full((o + rows * ld + 64,), 0x7F, dtype=torch.uint8, device="cuda")
        t[o:o + rows * ld].view(rows, ld)[:, :K] = lut.cuda()[torch.randint(0, 9, (rows, K), device="cuda", generator=g)]
        keep.append(t)
        ptr.append(t.data_ptr() + o)
    kb = -(-K // bk)
    ld_s = [kb + pick(0, 0, 3), kb + pick(0, 0, 5)]
    sa = torch.exp2(torch.randint(-6, -2, (-(-M // bm), ld_s[0]), device="cuda", generator=g).float())
    sb = torch.exp2(torch.randint(-5, 0, (-(-N // bn), ld_s[1]), device="cuda", generator=g).float())
    dtype = torch.bfloat16 if bf else torch.float16
    d0 = torch.randint(-8, 9, (N,), device="cuda", generator=g).to(dtype)
    stream = torch.cuda.current_stream().cuda_stream

    def run(flags, split, workspace):
        c = torch.full((M + 300, ldc), -77.0, dtype=dtype, device="cuda")
        p = capi.f8_problem(ptr[0], sa.data_ptr(), ptr[1], sb.data_ptr(), c.data_ptr(), M, N, K, lda=lda, ldb=ldb, ldc=ldc,
                            a_dtype=capi.F8_FNUZ if fnuz[0] else capi.F8_E4M3FN, b_dtype=capi.F8_FNUZ if fnuz[1] else capi.F8_E4M3FN,
                            c_dtype=capi.BF16 if bf else capi.F16, epilogue=epi, d0=d0.data_ptr(), k_batch=split, scale_block=(bm, bn, bk),
                            ld_a_scale=ld_s[0], ld_b_scale=ld_s[1], flags=flags | (capi.FLAG_BF16_RTN if rtn else 0) | capi.FLAG_F8_NO_SPECIALS)
        if not capi.is_supported(p):
            return None, capi.lib.wqgemm_last_error().decode(), 1
        n = capi.workspace_bytes(p) if workspace else 0
        ws = torch.full((n + 64,), 0xFF, dtype=torch.uint8, device="cuda")
        text = capi.type_string(p) if workspace else "KBatch1>"
        capi.launch(p, ws.data_ptr() if n else None, stream)
        torch.cuda.synchronize()
        assert bool((ws[n:] == 0xFF).all())
        return c, capi.kernel_name(p).split("+")[0], int(text.rsplit("KBatch", 1)[1].rstrip(">")) if "KBatch" in text else 1

    ref, _, _ = run(capi.FLAG_GENERIC, 1, False)
    got, kernel, slices = run(pin, k_batch, k_batch > 1 or bool(rng.integers(0, 4)))
    if got is None:
        return {"skipped": kernel}
    desc = dict(fmt="f8xf8", fnuz=fnuz, bf16=bf, rtn=rtn, M=M, N=N, K=K, lda=lda, ldb=ldb, ldc=ldc, offsets=off, block=[bm, bn, bk], ld_scales=ld_s,
                epilogue=epi, k_batch=slices, pinned=pin, kernel=kernel)
    desc["equal"] = bool(torch.equal(got[:M, :N], ref[:M, :N]))
    desc["padding_untouched"] = bool((got[:M, N:] == -77).all() and (got[M:] == -77).all())
    if not desc["equal"]:
        bad = torch.nonzero(got[:M, :N] != ref[:M, :N])
        desc["mismatches"], (i, j) = len(bad), bad[0].tolist() if len(bad) else (0, 0)
        desc["first"] = [i, j, float(got[i, j]), float(ref[i, j])]
    return desc


def main() -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--seconds", type=float, default=120)
    ap.add_argument("--seed", type=int, default=1)
    ap.add_argument("--out", default=None)
    ap.add_argument("--family", choices=("fp", "i8", "f8", "ab", "f8f8"), default="fp",
                    help="fp: fp16/bf16 x int4/int8; i8: int8 x int8 requantised; f8: fp8 x int4 MultiplyMultiply; "
                         "ab: fp8 x int4/int8 with block-wise scales of both operands; f8f8: fp8 x fp8 with them")
    args = ap.parse_args()
    rng = np.random.default_rng(args.seed)
    t0 = time.time()
    kernels, failures, skipped, n = {}, [], 0, 0
    while time.time() - t0 < args.seconds:
        d = {"fp": one_case, "i8": one_case_i8, "f8": one_case_f8, "ab": one_case_ab, "f8f8": one_case_f8f8}[args.family](rng)
        if "skipped" in d:
            skipped += 1
            continue
        n += 1
        key = d["kernel"] + ("" if d["k_batch"] == 1 else "+splitk")
        kernels[key] = kernels.get(key, 0) + 1
        if not (d["equal"] and d["padding_untouched"]):
            failures.append(d)
            print("FAIL", json.dumps(d), flush=True)
        if n % 50 == 0:
            print(f"[{time.time() - t0:6.0f} s] {n} cases, {len(failures)} failures, {skipped} skipped", flush=True)
    summary = dict(family=args.family, seed=args.seed, seconds=round(time.time() - t0, 1), cases=n, skipped=skipped, failures=failures, kernels=kernels)
    print(json.dumps(summary))
    if args.out:
        os.makedirs(os.path.dirname(args.out) or ".", exist_ok=True)
        with open(args.out, "w") as f:
            json.dump(summary, f, indent=1)
    return 1 if failures else 0


if __name__ == "__main__":
    sys.exit(main())
