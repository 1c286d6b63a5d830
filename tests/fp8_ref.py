"""64-bit definitions of the fp8 operators and the error bounds their tests use."""
from __future__ import annotations

import torch

U32 = 2.0 ** -24                                             # half a step of fp32
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
SMALLEST_HALF_STEP = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
F8_MAX, FLOOR, BLOCK = 448.0, 1e-12, 128


def f8_values(bits: torch.Tensor, fnuz: bool = False) -> torch.Tensor:
    """uint8 e4m3fn (or e4m3 FNUZ) bit patterns -> float64, from the formats' definitions."""
    b = bits.to(torch.int64)
    e, m = (b >> 3) & 15, b & 7
    bias = 8 if fnuz else 7
    v = torch.where(e == 0, m.double() * 2.0 ** (-2 - bias), (8 + m).double() * torch.pow(2.0, (e - 3 - bias).double()))
    v = torch.where(b >= 128, -v, v)
    nan = (b == 0x80) if fnuz else (b & 0x7F) == 0x7F
    return torch.where(nan, torch.full_like(v, float("nan")), v)


def expand(s: torch.Tensor, rows: int, cols: int, block_rows: int, block_cols: int) -> torch.Tensor:
    """Block table -> one value per element, float64."""
    return s.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(block_cols, 1)[:, :cols]


def fastgelu(v: torch.Tensor) -> torch.Tensor:
    return v * torch.special.expit(2 * (0.797885 * v + 0.035677 * v ** 3))


def linear(a: torch.Tensor, b: torch.Tensor, bias=None, act: str = "none"):
    """a (M, K), b (N, K) float64, scales applied -> (y, S): the product after epilogue, and sum_k |a b|."""
    y, size = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        y = y + bias.double()
        size = size + bias.double().abs()
    return (fastgelu(y) if act.endswith("fastgelu") else y), size


def linear_bound(y, size, K: int, dtype, act: str = "none") -> torch.Tensor:
    """Largest error of a kernel that sums each 128-k block on the matrix core, multiplies by the product of the scales (rounded
    once, then a fused multiply-add per block), sums the blocks and at most 64 slices in fp32 and rounds once to dtype.

    The fp8 matrix core takes 8 consecutive k together: it aligns their products to the largest one's exponent e and drops what
    lies below 2^(e - 13) (2^16 + 2^3 survives, 2^16 + 2^2 does not; 8 k apart 2^16 + 2^-7 does).  Each of the 7 others loses
    less than 2^(e - 13) <= 2^-13 of the largest product, so a group is off by 7 * 2^-13 of its largest product and a block by
    7 * 2^-13 of its S; then 128 / 8 additions off by at most a step, 2 * U, of at most S each.
    FastGelu: |slope| <= 1.13; its exponent is off by a few steps of an argument that matters up to |u| ~ 20, the exponential
    and the reciprocal by one each: 64 steps of |y| <= |x| <= S cover it."""
    kb = -(-K // BLOCK)
    err = (7 * 2.0 ** -13 + (2 * 16 + kb + 64 + 4) * U32) * size
    if act.endswith("fastgelu"):
        err = 1.13 * err + 64 * U32 * size
    return err + HALF_STEP[dtype] * (y.abs() + err) + SMALLEST_HALF_STEP[dtype]


def quant_scales(y: torch.Tensor, group: int) -> torch.Tensor:
    m, k = y.shape
    g = group or k
    n = -(-k // g)
    p = torch.nn.functional.pad(y, (0, n * g - k)).view(m, n, g)
    return p.abs().amax(2).clamp(min=FLOOR) / F8_MAX


def check_quantized(q: torch.Tensor, scale: torch.Tensor, y: torch.Tensor, group: int, rel: float, abs_err=0.0):
    """q, scale of a quantiser against y (float64): the scale is off by at most the error of y's largest magnitude (rel, and
    abs_err where y is a sum) and three fp32 roundings; q times the scale it stands beside by half an e4m3 step (2^-4 of the value,
    2^-10 of the scale below the normal numbers), the error of y, and the three fp32 roundings of the quotient."""
    m, k = y.shape
    want = quant_scales(y, group)
    assert scale.shape == want.shape, (scale.shape, want.shape)
    s = scale.double()
    slack = abs_err if isinstance(abs_err, torch.Tensor) else torch.full_like(y, abs_err)
    tol_s = want * (rel + 4 * U32) + quant_scales(slack, group) + 2.0 ** -149
    bad = (s - want).abs() > tol_s
    assert not bool(bad.any()), f"scale off by {float(((s - want).abs() / want).max())} relative"
    g = group or k
    wide = s.repeat_interleave(g, 1)[:, :k]
    got = q.float().double() * wide
    tol = (2.0 ** -4) * y.abs() * (1 + 2.0 ** -4) * (1 + 8 * U32 + rel) + 2.0 ** -10 * wide * (1 + 8 * U32) + (rel + 8 * U32) * y.abs() + slack
    # (half a step of the rounded value: a value just under a power of two rounds by the finer step, never a coarser one; the
    # 1 + 2^-4 lets |y| stand for the larger of y and its rounding)
    worst = ((got - y).abs() - tol).max()
    assert float(worst) <= 0, f"q * scale exceeds its bound by {float(worst)}"
