"""Calls of the fp8 operators at the edges of what they accept."""
import pytest
import torch

from composable_kernel_amd import capi, torch_ops, weights
import fp8_ref
from fp8_ref import U32
from test_gpu_fp8 import check, check_exact, gen, launch, problem, reference, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,k_batch", [(16, 512, 256, 3), (16, 512, 256, 8), (5, 64, 128, 2), (9, 4100, 400, 6), (16, 8200, 272, 5), (20, 512, 256, 8),
                                           (32, 4104, 384, 4), (8, 64, 128, 4000), (2, 64, 128, 7), (3, 8200, 256, 9), (40, 520, 256, 7), (300, 512, 384, 11)])
def test_slices_behind_the_end_of_k(m, n, k, k_batch):
    """More slices than K has blocks: the last ones are empty and add nothing, in every kernel."""
    P = problem(m, n, k, m + k_batch, exact=True)
    check_exact(launch(P, torch.bfloat16, k_batch=k_batch), P)
    P = problem(m, n, k, m + k_batch)
    check(launch(P, torch.float16, k_batch=k_batch), P, torch.float16)


@pytest.mark.parametrize("block", [(1, 128, 2 ** 31 - 1), (3, 40, 2 ** 31 - 1), (2 ** 31 - 1, 7, 2 ** 31 - 100), (2, 2 ** 31 - 1, 200)])
def test_scale_blocks_longer_than_the_operands(block):
    """One scale along K, as a block of any length says it: each row and column block with its own."""
    bm, bn, bk = block
    m, n, k = 10, 320, 384
    P = problem(m, n, k, 7, bm=min(bm, m), bn=min(bn, n), bk=min(bk, k))
    want, size = reference(P)
    P["block"] = block
    got = launch(P, torch.float16)
    # (the general kernel sums the K products one by one: K additions in place of 128 and the blocks')
    bound = fp8_ref.linear_bound(want, size, k, torch.float16) + 3 * k * U32 * size
    assert bool(((got.double() - want).abs() <= bound).all())
    Q = problem(m, n, k, 7, bm=min(bm, m), bn=min(bn, n), bk=min(bk, k))
    assert torch.equal(got, launch(Q, torch.float16, flags=capi.FLAG_GENERIC | capi.FLAG_BF16_RTN))


def same_bits(got, want):
    return all(torch.equal(g.view(torch.uint8), w.view(torch.uint8)) for g, w in zip(got, want) if w is not None)


@pytest.mark.parametrize("k", [300, 4096, 4097, 5000, 5120, 8192, 8200, 16384, 20000, 40000])
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("residual", [False, True])
def test_a_row_of_the_norm_is_the_same_in_every_batch(k, group, residual):
    """A token of a prefill and the same token alone: equal bytes and scales, whatever the launch's workgroups look like."""
    x, r = rows(600, k, k, torch.bfloat16), rows(600, k, k + 1, torch.bfloat16) if residual else None
    w = (1 + 0.3 * torch.randn(k, device="cuda", generator=gen(3))).to(torch.bfloat16)
    whole = torch_ops.rmsnorm_fp8(x, w, r, 1e-6, group)
    for a, b in ((0, 1), (599, 600), (37, 300), (0, 511), (1, 513), (88, 600)):
        part = torch_ops.rmsnorm_fp8(x[a:b], w, r[a:b] if residual else None, 1e-6, group)
        assert same_bits(part, [t[a:b] if t is not None else None for t in whole]), (a, b)


def test_the_rows_behind_the_last_full_launch_are_no_others():
    """2^21 rows go in one launch: the few behind them take the same sums."""
    k, many = 5000, 2 ** 21 + 5
    part = rows(1021, k, 8, torch.bfloat16)
    x = part.repeat(many // 1021 + 1, 1)[:many]
    w = torch.randn(k, device="cuda", generator=gen(2)).bfloat16()
    whole = torch_ops.rmsnorm_fp8(x, w)[:2]
    for a in (0, 2 ** 21 - 700, many - 700):
        alone = torch_ops.rmsnorm_fp8(x[a:a + 700].clone(), w)[:2]
        assert same_bits([t[a:a + 700] for t in whole], alone), a


def ties(m, k, group, dtype, seed):
    """Rows whose quotients by their scale lie halfway between two e4m3 values, but for the largest of each group.  The scale is s = odd
    * 2^e: the largest value, 448 s, and t s for a t of 5 significant bits have at most 8 bits, so they are bf16 and fp16 values."""
    g = gen(seed)
    width = group or k
    n = -(-k // width)
    pick = lambda lo, hi, shape: torch.randint(lo, hi + 1, shape, device="cuda", generator=g).double()  # noqa: E731
    s = (2 * pick(0, 3, (m, n)) + 1) * torch.exp2(pick(-3, 2, (m, n)))  # 1, 3, 5, 7
    wide = s.repeat_interleave(width, 1)[:, :k]
    t = (2 * pick(8, 15, (m, k)) + 1) * torch.exp2(pick(-10, 3, (m, k)))  # 17 .. 31, odd, up to 248: halfway between two normal values
    low = (2 * pick(0, 7, (m, k)) + 1) * 2.0 ** -10                       # and between two subnormal ones
    t = torch.where(torch.rand(m, k, device="cuda", generator=g) < 0.1, low, t)
    y = t * wide * torch.where(torch.rand(m, k, device="cuda", generator=g) < 0.5, -1.0, 1.0)
    for i in range(n):
        at = i * width + int(torch.randint(0, min(width, k - i * width), (1,), device="cuda", generator=g))
        y[:, at] = 448 * s[:, i]
    x = y.to(dtype)
    assert torch.equal(x.double(), y)
    return x


@pytest.mark.parametrize("m,k", [(3, 128), (40, 1000), (600, 640), (7, 9001), (2, 40000)])
@pytest.mark.parametrize("group", [128, 0])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_ties_of_the_8_bit_format(m, k, group, dtype):
    """Quotients as an IEEE division gives them, rounded to nearest even: bytes and scales bit for bit (the division on the host).  A
    product with the rounded reciprocal would fall to either side of a tie."""
    width = group or k
    n = -(-k // width)
    as_bytes = lambda v: v.view(m, n * width)[:, :k].to(torch.float8_e4m3fn).view(torch.uint8)  # noqa: E731
    for name, x in (("ties", ties(m, k, group, dtype, m + k)), ("any", rows(m, k, m * k, dtype))):
        v = torch.nn.functional.pad(x.float().cpu(), (0, n * width - k)).view(m, n, width)
        want_s = v.abs().amax(2).clamp(min=torch.tensor(1e-12)) / torch.tensor(448.0)
        want = as_bytes(v / want_s[:, :, None])
        if name == "ties" and bool((torch.frexp(want_s)[0] == 7 / 8).any()):  # (of the reciprocals of 1, 3, 5 and 7 only that of 7 misses ties, a quarter of them)
            assert not torch.equal(as_bytes(v * (1 / want_s)[:, :, None]), want)
        q, s = torch_ops.quantize_fp8(x, group)
        assert torch.equal(s.cpu(), want_s) and torch.equal(q.cpu().view(torch.uint8), want)


@pytest.mark.parametrize("flags", [capi.FLAG_TILE_128, capi.FLAG_TILE_256, capi.FLAG_TILE_128 | capi.FLAG_TILE_256])
@pytest.mark.parametrize("m,n,k", [(513, 512, 1024), (300, 520, 400)])
def test_a_row_of_the_product_is_the_same_anywhere(flags, m, n, k):
    """Rows in another order, and some of them alone, on the same kernel: the same bits."""
    P = problem(m, n, k, m + 1)
    whole = launch(P, torch.float16, flags=flags)
    order = torch.randperm(m, device="cuda", generator=gen(4))
    for at in (order, order[:200], order[:77]):
        bits, sa = P["a_bits"][at].contiguous(), P["sa"][at].contiguous()
        part = dict(P, m=len(at), a_bits=bits, a_ptr=bits.data_ptr(), sa=sa)
        assert torch.equal(launch(part, torch.float16, flags=flags), whole[at])


@pytest.mark.parametrize("m,few,n,k", [(4, 3, 4096, 2064), (16, 9, 4096, 640), (16, 7, 5000, 1040), (16, 5, 8200, 400), (32, 20, 4096, 784), (32, 17, 5000, 656)])
def test_a_row_of_few_is_the_same_anywhere(m, few, n, k):
    P = problem(m, n, k, m + 1)
    whole = launch(P, torch.float16)
    order = torch.randperm(m, device="cuda", generator=gen(4))
    for at in (order, order[:few]):
        bits, sa = P["a_bits"][at].contiguous(), P["sa"][at].contiguous()
        part = dict(P, m=len(at), a_bits=bits, a_ptr=bits.data_ptr(), sa=sa)
        assert torch.equal(launch(part, torch.float16), whole[at])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_reduction_needs_no_scales(dtype):
    """The slabs carry the scales: what the problem says of the tables, or does not say, is not looked at."""
    m, n = 37, 64
    slabs = torch.randint(-8, 9, (3, m, n), device="cuda", generator=gen(1)).float()
    out = torch.empty(m, n, dtype=dtype, device="cuda")
    for tables, block in ((slabs.data_ptr(), (0, 0, 0)), (None, (0, 0, 0)), (slabs.data_ptr(), (1, 128, 128))):
        p = capi.f8_problem(slabs.data_ptr(), tables, slabs.data_ptr(), tables, out.fill_(-77).data_ptr(), m, n, 384,
                            c_dtype=capi.F16 if dtype == torch.float16 else capi.BF16, scale_block=block)
        capi.reduce_finalize(p, slabs.data_ptr(), 3, torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out, slabs.sum(0).to(dtype))


@pytest.mark.parametrize("off", [0, 1, 8, 16])
def test_timing_over_copies_stays_in_the_workspace(off):
    """Copies of operands of any alignment: the kernel, and the workspace it asks for, are those of the problem itself.  (1528 x 3265 x 6640
    takes 57 MiB with aligned rows and 30 without.)"""
    m, n, k = 1528, 3265, 6640
    P = problem(m, n, k, 3, offset=off, exact=True)
    c = torch.full((m, n), -77.0, dtype=torch.bfloat16, device="cuda")
    p = capi.f8_problem(P["a_ptr"], P["sa"].data_ptr(), P["b_ptr"], P["sb"].data_ptr(), c.data_ptr(), m, n, k, flags=capi.FLAG_BF16_RTN)
    nbytes = capi.workspace_bytes(p)
    ws = torch.full((nbytes + (64 << 20),), 0xFF, dtype=torch.uint8, device="cuda")
    assert capi.run_timed_rotating(p, ws.data_ptr(), torch.cuda.current_stream().cuda_stream, 1, 5, 3) > 0
    torch.cuda.synchronize()
    assert bool((ws[nbytes:] == 0xFF).all())
    check_exact(c, P)


def test_out_of_memory_is_torchs_own_error():
    """Outputs that do not fit the card, in both ways into the library."""
    m, n, k = 2 ** 24, 2 ** 14, 16
    q, s = torch.zeros(m, k, device="cuda").to(torch.float8_e4m3fn), torch.ones(m, 1, device="cuda")
    w, ws = torch.zeros(n, k, device="cuda").to(torch.float8_e4m3fn), torch.ones(n // 128, 1, device="cuda")
    for call in (torch_ops.fp8_linear, lambda *a: torch_ops._fp8_linear(*a, None, "none", torch.bfloat16)):
        with pytest.raises(torch.OutOfMemoryError):
            call(q, s, w, ws)
    assert torch_ops.fp8_linear(q[:5], s[:5], w, ws).shape == (5, n)


def test_without_the_short_way(monkeypatch):
    """Where the C++ front was not built, the registered operators answer, with the same bits."""
    args = operands(4)
    want = layer(*args)
    monkeypatch.setattr(torch_ops, "_torch_front", torch_ops._NoFront)
    assert same_bits(layer(*args), want)
    x = args[0].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="inference-only"):
        torch_ops.quantize_fp8(x)
    with pytest.raises(ValueError):
        torch_ops.quantize_fp8(args[0], 64)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("stored", [torch.float16, torch.bfloat16, torch.float32])
def test_a_cast_layer_computes_as_before(dtype, stored):
    """A model's .half() or .bfloat16() behind the layer's making; biases of every type, rounded once to the output's."""
    w = torch.randn(300, 400, generator=torch.Generator().manual_seed(1)).numpy()
    bias = torch.randn(300, generator=torch.Generator().manual_seed(2)).to(stored)
    layer = torch_ops.Fp8Linear(weights.quantize_fp8_blocks(w), bias, "fastgelu")
    x = torch.randn(7, 400, device="cuda", generator=gen(3)).to(dtype)
    want = torch_ops.fp8_linear(*torch_ops.quantize_fp8(x), layer.weight, layer.weight_scale, bias.cuda().to(dtype), "add_fastgelu", dtype)
    assert torch.equal(layer(x), want)
    cast = layer.half() if dtype == torch.float16 else layer.bfloat16()
    assert cast.bias.dtype == dtype and torch.equal(cast(x), want)


# ---- calls that something records or transforms ----

def layer(x, norm, wt, ws):
    q, s, h = torch_ops.rmsnorm_fp8(x, norm, x)
    q2, s2 = torch_ops.quantize_fp8(h)
    q3, s3 = torch_ops.gated_fp8(x, h, "fastgelu")
    return torch_ops.fp8_linear(q, s, wt, ws) + torch_ops.fp8_linear(q2, s2, wt, ws), q3, s3


def operands(seed, m=6, k=512, n=72):
    g = gen(seed)
    return (torch.randn(m, k, device="cuda", generator=g).bfloat16(), 1 + 0.1 * torch.randn(k, device="cuda", generator=g),
            torch.randn(n, k, device="cuda", generator=g).to(torch.float8_e4m3fn), torch.rand(1, k // 128, device="cuda", generator=g))


@pytest.mark.parametrize("way", ["compile", "make_fx", "jit"])
def test_a_recorded_program_computes(way):
    """What a tracer has recorded holds the operators, and gives with other inputs what the plain calls give with them."""
    from torch.fx.experimental.proxy_tensor import make_fx

    first = operands(1)
    if way == "compile":
        torch._dynamo.reset()
        program = torch.compile(layer, backend="eager", fullgraph=True)
    else:
        program = make_fx(layer)(*first) if way == "make_fx" else torch.jit.trace(layer, first, check_trace=False)
        text = str(program.graph)
        assert all(f"wqgemm{sep}{op}" in text for op in ("rmsnorm_fp8", "quantize_fp8", "gated_fp8", "fp8_linear") for sep in (["."] if way == "make_fx" else ["::"]))
    for seed in (1, 2, 3):
        args = operands(seed)
        assert same_bits(program(*args), layer(*args))


def test_tangents_and_fake_tensors_of_a_gpu():
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.autograd import forward_ad

    x, w = operands(1)[:2]
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: torch_ops.quantize_fp8(d), lambda: torch_ops.gated_fp8(x, d), lambda: torch_ops.rmsnorm_fp8(d, w)):
            with pytest.raises(RuntimeError, match="inference-only"):
                call()
        assert same_bits(torch_ops.quantize_fp8(x), torch_ops.quantize_fp8(x.clone()))
    with FakeTensorMode(allow_non_fake_inputs=True):
        q, s = torch_ops.quantize_fp8(x)
        assert type(q).__name__ == type(s).__name__ == "FakeTensor" and s.shape == (6, 4)
    assert type(torch_ops.quantize_fp8(x)[0]) is torch.Tensor
