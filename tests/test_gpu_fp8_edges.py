"""Calls of the fp8 operators at the edges of what they accept."""
import pytest
import torch

from composable_kernel_amd import capi
import fp8_ref
from fp8_ref import U32
from test_gpu_fp8 import check, check_exact, launch, problem, reference

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
