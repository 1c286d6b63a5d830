"""Calls of the fp8 operators at the edges of what they accept."""
import pytest
import torch

from test_gpu_fp8 import check, check_exact, launch, problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k,k_batch", [(16, 512, 256, 3), (16, 512, 256, 8), (5, 64, 128, 2), (9, 4100, 400, 6), (16, 8200, 272, 5), (20, 512, 256, 8),
                                           (32, 4104, 384, 4), (8, 64, 128, 4000), (2, 64, 128, 7), (3, 8200, 256, 9), (40, 520, 256, 7), (300, 512, 384, 11)])
def test_slices_behind_the_end_of_k(m, n, k, k_batch):
    """More slices than K has blocks: the last ones are empty and add nothing, in every kernel."""
    P = problem(m, n, k, m + k_batch, exact=True)
    check_exact(launch(P, torch.bfloat16, k_batch=k_batch), P)
    P = problem(m, n, k, m + k_batch)
    check(launch(P, torch.float16, k_batch=k_batch), P, torch.float16)
