"""What the library accepts and refuses of the fp8 operators at the edges of their sizes.  No GPU call is made here."""
import pytest

from composable_kernel_amd import capi
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
