"""More of what K6, K7 and K8 refuse, and of their host-side logic. Nothing here needs a GPU; the addresses are never read."""
import pytest

from cubert_b200 import kernels

A = 0x10000                                    # an aligned address that nothing dereferences


@pytest.mark.parametrize("channels", [2 ** 30 + 1, 2 ** 30 + 8, 2 ** 31 - 1])
@pytest.mark.parametrize("t", ["f32", "f16"])
def test_rms_norm_refuses_rows_whose_columns_pass_32_bit_arithmetic(channels, t):
    lib = kernels.load()
    assert getattr(lib, "cubk_residual_rms_norm_" + t)(A, None, A, 1, channels, 1e-6, None, A, None) == kernels.CUBK_ERR_UNSUPPORTED
    for group in (0, 128):
        assert getattr(lib, "cubk_residual_rms_norm_e4m3_" + t)(A, None, A, 1, channels, 1e-6, group, None, A, A, None) == kernels.CUBK_ERR_UNSUPPORTED


def test_window_give_ups_needs_a_place_for_the_count():
    assert kernels.load().cubk_window_give_ups(None) == kernels.CUBK_ERR_INVALID_ARG
