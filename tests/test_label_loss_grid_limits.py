"""Sizes that one grid (fewer than 2^32 threads) cannot hold are refused before anything is launched.  No device is needed: the addresses are never read."""
import pytest

OK, UNSUPPORTED = 0, -2


@pytest.fixture(scope="module")
def lib():
    import torch
    if torch.cuda.is_available():
        pytest.skip("with addresses that are none: on a machine without a device")
    from em_adapt_tensorflow_amd import _lib
    return _lib.load()


@pytest.mark.parametrize("ldl,dtype,M", [(1, 0, 1 << 34), (1, 1, 1 << 34), (4, 0, 1 << 34), (9, 1, 1 << 33), (5, 0, 1 << 33), (1 << 30, 0, 64), (1 << 30, 1, 128)])
def test_gradients_of_more_vectors_than_a_grid_has_threads(lib, ldl, dtype, M):
    at = [k << 52 for k in range(1, 12)]
    size = 1 << 50
    assert lib.emadapt_label_logp_bwd(at[0], dtype, ldl, at[1], at[2], at[3], M, 1, at[4], dtype, None) == UNSUPPORTED
    assert lib.emadapt_policy_loss(at[0], dtype, ldl, at[1], at[2], None, at[3], None, M, 1, 0.2, 0.2, 0.0, 1.0, at[4], at[5], at[6], dtype, at[7], size, None) == UNSUPPORTED
    assert lib.emadapt_preference_loss(at[0], dtype, ldl, at[1], at[2], 1, at[3], M, 1, 0.1, 0.0, 1.0, at[4], at[5], at[6], dtype, at[7], size, None) == UNSUPPORTED


def test_sizes_below_are_not(lib):
    # (no rows: accepted and nothing to do; the limit is on rows times vectors)
    assert lib.emadapt_label_logp_bwd(None, 0, 1 << 30, None, None, None, 0, 1, None, 0, None) == OK
