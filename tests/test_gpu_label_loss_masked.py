"""Log-probabilities of labels at places that a mask has set to the type's lowest value, or that lie in a row with -inf elsewhere: finite, without exception."""
import pytest

from test_gpu_label_loss import H, _labels, _logits, _reference, _say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    import em_adapt_tensorflow_amd.ops as ops
    return ops, torch


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,C,ldl", [(300, 21, 24), (40, 5000, 5000), (6, 130000, 130000)])
def test_labels_at_masked_places(env, M, C, ldl, dtype):
    """Every second row masked over its first half; the labels of the masked rows on both sides of the border.  Tolerances as in test_gpu_label_loss.py."""
    ops, torch = env
    _say("masked labels", M, C, dtype)
    z = _logits(torch, M, ldl, dtype, 3)
    lab = _labels(torch, M, C, 3, outside=False)
    z[::2, : C // 2] = torch.finfo(z.dtype).min
    lab[0::4] = lab[0::4] % (C // 2)                     # masked
    lab[2::4] = C // 2 + lab[2::4] % (C - C // 2)        # not masked
    z[1::4, C - 1] = float("-inf")
    lab[1::4] = lab[1::4].clamp(max=C - 2)
    logp, lse = ops.label_logp(z, lab, C)
    assert bool(torch.isfinite(logp).all()) and bool(torch.isfinite(lse).all())
    assert bool((logp[0::4] < -1e38).all()) and bool((logp[2::4] > -1e3).all())
    for r in range(M):
        ok = torch.isfinite(z[r:r + 1, :C])[0]
        row, at = z[r:r + 1, :C][:, ok], ok[: int(lab[r])].sum().view(1)
        x, want_lse, want, used, tol = _reference(torch, row, at, row.shape[1])
        size = x[0, int(at)].abs() + want.abs()
        assert bool((lse[r].double() - want_lse).abs() <= tol) and bool((logp[r].double() - want).abs() <= tol + H * size)
