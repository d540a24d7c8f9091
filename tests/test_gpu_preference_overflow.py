"""preference_loss whose coefficient (grad_scale beta times a slope) is beyond f32: held to the largest finite value, no NaN where a probability underflows."""
import pytest

from test_gpu_label_loss import _check_grad, _logits, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [(40, 21, 24), (20, 700, 700), (10, 5001, 5001), (4, 140001, 140001)])
def test_a_coefficient_beyond_f32_is_held(shape):
    import torch
    assert torch.cuda.is_available()
    import em_adapt_tensorflow_amd.ops as ops
    M, C, ldl = shape
    z = _logits(torch, M, ldl, "float32", 31)
    z[:, 0] = -1000.0
    lab = torch.ones(M, dtype=torch.int64, device="cuda")
    at = torch.tensor([0, M // 2, M], device="cuda")
    x, lse, logp, used, tol = _reference(torch, z, lab, C)
    seq = torch.stack([logp[:M // 2].sum(), logp[M // 2:].sum()]).float()
    for ref, beta, scale in ((seq, 1e20, 1e20), (seq, 3e38, -3e38)):      # ratios of a rounding: whatever the slope's half, its product is beyond f32
        for smooth in (0.0, 1.0):
            _, _, d = ops.preference_loss(z, lab, at, ref + torch.tensor([1.0, 0.0] if smooth == 0.0 else [0.0, 1.0], device="cuda"), C, beta=beta,
                                          label_smoothing=smooth, grad_scale=scale)
            sign = (1.0 if scale > 0 else -1.0) * (-1.0 if smooth == 0.0 else 1.0) * torch.finfo(torch.float32).max
            coef = torch.full((M,), sign, dtype=torch.float64, device="cuda")
            coef[M // 2:] = -sign
            _check_grad(torch, d, x, lse, used, lab, coef, torch.zeros_like(lse), tol, C)
