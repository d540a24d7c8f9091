"""policy_loss where exp(logp - old_logp) or exp(ref_logp - logp) is beyond f32: an action that the old policy held for impossible, a reference far from
the network.  Against the formulas in 64 bits.

Tolerances, with h = 2^-24: an exponential of x is off by 3 h |x| + 16 h of itself (x rounded to f32, its eighth's product with log2 e and that constant,
then the eighth power of an f32 exponential that is off by 2 h), and by x's own error: that of the log-probability (test_gpu_label_loss.py) and h (|old| +
|ref|) of the inputs' differences; the products behind it are 64-bit ones, rounded once to f32: 20 h in all."""
import pytest

from test_gpu_label_loss import H, _check_grad, _labels, _logits, _reference, _say

pytestmark = pytest.mark.gpu

# rows by lanes with the 64-bit path in place (one workgroup, several), by lanes of a whole wave, in a workgroup's registers, few rows in parts, streamed rows
SHAPES = [(40, 21, 24), (3000, 21, 24), (20, 700, 700), (200, 5001, 5001), (6, 40000, 40000), (130, 140001, 140001)]


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    import em_adapt_tensorflow_amd.ops as ops
    return ops, torch


def _want(torch, z, lab, old, adv, C, ref, w, lo, hi, kl, scale):
    x, lse, logp, used, tol = _reference(torch, z, lab, C, w != 0)
    zero = torch.zeros_like(lse)
    off = tol + H * (old.double().abs() + ref.double().abs() + 3 * logp.abs())
    lr, q = torch.where(used, logp - old.double(), zero), torch.where(used, ref.double() - logp, zero)
    A, wt = adv.double(), torch.where(used, w.double(), zero)
    r, e = torch.exp(lr.clamp(max=700)), torch.exp(q)
    held = -A * r.clamp(1 - lo, 1 + hi)
    clip = held > -A * r
    part = torch.where(clip, held, -A * r)
    k = torch.expm1(q) - q
    e_r, e_e = torch.where(clip, zero, (A * r).abs() * (off + 3 * H * lr.abs() + 20 * H)), (e + 1) * (off + 3 * H * q.abs() + 20 * H)
    sums = torch.stack([(wt * (part + kl * k)).sum(), (wt * part).sum(), (wt * k).sum(), (wt * clip).sum()])
    sums_tol = torch.stack([(wt * (e_r + kl * e_e)).sum(), (wt * e_r).sum(), (wt * e_e).sum(), zero.sum()]) + 8 * H * sums.abs() + 1e-30
    coef = wt * scale * (torch.where(clip, zero, -A * r) + kl * (1 - e))
    return x, lse, used, tol, sums, sums_tol, coef, wt * abs(scale) * (e_r + kl * e_e)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_no_advantage_at_a_ratio_beyond_f32(env, shape, dtype):
    """A group whose rewards are all equal has advantages of exactly 0: no surrogate and no gradient, whatever the ratio."""
    ops, torch = env
    M, C, ldl = shape
    _say("no advantage", shape, dtype)
    z = _logits(torch, M, ldl, dtype, 21)
    lab = _labels(torch, M, C, 21, outside=False)
    logp = ops.label_logp(z, lab, C)[0]
    adv = torch.zeros(M, device="cuda")
    adv[1::3] = -0.5
    old = logp.clone()
    old[0::3], old[2::3] = logp[0::3] - 100.0, torch.finfo(torch.float32).min
    for want_grad in (True, False):
        sums0, lp0, _ = ops.policy_loss(z, lab, torch.where(adv == 0, logp, old), adv, C, grad_scale=1.0, want_grad=want_grad)
        sums, lp, d = ops.policy_loss(z, lab, old, adv, C, grad_scale=1.0, want_grad=want_grad)
        assert torch.equal(sums, sums0) and torch.equal(lp, lp0) and bool(torch.isfinite(sums).all())
        if want_grad:
            assert not bool(d[0::3].any()) and not bool(d[2::3].any()) and bool(torch.isfinite(d).all()) and bool((d[1::3] != 0).any())
    _, _, d = ops.policy_loss(z, lab, old, torch.full_like(adv, -1.0), C, grad_scale=0.0)
    assert not bool(d.any())      # a scale of 0 takes any gradient out


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_factors_bring_the_exponentials_back(env, shape, dtype):
    """Ratios of exp(100) on advantages, and KL factors of exp(95) on coefficients, whose products f32 holds: rows of each, of both and of neither."""
    ops, torch = env
    M, C, ldl = shape
    _say("factors", shape, dtype)
    z = _logits(torch, M, ldl, dtype, 22)
    lab = _labels(torch, M, C, 22, outside=M > 100)
    logp = _reference(torch, z, lab, C)[2].float()
    gen = torch.Generator(device="cuda").manual_seed(1)
    adv = torch.randn(M, generator=gen, device="cuda") * 1e-30
    w = torch.rand(M, generator=gen, device="cuda")
    rows = torch.arange(M, device="cuda")
    old = torch.where(rows % 2 == 0, logp - 100.0, logp - 0.05)
    ref = torch.where(rows % 4 < 2, logp + 95.0, logp + 0.3)
    kl, scale = 1e-25, 1.0 / M
    want_x = _want(torch, z, lab, old, adv, C, ref, w, 0.2, 0.28, float(torch.tensor(kl, dtype=torch.float32)), float(torch.tensor(scale, dtype=torch.float32)))
    x, lse, used, tol, want, want_tol, coef, coef_tol = want_x
    for ddt in (torch.float32, torch.bfloat16):
        sums, _, d = ops.policy_loss(z, lab, old, adv, C, ref_logp=ref, weights=w, clip_low=0.2, clip_high=0.28, kl_coef=kl, grad_scale=scale,
                                     dlogits=torch.full_like(z, 3.0, dtype=ddt))
        assert bool(((sums.double() - want).abs() <= want_tol)[[0, 1, 3]].all()), (sums, want, want_tol)
        assert float(sums[2]) == float(want[2].float())      # (its own sum is beyond f32)
        _check_grad(torch, d, x, lse, used, lab, coef, coef_tol, tol, C)
    sums, _, _ = ops.policy_loss(z, lab, old, adv, C, ref_logp=ref, weights=w, clip_low=0.2, clip_high=0.28, kl_coef=kl, want_grad=False)
    assert bool(((sums.double() - want).abs() <= want_tol)[[0, 1, 3]].all()), (sums, want, want_tol)


@pytest.mark.parametrize("shape", SHAPES)
def test_a_small_weight_on_a_large_kl(env, shape):
    """The KL part's own sum, without a KL coefficient: weights of 1e-30 on exp(95)."""
    ops, torch = env
    M, C, ldl = shape
    z = _logits(torch, M, ldl, "float32", 23)
    lab = _labels(torch, M, C, 23, outside=False)
    logp = _reference(torch, z, lab, C)[2].float()
    w, adv = torch.full((M,), 1e-30, device="cuda"), torch.ones(M, device="cuda")
    _, _, _, _, want, want_tol, _, _ = _want(torch, z, lab, logp - 0.05, adv, C, logp + 95.0, w, 0.2, 0.28, 0.0, 1.0)
    for want_grad in (True, False):
        sums, _, _ = ops.policy_loss(z, lab, logp - 0.05, adv, C, ref_logp=logp + 95.0, weights=w, clip_high=0.28, want_grad=want_grad)
        assert bool(((sums.double() - want).abs() <= want_tol).all()), (sums, want, want_tol)


@pytest.mark.parametrize("shape", SHAPES)
def test_a_coefficient_beyond_f32_is_held(env, shape):
    """Neither NaN nor infinite where the probability underflows: the row's coefficient is held to the largest finite value."""
    ops, torch = env
    M, C, ldl = shape
    z = _logits(torch, M, ldl, "float32", 24)
    lab = _labels(torch, M, C, 24, outside=False)
    z[:, 0] = -1000.0
    lab[:] = lab.clamp(min=1)
    big = torch.finfo(torch.float32).max
    x, lse, logp, used, tol = _reference(torch, z, lab, C)
    logp = logp.float()
    adv = torch.full((M,), -1.0, device="cuda")
    for old, ref, kl, sign in ((logp - 100.0, None, 0.0, 1.0), (torch.full_like(logp, torch.finfo(torch.float32).min), None, 0.0, 1.0),
                               (logp, logp + 300.0, 0.1, -1.0), (logp, torch.full_like(logp, big), 0.1, -1.0)):
        sums, _, d = ops.policy_loss(z, lab, old, adv, C, ref_logp=ref, kl_coef=kl, grad_scale=1.0)
        assert float(sums[0]) == float("inf") and not bool(torch.isnan(sums).any())
        _check_grad(torch, d, x, lse, used, lab, torch.full_like(lse, sign * big), torch.zeros_like(lse), tol, C)
    z[:, 1], lab[:] = float("-inf"), 1     # an action of probability 0 under the network, not under the reference
    sums, lp, d = ops.policy_loss(z, lab, torch.zeros_like(logp), adv, C, ref_logp=torch.full_like(logp, -1.0), kl_coef=0.1, grad_scale=1.0)
    assert bool((lp == float("-inf")).all()) and float(sums[0]) == float("inf") and not bool(torch.isnan(sums).any())
    assert bool(torch.isfinite(d).all()) and bool((d[:, 1] == -big).all())


@pytest.mark.parametrize("shape", SHAPES)
def test_nan_is_not_taken_for_an_overflow(env, shape):
    """A row of NaN logits that counts stays NaN, without an advantage too; the rows beside it do not see it."""
    ops, torch = env
    M, C, ldl = shape
    z = _logits(torch, M, ldl, "float32", 25)
    lab = _labels(torch, M, C, 25, outside=False)
    logp = ops.label_logp(z, lab, C)[0]
    z[1, C // 2] = float("nan")
    adv = torch.zeros(M, device="cuda")
    for value in (0.0, -1.0):
        adv[1] = value
        for ref in (None, logp):
            sums, lp, d = ops.policy_loss(z, lab, logp, adv, C, ref_logp=ref, kl_coef=0.0 if ref is None else 0.1, grad_scale=1.0)
            assert bool(torch.isnan(lp[1])) and bool(torch.isnan(sums[:2]).all()) and bool(torch.isnan(d[1, :C]).all())
            rest = torch.arange(M, device="cuda") != 1
            assert bool(torch.isfinite(lp[rest]).all()) and bool(torch.isfinite(d[rest]).all())
