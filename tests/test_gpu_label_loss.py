"""label_logp, policy_loss and preference_loss against the formulas in 64 bits.

Tolerances, with h = 2^-24 (half a step of f32) and n = the terms that one thread may add up one after the other (rows are spread over at least 4 lanes,
and at least over 64 where they are longer than 512):
  lse      a sum of n + 16 rounded adds, exponents off by the rounding of z - max and of its product with log2 e, exp itself 2 h:
           e_lse = h (n + 32 + 3 range(row) + 2 |lse| + |max|)
  logp     e_lse + h (|z| + |logp|)
  dlogits  ([c = label] - p) f: p off by e_lse + h (3 |z - lse| + 4) of itself, f by its own error, and the type's half step of the result"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
H = 2.0 ** -24


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    import em_adapt_tensorflow_amd.ops as ops
    return ops, torch


def _say(*a):
    print(*a, flush=True)


def _logits(torch, M, ldl, dtype, seed, scale=2.5, offset=0):
    """[M, ldl] logits whose first element lies `offset` elements into its buffer (any alignment the type allows)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    buf = torch.randn(M * ldl + offset, generator=gen, device="cuda").mul_(scale).to(getattr(torch, dtype))
    return buf[offset:].view(M, ldl)


def _reference(torch, z, labels, C, used=None):
    """(z f64 [M, C], lse, logp, used, tolerance of lse) in 64 bits."""
    x = z[:, :C].double()
    lse = torch.logsumexp(x, 1)
    ok = (labels >= 0) & (labels < C)
    used = ok if used is None else ok & used
    at = x.gather(1, torch.where(ok, labels, 0)[:, None])[:, 0]
    logp = torch.where(used, at - lse, torch.zeros_like(lse))
    fin = torch.where(x.abs() > 1e30, torch.zeros_like(x), x)   # (masked places weigh nothing)
    n = C / (64 if C > 512 else 4) + 1
    tol = H * (n + 32 + 3 * (fin.amax(1) - fin.amin(1)) + 2 * lse.abs() + x.amax(1).abs())
    return x, lse, logp, used, tol


def _half_step(torch, dtype):
    return torch.finfo(dtype).eps / 2


def _check_grad(torch, d, x, lse, used, labels, coef, coef_tol, tol, C):
    """d [M, ldl] against ([c = label] - p) coef."""
    p = torch.exp(x - lse[:, None])
    hot = torch.zeros_like(p)
    hot.scatter_(1, torch.where(used, labels, 0)[:, None], 1.0)
    f = torch.where(used, coef, torch.zeros_like(coef))
    want = torch.where(used[:, None], (hot - p) * f[:, None], torch.zeros_like(p))
    off = p * (tol[:, None] + H * (3 * torch.where(torch.isinf(x), torch.zeros_like(x), x - lse[:, None]).abs() + 4)) * f.abs()[:, None]
    off += (hot - p).abs() * torch.where(used, coef_tol, torch.zeros_like(coef))[:, None] + want.abs() * (_half_step(torch, d.dtype) + 3 * H) + 1e-38
    off = torch.where(used[:, None], off, torch.zeros_like(off))
    got = d[:, :C].double()
    bad = (got - want).abs() > off
    assert not bool(bad.any()), "gradient off at %s: %s, wanted %s +- %s" % (bad.nonzero()[0].tolist(), got[bad][0].item(), want[bad][0].item(), off[bad][0].item())
    assert not bool((d[:, C:] != 0).any()), "padding columns"


SHAPES = [   # rows, classes, ldl, offset of the buffer in elements
    (1, 1, 1, 0), (1, 2, 2, 1), (3, 21, 24, 0), (1000, 21, 24, 0), (257, 21, 21, 3), (70, 41, 48, 0), (5, 7, 64, 1), (130, 64, 64, 0), (33, 65, 65, 1),
    (64, 255, 256, 0), (9, 500, 513, 0), (17, 513, 513, 5), (6, 1000, 1000, 0), (5, 2047, 2050, 0), (300, 4096, 4096, 0), (4, 4099, 4099, 1),
    (3, 16383, 16384, 0), (2, 32769, 32769, 7), (1, 65537, 65537, 0), (2, 128001, 128001, 1), (1, 200003, 200008, 0), (600, 8191, 8192, 0),
]


def _labels(torch, M, C, seed, outside=True):
    gen = torch.Generator(device="cuda").manual_seed(seed + 1)
    lab = torch.randint(0, C, (M,), generator=gen, device="cuda")
    if outside and M > 4:
        lab[1], lab[2], lab[M - 1] = -1, C, 2 ** 40 + 3
    return lab


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_label_logp_and_gradient(env, shape, dtype):
    ops, torch = env
    M, C, ldl, offset = shape
    _say("label_logp", shape, dtype)
    z = _logits(torch, M, ldl, dtype, sum(shape), offset=offset)
    if ldl > C:
        z[:, C:] = float("nan")   # what lies in the padding does not count
    lab = _labels(torch, M, C, sum(shape))
    logp, lse = ops.label_logp(z, lab, C)
    x, want_lse, want, used, tol = _reference(torch, z, lab, C)
    assert bool(((lse.double() - want_lse).abs() <= tol).all())
    at = x.gather(1, torch.where(used, lab, 0)[:, None])[:, 0].abs()
    assert bool(((logp.double() - want).abs() <= torch.where(used, tol + H * (at + want.abs()), torch.zeros_like(tol))).all())
    gen = torch.Generator(device="cuda").manual_seed(5)
    coef = torch.randn(M, generator=gen, device="cuda")
    for ddt in (torch.float32, torch.bfloat16):
        d = ops.label_logp_bwd(z, lab, lse, coef, C, dlogits=torch.full_like(z, 7.0, dtype=ddt))
        _check_grad(torch, d, x, want_lse, used, lab, coef.double(), torch.zeros_like(tol), tol, C)
    again = ops.label_logp(z, lab, C)
    assert torch.equal(again[0], logp) and torch.equal(again[1], lse)


def test_rows_that_take_no_part_may_hold_anything(env):
    ops, torch = env
    for M, C, ldl in ((300, 21, 24), (40, 5000, 5000), (6, 130000, 130000)):
        _say("masked rows", M, C)
        z = _logits(torch, M, ldl, "float32", 3)
        lab = _labels(torch, M, C, 3, outside=False)
        z[0], z[1], z[2] = float("nan"), float("inf"), float("-inf")
        z[3, : C // 2] = torch.finfo(torch.float32).min
        z[4, C // 2] = float("-inf")
        lab[4] = 0
        lab[0], lab[1], lab[2] = -1, C, 255 if C == 21 else -100
        logp, lse = ops.label_logp(z, lab, C)
        assert bool((logp[:3] == 0).all()) and bool(torch.isfinite(logp[3:]).all() | (lab[3] < C // 2))
        coef = torch.ones(M, device="cuda")
        d = ops.label_logp_bwd(z, lab, lse, coef, C)
        assert bool((d[:3] == 0).all()) and bool(torch.isfinite(d[4:]).all()) and float(d[4, C // 2]) == 0.0
        w = torch.ones(M, device="cuda")
        lab2 = lab.clone()
        lab2[0], lab2[1], lab2[2] = 0, 1, 2
        w[:4] = 0
        nan = torch.full((M,), float("nan"), device="cuda")
        old, adv, ref = logp.clone(), torch.randn(M, device="cuda"), logp.clone()
        old[:4], adv[:4], ref[:4] = nan[:4], nan[:4], nan[:4]
        sums, lp, d = ops.policy_loss(z, lab2, old, adv, C, ref_logp=ref, weights=w, kl_coef=0.1)
        assert bool(torch.isfinite(sums).all()) and bool((d[:4] == 0).all()) and bool((lp[:4] == 0).all()) and bool(torch.isfinite(d).all())
        # the same with the sequence form: rows without a label add nothing to their sequence
        at = torch.tensor([0, M // 2, M], device="cuda")
        lab3 = lab.clone()
        lab3[3] = -1
        loss, seq, d = ops.preference_loss(z, lab3, at, torch.zeros(2, device="cuda"), C)
        assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(seq).all()) and bool((d[:4] == 0).all()) and bool(torch.isfinite(d).all())


@pytest.mark.parametrize("C", [21, 900, 5000, 130000, 300000])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_rows_at_the_types_lowest_and_largest_values(env, C, dtype):
    """A mask of the type's lowest value over a part of a row, over all of it (then every class is as likely), and logits near the largest."""
    ops, torch = env
    z = _logits(torch, 5, C, dtype, 14)
    lo, big = torch.finfo(z.dtype).min, torch.finfo(z.dtype).max
    z[0] = lo
    z[1, 1:] = lo
    z[2, 0] = big
    z[3, C // 2] = lo
    z[4] = big
    lab = torch.zeros(5, dtype=torch.int64, device="cuda")
    logp, lse = ops.label_logp(z, lab, C)
    sums, lp, d = ops.policy_loss(z, lab, logp - 0.1, torch.ones(5, device="cuda"), C, clip_high=10.0, grad_scale=1.0)
    assert bool(torch.isfinite(logp).all()) and bool(torch.isfinite(d).all()) and torch.equal(lp, logp)
    at = torch.tensor([0, 3, 5], device="cuda")
    loss, seq, d2 = ops.preference_loss(z, lab, at, torch.zeros(2, device="cuda"), C)
    assert bool(torch.isfinite(loss).all()) and bool(torch.isfinite(d2).all()) and bool(torch.isfinite(ops.label_logp_bwd(z, lab, lse, torch.ones(5, device="cuda"), C)).all())
    for r in (0, 4):   # every class is as likely
        assert abs(float(logp[r]) + np.log(C)) < 1e-5
        ratio = -float(d[r, 0])
        assert abs(float(d[r, 1]) * (C - 1) + float(d[r, 0])) < 0.02 * abs(ratio)
    assert abs(float(logp[1])) < 1e-6 and abs(float(logp[2])) < 1e-6
    x, want_lse, want, used, tol = _reference(torch, z[3:4], lab[3:4], C)
    assert abs(float(logp[3]) - float(want[0])) < float(tol[0]) * 2


def test_rows_that_count_keep_their_nan(env):
    ops, torch = env
    for C in (21, 3000, 130001):
        z = _logits(torch, 8, C, "bfloat16", 2)
        z[3, C // 2] = float("nan")
        lab = _labels(torch, 8, C, 2, outside=False)
        logp, lse = ops.label_logp(z, lab, C)
        assert bool(torch.isnan(logp[3])) and int(torch.isnan(logp).sum()) == 1
        d = ops.label_logp_bwd(z, lab, lse, torch.ones(8, device="cuda"), C)
        assert bool(torch.isnan(d[3]).all()) and int(torch.isnan(d).any(1).sum()) == 1


def _policy_reference(torch, z, lab, old, adv, C, ref, w, lo, hi, kl, scale):
    used = None if w is None else w != 0
    x, lse, logp, used, tol = _reference(torch, z, lab, C, used)
    zero = torch.zeros_like(lse)
    at = x.gather(1, torch.where(used, lab, 0)[:, None])[:, 0].abs()
    wt = torch.ones_like(lse) if w is None else w.double()
    A, o = adv.double(), old.double()
    ratio = torch.exp(torch.where(used, logp - o, zero))
    free, held = -A * ratio, -A * ratio.clamp(1 - lo, 1 + hi)
    clip = held > free
    q = torch.where(used, ref.double() - logp, zero) if ref is not None else zero
    k = torch.expm1(q) - q
    part = torch.where(clip, held, free)
    e = torch.where(used, tol + H * (2 * at + 2 * logp.abs() + 2 * o.abs() + (ref.double().abs() if ref is not None else 0)), zero)   # of logp - old, ref - logp
    wt = torch.where(used, wt, zero)
    sums = torch.stack([(wt * (part + kl * k)).sum(), (wt * part).sum(), (wt * k).sum(), (wt * clip).sum()])
    e_part = (free.abs() * (e + 8 * H) + part.abs() * 4 * H)
    e_k = (torch.exp(q) + 1) * (e + 8 * H) + 4 * H * (q.abs() + torch.exp(q))
    tot = wt.abs()
    sums_tol = torch.stack([(tot * (e_part + abs(kl) * e_k)).sum(), (tot * e_part).sum(), (tot * e_k).sum(), zero.sum()])
    sums_tol = sums_tol + sums.abs() * 2 * H + 1e-30
    coef = wt * scale * (torch.where(clip, zero, free) + kl * (1 - torch.exp(q)))
    coef_tol = tot * abs(scale) * (torch.where(clip, zero, free.abs()) * (e + 10 * H) + abs(kl) * ((torch.exp(q)) * (e + 10 * H) + 4 * H))
    return x, lse, logp, used, tol + H * (at + logp.abs()), tol, sums, sums_tol, coef, coef_tol


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("shape", SHAPES)
def test_policy_loss(env, shape, dtype):
    ops, torch = env
    M, C, ldl, offset = shape
    _say("policy_loss", shape, dtype)
    z = _logits(torch, M, ldl, dtype, sum(shape) + 1, offset=offset)
    if ldl > C:
        z[:, C:] = float("inf")
    lab = _labels(torch, M, C, sum(shape) + 1)
    gen = torch.Generator(device="cuda").manual_seed(11)
    true = _reference(torch, z, lab, C)[2]
    old = (true + torch.randn(M, generator=gen, device="cuda").double() * 0.2).float()
    ref = (true + torch.randn(M, generator=gen, device="cuda").double() * 0.3).float()
    adv = torch.randn(M, generator=gen, device="cuda")
    if M > 8:
        adv[5] = 0.0
    w = torch.rand(M, generator=gen, device="cuda") * (torch.rand(M, generator=gen, device="cuda") > 0.2)
    for use_ref, use_w, lo, hi, kl, ddt in ((True, True, 0.2, 0.28, 0.05, z.dtype), (False, False, 0.1, 0.0, 0.0, torch.float32), (True, False, 1.0, 0.2, 0.3, torch.bfloat16)):
        scale = 1.0 / M
        sums, logp, d = ops.policy_loss(z, lab, old, adv, C, ref_logp=ref if use_ref else None, weights=w if use_w else None, clip_low=lo, clip_high=hi, kl_coef=kl,
                                        grad_scale=scale, dlogits=torch.full_like(z, 3.0, dtype=ddt))
        x, lse, want_lp, used, lp_tol, tol, want, want_tol, coef, coef_tol = _policy_reference(torch, z, lab, old, adv, C, ref if use_ref else None,
                                                                                             w if use_w else None, lo, hi, kl, scale)
        assert bool(((logp.double() - want_lp).abs() <= torch.where(used, lp_tol, torch.zeros_like(lp_tol))).all())
        assert bool(((sums.double() - want).abs() <= want_tol).all()), (sums, want, want_tol)
        _check_grad(torch, d, x, lse, used, lab, coef, coef_tol, tol, C)
        again = ops.policy_loss(z, lab, old, adv, C, ref_logp=ref if use_ref else None, weights=w if use_w else None, clip_low=lo, clip_high=hi, kl_coef=kl,
                                grad_scale=scale, dlogits=torch.empty_like(d))
        assert torch.equal(again[0], sums) and torch.equal(again[1], logp) and torch.equal(again[2], d)
        sums2, logp2, none = ops.policy_loss(z, lab, old, adv, C, ref_logp=ref if use_ref else None, weights=w if use_w else None, clip_low=lo, clip_high=hi,
                                             kl_coef=kl, want_grad=False)
        assert none is None and bool(((sums2.double() - want).abs() <= want_tol).all())
        assert bool(((logp2.double() - want_lp).abs() <= torch.where(used, lp_tol, torch.zeros_like(lp_tol))).all())


@pytest.mark.parametrize("shape", [(4000, 21, 24), (300, 700, 700), (64, 40000, 40000), (5, 150001, 150001), (70001, 5, 5), (40000, 130, 130), (600, 5000, 5000)])
def test_policy_clip_is_decided_as_in_64_bits(env, shape):
    """old_logp such that the ratio lies a few f32 roundings to either side of a border, nearer than f32 can tell."""
    ops, torch = env
    M, C, ldl = shape
    _say("border", shape)
    z = _logits(torch, M, ldl, "float32", 8)
    lab = _labels(torch, M, C, 8, outside=False)
    true = _reference(torch, z, lab, C)[2]
    gen = torch.Generator(device="cuda").manual_seed(4)
    adv = torch.randn(M, generator=gen, device="cuda")
    lo, hi = 0.2, 0.28
    border = torch.where(adv > 0, np.log1p(hi), np.log1p(-lo)).double()
    old = (true - border).float()
    steps = torch.randint(-2, 3, (M,), generator=gen, device="cuda")
    for _ in range(2):
        old = torch.where(steps > 0, torch.nextafter(old, torch.full_like(old, 100.0)), torch.where(steps < 0, torch.nextafter(old, torch.full_like(old, -100.0)), old))
        steps -= steps.sign()
    sums, logp, d = ops.policy_loss(z, lab, old, adv, C, clip_low=lo, clip_high=hi, grad_scale=1.0)
    x, lse, want_lp, used, lp_tol, tol, want, want_tol, coef, coef_tol = _policy_reference(torch, z, lab, old, adv, C, None, None, lo, hi, 0.0, 1.0)
    assert float(sums[3]) == float(want[3]) and 0.2 * M < float(want[3]) < 0.8 * M + 2
    _check_grad(torch, d, x, lse, used, lab, coef, coef_tol, tol, C)


def _preference_reference(torch, z, lab, at, ref, C, beta, smooth, scale):
    x, lse, logp, used, tol = _reference(torch, z, lab, C)
    zero = torch.zeros_like(lse)
    atz = x.gather(1, torch.where(used, lab, 0)[:, None])[:, 0].abs()
    e = torch.where(used, tol + H * (2 * atz + logp.abs()), zero)
    bounds = at.tolist()
    seq = torch.stack([logp[bounds[i]:bounds[i + 1]].sum() for i in range(len(bounds) - 1)])
    seq_e = torch.stack([e[bounds[i]:bounds[i + 1]].sum() for i in range(len(bounds) - 1)])
    r = (seq - ref.double()).view(-1, 2)
    h = beta * (r[:, 0] - r[:, 1])
    h_e = abs(beta) * seq_e.view(-1, 2).sum(1) + 2 * H * h.abs()
    sp = torch.nn.functional.softplus
    loss = (1 - smooth) * sp(-h) + smooth * sp(h)
    slope = beta * (smooth - torch.sigmoid(-h)) * scale
    slope_tol = abs(beta * scale) * (0.25 * h_e + 4 * H)
    coef, coef_tol = zero.clone(), zero.clone()
    for j in range(len(h)):
        for q in (0, 1):
            i = slice(bounds[2 * j + q], bounds[2 * j + q + 1])
            coef[i] = -slope[j] if q else slope[j]
            coef_tol[i] = slope_tol[j]
    return x, lse, used, tol, seq, seq_e + 2 * H * seq.abs(), loss, h_e + 4 * H * loss + 1e-30, coef, coef_tol


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("C,ldl,lens,tail", [(21, 24, [5, 7], 0), (21, 24, [0, 3, 1, 1, 0, 0], 4), (21, 21, [1681, 900], 3), (600, 600, [33, 1, 2, 64], 0),
                                             (5001, 5001, [3, 9], 2), (40000, 40000, [20, 11, 5, 0], 1), (130001, 130001, [1, 2], 0), (8192, 8192, [300, 280], 0)])
def test_preference_loss(env, C, ldl, lens, tail, dtype):
    ops, torch = env
    _say("preference_loss", C, lens, dtype)
    M = sum(lens) + tail
    z = _logits(torch, M, ldl, dtype, C + M)
    if ldl > C:
        z[:, C:] = float("nan")
    lab = _labels(torch, M, C, 9, outside=sum(lens) > 6)
    at = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(6)
    true = _preference_reference(torch, z, lab, at, torch.zeros(len(lens), device="cuda"), C, 0.1, 0.0, 1.0)[4]
    ref = (true + torch.randn(len(lens), generator=gen, device="cuda").double() * 5).float()
    for beta, smooth, scale, ddt in ((0.1, 0.0, None, z.dtype), (0.5, 0.1, 2.0, torch.float32)):
        loss, seq, d = ops.preference_loss(z, lab, at, ref, C, beta=beta, label_smoothing=smooth, grad_scale=scale, dlogits=torch.full_like(z, 3.0, dtype=ddt))
        x, lse, used, tol, wseq, seq_tol, wloss, loss_tol, coef, coef_tol = _preference_reference(torch, z, lab, at, ref, C, beta, smooth,
                                                                                                 2.0 / len(lens) if scale is None else scale)
        assert bool(((seq.double() - wseq).abs() <= seq_tol).all()) and bool(((loss.double() - wloss).abs() <= loss_tol).all())
        _check_grad(torch, d, x, lse, used, lab, coef, coef_tol, tol, C)
        assert tail == 0 or bool((d[M - tail:] == 0).all())
        again = ops.preference_loss(z, lab, at, ref, C, beta=beta, label_smoothing=smooth, want_grad=False)
        assert again[2] is None and torch.equal(again[1], seq)


def test_preference_starts_out_of_range_touch_nothing_else(env):
    ops, torch = env
    z = _logits(torch, 10, 24, "float32", 1)
    lab = _labels(torch, 10, 21, 1, outside=False)
    room = torch.full((30, 24), 5.0, device="cuda")
    for starts in ([0, 4, 2 ** 40], [-7, 3, 8], [8, 4, 2], [20, 30, 40]):
        _say("starts", starts)
        d = room[10:20]
        ops.preference_loss(z, lab, torch.tensor(starts, device="cuda"), torch.zeros(2, device="cuda"), 21, dlogits=d)
        torch.cuda.synchronize()
        assert bool((room[:10] == 5).all()) and bool((room[20:] == 5).all()) and bool(torch.isfinite(d).all())


def test_gradients_against_differences(env):
    """Central differences of the losses themselves, over logits perturbed one at a time: h = 2^-6 leaves h^2 / 6 of a third derivative (at most 8
    here) and the rounding of the sums over 2 h."""
    ops, torch = env
    M, C = 6, 9
    z = _logits(torch, M, C, "float32", 21)
    lab = _labels(torch, M, C, 21, outside=False)
    gen = torch.Generator(device="cuda").manual_seed(3)
    logp = ops.label_logp(z, lab, C)[0]
    old = logp + 0.5 * (torch.rand(M, generator=gen, device="cuda") - 0.5).sign() + 0.02      # away from the borders
    ref, adv = logp + 0.2, torch.randn(M, generator=gen, device="cuda")
    at, sref = torch.tensor([0, 2, 6], device="cuda"), torch.tensor([-3.0, -8.0], device="cuda")
    up = torch.randn(M, generator=gen, device="cuda")
    losses = {
        "policy": (lambda x: ops.policy_loss(x, lab, old, adv, C, ref_logp=ref, kl_coef=0.3, want_grad=False)[0][0].double(),
                   ops.policy_loss(z, lab, old, adv, C, ref_logp=ref, kl_coef=0.3, grad_scale=1.0)[2]),
        "preference": (lambda x: ops.preference_loss(x, lab, at, sref, C, beta=0.4, label_smoothing=0.1, want_grad=False)[0].double().sum(),
                       ops.preference_loss(z, lab, at, sref, C, beta=0.4, label_smoothing=0.1, grad_scale=1.0)[2]),
        "logp": (lambda x: (ops.label_logp(x, lab, C)[0].double() * up.double()).sum(), ops.label_logp_bwd(z, lab, ops.label_logp(z, lab, C)[1], up, C)),
    }
    h = 2.0 ** -6
    for name, (f, d) in losses.items():
        base = abs(float(f(z))) + 20.0
        tol = h * h / 6 * 8 + base * 64 * H / h
        for r in range(M):
            for c in range(C):
                zp, zm = z.clone(), z.clone()
                zp[r, c] += h
                zm[r, c] -= h
                step = float(zp[r, c].double() - zm[r, c].double())
                assert abs(float(f(zp) - f(zm)) / step - float(d[r, c])) < tol, (name, r, c)


def test_empty_and_refused(env):
    ops, torch = env
    z, lab = torch.zeros(0, 24, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    f = torch.zeros(0, device="cuda")
    logp, lse = ops.label_logp(z, lab, 21)
    assert logp.numel() == 0 and lse.numel() == 0 and ops.label_logp_bwd(z, lab, lse, f, 21).numel() == 0
    sums, _, d = ops.policy_loss(z, lab, f, f, 21)
    assert sums.tolist() == [0.0] * 4 and d.numel() == 0
    one = torch.zeros(1, dtype=torch.int64, device="cuda")
    loss, seq, _ = ops.preference_loss(z, lab, one, f, 21)
    assert loss.numel() == 0 and seq.numel() == 0
    loss, seq, d = ops.preference_loss(z, lab, torch.zeros(3, dtype=torch.int64, device="cuda"), torch.tensor([1.0, 0.0], device="cuda"), 21, beta=1.0)
    assert abs(float(loss) - np.log1p(np.exp(1.0))) < 1e-6 and seq.tolist() == [0.0, 0.0]
    z, lab, f = torch.zeros(4, 24, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.zeros(4, device="cuda")
    at, ref = torch.tensor([0, 2, 4], device="cuda"), torch.zeros(2, device="cuda")
    for call in (lambda: ops.label_logp(z.half(), lab, 21), lambda: ops.label_logp(z, lab.int(), 21), lambda: ops.label_logp(z, f, 21)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ops.label_logp(z, lab, 25), lambda: ops.label_logp(z, lab, 0), lambda: ops.label_logp(z[:, :21], lab, 21), lambda: ops.label_logp(z, lab[:3], 21),
                 lambda: ops.label_logp(z.cpu(), lab.cpu(), 21), lambda: ops.label_logp_bwd(z, lab, f[:3], f, 21), lambda: ops.policy_loss(z, lab, f, f[:2], 21),
                 lambda: ops.policy_loss(z, lab, f, f, 21, clip_low=1.2), lambda: ops.policy_loss(z, lab, f, f, 21, kl_coef=0.1),
                 lambda: ops.policy_loss(z, lab, f, f, 21, clip_high=float("nan")), lambda: ops.policy_loss(z, lab, None, f, 21),
                 lambda: ops.policy_loss(z, lab, f, f, 21, dlogits=torch.zeros(4, 21, device="cuda")), lambda: ops.preference_loss(z, lab, at[:2], ref, 21),
                 lambda: ops.preference_loss(z, lab, at, ref[:1], 21), lambda: ops.preference_loss(z, lab, at, ref, 21, label_smoothing=2.0)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ops._lib.EmadaptError):   # in place
        ops.policy_loss(z, lab, f, f, 21, dlogits=z)


def test_on_another_stream_and_in_a_replayed_graph(env):
    """Eager calls on a side stream, two captured graphs, replays with new inputs between eager work: each equals the eager result."""
    ops, torch = env
    cases = []
    for k, (M, C) in enumerate(((700, 21), (40, 9000), (3, 140000))):
        z = _logits(torch, M, C, "bfloat16", 30 + k)
        lab = _labels(torch, M, C, 30 + k)
        f = [torch.randn(M, device="cuda") for _ in range(3)]
        at = torch.tensor([0, M // 3, M], device="cuda")

        def call(z=z, lab=lab, f=f, at=at, C=C):
            logp, lse = ops.label_logp(z, lab, C)
            a = ops.policy_loss(z, lab, logp + 0.1 * f[0], f[1], C, ref_logp=logp + f[2], kl_coef=0.1)
            b = ops.preference_loss(z, lab, at, f[0][:2].contiguous(), C)
            return [logp, lse, *a, *b]
        cases.append((z, call))
    want = [call() for _, call in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [call() for _, call in cases]
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, g))
    graphs = []
    for _, call in cases:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for turn in range(3):
        for z, _ in cases:
            z.mul_(0.9)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, call), (_, out) in zip(cases, graphs):
            assert all(torch.equal(x, y) for x, y in zip(call(), out)), turn


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,C,ldl", [(5, 3, 600), (9, 1, 5000), (40, 7, 300), (2, 5, 140001), (300, 8, 1001)])
def test_few_classes_in_long_rows(env, M, C, ldl, dtype):
    """Fewer classes than one 16-byte load holds, in rows far longer: no load may start in front of the row or behind it."""
    ops, torch = env
    _say("few classes", M, C, ldl, dtype)
    z = _logits(torch, M, ldl, dtype, M + ldl, offset=1)
    z[:, C:] = float("nan")
    lab = _labels(torch, M, C, M, outside=False)
    logp, lse = ops.label_logp(z, lab, C)
    x, want_lse, want, used, tol = _reference(torch, z, lab, C)
    at = x.gather(1, lab[:, None])[:, 0].abs()
    assert bool(((logp.double() - want).abs() <= tol + H * (at + want.abs())).all())
    gen = torch.Generator(device="cuda").manual_seed(2)
    adv = torch.randn(M, generator=gen, device="cuda")
    old = (want + 0.1).float()
    sums, lp, d = ops.policy_loss(z, lab, old, adv, C, grad_scale=1.0)
    x, _, want_lp, used, lp_tol, tol, wsums, wsums_tol, coef, coef_tol = _policy_reference(torch, z, lab, old, adv, C, None, None, 0.2, 0.2, 0.0, 1.0)
    assert bool(((sums.double() - wsums).abs() <= wsums_tol).all())
    _check_grad(torch, d, x, want_lse, used, lab, coef, coef_tol, tol, C)
    at, ref = torch.tensor([0, M // 2, M], device="cuda"), torch.zeros(2, device="cuda")
    loss, seq, d = ops.preference_loss(z, lab, at, ref, C, grad_scale=1.0)
    x, _, used, tol, wseq, seq_tol, wloss, loss_tol, coef, coef_tol = _preference_reference(torch, z, lab, at, ref, C, 0.1, 0.0, 1.0)
    assert bool(((loss.double() - wloss).abs() <= loss_tol).all())
    _check_grad(torch, d, x, want_lse, used, lab, coef, coef_tol, tol, C)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,C,ldl", [(300, 21, 24), (6, 700, 700), (3, 5001, 5001), (2, 130001, 130001)])
def test_gradient_far_from_zero(env, M, C, ldl, dtype):
    """Rows whose log-sum-exp in f32 lacks the sum's bits: the gradient is the row's own all the same.  Maximum and sum are then taken in the gradient's
    launch (differences to the maximum rounded once), so |lse| and |max| leave the tolerance."""
    ops, torch = env
    _say("far", M, C, dtype)
    z = _logits(torch, M, ldl, dtype, C)
    lo = torch.finfo(z.dtype).min
    for r in range(M):
        z[r] = (z[r].float() + (5000.0, -5000.0, 1e6)[r % 3]).to(z.dtype) if r % 4 else lo
    lab = _labels(torch, M, C, C, outside=False)
    _, lse = ops.label_logp(z, lab, C)
    x = z[:, :C].double()
    x = x - x.amax(1, keepdim=True)
    gen = torch.Generator(device="cuda").manual_seed(2)
    coef = torch.randn(M, generator=gen, device="cuda")
    d = ops.label_logp_bwd(z, lab, lse, coef, C)
    n = C / (64 if C > 512 else 4) + 1
    tol = H * (n + 32 + 3 * (x.amax(1) - x.amin(1)))
    _check_grad(torch, d, x, torch.logsumexp(x, 1), torch.ones_like(lab, dtype=torch.bool), lab, coef.double(), torch.zeros_like(tol), tol, C)
    # a log-sum-exp that is not the row's own (the classes are a part of all) is taken as it is: off by half a step of itself
    other = lse + 1.0 + lse.abs() * 2.0 ** -20
    d = ops.label_logp_bwd(z, lab, other, coef, C)
    full = z[:, :C].double()
    sane = lse.abs() < 1e30
    _check_grad(torch, d[sane], full[sane], other[sane].double(), sane[sane], lab[sane], coef[sane].double(), torch.zeros_like(tol[sane]), (H * 4 * other.abs().double())[sane], C)


@pytest.mark.parametrize("M,C,ldl", [(300, 21, 24), (20, 700, 700), (200, 5001, 5001), (3, 40000, 40000), (2, 300001, 300001)])
def test_policy_of_an_action_at_the_lowest_value(env, M, C, ldl):
    """clip_low 0 puts the border at ratio 1: all rows with old_logp = logp lie on it, also those whose action is masked with the type's lowest value
    (log-probability -3.4e38, ratio 1 all the same) or far below the others."""
    ops, torch = env
    z = _logits(torch, M, ldl, "float32", 6)
    lab = _labels(torch, M, C, 6, outside=False)
    rows = torch.arange(M, device="cuda")
    z[rows[::2], lab[::2]] = torch.finfo(torch.float32).min
    z[rows[1::2], lab[1::2]] = -1000.0
    logp = _reference(torch, z, lab, C)[2].float()
    adv = -torch.ones(M, device="cuda")
    for want_grad in (False, True):
        sums, lp, d = ops.policy_loss(z, lab, logp, adv, C, clip_low=0.0, grad_scale=1.0, want_grad=want_grad)
        # a ratio is off by exp(half a step of logp near 1000) at most; where f32 logp is above the exact one the ratio is below 1 and held there
        assert abs(float(sums[0]) - M) <= M * 2 * H * 1100
        assert bool(((lp - logp).abs() <= 2 * H * logp.abs()).all())
    x = z[:, :C].double()
    p = torch.softmax(x, 1)
    hot = torch.zeros_like(p)
    hot[rows, lab] = 1.0
    free = d[rows, lab] != 0
    assert bool(free[::2].all())
    assert bool(((d[:, :C].double() - (hot - p) * free[:, None]).abs() <= 1e-3 * (hot - p).abs() + 1e-38).all())


def test_kl_of_weight_zero_does_not_count(env):
    ops, torch = env
    for M, C in ((50, 21), (9, 5000), (2, 200001)):
        z = _logits(torch, M, C, "float32", 1)
        lab = _labels(torch, M, C, 1, outside=False)
        logp = ops.label_logp(z, lab, C)[0]
        adv = torch.ones(M, device="cuda")
        a = ops.policy_loss(z, lab, logp - 0.05, adv, C, kl_coef=0.0)
        b = ops.policy_loss(z, lab, logp - 0.05, adv, C, ref_logp=logp + 120.0, kl_coef=0.0)   # exp(120) is beyond f32
        assert torch.equal(a[0][:2], b[0][:2]) and torch.equal(a[2], b[2]) and bool(torch.isfinite(b[2]).all())


def test_preference_of_long_sequences(env):
    """Pairs long enough to be split over workgroups, of unlike lengths, an empty sequence among them, rows of no sequence in front and behind."""
    ops, torch = env
    C = 5
    lens = [40000, 25001, 0, 70003, 1, 8192]
    M = sum(lens) + 30
    z = _logits(torch, M, C, "float32", 12)
    lab = _labels(torch, M, C, 12)
    at = torch.tensor(10 + np.concatenate([[0], np.cumsum(lens)]), device="cuda")
    true = _preference_reference(torch, z, lab, at, torch.zeros(6, device="cuda"), C, 0.1, 0.0, 1.0)[4]
    ref = (true + torch.tensor([1.0, -1.0, 2.0, 3.0, -4.0, 0.5], device="cuda")).float()
    loss, seq, d = ops.preference_loss(z, lab, at, ref, C, beta=0.2, label_smoothing=0.1, grad_scale=1.0, dlogits=torch.full_like(z, 3.0))
    x, lse, used, tol, wseq, seq_tol, wloss, loss_tol, coef, coef_tol = _preference_reference(torch, z, lab, at, ref, C, 0.2, 0.1, 1.0)
    assert bool(((seq.double() - wseq).abs() <= seq_tol).all()) and bool(((loss.double() - wloss).abs() <= loss_tol).all())
    _check_grad(torch, d, x, lse, used, lab, coef, coef_tol, tol, C)
    assert bool((d[:10] == 0).all()) and bool((d[M - 20:] == 0).all())
    again = ops.preference_loss(z, lab, at, ref, C, beta=0.2, label_smoothing=0.1, grad_scale=1.0)
    assert torch.equal(again[0], loss) and torch.equal(again[2], d)
    # starts out of range and out of order: nothing outside the rows is touched
    room = torch.full((M + 20, C), 5.0, device="cuda")
    for starts in ([0, 2 ** 40, 2 ** 41], [-9, 50000, 20], [M + 5, M + 9, M + 12]):
        ops.preference_loss(z, lab, torch.tensor(starts, device="cuda"), ref[:2].contiguous(), C, dlogits=room[10:M + 10])
        torch.cuda.synchronize()
        assert bool((room[:10] == 5).all()) and bool((room[M + 10:] == 5).all())


@pytest.mark.parametrize("M,C,ldl", [(90_000_000, 21, 24), (33_000, 65_536, 65_600), (16_000, 140_000, 140_000)])
def test_rows_behind_2_31_elements(env, M, C, ldl):
    """Rows are worked on one by one: the last ones of a large call are, bit for bit, what a call on them alone gives."""
    ops, torch = env
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free memory")
    _say("large", M, C)
    assert M * ldl > 2 ** 31
    z = torch.empty(M, ldl, dtype=torch.bfloat16, device="cuda").normal_()
    lab = torch.randint(0, C, (M,), device="cuda")
    n = 300
    tail, tail_lab = z[M - n:].clone(), lab[M - n:].clone()
    logp, lse = ops.label_logp(z, lab, C)
    few, few_lse = ops.label_logp(tail, tail_lab, C)
    assert torch.equal(logp[M - n:], few) and torch.equal(lse[M - n:], few_lse)
    d = torch.empty_like(z)
    up = torch.ones(M, device="cuda")
    ops.label_logp_bwd(z, lab, lse, up, C, dlogits=d)
    assert torch.equal(d[M - n:], ops.label_logp_bwd(tail, tail_lab, few_lse, up[:n].contiguous(), C))
    old = logp - 0.1
    sums, lp, _ = ops.policy_loss(z, lab, old, up, C, grad_scale=1.0, dlogits=d)
    _, few_lp, few_d = ops.policy_loss(tail, tail_lab, old[M - n:].clone(), up[:n].contiguous(), C, grad_scale=1.0)
    assert torch.equal(lp[M - n:], few_lp) and torch.equal(d[M - n:], few_d)
    assert abs(float(sums[0]) / M + np.exp(0.1)) < 1e-5 and float(sums[3]) == 0
    at = torch.tensor([0, M - n, M], device="cuda")
    ref = torch.zeros(2, device="cuda")
    _, seq, _ = ops.preference_loss(z, lab, at, ref, C, beta=1e-9, grad_scale=1e9, dlogits=d)
    assert abs(float(seq[1]) - float(few.double().sum())) < 1e-6 * abs(float(seq[1]))
    x = tail[:, :C].double()
    lse64 = torch.logsumexp(x, 1)
    ok = torch.ones(n, dtype=torch.bool, device="cuda")
    h = 1e-9 * (float(seq[0]) - float(seq[1]))
    coef = torch.full((n,), 1.0 / (1.0 + np.exp(h)), dtype=torch.float64, device="cuda")
    tol = _reference(torch, tail, tail_lab, C)[4]
    _check_grad(torch, d[M - n:], x, lse64, ok, tail_lab, coef, coef.abs() * 1e-6, tol, C)
