"""AdamW over many tensors: moments bit for bit against IEEE arithmetic on the CPU (every product and sum is rounded on its own), the 8-bit codes against an
integer restatement of the formats and of the generator, weights within two roundings.

Weights: w - fade w is the same; the step rate * m / den is off by the rounding of its product, quotient and denominator, at most 4 h of itself
(h = 2^-24), and one rounding of the difference: 4 h |step| + 2 h |w|."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
H = 2.0 ** -24
SIZES = [1, 63, 64, 65, 4096, 4097, 300, 0, 12289, 7, 255, 257]


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    import em_adapt_tensorflow_amd.ops as ops
    assert ops.status_poll(raise_on_error=False) == 0
    return ops, torch


def _tensors(torch, sizes, gdtype, seed, odd=True, scale=1.0):
    """Weights and gradients as views at odd places of their buffers."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    ws, gs = [], []
    for k, n in enumerate(sizes):
        off = (k % 5) if odd else 0
        ws.append((torch.randn(n + off, generator=gen, device="cuda") * 0.1)[off:])
        gs.append((torch.randn(n + off, generator=gen, device="cuda") * scale * 10.0 ** (k % 4 - 3)).to(getattr(torch, gdtype))[off:])
    return ws, gs


def _mix(h):
    h = h ^ (h >> np.uint64(16))
    h = (h * np.uint64(0x85EBCA6B)) & np.uint64(0xFFFFFFFF)
    h = h ^ (h >> np.uint64(13))
    h = (h * np.uint64(0xC2B2AE35)) & np.uint64(0xFFFFFFFF)
    return h ^ (h >> np.uint64(16))


def _draws(seed, step, units):
    mask = np.uint64(0xFFFFFFFF)
    s1 = _mix(np.uint64(step) ^ _mix(np.uint64((seed + 0x9E3779B9) & 0xFFFFFFFF)))
    s2 = _mix((s1 + np.uint64(0x7F4A7C15)) & mask)
    h = ((units.astype(np.uint64) * np.uint64(0x9E3779B1)) & mask) ^ s1
    h = ((h ^ (h >> np.uint64(15))) * np.uint64(0x2C1B3C6D) + s2) & mask
    h = ((h ^ (h >> np.uint64(12))) * np.uint64(0x297A2D39)) & mask
    return (h ^ (h >> np.uint64(15))).astype(np.uint32)


def _encode(x, bits, draw):
    """x >= 0 f32 [n] of one tensor -> (codes, powers): by fp32 patterns, block by block."""
    n = len(x)
    pad = np.zeros((n + 63) // 64 * 64, np.float32)
    pad[:n] = x
    blocks = pad.reshape(-1, 64)
    top = blocks.max(1).view(np.uint32)
    e = np.minimum((top + np.uint32((1 << (23 - bits)) - 1)) >> np.uint32(23), 254).astype(np.int64)
    y = np.ldexp(blocks.astype(np.float64), (15 - e)[:, None]).astype(np.float32)
    d = np.zeros(pad.shape, np.uint32)
    d[:n] = draw
    c = np.minimum((y.view(np.uint32) + d.reshape(-1, 64)) >> np.uint32(23 - bits), (16 << bits) - 1).astype(np.uint8)
    if bits == 4:
        c = np.where((c == 0) & (blocks > 0), 1, c).astype(np.uint8)
    return c.reshape(-1)[:n], e.astype(np.uint8)


def _decode(codes, powers, bits):
    e = np.repeat(powers.astype(np.int64), 64)[:len(codes)]
    return np.ldexp((codes.astype(np.uint32) << np.uint32(23 - bits)).view(np.float32).astype(np.float64), e - 15).astype(np.float32)


def _f(x):
    return np.float32(x)


def _reference_step(w, g, m, v, t, lr, betas, eps, coef, wd, ls):
    """One tensor, f32 operation by operation."""
    with np.errstate(over="ignore", invalid="ignore"):
        gs = g * _f(coef)
        m1 = m * _f(betas[0]) + gs * _f(1 - betas[0])
        v1 = v * _f(betas[1]) + (gs * gs) * _f(1 - betas[1])
        u1 = np.sqrt(v1)
        ok = np.isfinite(m1) & np.isfinite(v1)
        rate = _f(lr / (1 - betas[0] ** t)) * _f(ls)
        root2 = _f(1 / np.sqrt(1 - betas[1] ** t))
        fade = _f(lr * float(_f(ls)) * float(_f(wd)))
        step = rate * (m1 / (u1 * root2 + _f(eps)))
        w1 = (w - fade * w) - step
    return np.where(ok, w1, w), np.where(ok, m1, m), np.where(ok, v1, v), np.where(ok, u1, np.sqrt(v)), np.where(ok, 4 * H * np.abs(step), 0) + 2 * H * np.abs(w)


def _np(t):
    return t.detach().float().cpu().numpy()


def _coef(gs, grad_scale, max_norm):
    if not max_norm:
        return _f(grad_scale), None
    norm = abs(float(_f(grad_scale))) * np.sqrt(sum(float((_np(g).astype(np.float64) ** 2).sum()) for g in gs))
    return (_f(float(_f(grad_scale)) * (max_norm / norm)) if norm > max_norm else _f(grad_scale)), norm


@pytest.mark.parametrize("gdtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("state", ["f32", "u8"])
@pytest.mark.parametrize("max_norm,grad_scale", [(0.0, 1.0), (0.5, 0.25), (1e9, 2.0)])
def test_steps(env, state, gdtype, max_norm, grad_scale):
    ops, torch = env
    print("adamw", state, gdtype, max_norm, flush=True)
    ws, gs = _tensors(torch, SIZES, gdtype, 5)
    wd = [0.01 * (k % 3) for k in range(len(SIZES))]
    ls = [1.0, 2.0, 10.0, 20.0] * 3
    opt = ops.AdamW(ws, gs, state=state, weight_decay=wd, lr_scale=ls, seed=99)
    ref = [dict(w=_np(w), m=np.zeros(w.numel(), np.float32), v=np.zeros(w.numel(), np.float32), u=np.zeros(w.numel(), np.float32)) for w in ws]
    lr = 1e-3
    for t in (1, 2, 3, 4):
        for g in gs:
            g.mul_(-0.7)
        coef, norm = _coef(gs, grad_scale, max_norm)
        opt.step(lr, grad_scale=grad_scale, max_norm=max_norm)
        assert int(opt.steps) == t
        if norm is not None:
            assert abs(float(opt.grad_norm) - norm) <= 2 * H * norm
        for k, (w, g, r) in enumerate(zip(ws, gs, ref)):
            n, off = w.numel(), opt.offsets[k]
            if state == "u8":
                r["v"] = r["u"] * r["u"]
            w1, m1, v1, u1, tol = _reference_step(r["w"], _np(g), r["m"], r["v"], t, lr, opt.betas, opt.eps, coef, wd[k], ls[k])
            got = _np(w)
            assert (np.abs(got.astype(np.float64) - w1) <= tol).all(), (k, t)
            if state == "f32":
                assert np.array_equal(_np(opt.m[off:off + n]), m1) and np.array_equal(_np(opt.v[off:off + n]), v1), (k, t)
                r.update(w=got, m=m1, v=v1)
            elif n:
                h = _draws(99, t, off + np.arange(n))
                cm, em = _encode(np.abs(m1), 3, (h & np.uint32(0xFFFF)) << np.uint32(4))
                cu, eu = _encode(u1, 4, (h >> np.uint32(16)) << np.uint32(3))
                nb = (n + 63) // 64
                pw = opt.powers[off // 64:off // 64 + nb].cpu().numpy()
                assert np.array_equal(pw[:, 0], em) and np.array_equal(pw[:, 1], eu), (k, t)
                assert np.array_equal(opt.m8[off:off + n].cpu().numpy(), cm | (np.signbit(m1).astype(np.uint8) << 7)), (k, t)
                assert np.array_equal(opt.u8[off:off + n].cpu().numpy(), cu), (k, t)
                m2, u2 = opt.unpack()
                r.update(w=got, m=np.copysign(_decode(cm, em, 3), m1), u=_decode(cu, eu, 4))
                assert np.array_equal(_np(m2[off:off + n]), r["m"]) and np.array_equal(_np(u2[off:off + n]), r["u"])
                b16 = opt.unpack(torch.bfloat16)
                assert torch.equal(b16[0].float(), m2) and torch.equal(b16[1].float(), u2)
    gaps = torch.ones(opt.total, dtype=torch.bool, device="cuda")
    for off, n in zip(opt.offsets, SIZES):
        gaps[off:off + n] = False
    for buf in ((opt.m, opt.v) if state == "f32" else (opt.m8, opt.u8)):
        assert not bool(buf[gaps].any())
    assert ops.status_poll(raise_on_error=False) == 0


def test_against_the_formula_in_64_bits(env):
    """Ten steps from zero; m and v are sums of t rounded terms, so off by at most 2 t h of the terms' magnitudes, w by the steps' errors."""
    ops, torch = env
    ws, gs = _tensors(torch, [5000, 33], "float32", 8)
    opt = ops.AdamW(ws, gs, weight_decay=0.05)
    w, m, v = [x.double().cpu().numpy() for x in ws], [np.zeros(5000), np.zeros(33)], [np.zeros(5000), np.zeros(33)]
    mag, moved = [np.zeros(5000), np.zeros(33)], [np.zeros(5000), np.zeros(33)]
    lr = 1e-2
    for t in range(1, 11):
        for k, g in enumerate(gs):
            g.mul_(-0.9).add_(0.01)
            x = g.double().cpu().numpy()
            m[k] = 0.9 * m[k] + 0.1 * x
            mag[k] = 0.9 * mag[k] + 0.1 * np.abs(x)
            v[k] = 0.999 * v[k] + 0.001 * x * x
            den = np.sqrt(v[k] / (1 - 0.999 ** t)) + 1e-8
            w[k] = w[k] - lr * 0.05 * w[k] - lr * (m[k] / (1 - 0.9 ** t)) / den
            # the constants' own roundings (b, 1 - b: half a step each) count with the sums'
            moved[k] += lr * (mag[k] / (1 - 0.9 ** t)) / den * (6 * t + 20) * H + 4 * H * np.abs(w[k])
        opt.step(lr)
    for k, n in enumerate((5000, 33)):
        off = opt.offsets[k]
        assert (np.abs(_np(opt.m[off:off + n]) - m[k]) <= 60 * H * mag[k]).all() and (np.abs(_np(opt.v[off:off + n]) - v[k]) <= 80 * H * v[k]).all()
        assert (np.abs(_np(ws[k]) - w[k]) <= moved[k]).all()


def test_every_code_survives_unpack_and_pack(env):
    ops, torch = env
    w = torch.zeros(64 * 512, device="cuda")
    opt = ops.AdamW([w], [w.clone()], state="u8")
    rng = np.random.default_rng(0)
    m8 = rng.integers(0, 256, 64 * 512).astype(np.uint8)
    u8 = rng.integers(0, 256, 64 * 512).astype(np.uint8)
    m8[:256], u8[:256] = np.arange(256), np.arange(256)
    m8[m8 == 0x80] = 0
    m8[0::64], u8[0::64] = 0x7F, 0xFF       # the block's largest code keeps its power of two
    pw = rng.integers(60, 200, (512, 2)).astype(np.uint8)
    opt.m8.copy_(torch.from_numpy(m8)); opt.u8.copy_(torch.from_numpy(u8)); opt.powers.copy_(torch.from_numpy(pw))
    m, u = opt.unpack()
    assert np.array_equal(_np(m), np.where(m8 & 0x80, -1, 1).astype(np.float32) * _decode(m8 & 0x7F, pw[:, 0], 3)) and np.array_equal(_np(u), _decode(u8, pw[:, 1], 4))
    opt.m8.fill_(1); opt.u8.fill_(1); opt.powers.fill_(1)
    opt.pack(m, u)
    assert np.array_equal(opt.m8.cpu().numpy(), m8) and np.array_equal(opt.u8.cpu().numpy(), u8) and np.array_equal(opt.powers.cpu().numpy(), pw)


def test_pack_rounds_to_nearest(env):
    """Half a step of `bits` mantissa bits of the value; below the smallest binade half of its step, and the whole step for a root that is not stored as zero.
    That step is 2^(k - 14 - bits), where the block's largest is at most (2 - 2^-bits) 2^k and above (2 - 2^-bits) 2^(k - 1): the whole step is at most
    2^-(14 + bits) * 2 / (2 - 2^-bits) of the largest (1.067 and 1.033 times 2^-(14 + bits))."""
    ops, torch = env
    w = torch.zeros(64 * 100, device="cuda")
    opt = ops.AdamW([w], [w.clone()], state="u8")
    gen = torch.Generator(device="cuda").manual_seed(1)
    m = torch.randn(opt.total, generator=gen, device="cuda") * torch.exp(4 * torch.randn(opt.total, generator=gen, device="cuda"))
    u = m.abs() * 3
    opt.pack(m, u)
    m2, u2 = opt.unpack()
    for x, y, bits in ((m, m2, 3), (u, u2, 4)):
        top = x.abs().view(-1, 64).amax(1, keepdim=True).expand(-1, 64).reshape(-1)
        assert bool(((x - y).abs() <= torch.maximum(x.abs() * 2.0 ** -(bits + 1), top * 2.0 ** -(14 + bits) * 2 / (2 - 2.0 ** -bits))).all())
    assert bool((u2[u > 0] > 0).all())


def test_eight_bit_moments_follow_the_average(env):
    """A constant gradient for 400 steps: rounding to nearest would stop v where its change falls below half a step (after about 16 steps for 4 mantissa bits
    of the root); rounding at random follows 1 - 0.999^t.  Averaged over 65536 elements: the spread of one element is below 8 %, of the mean below
    0.08 / 256 -- 1 % is asked."""
    ops, torch = env
    n = 65536
    w = torch.zeros(n, device="cuda")
    g = torch.exp(0.5 * torch.randn(n, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)))
    opt = ops.AdamW([w], [g], state="u8", seed=4)
    for _ in range(400):
        opt.step(0.0)
    m, u = opt.unpack()
    assert abs(float((m / g).double().mean()) - 1.0) < 0.01
    assert abs(float((u / g).double().square().mean()) / (1 - 0.999 ** 400) - 1.0) < 0.02
    a = ops.AdamW([torch.zeros(n, device="cuda")], [g], state="u8", seed=4)
    for _ in range(400):
        a.step(0.0)
    assert torch.equal(a.m8, opt.m8) and torch.equal(a.u8, opt.u8)


def test_gradients_that_are_not_finite(env):
    ops, torch = env
    try:
        for state in ("f32", "u8"):
            ws, gs = _tensors(torch, [300, 5000], "float32", 3)
            opt = ops.AdamW(ws, gs, state=state)
            opt.step(1e-3)
            before = [w.clone() for w in ws]
            gs[1][7], gs[1][4500], gs[0][0] = float("nan"), float("inf"), 3e38
            keep = [torch.ones(300, dtype=torch.bool, device="cuda"), torch.ones(5000, dtype=torch.bool, device="cuda")]
            keep[1][7] = keep[1][4500] = keep[0][0] = False
            opt.step(1e-3)                     # element by element
            assert int(opt.steps) == 2
            assert ops.status_poll(raise_on_error=False) == ops.STATUS_NAN_GRADIENT
            for k in (0, 1):
                assert torch.equal(ws[k][~keep[k]], before[k][~keep[k]]) and bool((ws[k][keep[k]] != before[k][keep[k]]).any()) and bool(torch.isfinite(ws[k]).all())
            before = [w.clone() for w in ws]
            opt.step(1e-3, max_norm=1.0)       # the norm is not a number: the whole step
            assert int(opt.steps) == 2 and not np.isfinite(float(opt.grad_norm))
            assert all(torch.equal(a, b) for a, b in zip(ws, before))
            opt.step(1e-3)                     # the word is still raised: nothing happens
            assert int(opt.steps) == 2 and all(torch.equal(a, b) for a, b in zip(ws, before))
            with pytest.raises(ops._lib.EmadaptDeviceError):
                ops.status_poll()
            for g in gs:
                g.fill_(0.5)
            opt.step(1e-3, max_norm=1.0)
            assert int(opt.steps) == 3 and ops.status_poll(raise_on_error=False) == 0
            # in collective mode the gradient carries the failure, the local word does not decide
            ops.status_collective(True)
            ops.status_raise(ops.STATUS_STREAMK_TIMEOUT)
            opt.step(1e-3)
            assert int(opt.steps) == 4
            ops.status_collective(False)
            assert ops.status_poll(raise_on_error=False) == ops.STATUS_STREAMK_TIMEOUT
    finally:
        ops.status_collective(False)
        ops.status_poll(raise_on_error=False)


def test_zero_grads_and_many_tensors(env):
    ops, torch = env
    for gdtype in ("float32", "bfloat16"):
        sizes = [1 + (k * 97) % 1500 for k in range(300)]
        ws, gs = _tensors(torch, sizes, gdtype, 9)
        one = ops.AdamW([w.clone() for w in ws], gs, weight_decay=0.1)
        one.step(1e-3)
        for k in (0, 150, 299):   # each alone
            w = ws[k].clone()
            o = ops.AdamW([w], [gs[k]], weight_decay=0.1)
            o.step(1e-3)
            assert torch.equal(w, one.params[k]) and torch.equal(o.m[:sizes[k]], one.m[one.offsets[k]:one.offsets[k] + sizes[k]])
        for state in ("f32", "u8"):
            mine = [g.clone() for g in gs]
            opt = ops.AdamW([w.clone() for w in ws], mine, state=state, weight_decay=0.1)
            opt.step(1e-3, zero_grads=True)
            assert all(not bool(g.any()) for g in mine)
            assert state == "u8" or all(torch.equal(a, b) for a, b in zip(opt.params, one.params))
        opt.set_grads(gs)
        opt.step(1e-3)
        assert int(opt.steps) == 2


def test_a_replayed_graph_steps_like_eager_calls(env):
    ops, torch = env
    for state in ("f32", "u8"):
        for max_norm in (0.0, 0.1):
            ws, gs = _tensors(torch, [700, 4097, 64], "float32", 12)
            eager = ops.AdamW([w.clone() for w in ws], gs, state=state, seed=3)
            ours = ops.AdamW([w.clone() for w in ws], gs, state=state, seed=3)
            eager.step(1e-3, max_norm=max_norm)
            ours.step(1e-3, max_norm=max_norm)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                ours.step(1e-3, max_norm=max_norm)
            for turn in range(4):
                for g in gs:
                    g.mul_(-0.8)
                graph.replay()
                torch.cuda.synchronize()
                eager.step(1e-3, max_norm=max_norm)
                assert int(ours.steps) == int(eager.steps) == turn + 2
                assert all(torch.equal(a, b) for a, b in zip(ours.params, eager.params)), (state, max_norm, turn)


def test_on_another_stream(env):
    ops, torch = env
    ws, gs = _tensors(torch, [9000, 5], "bfloat16", 1)
    a, b = ops.AdamW([w.clone() for w in ws], gs, state="u8"), ops.AdamW([w.clone() for w in ws], gs, state="u8")
    a.step(1e-3, max_norm=1.0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b.step(1e-3, max_norm=1.0)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(a.params, b.params)) and torch.equal(a.m8, b.m8)


def test_refusals(env):
    ops, torch = env
    w, g = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
    for call in (lambda: ops.AdamW([w], [g.half()]), lambda: ops.AdamW([w.bfloat16()], [g]), lambda: ops.AdamW([w, w.clone()], [g, g.bfloat16()])):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ops.AdamW([], []), lambda: ops.AdamW([w], [g], state="u4"), lambda: ops.AdamW([w], [g, g]), lambda: ops.AdamW([w], [g[:50]]),
                 lambda: ops.AdamW([w.cpu()], [g]), lambda: ops.AdamW([w], [g.cpu()]), lambda: ops.AdamW([w[::2]], [g[:50]]), lambda: ops.AdamW([w, w], [g, g]),
                 lambda: ops.AdamW([w[:60], w[50:]], [g[:60], g[50:]]), lambda: ops.AdamW([w], [g], betas=(1.0, 0.9)), lambda: ops.AdamW([w], [g], eps=0.0),
                 lambda: ops.AdamW([w], [g], weight_decay=[0.1, 0.2]), lambda: ops.AdamW([w], [g]).unpack(),
                 lambda: ops.AdamW([w, w.clone()], [g, g]).step(1e-3, zero_grads=True),
                 lambda: ops.AdamW([w], [g], state="u8").pack(torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda"))):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ops._lib.EmadaptError):
        ops.AdamW([w], [g]).step(1e-3, max_norm=-1.0)


def test_new_gradients_reach_a_captured_step(env):
    """set_grads() after a capture: replays read the new gradients (of the type they were captured with), never an address that is gone."""
    ops, torch = env
    for state in ("f32", "u8"):
        ws, gs = _tensors(torch, [700, 4097, 64], "float32", 13)
        ours = ops.AdamW([w.clone() for w in ws], [g.clone() for g in gs], state=state, seed=3)
        eager = ops.AdamW([w.clone() for w in ws], gs, state=state, seed=3)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ours.step(1e-3, max_norm=0.1)
        narrow = [(g * 0.5).bfloat16() for g in gs]
        for turn in range(3):
            for o in (ours, eager):
                o.set_grads(narrow)
                o.step(1e-3, max_norm=0.1)
            fresh = [g * (turn - 1.5) for g in gs]
            ours.set_grads([g.clone() for g in fresh])
            graph.replay()
            torch.cuda.synchronize()
            eager.set_grads(fresh)
            eager.step(1e-3, max_norm=0.1)
            assert int(ours.steps) == int(eager.steps) == 2 * turn + 2
            assert all(torch.equal(a, b) for a, b in zip(ours.params, eager.params)), (state, turn)


def test_gradients_in_the_weights_are_refused(env):
    ops, torch = env
    w, g = torch.zeros(100, device="cuda"), torch.zeros(100, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        ops.AdamW([w], [w])
    opt = ops.AdamW([w[:50], w[50:]], [g[:50], g[50:]])
    with pytest.raises(ValueError, match="share memory"):
        opt.set_grads([g[:50], w[10:60]])
    opt.step(1e-3)


def test_pack_takes_nan_as_zero(env):
    ops, torch = env
    opt = ops.AdamW([torch.zeros(128, device="cuda")], [torch.zeros(128, device="cuda")], state="u8")
    m, u = torch.ones(opt.total, device="cuda"), torch.ones(opt.total, device="cuda")
    m[3] = u[3] = m[70] = float("nan")
    m[5], u[5] = float("inf"), float("inf")
    opt.pack(m, u)
    m2, u2 = opt.unpack()
    assert float(m2[3]) == 0 and float(u2[3]) == 0 and float(m2[70]) == 0 and float(u2[70]) == 1
    assert bool(torch.isfinite(m2).all()) and bool(torch.isfinite(u2).all()) and bool((m2[64:70] == 1).all())


@pytest.mark.parametrize("state", ["f32", "u8"])
def test_a_tensor_of_more_than_2_31_elements(env, state):
    """Elements are worked on one by one (without a norm): the last ones of a large tensor go where they go in a tensor of their own.  (8 bits: the weights,
    which a first step moves by moments not yet rounded.)"""
    ops, torch = env
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of free memory")
    n, tail = 2 ** 31 + 4099, 5000
    w = torch.empty(n, device="cuda").normal_()
    g = torch.empty(n, dtype=torch.bfloat16, device="cuda").normal_()
    ws, gs = w[n - tail:].clone(), g[n - tail:].clone()
    large, small = ops.AdamW([w], [g], state=state, weight_decay=0.1), ops.AdamW([ws], [gs], state=state, weight_decay=0.1)
    large.step(1e-2)
    small.step(1e-2)
    assert torch.equal(w[n - tail:], ws)
    if state == "f32":
        assert torch.equal(large.m[n - tail:n], small.m[:tail]) and torch.equal(large.v[n - tail:n], small.v[:tail])
    else:
        m, u = large.unpack(torch.bfloat16)
        m2, u2 = small.unpack(torch.bfloat16)
        # either is within a whole step of what both round: 1/8 and 1/16 of the value, or of the block's smallest step
        for a, b, share in ((m[n - tail:n].float(), m2[:tail].float(), 1 / 8), (u[n - tail:n].float(), u2[:tail].float(), 1 / 16)):
            assert bool(((a - b).abs() <= 2 * share * torch.maximum(a.abs(), b.abs()) + float(b.abs().max()) * 2.0 ** -15).all())
    large.step(1e-2, max_norm=1.0)
    assert abs(float(large.grad_norm) - n ** 0.5) < 1e-3 * n ** 0.5
