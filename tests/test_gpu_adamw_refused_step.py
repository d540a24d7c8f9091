"""AdamW's clean op (zero_grads) where the gradients' norm is not finite: the update does not happen, the gradients are zeroed all the same, or an
accumulator that held a NaN once would hold it for good."""
import numpy as np
import pytest

from test_gpu_reward_training import B, _images, _net

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    from em_adapt_tensorflow_amd import ops
    from em_adapt_tensorflow_amd.deeplab import ADAPT
    from oracle import deeplab_oracle as do
    yield ADAPT, ops, do, torch
    ops.status_poll(raise_on_error=False)


SIZES = [1, 7, 64, 4096, 5000, 12289, 1021]


def _lists(torch, gdtype):
    gen = torch.Generator(device="cuda").manual_seed(2)
    buf = torch.randn(sum(SIZES) + 3, generator=gen, device="cuda")
    ws, gs, at = [], [], 3      # (behind one another from the third element on: any alignment)
    flat = (buf * 0.1).to(getattr(torch, gdtype))
    for n in SIZES:
        ws.append(buf[at:at + n])
        gs.append(flat[at:at + n])
        at += n
    return buf, flat, ws, gs


@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("gdtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("state", ["f32", "u8"])
def test_gradients_are_zeroed_behind_a_refused_step(env, state, gdtype, bad):
    _, ops, _, torch = env
    buf, flat, ws, gs = _lists(torch, gdtype)
    opt = ops.AdamW(ws, gs, state=state)
    opt.step(1e-3, max_norm=1.0)
    before, kept = buf.clone(), [t.clone() for t in ((opt.m, opt.v) if state == "f32" else (opt.m8, opt.u8, opt.powers))]
    head = flat[:3].clone()
    gs[4][4999] = float(bad)
    opt.step(1e-3, max_norm=1.0)                        # not asked to: they stay
    assert not bool(torch.isfinite(gs[4][4999])) and bool(flat[:3].ne(0).any())
    assert ops.status_poll(raise_on_error=False) == ops.STATUS_NAN_GRADIENT
    opt.step(1e-3, max_norm=1.0, zero_grads=True)
    assert not any(bool(g.any()) for g in gs) and torch.equal(flat[:3], head)
    assert torch.equal(buf, before) and int(opt.steps) == 1 and not np.isfinite(float(opt.grad_norm))
    assert all(torch.equal(a, b) for a, b in zip(kept, (opt.m, opt.v) if state == "f32" else (opt.m8, opt.u8, opt.powers)))
    for g in gs:
        g.fill_(0.25)
    opt.step(1e-3, max_norm=1.0, zero_grads=True)       # while the word is raised nothing happens, the clean op included
    assert all(bool((g == 0.25).all()) for g in gs) and int(opt.steps) == 1
    assert ops.status_poll(raise_on_error=False) == ops.STATUS_NAN_GRADIENT
    opt.step(1e-3, max_norm=1.0, zero_grads=True)
    assert int(opt.steps) == 2 and not any(bool(g.any()) for g in gs) and bool((buf[3:] != before[3:]).any())
    assert ops.status_poll(raise_on_error=False) == 0


@pytest.mark.parametrize("state", ["f32", "u8"])
def test_in_a_replayed_graph(env, state):
    _, ops, _, torch = env
    buf, flat, ws, gs = _lists(torch, "float32")
    opt = ops.AdamW(ws, gs, state=state)
    opt.step(1e-3, max_norm=1.0, zero_grads=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(1e-3, max_norm=1.0, zero_grads=True)
    for k in range(3):
        gs[2][5] = float("nan")
        before = buf.clone()
        graph.replay()
        assert not any(bool(g.any()) for g in gs) and torch.equal(buf, before) and int(opt.steps) == 1 + k
        assert ops.status_poll(raise_on_error=False) == ops.STATUS_NAN_GRADIENT
        for g in gs:
            g.fill_(0.5)
        graph.replay()
        assert not any(bool(g.any()) for g in gs) and not torch.equal(buf, before) and int(opt.steps) == 2 + k
        assert ops.status_poll(raise_on_error=False) == 0


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
@pytest.mark.parametrize("max_norm", [0.0, 1.0])
def test_training_goes_on_behind_a_bad_micro_batch(env, optimizer, max_norm):
    """Accumulators of the network's own: a micro-batch of NaN, then two clean ones, give what the two clean ones give alone."""
    ADAPT, ops, do, torch = env
    got = []
    for bad in (True, False):
        a, _, _ = _net(ADAPT, do, torch, accum_num=2, optimizer=optimizer, max_grad_norm=max_norm)
        lab = torch.ones((B, 9, 9), dtype=torch.int64, device="cuda")
        if bad and max_norm:     # (without a norm a refused element still counts the step)
            before = a._flat["params"].clone()
            for k in range(2):
                a.policy_step(_images(do, 70 + k), lab, torch.zeros((B, 9, 9), device="cuda"), torch.tensor([1.0, float("nan") if k == 0 else 1.0]).cuda())
            a.apply_update()
            assert torch.equal(a._flat["params"], before) and int(a._adamw.steps) == 0
            with pytest.raises(ops._lib.EmadaptDeviceError):
                ops.status_poll()
        elif bad:
            a._flat["accum"][:] = float("nan")
            a.apply_update()
            assert ops.status_poll(raise_on_error=False) == ops.STATUS_NAN_GRADIENT
            a._adamw.steps.zero_()
        assert not bool(a._flat["accum"][:a._adamw.params[0].numel()].any())
        for k in range(2):
            old = a.label_logp(_images(do, 80 + k), lab)
            a.policy_step(_images(do, 80 + k), lab, old, torch.tensor([1.0, -0.5]).cuda())
        a.apply_update()
        assert int(a._adamw.steps) == 1 and ops.status_poll(raise_on_error=False) == 0
        got.append([t.clone() for wb in a.weights.values() for t in wb])
    assert all(torch.equal(x, y) for x, y in zip(*got)) and all(bool(torch.isfinite(x).all()) for x in got[0])
