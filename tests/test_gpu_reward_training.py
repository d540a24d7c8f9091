"""Training on rewards and preferences end to end: label maps sampled from the network, the policy / preference loss on its logits, the hand-written
backward, AdamW.  Gradients against the CPU oracle's graph with the losses spelled out in 64 bits (the bars of test_gpu_model.py for the same backward),
the update against the formula on the gradients that the GPU has."""
import os
import sys

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
H = 2.0 ** -24
SIZE, C, WIDTH, B = 65, 5, 8, 2


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    from em_adapt_tensorflow_amd import ops
    from em_adapt_tensorflow_amd.deeplab import ADAPT
    from oracle import deeplab_oracle as do
    return ADAPT, ops, do, torch


def _net(ADAPT, do, torch, accum_num=1, **config):
    a = ADAPT(dict({"input_size": (SIZE, SIZE), "category_num": C, "width": WIDTH, "accum_num": accum_num, "batch_size": B, "device": "cuda:0"}, **config))
    a.build()
    oracle = do.DeepLabOracle(category_num=C, width=WIDTH, dtype=torch.float64)
    params = do.init_params(oracle.specs, seed=11, he=True)
    for layer, (w, b) in params.items():
        a.weights[layer][0].copy_(torch.tensor(w).cuda())
        a.weights[layer][1].copy_(torch.tensor(b).cuda())
    a.pre_train(base_lr=1e-3, weight_decay=1e-2, momentum=0.9, batch_size=B)
    return a, oracle, params


def _images(do, seed, n=B):
    return (do.synthetic_batch(n, SIZE, C, seed=seed)[0] / 50.0).astype(np.float32)


def _sample(torch, a, images, seed):
    """A label map per image drawn from the network's softmax, a part of it void."""
    logits = a.forward(images, 1.0)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    u = torch.rand(logits.shape, generator=gen, device="cuda").clamp(1e-9, 1 - 1e-7)
    lab = (logits - torch.log(-torch.log(u))).argmax(3)
    lab[:, 0, :2] = 255
    return lab


def _rel(got, want):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    return np.abs(got - want).max() / max(np.abs(want).max(), 1e-30)


def _accumulated(a, layer):
    seg = a._segments[layer]
    s, nw, (kh, kw, cin, cout) = seg["start"], seg["nw"], seg["shape"]
    return a._flat["accum"][s:s + nw].view(seg["pshape"])[:, :, :cin, :cout].cpu().numpy(), a._flat["accum"][s + nw:s + nw + cout].cpu().numpy()


def _oracle_logp(torch, oracle, params, images, lab):
    t = oracle.tensors(params)
    z = oracle.forward(t, images)["output"]
    lab = lab.cpu()
    used = lab < C
    logp = torch.log_softmax(z, 3).gather(3, torch.where(used, lab, 0)[..., None])[..., 0]
    return t, torch.where(used, logp, torch.zeros_like(logp)), used


def test_policy_step_against_the_oracle(env):
    ADAPT, ops, do, torch = env
    a, oracle, params = _net(ADAPT, do, torch, accum_num=2, optimizer="adamw")
    want = {}
    for mb in range(2):
        images = _images(do, 5 + mb)
        lab = _sample(torch, a, images, 3 + mb)
        old = a.label_logp(images, lab)
        rng = np.random.default_rng(mb)
        noise = torch.tensor(rng.normal(0, 0.25, tuple(lab.shape)).astype(np.float32)).cuda()
        ref, adv = old + 0.5 * noise.flip(0), torch.tensor([0.7, -1.3]).cuda()
        sums, logp = a.policy_step(images, lab, old - noise, adv, ref_logp=ref, clip_low=0.2, clip_high=0.2, kl_coef=0.1)
        t, lp, used = _oracle_logp(torch, oracle, params, images, lab)
        assert _rel(logp.cpu(), lp.detach()) < 1e-4
        ratio = torch.exp(lp - (old - noise).double().cpu())
        A = adv.double().cpu().view(-1, 1, 1)
        q = ref.double().cpu() - lp
        rows = torch.maximum(-A * ratio, -A * ratio.clamp(0.8, 1.2)) + 0.1 * (torch.exp(q) - q - 1)
        loss = (rows * used).sum()
        assert abs(float(sums[0]) - float(loss)) < 1e-3 * abs(float(loss)) + 1e-2
        (loss / lab.numel() / 2).backward()     # mean over the pixels, accum_num 2
        for layer, (w, b) in t.items():
            g = [w.grad.numpy(), b.grad.numpy()]
            want[layer] = g if layer not in want else [want[layer][0] + g[0], want[layer][1] + g[1]]
    for layer, (dw, db) in want.items():
        gw, gb = _accumulated(a, layer)
        assert _rel(gw, dw) < 2e-4 and _rel(gb, db) < 2e-4, layer


def test_preference_step_against_the_oracle(env):
    ADAPT, ops, do, torch = env
    a, oracle, params = _net(ADAPT, do, torch, optimizer="adamw")
    images = np.repeat(_images(do, 9, 1), 2, axis=0)
    lab = _sample(torch, a, images, 8)
    ref = a.label_logp(images, lab).sum((1, 2)) + torch.tensor([0.5, -2.0]).cuda()
    loss, seq = a.preference_step(images, lab, ref, beta=0.2, label_smoothing=0.1)
    t, lp, used = _oracle_logp(torch, oracle, params, images, lab)
    s = lp.sum((1, 2))
    assert _rel(seq.cpu(), s.detach()) < 1e-4
    r = s - ref.double().cpu()
    h = 0.2 * (r[0] - r[1])
    want = 0.9 * torch.nn.functional.softplus(-h) + 0.1 * torch.nn.functional.softplus(h)
    assert abs(float(loss) - float(want)) < 1e-3
    want.backward()
    for layer, (w, b) in t.items():
        gw, gb = _accumulated(a, layer)
        assert _rel(gw, w.grad.numpy()) < 2e-4 and _rel(gb, b.grad.numpy()) < 2e-4, layer


@pytest.mark.parametrize("max_norm", [0.0, 0.01])
def test_first_adamw_update_of_the_network(env, max_norm):
    """From zero moments the step is lr g / (|g| + eps) whatever the betas; 12 roundings (moments, corrections, quotient, product: each of the constants
    too) of the step and two of the weight; eps' share moves a gradient's own roundings by at most as much."""
    ADAPT, ops, do, torch = env
    a, oracle, params = _net(ADAPT, do, torch, optimizer="adamw", max_grad_norm=max_norm, betas=(0.8, 0.99))
    images = _images(do, 1)
    lab = _sample(torch, a, images, 1)
    old = a.label_logp(images, lab)
    a.policy_step(images, lab, old, torch.tensor([1.0, -0.5]).cuda())
    grads = {layer: [g.astype(np.float64) for g in _accumulated(a, layer)] for layer in params}
    norm = np.sqrt(sum((g ** 2).sum() for v in grads.values() for g in v))
    c = min(1.0, max_norm / norm) if max_norm else 1.0
    a.apply_update()
    assert float(a._flat["accum"].abs().max()) == 0.0 and int(a._adamw.steps) == 1
    if max_norm:
        assert abs(float(a._adamw.grad_norm) - norm) < 1e-6 * norm and c < 1
    for layer, wb in params.items():
        for k in (0, 1):
            g, w = c * grads[layer][k], wb[k].astype(np.float64)
            step = 1e-3 * g / (np.abs(g) + 1e-8)
            want = w - 1e-3 * (1e-2 if k == 0 else 0.0) * w - step
            got = a.weights[layer][k].cpu().numpy()
            assert (np.abs(got - want) <= 12 * H * np.abs(step) + 3 * H * np.abs(w)).all(), (layer, k)
        seg = a._segments[layer]
        kh, kw, cin, cout = seg["shape"]
        full = a._flat["params"][seg["start"]:seg["start"] + seg["nw"]].view(seg["pshape"])
        assert not bool(full[:, :, cin:].any()) and not bool(full[..., cout:].any())     # the padding stays zero


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_reward_loop_and_resume(env, tmp_path, optimizer, dtype):
    """Sample, score, update, save; a second network restored from the checkpoint takes the same further step, bit for bit."""
    ADAPT, ops, do, torch = env

    def step(a, k):
        images = _images(do, 40 + k)
        lab = _sample(torch, a, images, 60 + k)
        old = a.label_logp(images, lab)
        tags = torch.zeros(B, C, device="cuda")
        tags[:, 1] = 1
        seen = torch.stack([(lab == c).float().mean((1, 2)) for c in range(C)], 1)
        reward = 1 - (seen - tags).abs().sum(1)
        sums, logp = a.policy_step(images, lab, old, reward - reward.mean(), ref_logp=old, kl_coef=0.05, keep_prob=1.0)
        assert float(sums[3]) == 0.0    # on policy nothing is clipped
        a.apply_update()
        return sums, logp
    a, _, params = _net(ADAPT, do, torch, optimizer=optimizer, compute_dtype=dtype, max_grad_norm=1.0)
    for k in range(3):
        sums, logp = step(a, k)
    assert bool(torch.isfinite(sums).all()) and int(a._adamw.steps) == 3
    assert any(not np.array_equal(a.weights[layer][0].cpu().numpy(), w) for layer, (w, b) in params.items())
    path = a.saver["norm"].save(None, str(tmp_path / "norm"), global_step=3)
    b, _, _ = _net(ADAPT, do, torch, optimizer=optimizer, compute_dtype=dtype, max_grad_norm=1.0)
    b.restore_from_model(b.saver["norm"], path)
    assert int(b._adamw.steps) == 3
    for n in (a, b):
        step(n, 7)
    for layer in params:
        assert torch.equal(a.weights[layer][0], b.weights[layer][0]) and torch.equal(a.weights[layer][1], b.weights[layer][1]), layer
    assert ops.status_poll(raise_on_error=False) == 0


def test_a_momentum_checkpoint_restores_the_weights_alone(env, tmp_path):
    ADAPT, ops, do, torch = env
    a, _, _ = _net(ADAPT, do, torch)
    a.weights["fc8"][0].mul_(2.0)
    path = a.saver["norm"].save(None, str(tmp_path / "norm"), global_step=1)
    b, _, _ = _net(ADAPT, do, torch, optimizer="adamw8")
    with pytest.warns(UserWarning, match="moments"):
        b.restore_from_model(b.saver["norm"], path)
    assert torch.equal(a.weights["fc8"][0], b.weights["fc8"][0]) and not bool(b._adamw.m8.any())


def test_fused_and_accumulated_gradients_give_the_same_weights(env):
    """One micro-batch: its gradients read where backward leaves them, or from the accumulators that they were added to zero in."""
    ADAPT, ops, do, torch = env
    from oracle import estep_oracle as eo
    images, labels = do.synthetic_batch(B, SIZE, C, seed=5)
    images = (images / 50.0).astype(np.float32)
    perms = eo.draw_perms(5, C, seed=7)
    got = []
    for fused in (False, True):
        a, _, _ = _net(ADAPT, do, torch, optimizer="adamw", fused_update=fused)
        for _ in range(3):
            a.micro_step(images, labels, keep_prob=1.0, perms=perms)
            a.apply_update()
        got.append(a._flat["params"].clone())
    assert torch.equal(*got)


def test_train_with_adamw(env):
    ADAPT, ops, do, torch = env
    from em_adapt_tensorflow_amd.data import SyntheticData
    for optimizer, accum in (("adamw", 2), ("adamw8", 1)):
        cfg = {"input_size": (SIZE, SIZE), "category_num": 21, "width": WIDTH, "accum_num": accum, "batch_size": 2, "save_final": False, "optimizer": optimizer}
        a = ADAPT(dict(cfg, data=SyntheticData(dict(cfg, length=8))))
        assert a.train(base_lr=1e-3, weight_decay=1e-5, momentum=0.9, batch_size=2, epoches=1, log=lambda *x: None) == 4
        assert int(a._adamw.steps) == 4 // accum and bool(torch.isfinite(a._flat["params"]).all())
    with pytest.raises(ValueError):
        ADAPT({"input_size": (SIZE, SIZE), "optimizer": "adam"})


def _batch_of_four(do):
    """Images, label maps, log-probabilities and an advantage per image: nothing that a rounding of the logits could switch (no E-step, no clip)."""
    images = _images(do, 31, 2 * B)
    rng = np.random.default_rng(4)
    lab = rng.integers(0, C, (2 * B, 9, 9))
    return images, lab, (-np.log(C) + 0.1 * rng.normal(size=lab.shape)).astype(np.float32), np.array([1.0, -0.5, 0.25, 0.75], np.float32)


def _worker(rank, world, port, out_dir, exchange):
    sys.path.insert(0, ROOT)
    import torch
    import torch.distributed as dist
    from em_adapt_tensorflow_amd.deeplab import ADAPT
    from oracle import deeplab_oracle as do
    os.environ["MASTER_ADDR"], os.environ["MASTER_PORT"] = "127.0.0.1", str(port)
    torch.cuda.set_device(0)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    a, _, _ = _net(ADAPT, do, torch, optimizer="adamw", max_grad_norm=0.5, bucket_mb=1, **exchange)
    assert a._gradsync is not None
    mine = [x[rank * B:(rank + 1) * B] for x in _batch_of_four(do)]
    got = {}
    for step in range(2):
        a.policy_step(*mine, clip_low=1.0, clip_high=1e6)
        a.apply_update()
        torch.cuda.synchronize()
        got.update({"%s%d" % (k, step): t.cpu().numpy() for k, t in (("params", a._flat["params"]), ("m", a._adamw.m), ("v", a._adamw.v))})
    np.savez(os.path.join(out_dir, "adamw%d.npz" % rank), **got)
    assert float(a._flat["accum"].abs().max()) == 0.0 or a._gradsync.writeback is False
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize("exchange", [{}, {"allreduce_algo": "direct"}, {"allreduce_algo": "direct", "dp_prepack": False}])
def test_two_ranks_step_like_one(env, tmp_path, exchange):
    """Two ranks of half a batch each: the same weights and moments on both, step for step, and after the first step the moment of a single process on the
    whole batch, 0.1 of the clipped gradient: each side's gradient is within 2e-4 of exact arithmetic's (the backward's bar against the oracle), relative to
    its largest element.  (Not the weights: a first step is lr times the gradient's sign, which a gradient of rounding size does not have.)"""
    import socket
    import torch.multiprocessing as mp
    ADAPT, ops, do, torch = env
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    mp.spawn(_worker, args=(2, port, str(tmp_path), exchange), nprocs=2, join=True)
    p0, p1 = (dict(np.load(tmp_path / ("adamw%d.npz" % r))) for r in (0, 1))
    assert all(np.array_equal(p0[k], p1[k]) for k in p0)
    a, _, _ = _net(ADAPT, do, torch, optimizer="adamw", max_grad_norm=0.5, batch_size=2 * B)
    a.policy_step(*_batch_of_four(do), clip_low=1.0, clip_high=1e6)
    a.apply_update()
    assert a._gradsync is None
    m = a._adamw.m.cpu().numpy()
    assert np.abs(p0["m0"] - m).max() <= 4e-4 * np.abs(m).max() and np.abs(m).max() > 0
