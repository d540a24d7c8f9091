"""ADAPT with AdamW behind the gradient exchange, in one process (a job of one rank): the exchange's forms against the update without one, what the
collectives are given, and the accumulators behind each step."""
import socket

import pytest

from test_gpu_reward_training import B, C, _batch_of_four, _net

pytestmark = pytest.mark.gpu
FORMS = [{}, {"allreduce_algo": "direct"}, {"allreduce_algo": "direct", "dp_prepack": False}]


@pytest.fixture(scope="module")
def env():
    import torch
    import torch.distributed as dist
    assert torch.cuda.is_available()
    from em_adapt_tensorflow_amd import ops
    from em_adapt_tensorflow_amd.deeplab import ADAPT
    from oracle import deeplab_oracle as do
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    dist.init_process_group("gloo", init_method="tcp://127.0.0.1:%d" % port, rank=0, world_size=1)
    try:
        yield ADAPT, ops, do, torch, dist
    finally:
        ops.status_collective(False)
        ops.status_poll(raise_on_error=False)
        dist.destroy_process_group()


@pytest.mark.parametrize("accum_num", [1, 2])
@pytest.mark.parametrize("form", FORMS)
def test_one_rank_steps_as_without_an_exchange(env, monkeypatch, form, accum_num):
    ADAPT, ops, do, torch, dist = env
    devices = []
    for name in ("all_reduce", "all_to_all_single", "all_gather_into_tensor"):
        def wrap(*a, _f=getattr(dist, name), **kw):
            devices.extend(t.device.type for t in a if torch.is_tensor(t))
            assert "cuda" not in devices      # (looked at before the call: gloo is given CPU tensors only)
            return _f(*a, **kw)
        monkeypatch.setattr(dist, name, wrap)
    batch = [x[:B] for x in _batch_of_four(do)]
    got = []
    for exchange in (True, False):
        extra = dict(form, force_gradsync=True, bucket_mb=1) if exchange else {}
        a, _, _ = _net(ADAPT, do, torch, accum_num=accum_num, optimizer="adamw", max_grad_norm=0.5, **extra)
        assert (a._gradsync is not None) == exchange
        if not exchange:
            ops.status_collective(False)
        for _ in range(2):
            for _ in range(accum_num):
                a.policy_step(*batch, clip_low=1.0, clip_high=1e6)
            a.apply_update()
            assert not bool(a._flat["accum"].any())
        assert int(a._adamw.steps) == 2
        got.append([t.clone() for t in (a._flat["params"], a._adamw.m, a._adamw.v)])
    assert devices and all(torch.equal(x, y) for x, y in zip(*got))
    assert ops.status_poll(raise_on_error=False) == 0
