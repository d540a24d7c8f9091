"""A second pre_train() (train() called again on the same network) goes on with the optimizer's states, whichever the optimizer."""
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
    return ADAPT, ops, do, torch


@pytest.mark.parametrize("optimizer", ["momentum", "adamw", "adamw8"])
def test_states_go_on(env, optimizer):
    ADAPT, ops, do, torch = env
    lab = torch.ones((B, 9, 9), dtype=torch.int64, device="cuda")
    got = []
    for again in (True, False):
        a, _, _ = _net(ADAPT, do, torch, accum_num=2, optimizer=optimizer, max_grad_norm=1.0)
        for k in range(3):
            if again and k:
                a.pre_train(base_lr=1e-3, weight_decay=1e-2, momentum=0.9, batch_size=B)
            for m in range(2):
                a.policy_step(_images(do, 10 * k + m), lab, torch.full((B, 9, 9), -1.6, device="cuda"), torch.tensor([1.0, -0.5]).cuda())
            a.apply_update()
        if optimizer != "momentum":
            assert int(a._adamw.steps) == 3
        got.append(a._flat["params"].clone())
    assert torch.equal(*got) and ops.status_poll(raise_on_error=False) == 0
