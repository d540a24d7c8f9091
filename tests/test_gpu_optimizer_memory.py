"""What the optimizers hold on the device: AdamW's states stand in the place of the Momentum buffer, not beside it."""
import gc

import pytest

from test_gpu_reward_training import B, SIZE, C, WIDTH, _net

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def env():
    import torch
    assert torch.cuda.is_available()
    from em_adapt_tensorflow_amd import ops
    from em_adapt_tensorflow_amd.deeplab import ADAPT
    from oracle import deeplab_oracle as do
    return ADAPT, ops, do, torch


def test_bytes_per_parameter(env):
    """Beside weights, gradients and accumulators: 4 bytes a parameter with Momentum, 8 with AdamW, 2 + 2/64 with 8-bit states; the states' alignment adds 255
    elements a tensor at most, the table 64 bytes a chunk of 4096, the control block 16 KB and some, the allocator rounds each tensor up to 2 MB at most."""
    ADAPT, ops, do, torch = env
    held = {}
    for optimizer in ("momentum", "momentum", "adamw", "adamw8"):   # (the first for what is allocated once)
        gc.collect()                                                # (a network refers to itself)
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        a = ADAPT({"input_size": (SIZE, SIZE), "category_num": C, "width": 32, "batch_size": B, "device": "cuda:0", "optimizer": optimizer})
        a.build()
        a.pre_train(base_lr=1e-3, weight_decay=1e-2, momentum=0.9, batch_size=B)
        held[optimizer] = torch.cuda.memory_allocated() - before
        total = a._flat["total"]
        assert ("momentum" in a._flat) == (optimizer == "momentum")
        del a
    slack = 8 * 32 * 255 + 64 * (total // 4096 + 64) + (1 << 16) + 512 * 8
    assert total > 4 * slack
    assert abs((held["adamw"] - held["momentum"]) - 4 * total) < slack
    assert abs((held["momentum"] - held["adamw8"]) - (4 - 2 - 2 / 64) * total) < slack


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
def test_checkpoints_between_the_optimizers(env, tmp_path, optimizer):
    ADAPT, ops, do, torch = env
    a, _, _ = _net(ADAPT, do, torch, optimizer=optimizer)
    a._adamw.steps.fill_(7)
    a.weights["fc8"][0].mul_(3.0)
    path = a.saver["norm"].save(None, str(tmp_path / "norm"), global_step=1)
    b, _, _ = _net(ADAPT, do, torch)
    with pytest.warns(UserWarning, match="no momentum slots"):
        b.restore_from_model(b.saver["norm"], path)
    assert torch.equal(a.weights["fc8"][0], b.weights["fc8"][0]) and not bool(b._flat["momentum"].any())
    # a network that has its weights but no optimizer yet
    from em_adapt_tensorflow_amd.network import _Saver
    c = ADAPT({"input_size": (SIZE, SIZE), "category_num": C, "width": WIDTH, "batch_size": B, "device": "cuda:0", "optimizer": optimizer})
    c.build()
    c.restore_from_model(_Saver(c), path)
    again = _Saver(c).save(None, str(tmp_path / "again"))
    d, _, _ = _net(ADAPT, do, torch, optimizer=optimizer)
    with pytest.warns(UserWarning, match="moments"):
        d.restore_from_model(d.saver["norm"], again)
    assert torch.equal(a.weights["fc8"][0], c.weights["fc8"][0]) and torch.equal(a.weights["fc8"][0], d.weights["fc8"][0])
