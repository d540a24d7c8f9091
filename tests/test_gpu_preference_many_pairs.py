"""preference_loss of more pairs than one launch takes workgroups: a HIP grid has fewer than 2^32 threads, 2^22 workgroups of 1024."""
import pytest

pytestmark = pytest.mark.gpu
PAIRS = 2 ** 22 + 3


@pytest.mark.parametrize("want_grad", [False, True])
def test_four_million_pairs(want_grad):
    """Pairs of one row each, some empty; every pair's loss and gradient against the formula: ref_logp is 0, the logits are 0 (log 1/2 each), so that h =
    beta log(1/2) ([chosen has a row] - [rejected has one])."""
    import torch
    from em_adapt_tensorflow_amd import ops
    assert torch.cuda.is_available()
    pair = torch.arange(PAIRS, device="cuda")
    lens = torch.ones((PAIRS, 2), dtype=torch.int64, device="cuda")
    lens[:, 0] = (pair % 3 != 0).long()
    at = torch.zeros(2 * PAIRS + 1, dtype=torch.int64, device="cuda")
    at[1:] = lens.view(-1).cumsum(0)
    M = int(at[-1])
    z = torch.zeros((M, 2), device="cuda")
    lab = torch.zeros(M, dtype=torch.int64, device="cuda")
    print("preference_loss", M, flush=True)
    loss, seq, d = ops.preference_loss(z, lab, at, torch.zeros(2 * PAIRS, device="cuda"), 2, beta=0.5, grad_scale=1.0, want_grad=want_grad)
    h = 0.5 * torch.log(torch.tensor(0.5, dtype=torch.float64, device="cuda")) * (lens[:, 0] - 1)
    want = torch.nn.functional.softplus(-h)
    assert bool(((loss.double() - want).abs() < 1e-6).all())
    assert bool(((seq.view(PAIRS, 2).double() - lens * torch.log(torch.tensor(0.5, dtype=torch.float64, device="cuda"))).abs() < 1e-6).all())
    if want_grad:
        slope = -0.5 * torch.sigmoid(-h)               # of the chosen sequence, minus that of the rejected one
        coef = torch.repeat_interleave(torch.stack([slope, -slope], 1).view(-1), lens.view(-1))
        assert bool(((d[:, 0].double() - 0.5 * coef).abs() < 1e-6).all()) and bool(((d[:, 1].double() + 0.5 * coef).abs() < 1e-6).all())
