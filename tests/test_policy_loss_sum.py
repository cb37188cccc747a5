"""The policy loss's sum over rows, which the documents promise in 64 bits."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [3, 8, 1000, 9001])
@pytest.mark.parametrize("V", [1, 2000, 20000])
def test_terms_of_mixed_signs_cancel_exactly(rows, V):
    """One logit is possible in every row, so that lp = 0 and a token's loss is exactly -A (V = 1; otherwise the others are -inf).  Neighbours of
    2^25 and -2^25 enclose numbers 4 n + 1: 32 bits
    lose the ones, 64 bits hold the whole sum, which is rounded once."""
    from star_rwkv6_b200.loss import policy_loss
    if rows * V > 10 ** 8:
        rows = 10 ** 8 // V
    z = torch.full((rows, V), float("-inf"), device="cuda", dtype=torch.bfloat16)
    z[:, 0] = 0
    t, zero = torch.zeros(rows, dtype=torch.int64, device="cuda"), torch.zeros(rows, device="cuda")
    i = torch.arange(rows, device="cuda")
    adv = torch.where(i % 3 == 1, 4 * (i % 50) + 1, torch.where(i % 3 == 0, 2.0 ** 25, -2.0 ** 25)).float()
    adv[rows // 3 * 3:] = 1.0
    loss, lp = policy_loss(z, t, adv, zero, reduction="sum")
    assert not lp.any() and loss.item() == torch.tensor(-adv.double().sum().item()).float().item()
