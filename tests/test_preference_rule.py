"""The preference loss on both sides of the rule that chooses one block or two launches: the same sequences' sums, in 64 bits."""
import numpy as np
import pytest
import torch

from oracle import token_loss_oracle as O
from test_token_losses import LP, _np


@pytest.mark.gpu
@pytest.mark.parametrize("S,T", [(8, 512), (8, 513), (32, 128), (32, 129), (34, 120), (2, 512), (2, 513), (32, 1), (34, 1), (2, 1025), (32, 1024), (34, 1024)])
@pytest.mark.parametrize("average", [False, True])
def test_on_both_sides(S, T, average):
    from star_rwkv6_b200.loss import preference_loss
    g = torch.Generator().manual_seed(S + T)
    z, t = torch.randn(S, T, 7, generator=g), torch.randint(-1, 8, (S, T), generator=g)      # some targets are no tokens
    mask = torch.rand(S, T, generator=g) < 0.8
    beta = 1.0 if average else 0.01
    want, want_seq, want_g, c = O.preference(_np(z), _np(t), None, _np(mask), beta, 0.1, 0.2, average)
    zc = z.cuda().requires_grad_(True)
    loss, seq = preference_loss(zc, t.cuda(), None, mask.cuda(), beta=beta, label_smoothing=0.1, margin=0.2, average=average)
    off = LP if average else T * LP
    assert (np.abs(_np(seq) - want_seq) <= off + 2.0 ** -24 * np.abs(want_seq)).all()
    assert abs(loss.item() - want) <= 2 * beta * off + 2.0 ** -23 * abs(want)
    (gz,) = torch.autograd.grad(loss, zc)
    # a slope is off by a quarter of what D is off by, times 2 / S beta; every gradient by that and by what a probability is off by
    slope = 2 / S * beta
    assert (np.abs(_np(gz) - want_g) <= slope * (2 * beta * off + LP) + 2.0 ** -22 * np.abs(want_g)).all()
