"""The rounded square root in the 8-bit step is the correctly rounded one: read back as the scale of a block whose largest value it is."""
import numpy as np
import pytest
import torch

# v in [low, 2 low): beta2, and two values of sqrt(v) before the step, whose terms of the sum are an odd number of last places apart (a sum
# half way between two values goes to the even one)
HALVES = {1: (0.75, (np.float32(1.1547005), np.float32(1.1547004))), 2: (0.5, (np.float32(2.0), np.float32(1.9999999)))}


def _gradients(low, old, first, count):
    """Gradients g (0: none found) that take the second moment beta2 old^2 + (1 - beta2) g^2, rounded operation by operation, to the fp32
    values number first ... first + count - 1 of [low, 2 low), and those values."""
    f = np.float32
    b2 = HALVES[low][0]
    base = f(f(old * old) * f(b2))
    v = (np.float32(low).view(np.uint32) + np.arange(first, first + count, dtype=np.uint32)).view(f)
    near = np.sqrt(np.maximum(v.astype(np.float64) - base, 0.0) / (1 - b2)).astype(f)
    g = np.zeros_like(v)
    for k in (0, -1, 1, -2, 2):
        x = (np.maximum(near.view(np.int32) + k, 0)).view(f)
        g = np.where((base + (x * x) * f(1 - b2) == v) & (g == 0), x, g)
    return g, v


@pytest.mark.gpu
@pytest.mark.parametrize("low", [1, 2])
def test_every_square_root(low):
    """The values of [1, 2) and of [2, 4) that a gradient reaches (94 in 100 of their 2^24), one per block of 256; a scale is root / 448 rounded, which for roots
    below 1.75 no two roots have in common."""
    from star_rwkv6_b200.optim import adamw_step
    per = 1 << 18
    n = per * 256
    b2, olds = HALVES[low]
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m, v = (torch.zeros(n, dtype=torch.float8_e4m3fn, device="cuda") for _ in range(2))
    scales = [torch.zeros(per, device="cuda") for _ in range(2)]
    reached = 0
    for first in range(0, 1 << 23, per):
        there = np.zeros(per, bool)
        for old in olds:
            x, want_v = _gradients(low, old, first, per)
            g[::256] = torch.from_numpy(x).cuda()
            v.fill_(1.0)
            scales[1].fill_(float(old))
            adamw_step([p], [g], [m], [v], exp_avg_scales=scales[:1], exp_avg_sq_scales=scales[1:], step=1, lr=0.0, betas=(0.9, b2), weight_decay=0.0)
            root = np.sqrt(want_v.astype(np.float64)).astype(np.float32)      # rounding twice changes no square root: 53 >= 2 * 24 + 2
            want, got = root * np.float32(1.0 / 448.0), scales[1].cpu().numpy()
            assert np.array_equal(got[x != 0], want[x != 0])
            there |= x != 0
        reached += int(there.sum())
    assert reached >= 0.93 * 2 ** 23
