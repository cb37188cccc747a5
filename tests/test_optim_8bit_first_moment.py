"""How far the first moment can follow in 8 bits: e4m3 codes rounded to nearest, a step changes one by 1 - beta1 of what it lacks.  Codes with
a fraction of 1/8 are the last to move: their lower neighbour is at 8/9 of them, the border at 17/18.  So without gradients every code
above the subnormal ones falls for beta1 < 17/18 = 0.944, and some never do above it.  Below 2^-6 codes are 2^-9 apart and n of them
stay where n (1 - beta1) <= 1/2: at 0.94 the eight lowest, 3.5e-5 of a block's largest value."""
import numpy as np
import pytest
import torch

from oracle import adamw_oracle as O


def _decayed(beta1, steps=4000):
    q = np.unique(O.e4m3_nearest(np.linspace(0, 448, 1 << 16)))
    for _ in range(steps):
        q = O.e4m3_nearest(beta1 * q)
    return q


def test_which_betas_let_every_code_fall():
    assert _decayed(0.9).max() <= 5 * 2.0 ** -9 and _decayed(0.94).max() <= 8 * 2.0 ** -9
    assert _decayed(0.945).max() >= 200 and _decayed(0.95).max() >= 200


def test_others_are_refused():
    from star_rwkv6_b200 import _lib as L
    from star_rwkv6_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    for beta1 in (0.9401, 0.95, 0.99):
        with pytest.raises(ValueError, match="0.94"):
            AdamW([p], betas=(beta1, 0.999), state_bits=8)
        AdamW([p], betas=(beta1, 0.999))
    AdamW([p], betas=(0.94, 0.999), state_bits=8)
    with pytest.raises(ValueError, match="0.94"):             # a group's own settings
        AdamW([{"params": [p], "betas": (0.95, 0.999)}], state_bits=8)
    with pytest.raises(ValueError, match="0.94"):
        AdamW([{"params": [p], "state_bits": 8}], betas=(0.95, 0.999))
    c = L.AdamWConfig()
    c.dtype, c.state_bits, c.step, c.lr, c.beta1, c.beta2, c.eps = L.BF16, 8, 1, 1e-3, 0.95, 0.99, 1e-8
    assert L.lib.wkv6_adamw_step(c, 0, None, None) == -2 and b"0.94" in L.lib.wkv6_last_error()
    c.beta1 = 0.94
    assert L.lib.wkv6_adamw_step(c, 0, None, None) == 0
    c.state_bits, c.beta1 = 32, 0.95
    assert L.lib.wkv6_adamw_step(c, 0, None, None) == 0


@pytest.mark.gpu
def test_the_step():
    from star_rwkv6_b200.optim import AdamW, adamw_step
    n = 512
    p, g = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    m = torch.full((n,), 13.0, device="cuda").to(torch.float8_e4m3fn)
    v = m.clone()
    kw = dict(exp_avg_scales=[torch.ones(2, device="cuda")], exp_avg_sq_scales=[torch.ones(2, device="cuda")])
    for betas in ((0.95, 0.999), (0.9999, 0.9)):
        with pytest.raises(ValueError, match="0.94"):
            adamw_step([p], [g], [m], [v], step=1, betas=betas, **kw)
    q = torch.nn.Parameter(p.clone())
    opt = AdamW([q], state_bits=8)
    opt.param_groups[0]["betas"] = (0.95, 0.999)              # changed by a schedule
    q.grad = g
    with pytest.raises(ValueError, match="0.94"):
        opt.step()
    # one value per block holds the scale, the others' gradients are gone
    m.copy_(torch.linspace(1.0, 448.0, n, device="cuda"))
    g[::256] = 448.0
    m[::256] = 448.0
    for t in range(1, 601):
        adamw_step([p], [g], [m], [v], step=t, lr=0.0, betas=(0.94, 0.999), **kw)
    rest = torch.arange(n, device="cuda") % 256 != 0
    assert m.float()[rest].max() <= 8 * 2.0 ** -9 and (m.float()[::256] == 448).all()
    # the scale: blend's two constants, its products and their sum, code * scale, the scale's constant and product: at most 6 * 2^-24 a step
    assert ((kw["exp_avg_scales"][0] - 1).abs() <= 600 * 3 * 2.0 ** -23).all()
