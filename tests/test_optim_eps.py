"""eps below the smallest normal fp32 number would be zero in the step's reciprocal, and a value without any gradient so far 0 / 0."""
import pytest
import torch

BAD = (1e-38, 1e-45, 1e-300, -1e-8, float("nan"), float("inf"))


def test_refusals():
    from star_rwkv6_b200 import _lib as L
    from star_rwkv6_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(4))
    c = L.AdamWConfig()
    c.dtype, c.state_bits, c.step, c.lr, c.beta1, c.beta2 = L.BF16, 32, 1, 1e-3, 0.9, 0.99
    for eps in BAD:
        with pytest.raises(ValueError, match="eps"):
            AdamW([p], eps=eps)
        c.eps = eps
        assert L.lib.wkv6_adamw_step(c, 0, None, None) == -1 and b"eps" in L.lib.wkv6_last_error(), eps
    for eps in (0.0, 1.2e-38, 1e-8):
        AdamW([p], eps=eps)
        c.eps = eps
        assert L.lib.wkv6_adamw_step(c, 0, None, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_values_without_gradients(bits):
    from star_rwkv6_b200.optim import adamw_step
    p, g, v = torch.ones(600, device="cuda"), torch.zeros(600, device="cuda"), torch.zeros(600, device="cuda")
    m, more = v.clone(), {}
    if bits == 8:
        m, v = (x.to(torch.float8_e4m3fn) for x in (m, v))
        more = dict(exp_avg_scales=[torch.zeros(3, device="cuda")], exp_avg_sq_scales=[torch.zeros(3, device="cuda")])
    for eps in BAD:
        with pytest.raises(ValueError, match="eps"):
            adamw_step([p], [g], [m], [v], step=1, eps=eps, **more)
    g[3] = 1.0
    adamw_step([p], [g], [m], [v], step=1, lr=0.5, eps=1.2e-38, weight_decay=0.0, **more)
    assert p[3] != 1 and (p[torch.arange(600, device="cuda") != 3] == 1).all()
