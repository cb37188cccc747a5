"""Log-probabilities and both losses where max |z| / temperature is large: finite fills of any size among ordinary logits, rows that
are large throughout, temperatures down to the smallest that is accepted.

Tolerances, in half steps h = 2^-24 of fp32.  (z_a - max) / tau: temperature, its reciprocal or log2(e) / tau, the difference, the
product, the change of the logarithm's base (constant and product) and the two sums behind it: 8 h = 2^-21 of the log-probability.  The
logarithm of the sum: LP = 2.5e-6 as in test_token_losses.py, and as much again for the arguments of the exponentials, which have four
of these roundings instead of one (a term p 2^-d is off by d ln 2 2^-d times them, and d 2^-d is below 0.54).
A policy term is a product with exp(lp - old), where lp is above -50 or exp(lp - old) is below 2e-22: off by 50 * 2^-21 + 2 LP."""
import numpy as np
import pytest
import torch

from oracle import token_loss_oracle as O
from test_token_losses import LP, TYPES, _half_step, _np

REL, ABS = 2.0 ** -21, 2 * LP
RATIO = 50 * REL + ABS


def _close(got, want, off):
    got = _np(got)
    ok = (got == want) | (np.abs(got - want) <= off)
    assert ok.all(), (got[~ok][:4], np.asarray(want)[~ok][:4])


def _gradient_close(got, want, c, dtype, c_error):
    size = np.abs(np.broadcast_to(c, want.shape[:-1]))[..., None]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133 if dtype == torch.bfloat16 else 2.0 ** -149      # half steps of subnormal results
    _close(got, want, _half_step(dtype) * 1.01 * np.abs(want) + size * ABS + c_error * np.abs(c).max() + tiny)


def _check(z, targets, tau=1.0, both_losses=True):
    """Everything on logits z [S, T, V] against the float64 forms, gradients at sizes around 1 whatever the temperature."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    tau = float(np.float32(tau))
    S, T, V = z.shape
    g = torch.Generator().manual_seed(V)
    up, adv, noise = (torch.randn(S, T, generator=g) for _ in range(3))
    scale = min(tau, 1e37)       # gradients and losses times 3e38 would be infinite, an input of which nothing follows
    up = up * scale
    zc = z.cuda().requires_grad_(True)
    t = targets.cuda()
    lp, p, live = O.log_probs(_np(z), _np(targets), None, tau)
    assert np.isfinite(lp).all() and live.all()
    got = token_log_probs(zc, t, temperature=tau)
    _close(got, lp, ABS + REL * np.abs(lp))
    (gz,) = torch.autograd.grad(got, zc, up.cuda())
    _gradient_close(gz, O.logit_gradient(p, _np(targets), live, _np(up), tau), _np(up) / tau, z.dtype, REL)
    near = lp > -50
    old = torch.from_numpy(np.where(near, lp + 0.3 * _np(noise), 0.0)).float()
    for backward in (True, False):
        loss, want_lp, want, c = O.policy(_np(z), _np(targets), _np(adv), _np(old), tau=tau, scale=scale)
        with torch.set_grad_enabled(backward):
            got, got_lp = policy_loss(zc, t, adv.cuda(), old.cuda(), temperature=tau, scale=scale)
        _close(got_lp, want_lp, ABS + REL * np.abs(want_lp))
        sizes = O.policy(_np(z), _np(targets), np.abs(_np(adv)), _np(old), None, None, 0.999, 1e9, tau=tau, scale=scale)[0]
        # the clipped value of a ratio near zero is not among those sizes
        _close(got, loss, RATIO * (abs(sizes) + scale * float(adv.abs().mean())) + 2.0 ** -22 * abs(loss))
    loss, _ = policy_loss(zc, t, adv.cuda(), old.cuda(), temperature=tau, scale=scale)
    (gz,) = torch.autograd.grad(loss, zc, retain_graph=True)
    _gradient_close(gz, want, c / tau, z.dtype, RATIO)
    (again,) = torch.autograd.grad(loss * 2, zc)            # from the kept statistics
    _gradient_close(again, 2 * want, 2 * c / tau, z.dtype, RATIO)
    if tau == 1.0 and both_losses:
        mask = torch.from_numpy(near)
        loss, seq, want, c = O.preference(_np(z), _np(targets), None, _np(mask), 0.1)
        got, got_seq = preference_loss(zc, t, None, mask.cuda())
        off = T * ABS + REL * np.abs(np.where(near, lp, 0.0)).sum(-1).max()
        _close(got_seq, seq, off + 2.0 ** -24 * np.abs(seq))
        _close(got, loss, 2 * 0.1 * off + 2.0 ** -23 * abs(loss))
        (gz,) = torch.autograd.grad(got, zc)
        _gradient_close(gz, want, c[:, None], z.dtype, 2 * 0.1 * off + 2.0 ** -22)


FILLS = [-1e5, -3e7, -1e10, -1e12, -1e18, -1e20, -1e30]
SIZES = [40, 300, 4099, 9000, 20000, 70001]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", SIZES)
def test_large_finite_fills(V, dtype):
    """Banned tokens, a padded vocabulary, all but a few tokens: parts of a row, whole threads' shares among them, hold a large finite value."""
    g = torch.Generator().manual_seed(V)
    for fill in FILLS:
        z = 3 * torch.randn(2, 6, V, generator=g)
        at = torch.randint(0, V, (2, 6), generator=g)
        few = torch.rand(2, V, generator=g) < 5 / V
        few.scatter_(1, at[:, :1], True)
        z[:, 0] = torch.where(few, z[:, 0], fill)           # all but a few
        z[:, 1, :V // 2] = fill                             # the first half
        z[:, 2, V // 2:] = fill                             # the last half
        z[:, 3, (torch.arange(V) // 1024) % 2 == 0] = fill
        z[:, 4] = fill                                      # all: a uniform distribution
        z[:, 5] = fill                                      # all but one
        z[:, 5].scatter_(1, at[:, 5:6], 1.5)
        at[:, 1], at[:, 2] = V - 1 - at[:, 1] % (V // 4), at[:, 2] % (V // 4)
        _check(z.to(TYPES[dtype]), at)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("V", SIZES)
def test_rows_that_are_large_throughout(V, dtype):
    g = torch.Generator().manual_seed(V + 1)
    for top in (9e6, 1.3e7, 1.1e9, 5e9, -1.3e7, -1e10, 1e12, -1e15, 3e20, -1e30, 1e30):
        z = torch.zeros(2, 4, V)
        at = torch.randint(0, V, (2, 4), generator=g)
        z[:, 0] = top                                       # all alike
        z[:, 1].scatter_(1, at[:, 1:2], top)                # one among zeros: the target, then another token
        z[:, 2].scatter_(1, (at[:, 2:3] + 1) % V, top)
        z[:, 3] = top * (1 + torch.arange(V) % 7 * 1e-7)    # fp32: neighbours in the type, differences of a few units at 1e7
        _check(z.to(TYPES[dtype]), at, both_losses=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tau", [1e-3, 1e-4, 1e-5, 1e-6, 1e-7, 1e-9, 1e-10, 1e-12, 1e-20, 1e-30, 1e10, 1e38])
def test_temperatures(tau, dtype):
    """Ordinary logits over the whole accepted range; fp16 ones near the type's end, too."""
    for V in (40, 4099, 20001):
        g = torch.Generator().manual_seed(V + 2)
        z = 2.5 * torch.randn(2, 5, V, generator=g)
        at = torch.randint(0, V, (2, 5), generator=g)
        at[:, :3] = z[:, :3].argmax(-1)
        z[:, 1], z[:, 3, V // 2:] = 10.1, -60000.0
        z[:, 2].scatter_(1, at[:, 2:3], 60000.0)
        tau32 = float(np.float32(tau))
        z = z.to(TYPES[dtype])
        x = z.double() / tau32
        ok = (x.gather(-1, at[..., None])[..., 0] - x.amax(-1)).abs() < 1e38      # a log-probability that fp32 holds
        at = torch.where(ok, at, z.float().argmax(-1))
        _check(z, at, tau)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 4099, 70001])
def test_a_chosen_token_at_the_types_lowest_value(V, dtype):
    """Masked with the type's lowest value, or another one whose product with log2(e) leaves fp32, and chosen all the same: the
    log-probability is that value (temperature 1), infinite only where fp32 ends.  It must not turn a pair that holds it twice into NaN."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    dt = TYPES[dtype]
    lowest = torch.finfo(dt).min
    g = torch.Generator().manual_seed(V)
    z = 3 * torch.randn(2, 4, V, generator=g).to(dt)
    at = torch.randint(0, V, (2, 4), generator=g)
    fills = torch.tensor([[lowest, 0.75 * lowest, 0.0, lowest], [0.75 * lowest, lowest, 0.0, lowest]]).to(dt)
    z[:, [0, 1, 3]] = z[:, [0, 1, 3]].scatter(-1, at[:, [0, 1, 3], None], fills[:, [0, 1, 3], None])
    z[:, 3] = z[:, 3].scatter(-1, (at[:, 3:] + 1) % V, -lowest / 2)        # half the type's range above zero
    zc, t = z.cuda().requires_grad_(True), at.cuda()
    for tau in (1.0, 2.0, 0.5):
        lp, p, live = O.log_probs(_np(z), _np(at), None, tau)
        lp = np.where(lp < -float(np.finfo(np.float32).max) * (1 + 2.0 ** -24), -np.inf, lp)
        with np.errstate(invalid="ignore"):
            _close(token_log_probs(zc, t, temperature=tau), lp, ABS + REL * np.abs(lp))
        loss, got = policy_loss(zc, t, torch.ones(2, 4, device="cuda"), torch.zeros(2, 4, device="cuda"), temperature=tau)
        with np.errstate(invalid="ignore"):
            _close(got, lp, ABS + REL * np.abs(lp))
        assert loss.isfinite() and torch.autograd.grad(loss, zc)[0].isfinite().all()
    mask = torch.tensor([[True, False, True, False], [False, True, True, False]])
    _, want_seq, want, c = O.preference(_np(z), _np(at), None, _np(mask))
    loss, seq = preference_loss(zc, t, None, mask.cuda())
    _close(seq, want_seq, 3 * ABS + REL * np.abs(want_seq))
    (gz,) = torch.autograd.grad(loss, zc)
    assert loss.isfinite() and gz.isfinite().all()
    _gradient_close(gz, want, c[:, None], dt, 2.0 ** -22)        # |D| is above 1000: the slope is saturated


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_an_impossible_token_in_a_row_at_the_types_lowest_value(dtype):
    """-inf, whatever the temperature makes of the row's maximum; in a row of nothing but -inf NaN."""
    from star_rwkv6_b200.loss import policy_loss, token_log_probs
    z = torch.full((4, 333), torch.finfo(TYPES[dtype]).min, dtype=TYPES[dtype], device="cuda")
    z[:, 7] = float("-inf")
    z[1, 1], z[2, 9] = 3.0, torch.finfo(TYPES[dtype]).max
    z[3] = float("-inf")
    z.requires_grad_(True)
    t = torch.full((4,), 7, device="cuda")
    for tau in (1.0, 0.7, 1e-20, 1e-30, 7.0, 1e38):
        lp = token_log_probs(z, t, temperature=tau)
        assert lp[:3].isneginf().all() and lp[3].isnan()
        loss, again = policy_loss(z, t, torch.ones(4, device="cuda"), torch.zeros(4, device="cuda"), mask=lp.isneginf(), temperature=tau)
        assert again[:3].isneginf().all() and loss == 0 and not torch.autograd.grad(loss, z)[0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [40, 4099, 20001])
def test_both_ends_of_the_range_at_large_temperatures(V, dtype):
    """Values at both ends of the type's range are a few units apart at a temperature of 3e38: their difference is more than fp32 holds."""
    most = torch.finfo(TYPES[dtype]).max
    g = torch.Generator().manual_seed(V + 3)
    z = torch.where(torch.rand(2, 5, V, generator=g) < 0.5, most, -most)
    z[:, 1] = 3 * torch.randn(2, V, generator=g)
    z[:, 1, 3::7] = -most
    z[:, 2, 1:] = -most
    z[:, 2, 0] = most
    at = torch.randint(0, V, (2, 5), generator=g)
    for tau in (3e38, 1e38, 2e37):
        _check(z.to(TYPES[dtype]), at, tau)
