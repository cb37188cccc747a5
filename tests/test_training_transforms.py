"""Tensors that are not what their memory holds, or that carry more than a value: the losses and the optimizer step on lazily negated
ones (the bits of the negated copy), and on those with a forward-mode tangent (refused)."""
import types

import pytest
import torch

pytestmark = pytest.mark.gpu


def _lazily(x):
    """A tensor equal to x whose memory holds -x."""
    y = torch._neg_view(-x.detach())
    assert y.is_neg() and torch.equal(y, x)
    return y


def _inputs(V=301):
    g = torch.Generator(device="cuda").manual_seed(V)
    z = 2 * torch.randn(4, 5, V, generator=g, device="cuda")
    t = torch.randint(0, V, (4, 5), generator=g, device="cuda")
    adv, noise = (torch.randn(4, 5, generator=g, device="cuda") for _ in range(2))
    return z, t, adv, noise - 6, noise - 5.5, noise.sum(1)


@pytest.fixture(params=["native", "python"])
def path(request, monkeypatch):
    from star_rwkv6_b200 import loss, optim
    if request.param == "python":
        no = types.SimpleNamespace(**{n: lambda *a: None for n in ("token_log_probs", "policy_loss", "preference_loss", "adamw_step")})
        monkeypatch.setattr(loss, "_native", no)
        monkeypatch.setattr(optim, "_native", no)


def _losses(z, t, adv, old, ref, sums):
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    return [token_log_probs(z, t), *policy_loss(z, t, adv, old, ref_log_probs=ref, kl_coef=0.1), *preference_loss(z, t, sums)]


def test_lazily_negated_arguments_of_the_losses(path):
    given = list(_inputs())
    want = _losses(*given)
    for i in range(6):
        args = list(given)
        args[i] = _lazily(args[i])
        assert all(torch.equal(a, b) for a, b in zip(_losses(*args), want)), i
    for dtype in (torch.bfloat16, torch.float16):
        z = given[0].to(dtype)
        assert all(torch.equal(a, b) for a, b in zip(_losses(_lazily(z), *given[1:]), _losses(z, *given[1:])))


def test_gradients_of_lazily_negated_logits_and_lazily_negated_gradients(path):
    z, *rest = _inputs()
    x, y = (-z).requires_grad_(True), z.clone().requires_grad_(True)
    up = rest[1]
    for i in (0, 1, 3):
        a, b = _losses(torch._neg_view(x), *rest)[i], _losses(y, *rest)[i]
        up = rest[1] if i == 0 else torch.full((), 1.5, device="cuda")
        (ga,), (gb,) = torch.autograd.grad(a, x, up, retain_graph=True), torch.autograd.grad(b, y, up, retain_graph=True)
        assert torch.equal(ga, -gb) and gb.any()
        (gn,) = torch.autograd.grad(b, y, _lazily(up))
        assert torch.equal(gn, gb)


def _state():
    g = torch.Generator(device="cuda").manual_seed(7)
    return [torch.randn(700, generator=g, device="cuda") for _ in range(2)] + [torch.zeros(700, device="cuda") for _ in range(2)]


def test_lazily_negated_arguments_of_the_optimizer_step(path):
    from star_rwkv6_b200.optim import AdamW, adamw_step
    p, g, m, v = _state()
    p2, _, m2, v2 = _state()
    adamw_step([p], [g], [m], [v], step=1, lr=0.1)
    adamw_step([p2], [_lazily(g)], [m2], [v2], step=1, lr=0.1)
    assert all(torch.equal(a, b) for a, b in ((p, p2), (m, m2), (v, v2)))
    q, r = (torch.nn.Parameter(p.clone()) for _ in range(2))
    a, b = AdamW([q]), AdamW([r])
    q.grad, r.grad = g, _lazily(g)
    a.step()
    b.step()
    assert torch.equal(q, r)
    before = [x.clone() for x in (p, m, v)]
    for i in (0, 2, 3):
        lists = [[p], [g], [m], [v]]
        lists[i] = [torch._neg_view(lists[i][0])]
        with pytest.raises(ValueError, match="negated"):
            adamw_step(*lists, step=2)
    one, count = torch.ones((), device="cuda"), torch.ones((), dtype=torch.int64, device="cuda")
    for kw in (dict(step=2, lr=_lazily(one)), dict(step=_lazily(count)), dict(step=2, grad_scale=_lazily(one))):
        with pytest.raises(ValueError, match="negated"):
            adamw_step([p], [g], [m], [v], **kw)
    s = torch.ones(3, device="cuda")
    codes = [torch.zeros(700, device="cuda").to(torch.float8_e4m3fn) for _ in range(2)]
    with pytest.raises(ValueError, match="negated"):
        adamw_step([p], [g], codes[:1], codes[1:], exp_avg_scales=[_lazily(s)], exp_avg_sq_scales=[s], step=2)
    assert all(torch.equal(x, y) for x, y in zip((p, m, v), before))


def _dual(x):
    return torch.autograd.forward_ad.make_dual(x.detach(), torch.ones_like(x))


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_of_the_losses_are_refused(path, grad_mode):
    """Dual tensors do not require grad: their tangents must not be dropped on the path without a backward."""
    given = list(_inputs())
    want = _losses(*given)
    with torch.autograd.forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        for i in (0, 2, 3, 4, 5):
            args = list(given)
            args[i] = _dual(args[i])
            for f in (lambda: _losses(*args)[0], lambda: _losses(*args)[1], lambda: _losses(*args)[3]):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    f()
        assert all(torch.equal(a, b) for a, b in zip(_losses(*given), want))
    for f in (lambda x: torch.func.jvp(lambda z: _losses(z, *given[1:])[0], (x,), (x,)), lambda x: torch.func.vmap(lambda z: _losses(z, *given[1:])[0])(x[None])):
        with pytest.raises(RuntimeError):
            f(given[0])


def test_forward_mode_derivatives_of_the_gradients_are_refused(path):
    z, *rest = _inputs()
    z.requires_grad_(True)
    outs = _losses(z, *rest)
    with torch.autograd.forward_ad.dual_level():
        for i in (0, 1, 3):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(outs[i], z, _dual(torch.ones_like(outs[i])))


def test_forward_mode_derivatives_of_the_optimizer_step_are_refused(path):
    from star_rwkv6_b200.optim import adamw_step
    p, g, m, v = _state()
    before = [x.clone() for x in (p, m, v)]
    one = torch.ones((), device="cuda")
    with torch.autograd.forward_ad.dual_level():
        for i in range(4):
            lists = [[p], [g], [m], [v]]
            lists[i] = [_dual(lists[i][0])]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                adamw_step(*lists, step=1)
        for kw in (dict(lr=_dual(one)), dict(grad_scale=_dual(one))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                adamw_step([p], [g], [m], [v], step=1, **kw)
    assert all(torch.equal(x, y) for x, y in zip((p, m, v), before))


def test_the_next_token_loss_of_lazily_negated_tensors():
    from star_rwkv6_b200.loss import lm_loss
    z = torch.randn(4, 64, device="cuda").bfloat16()
    t = torch.arange(4, device="cuda")
    x, y = torch.neg(z).requires_grad_(True), z.clone().requires_grad_(True)
    a, b = lm_loss(torch._neg_view(x), t), lm_loss(y * 1, t)
    assert abs(a.item() - b.item()) <= 2 * 2.5e-6 + 2.0 ** -22 * b.item()        # two forms, each as in test_token_losses.py
    (ga,), (gb,) = torch.autograd.grad(a, x), torch.autograd.grad(b, y, _lazily(torch.full((), 1.0, device="cuda")))
    assert (ga.float() + gb.float()).abs().max() <= 2.0 ** -8 * gb.abs().max() and gb.any() and torch.equal(x, -z)
