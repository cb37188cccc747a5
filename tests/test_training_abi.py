"""Pointers that the C entries of the losses and the AdamW step turn down before anything is launched (the addresses are never read):
every array has to be aligned to its elements."""
import pytest

from star_rwkv6_b200 import _lib as L

A = 0x1000
INVALID = -1


def _rows(**kw):
    p = L.TokenLogits()
    p.S, p.T, p.V, p.dtype, p.temperature, p.logits, p.targets = 2, 3, 8, L.BF16, 1.0, A, A
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _log_probs(lp=A, stat=None, **kw):
    return L.lib.wkv6_token_log_probs(_rows(**kw), lp, stat, None)


def _gradient(stat=A, coefficient=A, factor=A, g=A, **kw):
    return L.lib.wkv6_token_log_probs_backward(_rows(**kw), stat, coefficient, 0, factor, 0, g, None)


def _policy(loss=A, lp=A, stat=A, coefficient=A, g=A, workspace=A, targets=A, **kw):
    c = L.Policy()
    c.advantages = c.old_log_probs = c.ref_log_probs = A
    c.kl_coef = c.scale = 1.0
    for k, v in kw.items():
        setattr(c, k, v)
    return L.lib.wkv6_policy_loss(_rows(targets=targets), c, loss, lp, stat, coefficient, g, workspace, 1 << 20, None)


def _preference(lp=A, loss=A, seq=A, coefficient=A, workspace=A, ref=A, targets=A):
    q = L.Preference()
    q.ref_log_probs, q.beta, q.scale = ref, 1.0, 1.0
    return L.lib.wkv6_preference_loss(_rows(targets=targets), lp, q, loss, seq, coefficient, workspace, 1 << 20, None)


def _adamw(**kw):
    c, t = L.AdamWConfig(), (L.AdamWTensor * 1)()
    c.dtype, c.state_bits, c.step, c.lr, c.beta1, c.beta2, c.eps = L.BF16, 32, 1, 1e-3, 0.9, 0.99, 1e-8
    t[0].p = t[0].g = t[0].m = t[0].v = A
    t[0].n = 8
    for k, v in kw.items():
        setattr(c, k, v)
    return L.lib.wkv6_adamw_step(c, 1, t, None)


@pytest.mark.parametrize("call,names", [
    (_log_probs, dict(targets=4, lp=2, stat=4)), (_gradient, dict(targets=4, stat=4, coefficient=2, factor=1, g=8)),
    (_policy, dict(targets=4, loss=2, lp=2, stat=4, coefficient=2, g=8, workspace=8, advantages=2, old_log_probs=1, ref_log_probs=2)),
    (_preference, dict(targets=2, lp=1, loss=2, seq=2, coefficient=2, workspace=4, ref=2)), (_adamw, dict(step_device=4, lr_device=2, grad_scale=2))])
def test_misaligned_pointers(call, names):
    for name, off in names.items():
        assert call(**{name: A + off}) == INVALID, name
        assert b"align" in L.lib.wkv6_last_error(), name
