"""The operators behind the logits and in front of the weights as a training program runs them one after the other: a reference
model's log-probabilities, policy updates and a preference update of a bf16 model, each followed by an AdamW step.  Every link is held to
its float64 form on what the link before it really gave (tolerances: tests/test_token_losses.py and tests/test_optim.py)."""
import numpy as np
import pytest
import torch

from oracle import adamw_oracle as A
from oracle import token_loss_oracle as O
from test_optim import _flat, _oracle, _check
from test_token_losses import LP, _check_gradient, _check_lp, _np

pytestmark = pytest.mark.gpu


def _model(layers=2, D=128, vocab=331):
    from star_rwkv6_b200.model import RWKV6
    torch.manual_seed(3)
    with torch.device("cuda"):
        return RWKV6(layers, vocab, D, decomposer_size=32, expand_size=3 * D, decay_rank=64).to_bf16_()


def _states(opt, ps, bits):
    l = dict(p=[p.detach().clone() for p in ps], g=[p.grad.clone() for p in ps], m=[], v=[], ms=[], vs=[])
    for p in ps:
        s = opt.state[p]
        for key, name in (("m", "exp_avg"), ("v", "exp_avg_sq")):
            l[key].append(s[name].detach().clone() if s else torch.zeros(p.shape, dtype=torch.float32 if bits == 32 else torch.float8_e4m3fn, device="cuda"))
            if bits == 8:
                l[key + "s"].append(s[name + "_scale"].clone() if s else torch.zeros(-(-p.numel() // A.BLOCK), device="cuda"))
    return l


@pytest.mark.parametrize("bits", [32, 8])
def test_policy_and_preference_updates(bits):
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    from star_rwkv6_b200.optim import AdamW
    S, T, vocab = 4, 37, 331
    model, reference = _model(), _model()
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.randint(0, vocab, (S, T + 1), generator=g, device="cuda")
    targets = tokens[:, 1:]                                    # a view: rows of T + 1
    mask = torch.zeros(S, T, dtype=torch.bool, device="cuda")
    for s in range(S):
        mask[s, 5 + s:T - 3 * s] = True
    adv = torch.randn(S, 1, generator=g, device="cuda").expand(S, T)
    with torch.no_grad():
        ref = token_log_probs(reference(tokens[:, :-1]), targets, mask)
        old = token_log_probs(model(tokens[:, :-1]), targets, mask)
        assert torch.equal(ref, old)                           # the same weights
        old = old + 0.2 * torch.randn(S, T, generator=g, device="cuda")
    ps = [p for p in model.parameters()]
    opt = AdamW(ps, lr=2e-3, weight_decay=0.05, state_bits=bits, seed=9)
    hyper = dict(lr=2e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)
    for step in range(1, 4):
        logits = model(tokens[:, :-1])
        logits.retain_grad()
        z, t, m = _np(logits), _np(targets), _np(mask)
        if step < 3:
            loss, lp = policy_loss(logits, targets, adv, old, ref_log_probs=ref, mask=mask, kl_coef=0.05, reduction="sequence_mean")
            want, want_lp, want_g, c = O.policy(z, t, _np(adv), _np(old), _np(ref), m, kl=0.05, reduction="sequence_mean")
            _check_lp(lp, want_lp)
            off = 2 * LP
        else:
            sums = ref.sum(-1)
            loss, seq = preference_loss(logits, targets, sums, mask)
            want, want_seq, want_g, c = O.preference(z, t, _np(sums), m)
            assert (np.abs(_np(seq) - want_seq) <= T * LP + 2.0 ** -22 * np.abs(want_seq)).all()
            c = c[:, None]
            off = 2 * 0.1 * (T * LP + 2.0 ** -23 * np.abs(want_seq).max()) * 2 + 2.0 ** -22
        assert abs(loss.item() - want) <= 1e-4 * max(abs(want), 1.0)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        _check_gradient(logits.grad, want_g, c, torch.bfloat16, off)
        l = _states(opt, ps, bits)
        forms = [_oracle(l, i, bits, step, 9, hyper) for i in range(len(ps))]
        opt.step()
        new = _states(opt, ps, bits)
        for i, (numbers, random, sizes) in enumerate(forms):
            _check(new, i, bits, True, numbers, random, sizes)
    assert all(torch.equal(a, b) for a, b in zip(reference.parameters(), _model().parameters()))
    assert {p.dtype for p in ps} == {torch.bfloat16, torch.float32} and _flat(ps[0]).size == vocab * 128
