"""Log-probabilities of given tokens, the clipped policy loss and the preference loss against their float64 forms.

Tolerances.  A log-probability is (z_a - c) / tau - log s in fp32.  s: each term has the error of the exponential (2^-22) and of
its argument's rounding (2^-24 |d|, |d| <= 16 log2 units where a term matters: 11 * 2^-24), and the sum's order adds up to
2^-20 over the chains of a few hundred terms here; the logarithm (at most 12) is off by one unit of its last place, 2^-21:
2.4e-6 in all, and 2^-22 of the result for the two subtractions.  LP = 2.5e-6 below.
A gradient c (1 - p) is off by the relative errors of p (the same 2.5e-6) and of c, and rounded once to its type.
"""
import numpy as np
import pytest
import torch

from oracle import token_loss_oracle as O

LP = 2.5e-6
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _inputs(S, T, V, dtype, seed=0, masked=True):
    g = torch.Generator().manual_seed(seed + 1000 * S + 10 * T + V)
    z = torch.randn(S, T, V, generator=g) * 3
    targets = torch.randint(0, V, (S, T), generator=g)
    z.scatter_add_(-1, targets[..., None], 3 * torch.rand(S, T, 1, generator=g))
    mask = torch.rand(S, T, generator=g) < 0.7 if masked else None
    return z.to(dtype), targets, mask, g


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def _check_lp(got, want):
    got, want = _np(got), np.asarray(want)
    assert got.shape == want.shape
    assert (np.abs(got - want) <= LP + np.abs(want) * 2.0 ** -22).all()


def _check_gradient(got, want, c, dtype, c_error):
    """c: coefficients [S, T] (or broadcast); c_error: relative to the largest coefficient."""
    size = np.abs(np.broadcast_to(c, want.shape[:-1]))[..., None]
    tol = _half_step(dtype) * 1.01 * np.abs(want) + size * LP + c_error * np.abs(c).max() + (2.0 ** -25 if dtype == torch.float16 else 0.0)
    assert got.dtype == dtype and got.shape == want.shape
    assert (np.abs(_np(got) - want) <= tol).all(), np.abs(_np(got) - want).max()


SIZES = [(1, 1, 1), (1, 1, 8), (2, 3, 7), (3, 5, 259), (2, 7, 2048), (1, 5, 2049), (2, 3, 4099), (1, 3, 65536), (2, 2, 50277)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("S,T,V", SIZES)
def test_token_log_probs(S, T, V, dtype):
    from star_rwkv6_b200.loss import token_log_probs
    z, targets, mask, g = _inputs(S, T, V, TYPES[dtype])
    up = torch.randn(S, T, generator=g)
    for m, tau in ((None, 1.0), (mask, 0.7)):
        lp, p, live = O.log_probs(_np(z), _np(targets), _np(m), tau)
        want = O.logit_gradient(p, _np(targets), live, _np(up), tau)
        zc = z.cuda().requires_grad_(True)
        mc = None if m is None else m.cuda()
        with torch.no_grad():
            alone = token_log_probs(zc, targets.cuda(), mc, temperature=tau)
        got = token_log_probs(zc, targets.cuda(), mc, temperature=tau)
        assert torch.equal(alone, got) and got.dtype == torch.float32
        _check_lp(got, lp)
        (gz,) = torch.autograd.grad(got, zc, up.cuda())
        _check_gradient(gz, want, _np(up) / tau, z.dtype, 2.0 ** -22)


@pytest.mark.gpu
@pytest.mark.parametrize("reduction", ["mean", "sequence_mean", "sum"])
@pytest.mark.parametrize("S,T,V,dtype,kl,tau", [(1, 1, 17, "f32", 0.0, 1.0), (3, 5, 259, "bf16", 0.1, 1.0), (2, 600, 100, "f32", 0.05, 0.8),
                                                (2, 9, 4099, "f16", 0.0, 1.3), (4, 3, 65536, "bf16", 0.04, 1.0), (5, 700, 9, "bf16", 0.0, 1.0)])
def test_policy_loss(S, T, V, dtype, kl, tau, reduction):
    from star_rwkv6_b200.loss import policy_loss
    z, targets, mask, g = _inputs(S, T, V, TYPES[dtype], seed=3)
    mask[0] = False                                         # an answer of which nothing counts
    if S > 1:
        mask[-1] = True
    lp, _, _ = O.log_probs(_np(z), _np(targets), None, tau)
    old = (torch.from_numpy(lp) + 0.3 * torch.randn(S, T, generator=g)).float()
    ref = (torch.from_numpy(lp) + 0.5 * torch.randn(S, T, generator=g)).float()
    adv = torch.randn(S, 1, generator=g).expand(S, T)       # broadcast, as a whole answer's advantage is
    scale = 64.0 if dtype == "f16" else 1.0
    loss, want_lp, want, c = O.policy(_np(z), _np(targets), _np(adv), _np(old), _np(ref), _np(mask), 0.2, 0.3, kl, tau, reduction, scale)
    zc = z.cuda().requires_grad_(True)
    args = (targets.cuda(), adv.cuda(), old.cuda())
    kw = dict(ref_log_probs=ref.cuda(), mask=mask.cuda(), clip_high=0.3, kl_coef=kl, temperature=tau, reduction=reduction, scale=scale)
    got, got_lp = policy_loss(zc, *args, **kw)
    _check_lp(got_lp, want_lp)
    assert not got_lp.requires_grad
    # every term is a product with exp(lp - old): its relative error is that of lp, and the terms' sizes add up
    sizes = O.policy(_np(z), _np(targets), np.abs(_np(adv)) + kl, _np(old), None, _np(mask), 0.999, 1e9, 0.0, tau, reduction, scale)[0]
    assert abs(got.item() - loss) <= 8 * LP * (abs(sizes) + kl * scale) + 2.0 ** -24 * abs(loss)
    (gz,) = torch.autograd.grad(got, zc, retain_graph=True)
    _check_gradient(gz, want, c / tau, z.dtype, 2 * LP)
    # another factor, and a second backward: the gradient is formed again, the one handed out stays
    kept = gz.clone()
    (third,) = torch.autograd.grad(got * 3, zc, retain_graph=True)
    _check_gradient(third, 3 * want, 3 * c / tau, z.dtype, 2 * LP)
    (again,) = torch.autograd.grad(got, zc)
    assert torch.equal(gz, kept) and torch.equal(again, kept) and again.data_ptr() != gz.data_ptr()
    (first_other,) = torch.autograd.grad(policy_loss(zc, *args, **kw)[0] * 3, zc)
    assert torch.equal(first_other, third)
    with torch.no_grad():
        plain = policy_loss(zc, *args, **kw)
    assert torch.equal(plain[0], got) and torch.equal(plain[1], got_lp)
    wide = torch.zeros(T, 2 * S, device="cuda").t()[::2]     # advantages with strides of their own, of another type
    wide.copy_(args[1])
    for a in (args[1].contiguous(), wide, args[1].double()):
        assert torch.equal(policy_loss(zc, args[0], a, args[2], **kw)[0], got)


@pytest.mark.gpu
@pytest.mark.parametrize("P,T,V,dtype,smoothing,average,reference,margin", [
    (1, 1, 5, "f32", 0.0, False, True, 0.0), (3, 7, 259, "bf16", 0.1, True, False, 0.5), (2, 300, 1000, "f32", 0.2, False, True, 0.0),
    (2, 3, 65536, "bf16", 0.0, False, True, 0.0), (300, 2, 9, "f16", 0.0, True, True, 0.0), (2, 1031, 40, "f32", 0.0, False, True, 0.1),
    (16, 300, 33, "bf16", 0.05, True, True, 0.0)])
def test_preference_loss(P, T, V, dtype, smoothing, average, reference, margin):
    from star_rwkv6_b200.loss import preference_loss
    z, targets, mask, g = _inputs(2 * P, T, V, TYPES[dtype], seed=4)
    mask[P] = False                                         # an empty answer
    beta = 1.0 if average else 0.1
    _, seq, _, _ = O.preference(_np(z), _np(targets), None, _np(mask), beta, 0.0, 0.0, average)
    ref = (torch.from_numpy(seq) + torch.randn(2 * P, generator=g)).float() if reference else None
    scale = 128.0 if dtype == "f16" else 1.0
    loss, want_seq, want, c = O.preference(_np(z), _np(targets), _np(ref), _np(mask), beta, smoothing, margin, average, scale)
    zc = z.cuda().requires_grad_(True)
    kw = dict(beta=beta, label_smoothing=smoothing, margin=margin, average=average, scale=scale)
    got, got_seq = preference_loss(zc, targets.cuda(), None if ref is None else ref.cuda(), mask.cuda(), **kw)
    # a sum of up to T log-probabilities, each off by at most LP
    off = T * LP if not average else LP
    assert (np.abs(_np(got_seq) - want_seq) <= off + 2.0 ** -22 * np.abs(want_seq)).all() and not got_seq.requires_grad
    d_off = 2 * beta * (off + 2.0 ** -23 * np.abs(want_seq).max())        # of a margin; |d loss / d D| <= 1, of the slope <= beta / 4
    assert abs(got.item() - loss) <= scale * d_off + 2.0 ** -23 * abs(loss)
    (gz,) = torch.autograd.grad(got, zc, retain_graph=True)
    _check_gradient(gz, want, c[:, None], z.dtype, 2 * d_off * beta * scale / P / max(np.abs(c).max(), 1e-30) + 2.0 ** -22)
    (twice,) = torch.autograd.grad(got * 0.5, zc)
    _check_gradient(twice, 0.5 * want, 0.5 * c[:, None], z.dtype, 2 * d_off * beta * scale / P / max(np.abs(c).max(), 1e-30) + 2.0 ** -22)
    with torch.no_grad():
        assert torch.equal(preference_loss(zc, targets.cuda(), None if ref is None else ref.cuda(), mask.cuda(), **kw)[0], got)


def test_gradients_against_differences():
    """The float64 forms' gradients against central differences of their losses, step 1e-5: the third derivative leaves 1e-9."""
    z, targets, mask, g = _inputs(4, 3, 11, torch.float32, seed=9)
    z, targets, mask = _np(z), _np(targets), _np(mask)
    lp, _, _ = O.log_probs(z, targets, None, 0.9)
    noise = torch.randn(3, 4, 3, generator=g).double().numpy()
    old, ref, adv = lp + 0.3 * noise[0], lp + 0.3 * noise[1], noise[2]
    forms = [lambda x: O.policy(x, targets, adv, old, ref, mask, 0.2, 0.2, 0.1, 0.9, r) for r in ("mean", "sequence_mean", "sum")]
    forms += [lambda x, a=a: O.preference(x, targets, None, mask, 0.3, 0.1, 0.2, a) for a in (False, True)]
    for f in forms:
        grad = f(z)[2]
        for at in ((0, 0, targets[0, 0]), (1, 2, 3), (2, 1, targets[2, 1]), (3, 0, 10), (3, 2, 0)):
            up, down = z.copy(), z.copy()
            up[at] += 1e-5
            down[at] -= 1e-5
            assert abs((f(up)[0] - f(down)[0]) / 2e-5 - grad[at]) <= 1e-7


@pytest.mark.gpu
@pytest.mark.parametrize("V", [300, 9000])
def test_rows_that_do_not_count_are_not_read(V):
    """NaN, infinities and the type's ends in masked rows and behind foreign targets; -inf and the lowest value among the logits."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    z, targets, _, _ = _inputs(2, 6, V, torch.bfloat16, seed=5)
    mask = torch.ones(2, 6, dtype=torch.bool)
    lowest = torch.finfo(torch.bfloat16).min
    z[0, 0], z[0, 1], z[0, 2] = float("nan"), float("inf"), float("-inf")
    mask[0, 0] = mask[0, 1] = mask[0, 2] = False
    z[0, 3], targets[0, 3] = float("nan"), -100
    z[0, 4], targets[0, 4] = float("nan"), V
    z[0, 5, 1:] = float("-inf")                     # one token is possible
    targets[0, 5] = 0
    z[1, 0] = lowest                                # all alike, at the type's end
    z[1, 1], z[1, 1, 3], targets[1, 1] = lowest, -lowest, 3
    z[1, 2, :V // 2], targets[1, 2] = float("-inf"), V - 1
    z[1, 3, 1], targets[1, 3] = float("-inf"), 1    # an impossible token was chosen
    zc = z.cuda().requires_grad_(True)
    with np.errstate(invalid="ignore", divide="ignore"):
        want, p, live = O.log_probs(_np(z), _np(targets), _np(mask))
        grad = O.logit_gradient(p, _np(targets), live, np.ones((2, 6)))
    assert list(live[0]) == [False] * 5 + [True] and live[1].all()
    lp = token_log_probs(zc, targets.cuda(), mask.cuda())
    ok = np.isfinite(want)
    assert np.array_equal(_np(lp)[~ok], want[~ok]) and not ok[1, 3] and ok.sum() == 11
    assert (np.abs(_np(lp)[ok] - want[ok]) <= LP + 2.0 ** -22 * np.abs(want[ok])).all()
    (g,) = torch.autograd.grad(lp, zc, torch.ones_like(lp))
    _check_gradient(g, grad, np.ones((2, 6)), torch.bfloat16, 2.0 ** -22)
    old = torch.zeros(2, 6, device="cuda")
    loss, _ = policy_loss(zc, targets.cuda(), torch.ones(2, 6, device="cuda"), old, mask=mask.cuda())
    (g,) = torch.autograd.grad(loss, zc)
    assert loss.isfinite() and g.isfinite().all() and not g[0, :5].any() and g[1, 4].any()
    everything = torch.zeros(2, 6, dtype=torch.bool, device="cuda")
    for f in (lambda m: policy_loss(zc, targets.cuda(), old + 1, old, mask=m)[0], lambda m: preference_loss(zc, targets.cuda(), None, m)[0]):
        loss = f(everything)
        (g,) = torch.autograd.grad(loss, zc)
        assert loss.isfinite() and not g.any()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [9, 300, 3000, 9000, 20000, 70001])
def test_one_possible_token(V):
    """All logits but one are -inf or the lowest value, wherever that one lies: its log-probability is 0, the others' gradient zero."""
    from star_rwkv6_b200.loss import policy_loss, token_log_probs
    at = sorted({0, 1, V // 3, V - 2, V - 1})
    for none in (float("-inf"), torch.finfo(torch.bfloat16).min):
        for tau in (0.3, 1.0, 7.0):
            z = torch.full((1, len(at), V), none, device="cuda", dtype=torch.bfloat16)
            t = torch.tensor([at], device="cuda")
            z.scatter_(-1, t[..., None], 1.5)
            z.requires_grad_(True)
            one = torch.ones(1, len(at), device="cuda")
            lp = token_log_probs(z, t, temperature=tau)
            loss, again = policy_loss(z, t, one, 0 * one, temperature=tau)
            assert (lp.abs() <= LP).all() and (again.abs() <= LP).all() and not (lp > 0).any() and abs(loss.item() + 1) <= 4 * LP
            g, h = torch.autograd.grad(lp, z, one)[0], torch.autograd.grad(loss, z)[0]
            assert g.abs().max() <= LP / tau and h.abs().max() <= LP / tau


@pytest.mark.gpu
def test_rows_without_a_distribution_give_nan():
    from star_rwkv6_b200.loss import policy_loss, token_log_probs
    for V in (40, 5000):
        z = torch.randn(1, 4, V, device="cuda")
        z[0, 0, 3], z[0, 1, 3], z[0, 2] = float("nan"), float("inf"), float("-inf")
        z.requires_grad_(True)
        t = torch.ones(1, 4, dtype=torch.int64, device="cuda")
        lp = token_log_probs(z, t)
        assert lp[0, :3].isnan().all() and lp[0, 3].isfinite()
        (g,) = torch.autograd.grad(lp, z, torch.ones_like(lp))
        assert g[0, :3].isnan().all() and g[0, 3].isfinite().all()
        loss, _ = policy_loss(z, t, torch.ones_like(lp), torch.zeros_like(lp), reduction="sum")
        assert loss.isnan()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts(dtype):
    """Views whose rows start anywhere against dense copies.  A row that starts elsewhere is summed up in another order: both results
    are within LP + 2^-22 of the true log-probability, the policy loss (one term, exp(lp + 5), per token) within 2 LP per term of
    its size, and the gradients within those shares and a rounding each."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    dt = TYPES[dtype]
    base = torch.randn(4, 9, 5100, device="cuda").to(dt)
    t = torch.randint(0, 500, (4, 9), device="cuda")
    views = [base[:, :-1, 3:4003], base[:, 1:, :501], base[::2, ::2, 7:907], base.transpose(0, 1)[:, :, 1:600], base[:1, :1, 5:].expand(4, 3, -1),
             base.permute(0, 2, 1)[:, :7, :], base[0], base[0, 0], base[:, None, :, 1:2001]]
    for z in views:
        z = z.detach().requires_grad_(True)
        shape = z.shape[:-1]
        targets = t.flatten()[:shape.numel()].reshape(shape) % z.shape[-1]
        dense = z.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True)
        a, b = token_log_probs(z, targets), token_log_probs(dense, targets)
        assert ((a - b).abs() <= 2 * (LP + 2.0 ** -22 * b.abs())).all()

        def close(ga, gb, size):
            ga, gb = ga.double(), gb.double()
            off = 2 * _half_step(dt) * torch.maximum(ga.abs(), gb.abs()) + 4 * LP * size + (2.0 ** -24 if dt == torch.float16 else 0.0)
            assert ((ga - gb).abs() <= off).all()

        close(*(torch.autograd.grad(x, y, torch.ones_like(x))[0] for x, y in ((a, z), (b, dense))), 1.0)
        old = torch.zeros(shape, device="cuda") - 5
        la, lb = (policy_loss(x, targets, old + 4, old, clip_low=1.0, clip_high=1e9)[0] for x in (z, dense))
        assert (la - lb).abs() <= 8 * LP * la.abs()
        close(*(torch.autograd.grad(l, x)[0] for l, x in ((la, z), (lb, dense))), float((b.detach() + 5).exp().max()) / b.numel())
        if z.dim() == 3 and shape[0] % 2 == 0:
            la, lb = (preference_loss(x, targets)[0] for x in (z, dense))
            off = 0.1 * 4 * shape[1] * (LP + 2.0 ** -22 * float(b.detach().abs().max()))       # of a margin D, and more than of the slope
            assert (la - lb).abs() <= off + 2.0 ** -22
            close(*(torch.autograd.grad(l, x)[0] for l, x in ((la, z), (lb, dense))), 0.1 * (1 + off / LP))


@pytest.mark.gpu
def test_no_tokens():
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    for shape in ((0, 5), (3, 0), (0,)):
        z = torch.randn(*shape, 11, device="cuda", requires_grad=True)
        t, x = torch.zeros(shape, dtype=torch.int64, device="cuda"), torch.zeros(shape, device="cuda")
        lp = token_log_probs(z, t)
        assert lp.shape == shape and torch.autograd.grad(lp, z, x)[0].shape == z.shape
        loss, _ = policy_loss(z, t, x, x)
        assert loss.item() == 0.0 and torch.autograd.grad(loss, z)[0].shape == z.shape
    for S in (0, 4):
        z = torch.randn(S, 0, 11, device="cuda", requires_grad=True)
        loss, seq = preference_loss(z, torch.zeros(S, 0, dtype=torch.int64, device="cuda"))
        assert abs(loss.item() - (np.log(2.0) if S else 0.0)) <= 1e-7 and seq.shape == (S,) and not seq.any()
        assert torch.autograd.grad(loss, z)[0].shape == z.shape


@pytest.mark.gpu
def test_offsets_beyond_32_bits():
    """Rows behind the first 2^31 elements, forward and backward (an 8.6 GB view, two rows of which are looked at)."""
    from star_rwkv6_b200.loss import policy_loss
    V, rows = 65536, 32768 + 2
    base = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    base[-2:] = torch.randn(2, V, device="cuda").to(torch.bfloat16) * 3
    t = torch.full((rows,), 7, dtype=torch.int64, device="cuda")
    mask = torch.zeros(rows, dtype=torch.bool, device="cuda")
    mask[-2:] = True
    z = base.requires_grad_(True)
    one = torch.ones(rows, device="cuda")
    loss, lp = policy_loss(z, t, one, -10 * one, mask=mask, clip_high=1e9)
    (g,) = torch.autograd.grad(loss, z)
    small = base.detach()[-2:].clone().requires_grad_(True)
    want, want_lp = policy_loss(small, t[-2:], one[-2:], -10 * one[-2:], clip_high=1e9)
    assert torch.equal(loss, want) and torch.equal(lp[-2:], want_lp)
    assert torch.equal(g[-2:], torch.autograd.grad(want, small)[0])
    assert not lp[:-2].any() and g[:-2].abs().max().item() == 0


@pytest.mark.gpu
def test_captured_and_on_other_streams():
    """Forward and backward in a CUDA graph, replayed on new logits; two graphs; a call on a side stream."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss
    S, T, V = 4, 5, 3000
    z, targets, mask, _ = _inputs(S, T, V, torch.bfloat16, seed=6)
    targets, mask = targets.cuda(), mask.cuda()
    old, adv = torch.full((S, T), -7.0, device="cuda"), torch.randn(S, T, device="cuda")
    static = z.cuda().requires_grad_(True)

    def both():
        a, _ = policy_loss(static, targets, adv, old, mask=mask)
        b, _ = preference_loss(static, targets, None, mask)
        return a, torch.autograd.grad(a * 2, static)[0], b, torch.autograd.grad(b, static)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            both()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(both())
        graphs.append(graph)
    for k in range(3):
        with torch.no_grad():
            static.copy_(z.cuda() * (1 + k))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = both()
        for out in outs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))
    torch.cuda.synchronize()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(out, want))


@pytest.mark.gpu
def test_two_calls_at_once():
    """Calls on two streams with nothing between them: each has its own workspace."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss
    sets, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for k in range(2):
        z, targets, mask, g = _inputs(6, 150, 2000 + 3000 * k, torch.bfloat16, seed=20 + k)
        adv, old = torch.randn(6, 150, generator=g), torch.full((6, 150), -6.0)
        sets.append([t.cuda() for t in (z, targets, mask, adv, old)])

    def both(z, targets, mask, adv, old):
        z = z.detach().requires_grad_(True)
        a, lp = policy_loss(z, targets, adv, old, mask=mask)
        b, seq = preference_loss(z, targets, None, mask)
        return a.detach(), lp, torch.autograd.grad(a, z)[0], b.detach(), seq, torch.autograd.grad(b, z)[0]

    want = [both(*s) for s in sets]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, stream in zip(sets, streams):
            with torch.cuda.stream(stream):
                got.append(both(*s))
    torch.cuda.synchronize()
    for i, out in enumerate(got):
        assert all(torch.equal(x, y) for x, y in zip(out, want[i % 2]))


def _outputs_of_one_run():
    """What the native and the Python call path are compared on."""
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    from star_rwkv6_b200.optim import AdamW
    out = []
    for V, dtype in ((50, torch.float32), (1001, torch.bfloat16), (9000, torch.float16)):
        z, targets, mask, g = _inputs(4, 6, V, dtype, seed=30)
        z, targets, mask = z.cuda().requires_grad_(True), targets.cuda(), mask.cuda()
        adv, old = torch.randn(4, 1, generator=g).cuda().expand(4, 6), torch.full((4, 6), -5.0, device="cuda")
        lp = token_log_probs(z, targets, mask, temperature=0.9)
        a, alp = policy_loss(z, targets, adv, old, ref_log_probs=old + 0.5, mask=mask, kl_coef=0.1, reduction="sequence_mean")
        b, seq = preference_loss(z, targets, None, mask, average=True, margin=0.1)
        out += [lp, alp, seq, a, b] + [torch.autograd.grad(x, z)[0] for x in (lp.sum(), a, b * 2)]
    for bits in (32, 8):
        torch.manual_seed(0)
        ps = [torch.nn.Parameter(torch.randn(n, device="cuda").to(dt)) for n, dt in ((700, torch.bfloat16), (33, torch.float32), (4096, torch.bfloat16))]
        opt = AdamW(ps, state_bits=bits, seed=3)
        for _ in range(3):
            for p in ps:
                p.grad = torch.randn_like(p)
            opt.step()
        out += ps + [t.float() for s in opt.state.values() for t in s.values() if torch.is_tensor(t)]
    return [t.detach().cpu() for t in out]


@pytest.mark.gpu
def test_both_call_paths_give_the_same_bits(tmp_path):
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = ("import sys, warnings; warnings.simplefilter('ignore'); sys.modules['star_rwkv6_b200._native'] = None\n"
            f"sys.path[:0] = [{os.path.dirname(here)!r}, {here!r}]\nimport torch, test_token_losses as t\n"
            f"torch.save(t._outputs_of_one_run(), {str(tmp_path / 'out.pt')!r})")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    python, native = torch.load(tmp_path / "out.pt"), _outputs_of_one_run()
    assert len(python) == len(native) and all(torch.equal(a, b) for a, b in zip(python, native))


@pytest.mark.gpu
def test_derivatives_of_the_gradients_are_refused():
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    z = torch.randn(2, 3, 50, device="cuda", requires_grad=True)
    t, x = torch.ones(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda")
    for f in (lambda: token_log_probs(z, t).sum(), lambda: policy_loss(z, t, x + 1, x - 9)[0], lambda: preference_loss(z, t)[0]):
        with pytest.raises(RuntimeError):
            (g,) = torch.autograd.grad(f(), z, create_graph=True)
            torch.autograd.grad(g.square().sum(), z)


@pytest.mark.gpu
def test_logits_changed_before_the_backward_are_refused():
    from star_rwkv6_b200.loss import policy_loss
    leaf = torch.randn(2, 3, 50, device="cuda", requires_grad=True)
    z = leaf * 1
    t, x = torch.ones(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda")
    loss, _ = policy_loss(z, t, x + 1, x - 9)
    z.detach().add_(1)
    z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_cpu_tensors_are_refused():
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    z, t, x = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)
    for f in (lambda: token_log_probs(z, t), lambda: policy_loss(z, t, x, x), lambda: preference_loss(z, t)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            f()


@pytest.mark.gpu
def test_refusals():
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    z, t = torch.zeros(2, 3, 5, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    x, m = torch.zeros(2, 3, device="cuda"), torch.ones(2, 3, dtype=torch.bool, device="cuda")
    bad = [(TypeError, lambda: token_log_probs(z.double(), t)), (TypeError, lambda: token_log_probs(z, t.int())),
           (ValueError, lambda: token_log_probs(z, t[:, :2])), (ValueError, lambda: token_log_probs(z[..., :0], t)),
           (TypeError, lambda: token_log_probs(z, t, m.int())), (ValueError, lambda: token_log_probs(z, t, m[:1])),
           (ValueError, lambda: token_log_probs(z, t, temperature=0.0)), (ValueError, lambda: token_log_probs(z, t, temperature=1e-40)), (ValueError, lambda: token_log_probs(z, t, temperature=float("nan"))),
           (RuntimeError, lambda: token_log_probs(z, t.cpu())), (RuntimeError, lambda: policy_loss(z, t, x.cpu(), x)),
           (ValueError, lambda: policy_loss(z, t, x[:, :1], x)), (TypeError, lambda: policy_loss(z, t, t, x)),
           (ValueError, lambda: policy_loss(z, t, x.clone().requires_grad_(True), x)), (ValueError, lambda: policy_loss(z, t, x, x, kl_coef=0.1)),
           (ValueError, lambda: policy_loss(z, t, x, x, reduction="max")), (ValueError, lambda: policy_loss(z, t, x, x, clip_low=1.5)),
           (ValueError, lambda: policy_loss(z, t, x, x, clip_high=-0.1)), (ValueError, lambda: policy_loss(z, t, x, x, scale=float("inf"))),
           (ValueError, lambda: preference_loss(z[:1], t[:1])), (ValueError, lambda: preference_loss(z[0], t[0])),
           (ValueError, lambda: preference_loss(z, t, x[0])), (ValueError, lambda: preference_loss(z, t, beta=0.0)),
           (ValueError, lambda: preference_loss(z, t, label_smoothing=1.0)), (ValueError, lambda: preference_loss(z, t, margin=float("nan")))]
    for error, f in bad:
        with pytest.raises(error):
            f()


def test_refusals_of_the_library():
    """Calls that the C ABI turns down before anything is launched (the addresses are never read)."""
    import ctypes
    from star_rwkv6_b200 import _lib as L
    lib, a = L.lib, 0x1000

    def rows(**kw):
        p = L.TokenLogits()
        p.S, p.T, p.V, p.dtype, p.temperature, p.logits, p.targets = 2, 3, 8, L.BF16, 1.0, a, a
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    for kw in (dict(S=-1), dict(V=0), dict(dtype=9), dict(temperature=0.0), dict(temperature=1e-40), dict(temperature=float("inf")), dict(logits=0), dict(targets=0),
               dict(row_stride=-8), dict(logits=a + 1)):
        assert lib.wkv6_token_log_probs(rows(**kw), a, None, None) == -1, kw
    assert lib.wkv6_token_log_probs(rows(S=70000, T=70000), a, None, None) == -2
    assert lib.wkv6_token_log_probs(rows(V=(1 << 30) + 1), a, None, None) == -2
    assert lib.wkv6_token_log_probs(rows(), None, None, None) == -1
    assert lib.wkv6_token_log_probs(rows(), a, a + 4, None) == -1 and b"stat" in lib.wkv6_last_error()
    assert lib.wkv6_token_log_probs(rows(S=0, logits=0, targets=0), None, None, None) == 0
    assert lib.wkv6_token_log_probs_backward(rows(), a, a, 0, None, 0, a + 2, None) == -1
    assert lib.wkv6_token_log_probs_backward(rows(), a, a, 0, None, 1, a, None) == -1          # unless_one without a factor
    c = L.Policy()
    c.advantages, c.old_log_probs, c.scale, c.reduction = a, a, 1.0, 1
    n = lib.wkv6_policy_loss_workspace_bytes(2, 3, 1)
    assert lib.wkv6_policy_loss(rows(), c, a, a, None, a, None, a, n - 1, None) == -3
    assert lib.wkv6_policy_loss(rows(), c, a, a, None, a, a + 8, a, n, None) == -1
    assert lib.wkv6_policy_loss(rows(), c, None, a, None, a, None, a, n, None) == -1
    c.kl_coef = 0.1
    assert lib.wkv6_policy_loss(rows(), c, a, a, None, a, None, a, n, None) == -1 and b"ref_log_probs" in lib.wkv6_last_error()
    c.reduction = 7
    assert lib.wkv6_policy_loss(rows(), c, a, a, None, a, None, a, n, None) == -1
    q = L.Preference()
    assert lib.wkv6_preference_loss(rows(S=3), a, q, a, a, a, a, 100, None) == -1
    assert lib.wkv6_preference_loss(rows(), a, q, a, a, a, a, 23, None) == -3
    assert lib.wkv6_preference_loss(rows(), None, q, a, a, a, a, 24, None) == -1
    assert ctypes.sizeof(L.TokenLogits) == 64 and ctypes.sizeof(L.Policy) == 80 and ctypes.sizeof(L.Preference) == 48


@pytest.mark.gpu
@pytest.mark.parametrize("native", [True, False])
def test_forward_and_backward_in_graphs_of_their_own(native, monkeypatch):
    """The backward is replayed with several factors for one forward, and what received a gradient may write over it."""
    import types
    from star_rwkv6_b200 import loss as L
    if not native:
        monkeypatch.setattr(L, "_native", types.SimpleNamespace(policy_loss=lambda *a: None))
    S, T, V = 3, 5, 900
    z, targets, mask, g = _inputs(S, T, V, torch.bfloat16, seed=40)
    static, targets, mask = z.cuda().requires_grad_(True), targets.cuda(), mask.cuda()
    adv, old = torch.randn(S, T, generator=g).cuda(), torch.full((S, T), -6.5, device="cuda")
    call = lambda: L.policy_loss(static, targets, adv, old, mask=mask)[0]
    factor = torch.ones((), device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(call(), static, factor)
    torch.cuda.synchronize()
    forward, backward = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(forward, stream=side):
        loss = call()
    with torch.cuda.graph(backward, stream=side, pool=forward.pool()):
        (got,) = torch.autograd.grad(loss, static, factor)
    torch.cuda.synchronize()
    for k in range(2):
        with torch.no_grad():
            static.copy_(z.cuda() * (1 + k))
        forward.replay()
        for x in (1.0, 3.0, 1.0, 0.5, 1.0):
            factor.fill_(x)
            backward.replay()
            eager = call()
            torch.autograd.grad(eager, static, factor, retain_graph=True)
            (want,) = torch.autograd.grad(eager, static, factor)       # the second one is formed from the logits, too
            assert torch.equal(loss, eager) and torch.equal(got, want) and got.any()
            got.zero_()
    torch.cuda.synchronize()
