"""The AdamW step over many tensors against its float64 form.

Tolerances, in half steps h = 2^-24 of fp32.  m = b1 m + c1 g: the constants h of their terms, a product h, the sum h: 3 h of the
terms' sizes (which may cancel): 2^-22 of them.  v: constants, two products and the sum, 4 h: 2^-21 of v.  The update is
m s / (sqrt(v) i + eps): m 3 h (with 8 bits 4 h, a code's product with its scale), s and its product 2 h; sqrt(v) half of v's 4 h (8 bits:
7 h), its own 2 h, i and the sum 2 h; the quotient 4 h (two units of the last place): 15 h, with 8 bits 17.5 h, of the update that the
terms' sizes give: 20 h of it below.  p: its factor's constant, product and the last sum, 3 h: 2^-22 of p.
Rounded values (bf16 parameters, e4m3 moments) have to be what their rounding, which is monotonic, gives of a value within those
bounds."""
import numpy as np
import pytest
import torch

from oracle import adamw_oracle as O

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
SIZES = [1, 7, 8, 255, 256, 257, 1000, 4096, 4097, 70001]


def _flat(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _make(sizes, dtypes, bits, seed=0, offset=0, shift=0):
    """Parameters, gradients and states of a run under way; `offset` values in front of every tensor, so that it starts off the boundary."""
    g = torch.Generator().manual_seed(seed)

    def tensor(x, dtype):
        whole = torch.zeros(offset + len(x), dtype=dtype, device="cuda")
        whole[offset:].copy_(x)
        return whole[offset:]

    lists = {k: [] for k in ("p", "g", "m", "v", "ms", "vs")}
    for i, n in enumerate(sizes):
        dt = dtypes[i % len(dtypes)]
        lists["p"].append(tensor(torch.randn(n, generator=g) * 0.1, dt))
        lists["g"].append(tensor(torch.randn(n, generator=g) * 10.0 ** (i % 4 - 3), dt))
        m, r = torch.randn(n, generator=g) * 1e-2, torch.rand(n, generator=g) * 2e-2 + 1e-4
        if bits == 32:
            lists["m"].append(tensor(m, torch.float32))
            lists["v"].append(tensor(r * r, torch.float32))
        else:
            for key, x in (("m", m), ("v", r)):
                pad = torch.nn.functional.pad(x, (0, -n % 256)).view(-1, 256)
                scale = pad.abs().amax(1) / 448
                lists[key + "s"].append(scale.cuda())
                codes = (pad / scale[:, None]).to(torch.float8_e4m3fn).view(-1)[:n]
                lists[key].append(tensor(codes.float(), torch.float8_e4m3fn))
    return lists


def _oracle(l, i, bits, step, seed, hyper, index=None, lr=None, grad_scale=1.0):
    """(p, m, v as stored) in float64 of tensor i before rounding, and its random bits."""
    p, g, m, v = (_flat(l[k][i]) for k in ("p", "g", "m", "v"))
    if bits == 8:
        m, v = O.values_of(m, _flat(l["ms"][i])), O.values_of(v, _flat(l["vs"][i])) ** 2
    lr, (b1, b2) = hyper["lr"] if lr is None else lr, hyper["betas"]
    new = O.update(p, g * grad_scale, m, v, step, lr, b1, b2, hyper["eps"], hyper["weight_decay"])
    terms = b1 * np.abs(m) + (1 - b1) * np.abs(g * grad_scale)
    update = lr / (1 - b1 ** step) * terms / (np.sqrt(new[2] / (1 - b2 ** step)) + hyper["eps"])
    off = 2.0 ** -22 * np.abs(p) + 20 * 2.0 ** -24 * update
    return new, O.random_bits(len(p), i if index is None else index, step, seed), (off, terms)


def _one_of(got, form, x, off):
    """got is what a monotonic rounding gives of a value within `off` of x."""
    ok = (form(x - off) <= got) & (got <= form(x + off))
    assert ok.all(), (got[~ok][:5], x[~ok][:5], off[~ok][:5])


def _check(l, i, bits, stochastic, want, random, sizes):
    (p, m, v), (off, terms), dt = want, sizes, l["p"][i].dtype
    if dt == torch.float32:
        assert (np.abs(_flat(l["p"][i]) - p) <= off).all()
    elif stochastic:
        _one_of(_flat(l["p"][i]), lambda x: O.bf16_stochastic(x, random), p, off)
    else:
        _one_of(_flat(l["p"][i]), lambda x: _flat(torch.from_numpy(x).float().bfloat16()), p, off)
    if bits == 32:
        assert (np.abs(_flat(l["m"][i]) - m) <= 2.0 ** -22 * terms).all()
        assert (np.abs(_flat(l["v"][i]) - v) <= 2.0 ** -21 * v).all()
        return
    root = np.sqrt(v)
    for key, x in (("m", m), ("v", root)):
        scale = _flat(l[key + "s"][i])
        assert (np.abs(scale - O.block_scales(x)) <= 2.0 ** -21 * scale).all()
        unit = np.repeat(O.block_scales(x), 256)[:len(x)]
        unit = np.where(unit > 0, unit, 1.0)                 # a block of zeros
        q = x / unit
        form = O.e4m3_nearest if key == "m" else (lambda y: O.e4m3_stochastic(np.maximum(y, 0.0), random))
        size = (terms if key == "m" else root) / unit
        _one_of(_flat(l[key][i]), form, q, 2.0 ** -20 * np.maximum(np.abs(q), size))


def _step(l, bits, **kw):
    from star_rwkv6_b200.optim import adamw_step
    more = dict(exp_avg_scales=l["ms"], exp_avg_sq_scales=l["vs"]) if bits == 8 else {}
    adamw_step(l["p"], l["g"], l["m"], l["v"], **more, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtypes,stochastic", [((torch.float32,), True), ((torch.bfloat16,), True), ((torch.bfloat16,), False),
                                               ((torch.bfloat16, torch.float32), True)])
def test_step(dtypes, stochastic, bits, offset):
    l = _make(SIZES, dtypes, bits, offset=offset)
    for step in (1, 2, 777):
        want = [_oracle(l, i, bits, step, 5, HYPER) for i in range(len(SIZES))]
        _step(l, bits, step=step, seed=5, stochastic_rounding=stochastic, **HYPER)
        for i, (new, random, sizes) in enumerate(want):
            _check(l, i, bits, stochastic, new, random, sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_and_empty_ones(bits):
    """More tensors than one launch holds, some without values; neighbours in memory are left alone."""
    sizes = [(37 * i) % 300 for i in range(1100)]
    l = _make(sizes, (torch.bfloat16,), bits, seed=1, offset=2)
    front = [t._base[:2].clone() if t._base is not None else None for t in l["p"]]
    want = {i: _oracle(l, i, bits, 3, 0, HYPER, index=i + 10) for i in (1, 2, 499, 500, 501, 777, 1099)}
    _step(l, bits, step=3, first_index=10, **HYPER)
    for i, (new, random, sizes) in want.items():
        _check(l, i, bits, True, new, random, sizes)
    assert all(f is None or torch.equal(f, t._base[:2]) for f, t in zip(front, l["p"]))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_values_on_the_device(bits):
    """Step number, learning rate and gradient scale on the device, captured and replayed with other values."""
    from star_rwkv6_b200.optim import adamw_step
    l = _make([5, 300, 9000], (torch.bfloat16, torch.float32), bits, seed=2)
    step = torch.zeros((), dtype=torch.int64, device="cuda")
    lr, scale = torch.zeros((), device="cuda"), torch.zeros(1, device="cuda")
    kw = dict(HYPER, lr=lr)
    side = torch.cuda.Stream()
    with pytest.raises(ValueError, match="replay"), torch.cuda.stream(side):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            _step(l, bits, step=4, **HYPER)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step.add_(1)
        _step(l, bits, step=step, grad_scale=scale, **kw)
    for k in range(3):
        lr.fill_(0.01 * (k + 1))
        scale.fill_(0.5 + k)
        want = [_oracle(l, i, bits, k + 1, 0, HYPER, lr=float(lr), grad_scale=float(scale)) for i in range(3)]
        graph.replay()
        for i, (new, random, sizes) in enumerate(want):
            _check(l, i, bits, True, new, random, sizes)


@pytest.mark.gpu
def test_infinities_and_nan_stay_where_they_are():
    for bits in (32, 8):
        l = _make([1000], (torch.float32,), bits, seed=3)
        l["g"][0][300], l["g"][0][600] = float("nan"), float("inf")
        _step(l, bits, step=9, **HYPER)
        bad = ~l["p"][0].isfinite()
        assert bad.nonzero().flatten().tolist() == [300, 600]
        state = l["m"][0].float()
        if bits == 32:
            assert (~state.isfinite()).nonzero().flatten().tolist() == [300, 600]
        else:     # the blocks of 256 around them
            assert (~(state * l["ms"][0].repeat_interleave(256)[:1000]).isfinite()).nonzero().flatten().tolist() == list(range(256, 768))
    b = _make([64], (torch.bfloat16,), 32, seed=3)
    b["g"][0][7] = float("nan")
    _step(b, 32, step=9, **HYPER)
    assert b["p"][0].isnan().nonzero().flatten().tolist() == [7]


@pytest.mark.gpu
def test_new_states_and_quiet_blocks():
    """From zeros, and back to them: a block whose gradients stay zero keeps codes and scales of zero, its parameters only decay."""
    l = _make([600], (torch.float32,), 8, seed=4)
    for k in ("m", "v"):
        l[k][0].zero_()
        l[k + "s"][0].zero_()
    l["g"][0][:256] = 0
    before = _flat(l["p"][0])
    want = _oracle(l, 0, 8, 1, 0, HYPER)[0][0]
    _step(l, 8, step=1, **HYPER)
    assert not l["m"][0][:256].float().any() and not l["v"][0][:256].float().any() and l["ms"][0][0] == 0 and l["vs"][0][0] == 0
    assert l["ms"][0][1] > 0 and (l["v"][0][256:].float() > 0).all()
    assert np.abs(_flat(l["p"][0])[:256] - before[:256] * (1 - 1e-3)).max() <= 1e-7
    assert np.abs(_flat(l["p"][0]) - want).max() <= 1e-7


@pytest.mark.gpu
def test_small_updates_reach_bf16_parameters():
    """Updates of a twentieth of a parameter's last bit: to nearest nothing would move; stochastically the mean does.
    Variance of a rounding: f (1 - f) steps^2, f = 0.05; 40 steps of 65536 values: five standard errors are 0.006 steps x 40^0.5."""
    n, steps = 65536, 40
    p = [torch.full((n,), 1.25, dtype=torch.bfloat16, device="cuda")]
    l = dict(p=p, g=[torch.full((n,), 1.0, dtype=torch.bfloat16, device="cuda")], m=[torch.ones(n, device="cuda")], v=[torch.ones(n, device="cuda")])
    last = 2.0 ** -7
    hyper = dict(lr=last / 20, betas=(0.0, 0.0), eps=0.0, weight_decay=0.0)
    for t in range(1, steps + 1):
        _step(l, 32, step=t, **hyper)
    moved = (1.25 - _flat(p[0])).mean() / last
    assert abs(moved - steps / 20) <= 5 * (steps * 0.05 * 0.95 / n) ** 0.5
    assert len(np.unique(_flat(p[0]))) > 4           # values move independently
    q = [torch.full((n,), 1.25, dtype=torch.bfloat16, device="cuda")]
    _step(dict(l, p=q), 32, step=1, stochastic_rounding=False, **hyper)
    assert (q[0] == 1.25).all()


@pytest.mark.gpu
def test_second_moments_in_8_bits_follow_the_gradients():
    """Gradients fall to a hundredth while one value per block keeps its size, so that the scales stay: v has to decay by beta2 per step
    although a step changes sqrt(v) by 0.25 % and an e4m3 step is 6 to 12 %.  Two thousand values average the rounding's noise: a
    value's rms relative deviation is below sqrt(0.09 / 2 * 0.0025 / (2 * 0.0025)) = 0.2, its bias on v (noise squared per decay) below 10 %."""
    n, b2 = 8 * 256, 0.995
    l = _make([n], (torch.float32,), 8, seed=6)
    l["g"][0].fill_(1.0)
    hyper = dict(lr=0.0, betas=(0.9, b2), eps=1e-8, weight_decay=0.0)
    for t in range(1, 1001):
        if t == 700:
            l["g"][0].fill_(0.01)
            l["g"][0][::256] = 1.0
        _step(l, 8, step=t, **hyper)
    values = (_flat(l["v"][0]) * np.repeat(_flat(l["vs"][0]), 256)) ** 2
    rest = np.arange(n) % 256 != 0
    expected = 1.0 * b2 ** 301 + 1e-4 * (1 - b2 ** 301)
    assert abs(values[rest].mean() / expected - 1) <= 0.15
    assert abs(values[::256].mean() - 1) <= 0.15


def test_random_bits_are_even():
    """Each of the 32 bits is set in half of a tensor's values, and changes with step, tensor and seed.  2^16 values: a share's standard
    error is 2^-9; six of them."""
    n = 1 << 16
    seen = []
    for index, step, seed in ((0, 1, 0), (0, 2, 0), (1, 1, 0), (0, 1, 1), (5, 100000, 12345)):
        bits = (O.random_bits(n, index, step, seed)[:, None] >> np.arange(32, dtype=np.uint64)) & np.uint64(1)
        assert np.abs(bits.mean(0) - 0.5).max() <= 6 * 2.0 ** -9
        assert np.abs((bits[1:] == bits[:-1]).mean(0) - 0.5).max() <= 6 * 2.0 ** -9
        seen.append(bits)
    for i in range(len(seen)):
        for j in range(i):
            assert np.abs((seen[i] == seen[j]).mean(0) - 0.5).max() <= 6 * 2.0 ** -9


def _net(dtype=torch.bfloat16):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(33, 65), torch.nn.Tanh(), torch.nn.Linear(65, 9)).cuda().to(dtype)


def _gradients(net, k):
    torch.manual_seed(100 + k)
    for p in net.parameters():
        p.grad = torch.randn_like(p)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer(bits):
    """The class against adamw_step: groups with their own settings, a parameter whose gradients start late, saving and loading."""
    from star_rwkv6_b200.optim import AdamW
    net = _net()
    ps = list(net.parameters())

    def make(ps):
        return AdamW([{"params": ps[:2], "lr": 1e-2}, {"params": ps[2:], "weight_decay": 0.0}], lr=3e-3, state_bits=bits, seed=4)

    opt, l = make(ps), None
    for k in range(4):
        _gradients(net, k)
        if k < 2:
            ps[3].grad = None
        before = [p.detach().clone() for p in ps]
        if k == 2:
            saved = opt.state_dict()
            twin = _net()
            with torch.no_grad():
                for a, b in zip(twin.parameters(), ps):
                    a.copy_(b)
            twin_opt = make(list(twin.parameters()))
            twin_opt.load_state_dict(saved)
            assert all(s["exp_avg"].dtype == (torch.float32 if bits == 32 else torch.float8_e4m3fn) for s in twin_opt.state.values())
        opt.step()
        assert all(torch.equal(p, b) == (p.grad is None) for p, b in zip(ps, before))
        if k >= 2:
            for a, b in zip(twin.parameters(), ps):
                a.grad = b.grad.clone()
            twin_opt.step()
            assert all(torch.equal(a, b) for a, b in zip(twin.parameters(), ps))
    assert [opt.state[p]["step"] for p in ps] == [4, 4, 4, 2]
    # one more step by hand
    _gradients(net, 9)
    l = dict(p=[ps[3].detach().clone()], g=[ps[3].grad], m=[opt.state[ps[3]]["exp_avg"].clone()], v=[opt.state[ps[3]]["exp_avg_sq"].clone()])
    if bits == 8:
        l["ms"], l["vs"] = [opt.state[ps[3]]["exp_avg_scale"].clone()], [opt.state[ps[3]]["exp_avg_sq_scale"].clone()]
    hyper = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0)
    want = _oracle(l, 0, bits, 3, 4, hyper, index=3)
    opt.step()
    l.update(p=[ps[3]], m=[opt.state[ps[3]]["exp_avg"]], v=[opt.state[ps[3]]["exp_avg_sq"]])
    if bits == 8:
        l["ms"], l["vs"] = [opt.state[ps[3]]["exp_avg_scale"]], [opt.state[ps[3]]["exp_avg_sq_scale"]]
    _check(l, 0, bits, True, *want)


@pytest.mark.gpu
def test_optimizer_captured():
    from star_rwkv6_b200.optim import AdamW
    net, twin = _net(), _net()
    opt = AdamW(net.parameters(), lr=1e-2, state_bits=8, capturable=True)
    eager = AdamW(twin.parameters(), lr=1e-2, state_bits=8)
    _gradients(net, 0)
    for p, q in zip(net.parameters(), twin.parameters()):
        q.grad = p.grad.clone()
    opt.step()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(3):
        for i, (p, q) in enumerate(zip(net.parameters(), twin.parameters())):
            torch.manual_seed(10 * k + i)
            p.grad.copy_(torch.randn_like(p))
            q.grad.copy_(p.grad)
        graph.replay()
        eager.step()
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), twin.parameters()))
    late = torch.nn.Parameter(torch.zeros(3, device="cuda"))
    opt.param_groups[0]["params"].append(late)
    late.grad = torch.ones(3, device="cuda")
    with pytest.raises(RuntimeError, match="first step"):
        opt.step()
    fresh = AdamW([late], capturable=True)
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.step()
    assert not late.any()


@pytest.mark.gpu
def test_gradient_layouts_and_closure():
    from star_rwkv6_b200.optim import AdamW
    p = torch.nn.Parameter(torch.randn(6, 10, device="cuda"))
    q = torch.nn.Parameter(p.detach().clone())
    g = torch.randn(10, 6, device="cuda")
    a, b = AdamW([p]), AdamW([q])
    b.grad_scale = torch.full((), 2.0, device="cuda")
    p.grad, q.grad = g.t(), (g.t() / 2).contiguous()
    assert a.step(lambda: 5) == 5
    b.step()
    assert torch.equal(p, q)
    version = p._version
    a.step()
    assert p._version > version


@pytest.mark.gpu
def test_refusals():
    from star_rwkv6_b200.optim import adamw_step
    f = lambda n=8, dt=torch.float32: torch.zeros(n, dtype=dt, device="cuda")
    p, g, m, v = f(), f(), f(), f()
    c1, c2, s1, s2 = f(8, torch.float8_e4m3fn), f(8, torch.float8_e4m3fn), f(1), f(1)
    two = f(16)
    bad = [(ValueError, lambda: adamw_step([p], [], [m], [v], step=1)), (TypeError, lambda: adamw_step([p.double()], [g], [m], [v], step=1)),
           (TypeError, lambda: adamw_step([p.half()], [g.half()], [m], [v], step=1)), (TypeError, lambda: adamw_step([p], [g.bfloat16()], [m], [v], step=1)),
           (TypeError, lambda: adamw_step([p], [g], [m.bfloat16()], [v], step=1)), (ValueError, lambda: adamw_step([p], [f(7)], [m], [v], step=1)),
           (ValueError, lambda: adamw_step([f(16)[::2]], [g], [m], [v], step=1)), (ValueError, lambda: adamw_step([p], [g], [m], [v], step=0)),
           (ValueError, lambda: adamw_step([p], [g], [m], [v], step=1, betas=(1.0, 0.9))), (ValueError, lambda: adamw_step([p], [g], [m], [v], step=1, eps=-1.0)),
           (ValueError, lambda: adamw_step([p, p], [g, g], [m, f()], [v, f()], step=1)), (ValueError, lambda: adamw_step([two[:8]], [g], [two[4:12]], [v], step=1)),
           (ValueError, lambda: adamw_step([p], [g], [m], [v], exp_avg_scales=[s1], step=1)),
           (TypeError, lambda: adamw_step([p], [g], [m], [v], exp_avg_scales=[s1], exp_avg_sq_scales=[s2], step=1)),
           (ValueError, lambda: adamw_step([p], [g], [c1], [c2], exp_avg_scales=[f(2)], exp_avg_sq_scales=[s2], step=1)),
           (RuntimeError, lambda: adamw_step([p.cpu()], [g], [m], [v], step=1)), (RuntimeError, lambda: adamw_step([p], [g], [m.cpu()], [v], step=1)),
           (ValueError, lambda: adamw_step([p], [g], [m], [v], step=torch.ones((), device="cuda"))),
           (ValueError, lambda: adamw_step([p], [g], [m], [v], step=1, lr=torch.ones(2, device="cuda"))),
           (ValueError, lambda: adamw_step([p], [g], [m], [v], step=1, grad_scale=torch.ones(1))),
           (ValueError, lambda: adamw_step([p], [g], [m], [v], step=1, lr=float("nan")))]
    for error, call in bad:
        with pytest.raises(error):
            call()
    adamw_step([], [], [], [], step=1)
    assert not p.any()


def test_refusals_without_a_gpu():
    from star_rwkv6_b200 import _lib as L
    from star_rwkv6_b200.optim import AdamW, adamw_step
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(state_bits=16), dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(eps=float("nan")), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([p], **kw)
    opt = AdamW([p])
    opt.step()                                       # no gradients: nothing to do
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()
    lib, a = L.lib, 0x1000

    def call(count=1, n=8, index=0, p=a, ms=a, **kw):
        c, t = L.AdamWConfig(), (L.AdamWTensor * 1)()
        c.dtype, c.state_bits, c.step, c.lr, c.beta1, c.beta2, c.eps = L.BF16, 8, 1, 1e-3, 0.9, 0.99, 1e-8
        for k, v in kw.items():
            setattr(c, k, v)
        e = t[0]
        e.p, e.g, e.m, e.v, e.m_scale, e.v_scale, e.n, e.index = p, a, a, a, ms, a, n, index
        return lib.wkv6_adamw_step(c, count, t, None)

    for kw in (dict(count=-1), dict(n=-1), dict(index=-1), dict(index=1 << 31), dict(p=0), dict(p=a + 1), dict(ms=0), dict(ms=a + 2), dict(step=0),
               dict(beta1=1.0), dict(beta2=float("nan"))):
        assert call(**kw) == -1, kw
    assert call(dtype=L.F16) == -2 and call(state_bits=16) == -2
    assert call(n=0, p=0) == 0 and call(count=0) == 0
    assert lib.wkv6_adamw_step(None, 0, None, None) == -1


@pytest.mark.gpu
def test_gradients_may_share_memory_among_themselves_only():
    from star_rwkv6_b200.optim import adamw_step
    f = lambda n: torch.zeros(n, device="cuda")
    one, two = torch.ones(8, device="cuda"), f(24)
    ps, qs = [f(8), f(5), f(0)], [f(8), f(5), f(0)]
    states = [[f(len(p)) for p in ps] for _ in range(4)]
    adamw_step(ps, [one, one[3:], one[:0]], states[0], states[1], step=1)
    adamw_step(qs, [one.clone(), one[3:].clone(), f(0)], states[2], states[3], step=1)
    assert all(torch.equal(p, q) for p, q in zip(ps, qs)) and ps[0].all()
    for p, g, m, v in ((two[:8], two[:8], f(8), f(8)), (two[:8], two[7:15], f(8), f(8)), (two[8:16], two[1:9], f(8), f(8)),
                       (f(8), two[:8], two[4:12], f(8)), (f(8), two[:8], f(8), two[:8]), (f(24), two, two.new_zeros(24), two)):
        with pytest.raises(ValueError, match="share memory"):
            adamw_step([p], [g], [m], [v], step=1)
    narrow = dict(dtype=torch.float8_e4m3fn, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        adamw_step([f(8)], [two[:8]], [torch.zeros(8, **narrow)], [torch.zeros(8, **narrow)], exp_avg_scales=[two[3:4]], exp_avg_sq_scales=[f(1)], step=1)
    adamw_step([two[:8]], [two[8:16]], [f(8)], [two[16:]], step=1)      # side by side
    assert not two.any()


@pytest.mark.gpu
def test_a_group_made_capturable_goes_on_from_its_step():
    from star_rwkv6_b200.optim import AdamW
    p, q = (torch.nn.Parameter(torch.ones(40, device="cuda")) for _ in range(2))
    a, b = AdamW([p], lr=0.1), AdamW([q], lr=0.1)
    for k in range(4):
        p.grad = torch.full_like(p, 1.0 + k)
        q.grad = p.grad.clone()
        if k == 2:
            a.param_groups[0]["capturable"] = True
            with pytest.raises(RuntimeError, match="before the capture"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    a.step()
        a.step()
        b.step()
    assert torch.equal(p, q) and int(a.param_groups[0]["step"]) == 4


@pytest.mark.gpu
def test_a_tensor_of_more_than_32_bits():
    """The last 700 values of a tensor of 2^32 + 700 (26 GB with its gradient and states); all others are zeros and stay so."""
    l, tail, n = _make([700], (torch.bfloat16,), 8, seed=5), 700, 2 ** 32 + 700
    seed, step, index = 77, 6, 0
    big = {}
    for key in ("p", "g", "m", "v"):
        big[key] = [torch.zeros(n, dtype=l[key][0].dtype, device="cuda")]
        big[key][0][-tail:] = l[key][0]
    for key in ("ms", "vs"):
        big[key] = [torch.zeros((n + 255) // 256, device="cuda")]
        big[key][0][-3:] = l[key][0]
    new, _, sizes = _oracle(l, 0, 8, step, seed, HYPER)
    key = O.stir(np.uint64(index) ^ O.stir(np.uint64(step) ^ O.stir(np.uint64(seed))))
    random = O.stir(np.arange(tail, dtype=np.uint64) ^ O.stir(key + np.uint64(1)))
    _step(big, 8, step=step, seed=seed, **HYPER)
    for key, count in (("p", tail), ("m", tail), ("v", tail), ("ms", 3), ("vs", 3)):
        l[key][0].copy_(big[key][0][-count:])
        for at in (0, 2 ** 31 // (n // len(big[key][0])), len(big[key][0]) - count - 1000):
            assert not big[key][0][at:at + 1000].float().any()
    _check(l, 0, 8, True, new, random, sizes)
