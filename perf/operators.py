"""What the operators behind a model's logits and in front of its weights are measured on: log-probabilities of given tokens,
the clipped policy loss, the preference loss (``star_rwkv6_b200.loss``) and the AdamW step over many tensors
(``star_rwkv6_b200.optim``), each through its public entry point (``own``) and as plain tensor operations.

Logits are N(0, 2.5^2) with the chosen token's raised, as a trained model's are (log-probabilities around -1); every
sequence starts with a prompt and ends with padding, which the mask leaves out.  Optimizer states are those of a run under way
(step 1000).
"""
import torch

own = False

VOCAB = 65536               # of every model of this package
BLOCK = 256                 # values that share a scale where states have 8 bits
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LR, BETAS, EPS, DECAY, SEED = 3e-4, (0.9, 0.999), 1e-8, 0.1, 77


# ------------------------------------------------------------------------------------------------------------------ cases

def _tokens(name, op, S, T, V, dtype="bf16", **more):
    c = {"op": op, "S": S, "T": T, "V": V, "dtype": dtype, "backward": True, "temperature": 1.0,
         "scale": 1024.0 if dtype == "f16" else 1.0, **more}     # fp16 gradients are scaled away from the type's lower end
    return dict(c, name=name) if name else c


def _policy(name, S, T, V, dtype="bf16", reduction="mean", kl=0.02, temperature=1.0):
    return _tokens(name, "policy", S, T, V, dtype, reduction=reduction, kl=kl, temperature=temperature)


def _preference(name, pairs, T, V, dtype="bf16", smoothing=0.0, average=False, reference=True):
    return _tokens(name, "preference", 2 * pairs, T, V, dtype, smoothing=smoothing, average=average, reference=reference)


def _adamw(name, D, layers, vocab, types, bits, tight=False):
    c = {"op": "adamw", "D": D, "layers": layers, "vocab": vocab, "types": types, "bits": bits, "tight": tight}
    return dict(c, name=name) if name else c


def listed():
    return [
        # scoring the tokens that a serving batch has just sampled: one row per sequence, latency
        _tokens("logp S16 T1 forward", "logp", 16, 1, VOCAB, backward=False),
        # a reference model's pass over a batch of answers, no gradient
        _tokens("logp S4 T1003 forward", "logp", 4, 1003, VOCAB, backward=False),
        # log-probabilities as part of another loss, fp32 logits of a vocabulary that is not a multiple of anything
        _tokens("logp S3 T333 V50277 f32", "logp", 3, 333, 50277, "f32"),
        # a short answer or two: the smallest policy update
        _policy("policy S2 T33", 2, 33, VOCAB),
        # fp16 logits, odd vocabulary, a sampling temperature, answers weighted alike whatever their length
        _policy("policy S3 T517 V50277 f16", 3, 517, 50277, "f16", "sequence_mean", 0.0, 0.7),
        # a group of answers to one question
        _policy("policy S8 T1024", 8, 1024, VOCAB),
        # one pair of short answers
        _preference("preference P1 T65", 1, 65, VOCAB),
        # a byte-level model's pairs in fp32: no reference model, mean log-probabilities, noisy labels
        _preference("preference P16 T700 V259 f32", 16, 700, 259, "f32", 0.1, True, False),
        # an ordinary batch of pairs
        _preference("preference P4 T1024", 4, 1024, VOCAB),
        # a toy model's step: many tensors, none of them large
        _adamw("adamw D128 f32", 128, 2, 512, "f32", 32),
        # embedding, head and two layers of the 1.6B shape, as the package's model types its parameters
        _adamw("adamw D2048", 2048, 2, VOCAB, "mixed", 32),
        # the same with states in 8 bits
        _adamw("adamw D2048 8 bits", 2048, 2, VOCAB, "mixed", 8),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _odd_tokens(rng, most):
    V = rng.choice((VOCAB, VOCAB, 50277, _log(rng, 100, 130000)))
    dtype = rng.choice(("bf16", "bf16", "bf16", "f16", "f32"))
    rows = _log(rng, 2, max(3, min(most, most * VOCAB * 2 // (V * DTYPES[dtype].itemsize))))
    S = min(rows, rng.choice((1, 2, 3, 4, 8, 16)))
    return S, max(1, rows // S), V, dtype


def draw(rng):
    op = rng.choice(("logp", "policy", "policy", "preference", "preference", "adamw", "adamw"))
    if op == "adamw":
        D = 64 * _log(rng, 1, 32)
        return _adamw(None, D, rng.randint(1, 2), min(VOCAB, _log(rng, 100, VOCAB)), rng.choice(("f32", "bf16", "mixed")),
                      rng.choice((32, 8)), rng.random() < 0.2)
    S, T, V, dtype = _odd_tokens(rng, 6000)
    if op == "logp":
        return _tokens(None, "logp", S, T, V, dtype, backward=rng.random() < 0.5, temperature=rng.choice((1.0, 0.8)))
    if op == "policy":
        return _policy(None, S, T, V, dtype, rng.choice(("mean", "sequence_mean", "sum")), rng.choice((0.0, 0.04)),
                       rng.choice((1.0, 1.0, 0.9)))
    return _preference(None, max(1, S // 2), T, V, dtype, rng.choice((0.0, 0.1)), rng.random() < 0.3, rng.random() < 0.8)


# ----------------------------------------------------------------------------------------------------------------- inputs

def _live(c):
    """(prompt length, end) of every sequence: tokens between them count.  The shares are those of chat data: an eighth to a
    quarter of the row is prompt, up to a quarter padding."""
    S, T = c["S"], c["T"]
    return [((T // 8) + (37 * s) % (T // 8 + 1), T - (53 * s) % (T // 4 + 1)) for s in range(S)]


def _prepare_tokens(c, g):
    S, T, V, dt = c["S"], c["T"], c["V"], DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    targets = torch.randint(0, V, (S, T), generator=g, device="cuda")
    z = 2.5 * normal(S, T, V)
    z.scatter_(-1, targets[..., None], torch.logsumexp(z, -1, keepdim=True) + 1.0 + 2.0 * normal(S, T, 1))
    z = z.to(dt)
    at, ends = torch.arange(T, device="cuda"), torch.tensor(_live(c), device="cuda")
    mask = (at >= ends[:, :1]) & (at < ends[:, 1:])
    s = dict(c, targets=targets, mask=mask)
    tau = c["temperature"]
    lp = torch.stack([torch.log_softmax(r.float() / tau, -1).gather(-1, t[:, None])[:, 0] for r, t in zip(z, targets)])
    if c["op"] == "logp":
        s["grad"] = normal(S, T) if c["backward"] else None
    if c["op"] == "policy":   # an update or two after the answers were sampled; one advantage for each answer
        s["old"] = lp + 0.15 * normal(S, T)
        s["ref"] = lp + 0.3 * normal(S, T) if c["kl"] else None
        s["advantages"] = normal(S, 1).expand(S, T)
    if c["op"] == "preference":
        total, n = torch.where(mask, lp, 0.0).sum(-1), mask.sum(-1)
        noise = normal(S) * (0.1 if c["average"] else 5.0)
        s["ref"] = total / (n.clamp(min=1) if c["average"] else 1) + noise if c["reference"] else None
    s["logits"] = z.requires_grad_(c["backward"])
    return s


def _shapes(c):
    """(shape, kept in fp32) of the parameters of an RWKV-6 model of this package."""
    D, V, H = c["D"], c["vocab"], max(1, c["D"] // 64)
    F = D * 7 // 2
    vector, small = ((D,), False), ((D,), True)
    time_mix = [small, ((D, 160), False), ((5, 32, D), False), ((5, 1, D), False)] + 5 * [((D, D), False)]
    time_mix += [((64, D), False), ((D, 64), False), vector, ((H, 64), True), ((H, 64), True), ((H, 64), True)]
    channel_mix = [small, small, ((F, D), False), ((D, F), False), ((D, D), False)]
    block = 4 * [vector] + time_mix + channel_mix
    return [((V, D), False)] + 2 * [vector] + c["layers"] * block + 2 * [vector] + [((V, D), False)]


def _size(shape):
    n = 1
    for k in shape:
        n *= k
    return n


def _places(sizes, step):
    """Where tensors of these sizes start in one buffer, at multiples of `step` values, and the buffer's size."""
    at, end = [], 0
    for n in sizes:
        at.append(end)
        end += -(-n // step) * step
    return at, end


def _views(flat, sizes, step):
    return [flat[a:a + n] for a, n in zip(_places(sizes, step)[0], sizes)]


def _prepare_adamw(c, g):
    """Parameters, gradients and states as views of flat buffers, as data-parallel training keeps them."""
    shapes = _shapes(c)
    sizes = [_size(s) for s, _ in shapes]
    wide = [c["types"] == "f32" or (c["types"] == "mixed" and keep) for _, keep in shapes]
    step = 1 if c["tight"] else BLOCK
    total = _places(sizes, step)[1]

    def normal(n):
        return torch.randn(n, generator=g, device="cuda")

    p = {True: None, False: None}
    grad = {True: None, False: None}
    views, grads = [None] * len(sizes), [None] * len(sizes)
    for w in (True, False):
        which = [k for k in range(len(sizes)) if wide[k] == w]
        if which:
            mine = [sizes[k] for k in which]
            n, dt = _places(mine, step)[1], torch.float32 if w else torch.bfloat16
            p[w], grad[w] = (0.02 * normal(n)).to(dt), (1e-3 * normal(n)).to(dt)
            for k, a, b in zip(which, _views(p[w], mine, step), _views(grad[w], mine, step)):
                views[k], grads[k] = a.view(shapes[k][0]), b.view(shapes[k][0])
    m, r = 3e-4 * normal(total), 1e-3 * (0.3 + torch.rand(total, generator=g, device="cuda"))
    s = dict(c, sizes=sizes, step=1000, flat=[p[w] for w in (True, False) if p[w] is not None], keep=grad, params=views, grads=grads)
    if c["bits"] == 32:
        s["m"], s["v"] = m, r * r
        s["m_scale"] = s["v_scale"] = None
    else:
        blocks = [-(-n // BLOCK) for n in sizes]
        for key, x in (("m", m), ("v", r)):   # the second moment is held as its square root
            parts = [_to_blocks(t) for t in _views(x, sizes, step)]
            codes, scales = torch.zeros(total, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(sum(blocks), device="cuda")
            for part, a, b, n in zip(parts, _views(codes, sizes, step), _views(scales, blocks, 1), sizes):
                scale = part.abs().amax(-1) / 448.0
                b.copy_(scale)
                a.copy_((part / scale[:, None]).to(torch.float8_e4m3fn).reshape(-1)[:n])
            s[key], s[key + "_scale"] = codes, scales
        s["m_scales"], s["v_scales"] = _views(s["m_scale"], blocks, 1), _views(s["v_scale"], blocks, 1)
    s["m_views"], s["v_views"] = ([t.view(sh[0]) for t, sh in zip(_views(s[k], sizes, step), shapes)] for k in ("m", "v"))
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_adamw(case, g) if case["op"] == "adamw" else _prepare_tokens(case, g)


# ------------------------------------------------------------------------------------------------------------ plain forms

def _row_parts(z, targets, tau):
    """exp((z - max) / tau), its sum, and the targets' log-probabilities, over the last axis in fp32."""
    z = z.detach().float()
    d = z - z.amax(-1, keepdim=True)
    if tau != 1.0:
        d = d / tau
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    return e, total, (d.gather(-1, targets[..., None]) - torch.log(total))[..., 0]


def _logit_gradient(s, e, total, coefficient):
    """coefficient (1[j = target] - p_j) / tau, in the logits' type."""
    c = (coefficient / s["temperature"])[..., None]
    g = e.mul_(-c / total)
    g.scatter_add_(-1, s["targets"][..., None], c)
    return g.to(s["logits"].dtype)


def _plain_logp(s):
    e, total, lp = _row_parts(s["logits"], s["targets"], s["temperature"])
    lp = torch.where(s["mask"], lp, 0.0)
    if not s["backward"]:
        return lp
    return lp, _logit_gradient(s, e, total, torch.where(s["mask"], s["grad"], 0.0))


def _plain_policy(s):
    mask, adv = s["mask"], s["advantages"]
    e, total, lp = _row_parts(s["logits"], s["targets"], s["temperature"])
    ratio = torch.exp(lp - s["old"])
    free, clipped = ratio * adv, ratio.clamp(0.8, 1.2) * adv
    loss, slope = -torch.minimum(free, clipped), torch.where(free <= clipped, -free, 0.0)
    if s["kl"]:
        d = s["ref"] - lp
        loss, slope = loss + s["kl"] * (torch.exp(d) - d - 1.0), slope + s["kl"] * (1.0 - torch.exp(d))
    n = mask.sum(-1, keepdim=True).double()
    weight = {"mean": 1.0 / n.sum().clamp(min=1.0), "sequence_mean": 1.0 / (n.clamp(min=1.0) * len(n)), "sum": torch.ones_like(n)}[s["reduction"]]
    weight = torch.where(mask, weight * s["scale"], 0.0)
    total_loss = torch.where(mask, loss * weight, 0.0).sum().float()
    grad = _logit_gradient(s, e, total, torch.where(mask, slope * weight, 0.0).float())
    return total_loss, torch.where(mask, lp, 0.0), grad


def _plain_preference(s):
    mask, beta, eps = s["mask"], 2.0 if s["average"] else 0.1, s["smoothing"]
    e, total, lp = _row_parts(s["logits"], s["targets"], 1.0)
    n = mask.sum(-1).clamp(min=1).double() if s["average"] else torch.ones(len(mask), dtype=torch.float64, device=lp.device)
    seq = torch.where(mask, lp, 0.0).double().sum(-1) / n
    ratio = seq - s["ref"].double() if s["reference"] else seq
    good, bad = ratio.chunk(2)
    d = beta * (good - bad)
    tail = torch.log1p(torch.exp(-d.abs()))
    loss = ((1.0 - eps) * (tail + (-d).clamp(min=0.0)) + eps * (tail + d.clamp(min=0.0))).mean()
    slope = -beta * (1.0 - eps - 1.0 / (1.0 + torch.exp(-d))) * (s["scale"] / len(d))
    coefficient = (torch.cat((slope, -slope)) / n).float()
    return (loss * s["scale"]).float(), seq.float(), _logit_gradient(s, e, total, torch.where(mask, coefficient[:, None], 0.0))


MASK32 = 0xFFFFFFFF


def _mix(x):
    """A 32-bit integer's bits stirred (an int, or an int64 tensor)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & MASK32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & MASK32
    return x ^ (x >> 16)


def _key(k, step):
    """The random stream of tensor k at this step."""
    return _mix(k ^ _mix(step ^ _mix(SEED)))


def _random_bits(n, key):
    """32 bits for each of a tensor's values."""
    return _mix(torch.arange(n, device="cuda") ^ key)


def _to_blocks(x):
    """x [n] as [blocks, BLOCK], zeros behind the last value."""
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -len(x) % BLOCK)).view(-1, BLOCK)


def _plain_from_blocks(codes, scales):
    return (_to_blocks(codes.float()) * scales[:, None]).reshape(-1)[:codes.numel()]


def _plain_scales(x):
    """[blocks, BLOCK] values as multiples of their block's scale (448 of it is the largest value), and the scales."""
    top = x.abs().amax(-1)
    top = torch.where(top < 2.0 ** -100, 0.0, top)
    return torch.where(top[:, None] > 0.0, x * (448.0 / top)[:, None], 0.0), top * (1.0 / 448.0)


def _plain_update(p, g, m, v, m_scale, v_scale, k, step):
    """One AdamW step of one tensor, in place."""
    n = p.numel()
    bits = _random_bits(n, _key(k, step)) if p.dtype == torch.bfloat16 or m_scale is not None else None
    x, g = p.float().reshape(-1), g.float().reshape(-1)
    if m_scale is None:
        a, b = m.reshape(-1), v.reshape(-1)
    else:
        a, b = _plain_from_blocks(m.reshape(-1), m_scale), _plain_from_blocks(v.reshape(-1), v_scale)
        b = b * b
    a = a * BETAS[0] + g * (1.0 - BETAS[0])
    b = b * BETAS[1] + (g * g) * (1.0 - BETAS[1])
    root = torch.sqrt(b)
    x = x * (1.0 - LR * DECAY)
    x = x - (a * (LR / (1.0 - BETAS[0] ** step))) / (root * ((1.0 - BETAS[1] ** step) ** -0.5) + EPS)
    if p.dtype == torch.bfloat16:      # up or down with the probabilities that keep the mean
        x = _plain_truncate(x, bits)
    p.copy_(x.view(p.shape))
    if m_scale is None:
        m.copy_(a.view(m.shape))
        v.copy_(b.view(v.shape))
        return
    q, scale = _plain_scales(_to_blocks(a))
    m_scale.copy_(scale)
    m.copy_(q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).reshape(-1)[:n].view(m.shape))
    q, scale = _plain_scales(_to_blocks(root))
    v_scale.copy_(scale)
    q, r = q.reshape(-1)[:n], bits >> 16
    normal = ((q.view(torch.int32).long() + (r << 4)) >> 20 << 20).to(torch.int32).view(torch.float32)
    tiny = torch.floor(q * 512.0 + r.float() * 2.0 ** -16) * (1.0 / 512.0)
    q = torch.where(q >= 2.0 ** -6, normal, torch.where(q > 0.0, tiny.clamp(min=1.0 / 512.0), 0.0))
    v.copy_(q.clamp(max=448.0).to(torch.float8_e4m3fn).view(v.shape))


def _plain_truncate(x, bits):
    """fp32 values rounded to bf16 by adding 16 random bits below its last one and dropping them."""
    u = ((x.view(torch.int32).long() & MASK32) + (bits & 0xFFFF)) & 0xFFFF0000
    return torch.where(u >= 1 << 31, u - (1 << 32), u).to(torch.int32).view(torch.float32).to(torch.bfloat16)


def _adamw_outputs(s):
    return s["flat"], s["m"], s["v"], s["m_scale"], s["v_scale"]


def _run_adamw(s):
    s["step"] += 1
    if own:
        from star_rwkv6_b200.optim import adamw_step
        adamw_step(s["params"], s["grads"], s["m_views"], s["v_views"], exp_avg_scales=s.get("m_scales"),
                   exp_avg_sq_scales=s.get("v_scales"), step=s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, seed=SEED)
    else:
        none = [None] * len(s["params"])
        every = zip(s["params"], s["grads"], s["m_views"], s["v_views"], s.get("m_scales", none), s.get("v_scales", none))
        for k, t in enumerate(every):
            _plain_update(*t, k, s["step"])
    return _adamw_outputs(s)


def run(s):
    op = s["op"]
    if op == "adamw":
        return _run_adamw(s)
    if not own:
        return {"logp": _plain_logp, "policy": _plain_policy, "preference": _plain_preference}[op](s)
    from star_rwkv6_b200.loss import policy_loss, preference_loss, token_log_probs
    z = s["logits"]
    if op == "logp":
        lp = token_log_probs(z, s["targets"], s["mask"], temperature=s["temperature"])
        return (lp, *torch.autograd.grad(lp, z, s["grad"])) if s["backward"] else lp
    if op == "policy":
        loss, lp = policy_loss(z, s["targets"], s["advantages"], s["old"], ref_log_probs=s["ref"], mask=s["mask"],
                               kl_coef=s["kl"], temperature=s["temperature"], reduction=s["reduction"], scale=s["scale"])
        return (loss, lp, *torch.autograd.grad(loss, z))
    loss, seq = preference_loss(z, s["targets"], s["ref"], s["mask"], beta=2.0 if s["average"] else 0.1,
                                label_smoothing=s["smoothing"], average=s["average"], scale=s["scale"])
    return (loss, seq, *torch.autograd.grad(loss, z))


# ------------------------------------------------------------------------------------------------------- work and 64 bits

def work(case):
    if case["op"] == "adamw":
        shapes = _shapes(case)
        n = sum(_size(s) for s, _ in shapes)
        wide = sum(_size(s) for s, keep in shapes if case["types"] == "f32" or (case["types"] == "mixed" and keep))
        states = 16 * n if case["bits"] == 32 else 4 * n + 16 * sum(-(-_size(s) // BLOCK) for s, _ in shapes)
        return {"bytes": 3 * (4 * wide + 2 * (n - wide)) + states, "flops": 14 * n}
    rows, row = case["S"] * case["T"], case["V"] * DTYPES[case["dtype"]].itemsize
    live = sum(max(0, b - a) for a, b in _live(case))
    small = rows * (8 + 1 + 4) + (rows * 4 if case["op"] == "logp" and case["backward"] else 0)
    small += live * 12 if case["op"] == "policy" else 0
    moved = live * row + (rows * row if case["backward"] else 0)
    return {"bytes": moved + small, "flops": live * case["V"] * (8 if case["backward"] else 4)}


def _exact_tokens(c, s):
    """From the definitions, gradients by differentiating them."""
    z = s["logits"].detach().double().requires_grad_(c["backward"])
    mask = s["mask"]
    all_lp = torch.log_softmax(z / c["temperature"], -1).gather(-1, s["targets"].unsqueeze(-1)).squeeze(-1)
    lp = all_lp * mask
    if c["op"] == "logp":
        return (lp.detach(), *torch.autograd.grad(lp, z, s["grad"].double())) if c["backward"] else lp
    if c["op"] == "policy":
        A, rho = s["advantages"].double(), (all_lp - s["old"].double()).exp()
        each = -torch.min(rho * A, torch.clamp(rho, 1 - 0.2, 1 + 0.2) * A)
        if c["kl"]:
            log_ratio = s["ref"].double() - all_lp
            each = each + c["kl"] * (torch.expm1(log_ratio) - log_ratio)
        each, n = each * mask, mask.sum(1)
        if c["reduction"] == "mean":
            loss = each.sum() / n.sum().clamp(min=1)
        elif c["reduction"] == "sum":
            loss = each.sum()
        else:
            loss = (each.sum(1) / n.clamp(min=1)).mean()
        loss = loss * c["scale"]
        return (loss.detach(), lp.detach(), *torch.autograd.grad(loss, z))
    seq = lp.sum(1) / mask.sum(1).clamp(min=1) if c["average"] else lp.sum(1)
    over = seq - s["ref"].double() if c["reference"] else seq
    pairs = c["S"] // 2
    margin = (2.0 if c["average"] else 0.1) * (over[:pairs] - over[pairs:])
    logsigmoid = torch.nn.functional.logsigmoid
    loss = -((1 - c["smoothing"]) * logsigmoid(margin) + c["smoothing"] * logsigmoid(-margin)).mean() * c["scale"]
    return (loss.detach(), seq.detach(), *torch.autograd.grad(loss, z))


def _exact_grid(x, digits, least):
    """The spacing, at x, of a binary format with `digits` bits behind the leading one and 2^least as its smallest normal."""
    return torch.exp2((torch.frexp(x)[1] - 1).clamp(min=least).double() - digits)


def _exact_adamw(c, s):
    t = s["step"] + 1
    flat, m_all, v_all = [x.double() for x in s["flat"]], s["m"].double(), s["v"].double()
    ms, vs = (None, None) if c["bits"] == 32 else (s["m_scale"].double(), s["v_scale"].double())
    step = 1 if c["tight"] else BLOCK
    sizes = s["sizes"]
    block_at, value_at = _places([-(-n // BLOCK) for n in sizes], 1)[0], _places(sizes, step)[0]
    start = {f.dtype: 0 for f in s["flat"]}
    for k, n in enumerate(sizes):
        p, g = s["params"][k].double().flatten(), s["grads"][k].double().flatten()
        dtype = s["params"][k].dtype
        here, blocks = slice(value_at[k], value_at[k] + n), slice(block_at[k], block_at[k] + -(-n // BLOCK))
        m, v = m_all[here], v_all[here]
        if ms is not None:
            each = torch.arange(n, device="cuda") // BLOCK
            m, v = m * ms[blocks][each], (v * vs[blocks][each]) ** 2
        m, v = torch.lerp(g, m, BETAS[0]), torch.lerp(g * g, v, BETAS[1])
        p = p - LR * DECAY * p - LR * (m / (1 - BETAS[0] ** t)) / ((v / (1 - BETAS[1] ** t)).sqrt() + EPS)
        random = _random_bits(n, _key(k, t))
        if dtype == torch.bfloat16:
            grid = _exact_grid(p, 7, -126)
            p = torch.copysign(torch.floor(p.abs() / grid + (random % 65536).double() / 65536) * grid, p)
        which = [f.dtype for f in s["flat"]].index(dtype)
        flat[which][start[dtype]:start[dtype] + n] = p
        start[dtype] += -(-n // step) * step
        if ms is None:
            m_all[here], v_all[here] = m, v
            continue
        root = v.sqrt()
        ms[blocks], vs[blocks] = (_to_blocks(x).abs().max(-1).values / 448 for x in (m, root))
        q, r = m / ms[blocks][each], root / vs[blocks][each]
        grid = _exact_grid(q, 3, -6)
        m_all[here] = torch.round(q / grid) * grid
        grid = _exact_grid(r, 3, -6)
        v_all[here] = (torch.floor(r / grid + torch.div(random, 65536, rounding_mode="floor").double() / 65536) * grid).clamp(2.0 ** -9, 448.0)
    return flat, m_all, v_all, ms, vs


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(case, s) if case["op"] == "adamw" else _exact_tokens(case, s)
