"""Optimizer objects that are copied, saved, loaded and switched, and calls that fail half way: what they go on with."""
import copy
import pickle

import pytest
import torch


def _pair(n=40, **kw):
    from star_rwkv6_b200.optim import AdamW
    ps = [torch.nn.Parameter(torch.linspace(-1, 1, n, device="cuda")) for _ in range(2)]
    return ps, [AdamW([p], **kw) for p in ps]


def _grad(ps, k):
    for p in ps:
        p.grad = torch.full_like(p, 1.0 + k)


@pytest.mark.gpu
@pytest.mark.parametrize("before", [0, 2])
def test_a_group_taken_out_of_capturable_goes_on_from_its_step(before):
    """Bias corrections and random bits of step 5 and on, not those of the first step; and back again."""
    (p, q), (a, b) = _pair(lr=0.1)
    for k in range(10):
        _grad((p, q), k % 3)
        a.param_groups[0]["capturable"] = before <= k < 4 or k >= 7
        if k == 4:
            with pytest.raises(RuntimeError, match="outside of the capture"):
                with torch.cuda.graph(torch.cuda.CUDAGraph()):
                    a.step()
        a.step()
        b.step()
        assert torch.equal(p, q), k
        if k in (5, 8):           # a copy goes on alike
            r = torch.nn.Parameter(p.detach().clone())
            c = type(a)([r], lr=0.1)
            c.load_state_dict(a.state_dict())
            assert c.param_groups[0]["capturable"] == (k == 8)
            c.param_groups[0]["capturable"] = False
            r.grad, q.grad = torch.ones_like(r), torch.ones_like(r)
            d = copy.deepcopy(b.state_dict())
            kept = q.detach().clone()
            c.step()
            b.step()
            assert torch.equal(r, q)
            b.load_state_dict(d)
            with torch.no_grad():
                q.copy_(kept)
    assert a.state[p]["step"] == 7 and int(a.param_groups[0]["step"]) == 10


def test_copied_and_unpickled_optimizers_have_their_attributes():
    from star_rwkv6_b200.optim import AdamW
    opt = AdamW([torch.nn.Parameter(torch.zeros(4))])
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.grad_scale is None
        other.step()


@pytest.mark.gpu
def test_copied_and_unpickled_optimizers_step():
    for again in (copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))):
        (p, _), (opt, _) = _pair(lr=0.1)
        _grad((p,), 0)
        opt.step()
        other = again(opt)
        q = other.param_groups[0]["params"][0]
        assert q is not p and torch.equal(p, q)
        _grad((p, q), 1)
        opt.step()
        other.step()
        assert torch.equal(p, q) and other.state[q]["step"] == 2


@pytest.mark.gpu
def test_a_checkpoint_loaded_to_the_host(tmp_path):
    """Learning rate and step number on the device, read back with map_location="cpu"."""
    (p, q), (a, b) = _pair(lr=torch.full((), 0.1, device="cuda"), capturable=True)
    _grad((p, q), 0)
    a.step()
    torch.save(a.state_dict(), tmp_path / "opt.pt")
    saved = torch.load(tmp_path / "opt.pt", map_location="cpu")
    assert saved["param_groups"][0]["lr"].device.type == "cpu"
    b.load_state_dict(saved)
    with torch.no_grad():
        q.copy_(p)
    _grad((p, q), 1)
    a.step()
    b.step()
    assert torch.equal(p, q) and b.param_groups[0]["lr"].is_cuda
    a.param_groups[0]["lr"].fill_(5.0)           # a copy, as the other values are
    assert b.param_groups[0]["lr"].item() == torch.tensor(0.1).item() and saved["param_groups"][0]["lr"].device.type == "cpu"


@pytest.mark.gpu
def test_a_refused_step_is_not_counted():
    (p, q), (a, b) = _pair(lr=0.1, capturable=True)
    for k in range(3):
        _grad((p, q), k)
        good = p.grad
        p.grad = p.detach()                      # shares memory with what the step writes
        with pytest.raises(ValueError, match="share memory"):
            a.step()
        p.grad = good
        a.step()
        b.step()
        assert torch.equal(p, q) and int(a.param_groups[0]["step"]) == k + 1


def test_hooks_of_loading():
    """What a hook makes of a state dict is what is loaded, in the states' own types; hooks behind the loading see those."""
    from star_rwkv6_b200.optim import AdamW
    p, q = (torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16)) for _ in range(2))
    opt = AdamW([p, q])
    group = {k: v for k, v in opt.param_groups[0].items() if k != "params"}
    x = torch.arange(300.0) + 0.001
    saved = {"state": {0: {"exp_avg": x, "exp_avg_sq": x, "step": 3}}, "param_groups": [dict(group, params=[0, 1])]}

    def swap(optimizer, d):
        return dict(d, state={1: dict(d["state"][0], step=4)})

    def look(optimizer):
        seen.append(optimizer.state[q]["exp_avg"].dtype)
        optimizer.state[q]["exp_avg_sq"].zero_()

    seen = []
    opt.register_load_state_dict_pre_hook(swap)
    opt.register_load_state_dict_post_hook(look)
    opt.load_state_dict(saved)
    s = opt.state[q]
    assert seen == [torch.float32] and p not in opt.state and s["step"] == 4
    assert torch.equal(s["exp_avg"], x) and s["exp_avg"] is not x and not s["exp_avg_sq"].any() and x.all()


@pytest.mark.gpu
def test_numbers_beyond_64_bits_are_refused():
    from star_rwkv6_b200.optim import adamw_step
    f = lambda: torch.zeros(8, device="cuda")
    p = f()
    for kw in (dict(step=2 ** 63), dict(step=2 ** 64 + 1), dict(step=1, first_index=-1), dict(step=1, first_index=2 ** 31),
               dict(step=1, first_index=2 ** 64), dict(step=1, first_index=2 ** 31 - 1, more=True)):
        ps = [p, f()] if kw.pop("more", False) else [p]
        with pytest.raises(ValueError):
            adamw_step(ps, [f() + 1 for _ in ps], [f() for _ in ps], [f() for _ in ps], **kw)
    assert not p.any()
    adamw_step([p], [f() + 1], [f()], [f()], step=2 ** 63 - 1, first_index=2 ** 31 - 1, seed=2 ** 70 + 5)
    assert p.all()


def test_the_capture_that_counts_is_the_parameters_devices(monkeypatch):
    """Host logic on a stand-in for a second device: its stream is being captured, the current device's is not."""
    from star_rwkv6_b200.optim import AdamW

    class Parameter:
        is_cuda, device, shape = True, torch.device("cuda:1"), (4,)

    current = [torch.device("cuda:0")]

    class Device:
        def __init__(self, dev):
            self.dev = torch.device(dev)

        def __enter__(self):
            current.append(self.dev)

        def __exit__(self, *args):
            current.pop()

    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: current[-1].index == 1)
    opt = AdamW([torch.nn.Parameter(torch.zeros(4))])
    with pytest.raises(RuntimeError, match="before the capture"):
        opt._state_of(Parameter(), opt.param_groups[0])
