"""zmoe.adamw.AdamW's states without a GPU: what load_state_dict takes, and that a load that it refuses changes nothing."""

import copy

import pytest
import torch

SHAPES = [(5, 7), (600,), (300,)]


def states(bits, seed=0, shapes=SHAPES):
    """A state dict's entries, as steps make them."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for i, s in enumerate(shapes):
        n = torch.Size(s).numel()
        if bits == 32:
            out[i] = {"step": torch.tensor(3.0), "exp_avg": torch.randn(s, generator=g), "exp_avg_sq": torch.rand(s, generator=g)}
        else:
            out[i] = {"step": torch.tensor(3.0), "exp_avg": torch.randint(-127, 128, s, generator=g, dtype=torch.int8),
                      "exp_avg_sq": torch.randint(0, 256, s, generator=g, dtype=torch.uint8),
                      "exp_avg_scale": torch.rand(-(-n // 256), generator=g),
                      "exp_avg_sq_scale": torch.rand(-(-n // 256), generator=g)}
    return out


def made(bits=32, dtype=torch.float32):
    from zmoe.adamw import AdamW

    params = [torch.zeros(s, dtype=dtype, requires_grad=True) for s in SHAPES]
    return params, AdamW([{"params": params[:2]}, {"params": params[2:], "weight_decay": 0.0}], lr=0.5, state_bits=bits)


def dict_of(opt, state, **group):
    d = opt.state_dict()
    return {"state": state, "param_groups": [{**g, **group} for g in d["param_groups"]]}


def same(a, b):
    if isinstance(a, torch.Tensor):
        return isinstance(b, torch.Tensor) and a.dtype == b.dtype and a.stride() == b.stride() and torch.equal(a, b)
    if isinstance(a, dict):
        return a.keys() == b.keys() and all(same(v, b[k]) for k, v in a.items())
    if isinstance(a, (list, tuple)):
        return len(a) == len(b) and all(map(same, a, b))
    return a == b


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_states_keep_their_types(bits, dtype):
    params, opt = made(bits, dtype)
    want = states(bits)
    opt.load_state_dict(dict_of(opt, want))
    assert same({i: dict(opt.state[p]) for i, p in enumerate(params)}, want)
    again = copy.deepcopy(opt)
    again.load_state_dict(opt.state_dict())
    assert same(again.state_dict(), opt.state_dict())


def change(i, **kw):
    def f(d):
        d["state"][i] = {k: v for k, v in {**d["state"][i], **kw}.items() if v is not None}

    return f


def groups(**kw):
    return lambda d: [g.update(kw) for g in d["param_groups"]]


REFUSED = {
    32: [lambda d: d.update(state=states(8)), change(2, **states(8)[2]), change(1, exp_avg=torch.zeros(5)),
         change(2, exp_avg_sq=torch.zeros(300, dtype=torch.int64)), change(1, exp_avg=None), change(1, step=None),
         change(2, step=torch.zeros(2)), change(2, exp_avg_sq=0.5), groups(state_bits=16), groups(state_bits=8),
         groups(lr=-1.0), groups(betas=(0.9, 1.0)), groups(eps=-1e-8), groups(weight_decay=-0.1), groups(amsgrad=True),
         groups(maximize=True), groups(decoupled_weight_decay=False, weight_decay=0.1)],
    8: [lambda d: d.update(state=states(32)), change(1, **states(32)[1]), change(1, exp_avg_scale=torch.zeros(2)),
        change(2, exp_avg_sq_scale=torch.zeros(3)), change(1, exp_avg_scale=None),
        change(1, exp_avg_scale=torch.zeros(3, dtype=torch.int64)), change(2, exp_avg=torch.zeros(300, dtype=torch.uint8)),
        change(0, exp_avg=states(8)[0]["exp_avg"].t().contiguous().t()), groups(state_bits=32)],
}


@pytest.mark.parametrize("bits,which", [(b, i) for b, r in REFUSED.items() for i in range(len(r))])
def test_a_refused_load_changes_nothing(bits, which):
    params, opt = made(bits)
    opt.load_state_dict(dict_of(opt, states(bits, seed=1)))
    before = copy.deepcopy(opt.state_dict())
    held = [opt.state[p]["exp_avg"] for p in params]
    bad = dict_of(opt, states(bits, seed=2), lr=0.25)
    REFUSED[bits][which](bad)
    given = copy.deepcopy(bad)
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    assert same(opt.state_dict(), before) and same(bad, given)
    assert all(opt.state[p]["exp_avg"] is t for p, t in zip(params, held))
    opt.load_state_dict(dict_of(opt, states(bits, seed=2), lr=0.25))  # and it still takes what fits
    assert opt.param_groups[0]["lr"] == 0.25 and same(opt.state_dict()["state"], states(bits, seed=2))


def test_groups_that_do_not_match():
    _, opt = made()
    opt.load_state_dict(dict_of(opt, states(32)))
    before = copy.deepcopy(opt.state_dict())
    d = dict_of(opt, states(32, seed=5))
    for bad in (d["param_groups"][:1], [d["param_groups"][0], {**d["param_groups"][1], "params": [2, 3]}]):
        with pytest.raises(ValueError):
            opt.load_state_dict({**d, "param_groups": bad})
        assert same(opt.state_dict(), before)


def test_parameters_without_a_state():
    """Those that had no step yet: no entry, or an empty one (which reading opt.state leaves)."""
    params, opt = made()
    some = states(32)
    some[1] = {}
    del some[2]
    opt.load_state_dict(dict_of(opt, some))
    assert same(dict(opt.state[params[0]]), some[0]) and not opt.state[params[1]] and not opt.state[params[2]]
    assert len(opt.moments()) == 3


def test_hooks():
    """A caller's hooks in front of a load change what is loaded, those behind it see the state as it stays."""
    params, opt = made(8)
    seen = []
    opt.register_load_state_dict_pre_hook(lambda o, d: {**d, "state": states(8, seed=9)})
    opt.register_load_state_dict_post_hook(lambda o: seen.append(o.state[params[1]]["exp_avg"].dtype))
    opt.load_state_dict(dict_of(opt, states(8, seed=3)))
    assert same(opt.state_dict()["state"], states(8, seed=9)) and seen == [torch.int8]


def test_torchs_states():
    params, opt = made()
    theirs = torch.optim.AdamW(torch.optim.AdamW(params).param_groups[0]["params"], lr=0.1)
    for p in params:
        p.grad = torch.ones_like(p)
    theirs.step()
    state = theirs.state_dict()["state"]
    opt.load_state_dict(dict_of(opt, state))
    assert same(opt.state_dict()["state"], {i: {k: v.float() for k, v in s.items()} for i, s in state.items()})
    # Adam's decay goes through its moments, which this step does not do; without decay the two steps are one
    for decay, ok in ((0.0, True), (0.1, False)):
        adam = torch.optim.Adam(params, lr=0.1, weight_decay=decay)
        adam.step()
        from zmoe.adamw import AdamW

        ours = AdamW(params)
        if ok:
            ours.load_state_dict(adam.state_dict())
        else:
            with pytest.raises(ValueError, match="decay"):
                ours.load_state_dict(adam.state_dict())
            assert not ours.state


def test_what_the_step_refuses_of_eps():
    """Without tensors, so that nothing could be launched."""
    from zmoe import _lib

    lib = _lib.load()
    call = lambda eps: lib.zmoe_adamw(None, 0, 0, 32, None, 1e-3, 0.9, 0.999, eps, 0.0, None, None, 0, None)  # noqa: E731
    assert call(0.0) == call(1e-40) == call(1e-8) == 0
    assert call(-1e-8) == call(float("nan")) == 2


class Wrapped(torch.Tensor):
    """A tensor that holds another and has a dispatch of its own, as sharded and quantised ones do."""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device,
                                                   requires_grad=inner.requires_grad)

    def __init__(self, inner):
        self.inner = inner

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        plain = lambda t: t.inner if isinstance(t, Wrapped) else t  # noqa: E731
        return func(*map(plain, args), **{k: plain(v) for k, v in (kwargs or {}).items()})


class Marked(torch.nn.Parameter):
    """A parameter by another name, whose memory is its own."""


def test_tensors_with_a_dispatch_of_their_own():
    from zmoe.adamw import AdamW

    p = torch.zeros(4, requires_grad=True)
    w = Wrapped(torch.zeros(4)).requires_grad_(True)
    with pytest.raises(ValueError, match="Wrapped"):
        AdamW([p, w])
    opt = AdamW([p, Marked(torch.zeros(3))])
    with pytest.raises(ValueError, match="Wrapped"):
        opt.add_param_group({"params": [w]})
    assert len(opt.param_groups) == 1
