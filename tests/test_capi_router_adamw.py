"""What the entry points of the router's forms, its losses and the AdamW step refuse, without a GPU: sizes, types, null
pointers and alignment are checked on the host before any launch."""

import ctypes

import pytest
import torch

P = ctypes.c_void_p
ERR_NULL, ERR_SHAPE, ERR_DTYPE, ERR_ALIGN, ERR_WORKSPACE = 1, 2, 3, 4, 5
p = P(256)


@pytest.fixture(scope="module")
def lib():
    from zmoe import _lib

    return _lib.load()


def route(lib, logits=p, dtype=0, T=4, E=32, k=4, score=0, bias=None, groups=1, top=1, scores=1, idx=p, w=p):
    return lib.zmoe_route(logits, dtype, T, E, k, score, bias, groups, top, scores, 1, 1.0, idx, w, None, None)


def test_route(lib):
    for kw in (dict(E=0), dict(E=1025), dict(k=0), dict(k=33), dict(E=128, k=65), dict(T=-1), dict(score=2), dict(score=-1),
               dict(groups=0), dict(groups=65, E=130), dict(groups=5), dict(groups=4, top=5), dict(groups=4, top=0),
               dict(groups=8, top=1, k=5), dict(groups=32, top=32, scores=2), dict(groups=4, top=1, scores=3), dict(scores=0)):
        assert route(lib, **kw) == ERR_SHAPE, kw
    assert route(lib, dtype=2) == ERR_DTYPE
    for kw in (dict(logits=None), dict(idx=None), dict(w=None)):
        assert route(lib, **kw) == ERR_NULL, kw
    assert route(lib, T=0, logits=None, idx=None, w=None) == 0


def backward(lib, dw=p, prob=p, idx=p, T=4, E=32, k=4, score=0, logits=None, add=None, ld_add=0, out=p, ld=32, dtype=0):
    return lib.zmoe_route_backward(dw, prob, idx, T, E, k, score, logits, 1, 1.0, add, ld_add, out, ld, dtype, None)


def test_route_backward(lib):
    for kw in (dict(E=1025, ld=1025), dict(k=0), dict(k=33), dict(T=-1), dict(ld=31), dict(add=p, ld_add=31), dict(score=2)):
        assert backward(lib, **kw) == ERR_SHAPE, kw
    assert backward(lib, dtype=-1) == ERR_DTYPE
    for kw in (dict(dw=None), dict(prob=None), dict(idx=None), dict(out=None), dict(score=1)):  # a softmax needs the logits
        assert backward(lib, **kw) == ERR_NULL, kw
    assert backward(lib, T=0, dw=None) == 0


def losses(lib, logits=p, dtype=0, T=100, E=32, idx=p, k=4, score=0, cu=p, S=3, out=p, grad=p, inv=p, ws=p, nbytes=1 << 30):
    return lib.zmoe_router_losses(logits, dtype, T, E, idx, k, score, cu, 0, S, out, grad, inv, ws, nbytes, None)


def test_router_losses(lib):
    for kw in (dict(E=0), dict(E=1025), dict(T=-1), dict(score=2), dict(S=0), dict(S=(1 << 20) + 1), dict(k=0), dict(k=33),
               dict(T=1 << 31)):
        assert losses(lib, **kw) == ERR_SHAPE, kw
    assert losses(lib, dtype=5) == ERR_DTYPE
    for kw in (dict(logits=None), dict(idx=None), dict(out=None), dict(grad=None), dict(inv=None), dict(ws=None), dict(cu=None)):
        assert losses(lib, **kw) == ERR_NULL, kw
    assert losses(lib, ws=P(264)) == ERR_ALIGN
    need = lib.zmoe_router_losses_workspace_bytes(100, 32, 3)
    assert losses(lib, nbytes=need - 1) == ERR_WORKSPACE
    for bad in ((-1, 32, 1), (10, 0, 1), (10, 1025, 1), (10, 32, 0), (1 << 40, 32, 1)):
        assert lib.zmoe_router_losses_workspace_bytes(*bad) == 0
    # two tiles and three sequences meet in at most five places
    assert need >= 5 * 32 * 8 and lib.zmoe_router_losses_workspace_bytes(0, 32, 1) > 0
    back = lambda **kw: lib.zmoe_router_losses_backward(*{**dict(  # noqa: E731
        logits=p, dtype=0, T=100, E=32, score=0, cu=p, wide=0, S=3, grad=p, inv=p, gb=p, gz=p, out=p, stream=None), **kw}.values())
    assert back(E=0) == back(S=0) == back(score=3) == back(T=-1) == ERR_SHAPE
    assert back(logits=None) == back(grad=None) == back(inv=None) == back(out=None) == back(cu=None) == ERR_NULL
    assert back(T=0, logits=None) == 0


def adamw(lib, change=None, count=1, dtype=0, bits=32, betas=(0.9, 0.99), ws=p, nbytes=1 << 20, **fields):
    from zmoe import _lib

    table = (_lib.AdamwTensor * max(1, count))()
    for e in table:
        for name, v in {**dict(param=256, grad=256, exp_avg=256, exp_avg_sq=256, scale_avg=256, scale_sq=256, step=256, n=10),
                        **fields}.items():
            setattr(e, name, v)
    return lib.zmoe_adamw(table, count, dtype, bits, None, 1e-3, *betas, 1e-8, 0.1, None, ws, nbytes, None)


def test_adamw(lib):
    assert adamw(lib, count=0) == 0
    for kw in (dict(count=-1), dict(n=-1), dict(n=1 << 40), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.5)),
               dict(betas=(float("nan"), 0.9))):
        assert adamw(lib, **kw) == ERR_SHAPE, kw
    for kw in (dict(dtype=2), dict(bits=16), dict(bits=4)):
        assert adamw(lib, **kw) == ERR_DTYPE, kw
    for name in ("param", "grad", "exp_avg", "exp_avg_sq", "step"):
        assert adamw(lib, **{name: None}) == ERR_NULL, name
    for name in ("scale_avg", "scale_sq"):
        assert adamw(lib, bits=8, **{name: None}) == ERR_NULL, name
    assert adamw(lib, ws=None) == ERR_NULL
    for kw in (dict(param=258), dict(grad=257, dtype=1), dict(exp_avg=257), dict(scale_sq=258, bits=8), dict(ws=P(264))):
        assert adamw(lib, **kw) == ERR_ALIGN, kw
    assert adamw(lib, count=3, nbytes=47) == ERR_WORKSPACE
    assert lib.zmoe_adamw(None, 1, 0, 32, None, 1e-3, 0.9, 0.9, 1e-8, 0.0, None, p, 16, None) == ERR_NULL


def test_moments_and_norm(lib):
    from zmoe import _lib

    def moments(**fields):
        table = (_lib.Moment * 1)()
        for name, v in {**dict(codes=256, scale=256, out=256, n=10, second=0), **fields}.items():
            setattr(table[0], name, v)
        return lib.zmoe_adamw_moments(table, 1, None)

    assert moments(n=-1) == ERR_SHAPE and lib.zmoe_adamw_moments(None, -1, None) == ERR_SHAPE
    assert moments(codes=None) == moments(scale=None) == moments(out=None) == ERR_NULL
    assert moments(out=258) == moments(scale=258) == ERR_ALIGN
    assert lib.zmoe_adamw_moments(None, 0, None) == 0 and lib.zmoe_adamw_moments(None, 2, None) == ERR_NULL

    size = lib.zmoe_sum_squares_workspace_bytes
    assert size(0) == size(-1) == size(1 << 40) == 0 and size(1) == 8 and size(1 << 30) == 8 * (1 << 30) // 16384
    ptrs, n = (P * 1)(256), (ctypes.c_int64 * 1)(-1)
    assert lib.zmoe_sum_squares(ptrs, n, 1, 0, p, None) == ERR_SHAPE
    assert lib.zmoe_sum_squares(ptrs, n, 1, 3, p, None) == ERR_DTYPE
    assert lib.zmoe_sum_squares((P * 1)(None), (ctypes.c_int64 * 1)(4), 1, 0, p, None) == ERR_NULL
    assert lib.zmoe_sum_squares(None, None, 1, 0, p, None) == ERR_NULL and lib.zmoe_sum_squares(None, None, 0, 0, None, None) == 0
    assert lib.zmoe_clip_factor(None, 1, 1.0, p, None) == lib.zmoe_clip_factor(p, 1, 1.0, None, None) == ERR_NULL
    assert lib.zmoe_clip_factor(p, -1, 1.0, p, None) == ERR_SHAPE


def test_python_entry_points_refuse_host_tensors():
    from zmoe.adamw import AdamW
    from zmoe.functional import route, router_losses

    z = torch.zeros(3, 32)
    with pytest.raises(ValueError):
        route(z, 4)
    with pytest.raises(ValueError):
        route(z, 4, score="tanh")
    with pytest.raises(ValueError):
        router_losses(z, torch.zeros(3, 4, dtype=torch.int64))
    w = torch.zeros(3, requires_grad=True)
    w.grad = torch.zeros(3)
    with pytest.raises(ValueError):
        AdamW([w]).step()
    with pytest.raises(ValueError):
        AdamW([w], max_grad_norm=1.0).step()
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16),
               dict(max_grad_norm=0.0), dict(max_grad_norm=float("nan"))):
        with pytest.raises(ValueError):
            AdamW([w], **kw)
    with pytest.raises(ValueError), pytest.warns(UserWarning):
        AdamW([w, w])
    opt = AdamW([w])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [torch.zeros(3, dtype=torch.float64, requires_grad=True)]})
    assert len(opt.param_groups) == 1


def test_router_config():
    from modeling.model_config import ModelConfig
    from modeling.moe_gate import MoEGate, RouteForm

    base = dict(hidden_size=64, intermediate_size=32, n_experts=17, n_shared_experts=1, n_experts_per_token=4)
    for bad in (dict(router_score="relu"), dict(router_groups=3), dict(router_groups=0), dict(router_groups=4, router_top_groups=5),
                dict(router_groups=8, router_top_groups=1), dict(router_group_scores=3),
                dict(router_groups=16, router_top_groups=8)):
        with pytest.raises(ValueError):
            ModelConfig(**{**base, **bad})
    assert MoEGate(ModelConfig(**base)).form is None
    form = MoEGate(ModelConfig(**base, router_score="softmax", router_groups=4, router_top_groups=2, router_scale=2.5)).form
    assert form == RouteForm(1, 4, 2, 2, True, 2.5, True)

    class Bare:  # the reference's own config has none of the fields
        hidden_size, n_experts_per_token, n_routed_experts, initializer_range = 64, 4, 16, 0.1

    assert MoEGate(Bare()).form is None


def test_adamw_copies_and_states_of_other_forms():
    import copy
    import pickle

    from zmoe.adamw import AdamW

    w = torch.zeros(3, requires_grad=True)
    opt = AdamW([w], max_grad_norm=0.5, state_bits=8)
    for other in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert other.max_grad_norm == 0.5 and other.grad_norm is None and other.param_groups[0]["state_bits"] == 8
    for name in ("amsgrad", "maximize"):
        with pytest.raises(ValueError, match=name):
            opt.load_state_dict(torch.optim.AdamW([w], **{name: True}).state_dict())
