"""CPU: calls of the optimizer (duck_gym_b200/optim.py) at the edges of what its
documentation allows."""

import pytest
import torch

from duck_gym_b200 import optim


def count():
    return torch.zeros((), dtype=torch.int64)


@pytest.mark.parametrize("bits", [32, 8])
def test_iterators_are_taken_as_lists_are(bits):
    def tensors():
        p, g = [torch.ones(5), torch.ones(3)], [torch.full((5,), 0.5), torch.full((3,), -2.0)]
        if bits == 8:
            return p, g, [optim.state8_zeros(x, True) for x in p], [optim.state8_zeros(x, False) for x in p]
        return p, g, [torch.zeros_like(x) for x in p], [torch.zeros_like(x) for x in p]

    lists, iterators, a, b = tensors(), tensors(), count(), count()
    optim.adamw_step(*lists, a, 0.1, max_norm=1.0)
    optim.adamw_step(*map(iter, iterators), b, 0.1, max_norm=1.0)
    assert int(a) == int(b) == 1 and not torch.equal(lists[0][0], torch.ones(5))
    flat = lambda x: [t for s in x for t in (flat(s) if isinstance(s, (list, tuple)) else [s])]
    assert all(torch.equal(x, y) for x, y in zip(flat(lists), flat(iterators)))


@pytest.mark.parametrize("lr", [float("nan"), float("inf"), -float("inf")])
def test_a_learning_rate_that_is_not_finite_is_refused(lr):
    p, step = torch.ones(4), count()
    with pytest.raises(RuntimeError, match="finite"):
        optim.adamw_step([p], [torch.ones(4)], [torch.zeros(4)], [torch.zeros(4)], step, lr)
    assert torch.equal(p, torch.ones(4)) and int(step) == 0


def trained(kind, **options):
    p = torch.nn.Parameter(torch.ones(3))
    opt = kind([p], **options)
    for _ in range(3):
        p.grad = torch.tensor([1.0, -0.5, 0.1])
        opt.step()
    return p, opt


@pytest.mark.parametrize("kind,options", [
    (torch.optim.Adam, dict(maximize=True)), (torch.optim.AdamW, dict(maximize=True)), (torch.optim.Adam, dict(amsgrad=True)),
    (torch.optim.AdamW, dict(amsgrad=True)), (torch.optim.Adam, dict(weight_decay=0.1)), (torch.optim.RAdam, {}),
    (torch.optim.SGD, dict(momentum=0.9)), (torch.optim.NAdam, {}), (torch.optim.Adamax, {})])
def test_a_state_dict_that_cannot_be_gone_on_from_is_refused(kind, options):
    p, opt = trained(kind, lr=1e-2, **options)
    mine = optim.AdamW([p], lr=5.0)
    with pytest.raises(RuntimeError, match="AdamW:"):
        mine.load_state_dict(opt.state_dict())
    assert not mine.state and mine.param_groups[0]["lr"] == 5.0   # as it was


def test_weight_decay_of_torch_is_taken_where_it_is_decoupled():
    results = []
    for switch in (False, True):
        p, opt = trained(torch.optim.AdamW, lr=1e-2, weight_decay=0.3)
        if switch:
            saved, opt = opt.state_dict(), optim.AdamW([p])
            older = {**saved, "param_groups": [{k: v for k, v in saved["param_groups"][0].items() if k != "decoupled_weight_decay"}]}
            with pytest.raises(RuntimeError, match="decoupled_weight_decay"):   # Adam's looks the same
                opt.load_state_dict(older)
            opt.load_state_dict(saved)
        for _ in range(3):
            opt.step()
        results.append(p.detach())
    # Three steps of some eight roundings of 2^-24, of a value and of steps of lr.
    assert bool(((results[0] - results[1]).abs() <= 24 * 2.0 ** -24 * (1 + 1e-2)).all())


def test_moments_of_torch_in_bfloat16_become_float32():
    p = torch.nn.Parameter(torch.ones(300, dtype=torch.bfloat16))
    opt = torch.optim.AdamW([p], lr=1e-2, weight_decay=0.1)
    grad = (torch.arange(300) / 100 - 1.5).bfloat16()
    for _ in range(2):
        p.grad = grad
        opt.step()
    saved = opt.state_dict()
    m, v, before = (saved["state"][0][k].clone() for k in ("exp_avg", "exp_avg_sq", "step"))
    was = p.detach().float()
    mine = optim.AdamW([p])
    mine.load_state_dict(saved)
    mine.step()
    state = mine.state[p]
    assert m.dtype == torch.bfloat16 and state["exp_avg"].dtype == state["exp_avg_sq"].dtype == torch.float32
    assert int(before) == 2 and int(mine.param_groups[0]["step"]) == 3
    g, m, v = grad.double(), m.double(), v.double()
    m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
    assert torch.allclose(state["exp_avg"].double(), m, rtol=1e-6, atol=1e-7) and torch.allclose(state["exp_avg_sq"].double(), v, rtol=1e-6)
    want = was * (1 - 1e-3) - 1e-2 * m / (1 - 0.9 ** 3) / ((v / (1 - 0.999 ** 3)).sqrt() + 1e-8)
    # Up or down by less than a place of bfloat16.
    assert bool(((p.detach().double() - want).abs() <= 2.0 ** -7 * want.abs()).all())


# Steps in which each of four parameters has a gradient: always, from the eleventh on, with gaps, and never.
PATTERN = [lambda k: True, lambda k: k >= 10, lambda k: k % 3 != 1, lambda k: False]


def gappy(make, steps, clip=None, switch=None):
    torch.manual_seed(3)
    params = [torch.nn.Parameter(torch.randn(40)) for _ in PATTERN]
    opt = make([dict(params=params[:3]), dict(params=params[3:])])
    for k in range(steps):
        for p, has in zip(params, PATTERN):
            p.grad = torch.randn(40) * (1 + k % 5) if has(k) else None
        if clip is not None:
            torch.nn.utils.clip_grad_norm_(params, clip)
        if switch is not None:
            opt = switch(k, opt, params)
        opt.step()
    return opt, params


@pytest.mark.parametrize("clip", [None, 0.5])
def test_a_parameter_that_comes_late_or_pauses_steps_as_with_torch(clip):
    opt, params = gappy(lambda groups: optim.AdamW(groups, lr=1e-2, max_grad_norm=clip), 400)
    _, wants = gappy(lambda groups: torch.optim.AdamW(groups, lr=1e-2), 400, clip)
    # 400 steps of about lr, each off by some ten roundings of 2^-24 (clipped ones of the norm, too), and the parameter's own.
    for p, want in zip(params, wants):
        assert bool(((p - want).abs() <= 400 * (1e-2 * 16 + 4) * 2.0 ** -24).all())
    steps = [int(opt.state[p].get("step", opt.param_groups[0]["step"])) for p in params[:3]]
    assert steps == [400, 390, 267] and params[3] not in opt.state and "step" not in opt.param_groups[1]


@pytest.mark.parametrize("bits", [32, 8])
def test_own_counts_of_steps_pass_through_state_dicts(bits):
    def switch(k, opt, params):
        if k in (5, 12, 20):
            saved, opt = opt.state_dict(), optim.AdamW([dict(params=params[:3]), dict(params=params[3:])], bits=bits)
            opt.load_state_dict(saved)
        return opt

    make = lambda groups: optim.AdamW(groups, lr=1e-2, bits=bits)
    (a, p), (b, q) = gappy(make, 30), gappy(make, 30, switch=switch)
    assert all(torch.equal(x, y) for x, y in zip(p, q))
    for x, y in zip(p[:3], q[:3]):
        for name in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(a.state[x][name], b.state[y][name])
        count = lambda opt, z: int(opt.state[z].get("step", opt.param_groups[0]["step"]))
        assert count(a, x) == count(b, y)


def test_different_counts_of_torch_are_gone_on_from():
    def switch(k, opt, params):
        if k == 20:
            saved, opt = opt.state_dict(), optim.AdamW([dict(params=params[:3]), dict(params=params[3:])])
            opt.load_state_dict(saved)
        return opt

    make = lambda groups: torch.optim.AdamW(groups, lr=1e-2)
    (_, p), (opt, q) = gappy(make, 40), gappy(make, 40, switch=switch)
    for x, y in zip(p, q):
        assert bool(((x - y).abs() <= 20 * (1e-2 * 16 + 4) * 2.0 ** -24).all())
    assert [int(opt.state[x].get("step", opt.param_groups[0]["step"])) for x in q[:3]] == [40, 30, 27]


def test_a_step_that_was_refused_counts_nothing():
    p = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(3))]
    opt = optim.AdamW(p, lr=1e-2)
    for x in p:
        x.grad = torch.ones(3)
    opt.param_groups[0]["eps"] = -1.0
    with pytest.raises(RuntimeError):
        opt.step()
    opt.param_groups[0]["eps"] = 1e-8
    opt.step()
    assert int(opt.param_groups[0]["step"]) == 1 and all("step" not in opt.state[x] for x in p)
    assert torch.allclose(p[0], torch.full((3,), (1 - 1e-4) - 1e-2))
