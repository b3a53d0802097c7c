"""CPU: the optimizer (duck_gym_b200/optim.py) against float64 restatements
(tests/gated_math.py) and torch's, its moments in 8 bits, its refusals."""

import copy
import math

import pytest
import torch

import gated_math
from duck_gym_b200 import optim
from test_gated import offsets


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def model(seed, shapes, dtype=torch.float32):
    g = gen(seed)
    return ([(0.1 * torch.randn(s, generator=g)).to(dtype) for s in shapes],
            [(0.01 * torch.randn(s, generator=g) * torch.exp(torch.randn(s, generator=g))).to(dtype) for s in shapes])


def zeros(params, bits):
    if bits == 8:
        return [optim.state8_zeros(p, True) for p in params], [optim.state8_zeros(p, False) for p in params]
    return [torch.zeros(p.shape) for p in params], [torch.zeros(p.shape) for p in params]


SHAPES = [(), (3,), (129,), (5, 7), (0,), (300,)]


@pytest.mark.parametrize("max_norm", [None, 0.5, 100.0])
def test_step_matches_restatement(max_norm):
    p, g = model(1, SHAPES)
    m, v = zeros(p, 32)
    step, lr, wd, betas = torch.zeros((), dtype=torch.int64), 3e-3, 0.1, (0.8, 0.95)
    want = [(a.double(), b.double(), c.double()) for a, b, c in zip(p, m, v)]
    clip = 1.0
    if max_norm is not None:
        clip = min(1.0, max_norm / (math.sqrt(sum(float(x.double().square().sum()) for x in g)) + 1e-6))
    for t in (1, 2, 3):
        optim.adamw_step(p, g, m, v, step, lr, betas, 1e-6, wd, max_norm)
        want = [gated_math.adamw(a, x, b, c, t, lr, betas, 1e-6, wd, clip) for x, (a, b, c) in zip(g, want)]
    assert int(step) == 3
    for got, exact in zip(zip(p, m, v), want):
        for a, b in zip(got, exact):
            # Three steps of some eight roundings of 2^-24.
            assert bool(((a.double() - b).abs() <= 24 * 2.0 ** -24 * b.abs() + 24 * 2.0 ** -24 * lr).all())


def test_codes_by_hand():
    """One group's codes against the definition, value by value."""
    g = gen(2)
    x = torch.randn(300, generator=g) * torch.exp(3 * torch.randn(300, generator=g))
    x[5], x[6], x[7] = 0.0, 1e-30, -0.0
    for signed in (True, False):
        values = x if signed else x.abs()
        state = optim.state8_zeros(x, signed)
        noise = torch.randint(0, 1 << 20, (300,), generator=g)
        optim._encode(values, state, noise)
        most = 127 if signed else 255
        for i in range(300):
            group = values[i // 128 * 128:i // 128 * 128 + 128]
            e = int(group.abs().max().view(torch.int32)) >> 23
            bits = int(values[i].abs().view(torch.int32))
            code = (bits + int(noise[i])) // 2**20 - max(0, 8 * e + 8 - most)
            code = max(0, code) if signed else 0 if bits == 0 else max(1, code)
            assert int(state.exponents[i // 128]) == e and abs(int(state.codes[i])) == code <= most
            assert code == 0 or (int(state.codes[i]) < 0) == (float(values[i]) < 0)
        got, = optim.state8_values([state])
        assert torch.equal(got.double(), gated_math.code_values(*state))


def test_codes_are_unbiased():
    """A value's codes are its neighbours, each as often as it is near."""
    n = 1 << 16
    x = torch.full((n,), 1.3)
    state = optim.state8_zeros(x, False)
    optim._encode(x, state, torch.randint(0, 1 << 20, (n,), generator=gen(3)))
    got, = optim.state8_values([state])
    assert got.unique().tolist() == [1.25, 1.375]
    # 1.3 is 0.4 of the way: the mean's deviation is 0.125 sqrt(0.24 / n); five of them.
    assert abs(float(got.double().mean()) - 1.3) <= 5 * 0.125 * math.sqrt(0.24 / n) + 1e-6


def test_second_moment_in_8_bits_follows_small_changes():
    """beta2 = 0.999 changes it by a thousandth a step, a code by an eighth of an octave."""
    p, g = [torch.zeros(1 << 12)], [torch.full((1 << 12,), 0.01)]
    m, v = zeros(p, 8)
    step = torch.zeros((), dtype=torch.int64)
    for _ in range(400):
        optim.adamw_step(p, g, m, v, step, 0.0)
    got = float(optim.state8_values(v)[0].double().mean())
    want = 1e-4 * (1 - 0.999 ** 400)
    # Each step's rounding is off by 0.04 of the value in the mean square; 400 of them that decay slowly add up to
    # 0.8 at most in one value, and 0.013 in the mean of 4096; five of them.
    assert abs(got / want - 1) <= 0.065


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step_in_8_bits(dtype):
    p, g = model(4, [(700,), (130,)], dtype)
    m, v = zeros(p, 8)
    step, lr = torch.zeros((), dtype=torch.int64), 1e-2
    for t in (1, 2, 3):
        before = [(a.clone(), gated_math.code_values(*b), gated_math.code_values(*c)) for a, b, c in zip(p, m, v)]
        optim.adamw_step(p, g, m, v, step, lr)
        for i, (x, (a, b, c)) in enumerate(zip(g, before)):
            pw, mw, vw = gated_math.adamw(a, x, b, c, t, lr, (0.9, 0.999), 1e-8, 0.0)
            if dtype == torch.float32:
                assert bool(((p[i].double() - pw).abs() <= 8 * 2.0 ** -24 * (pw.abs() + lr * 10)).all())
            else:   # up or down by less than a place: at most 2^-7 of the value
                assert bool(((p[i].double() - pw).abs() <= 2.0 ** -7 * pw.abs() + 1e-6).all())
            # A code's neighbours are an eighth of the octave apart: at most an eighth of the value.
            for got, want, floor in ((m[i], mw, 2.0 ** -14), (v[i], vw, 2.0 ** -30)):
                lowest = torch.cat([part.abs().max().expand(part.numel()) for part in want.split(128)]) * floor
                off = (gated_math.code_values(*got) - want).abs()
                assert bool((off <= 0.126 * want.abs() + lowest).all())
            # The very rounding: codes are the float's leading bits after the hash is added, and the lowest one at least.
            low = torch.tensor(gated_math.hashed(t, i, x.numel())) & 0xFFFFF
            v32 = (c.float() * 0.999 + x.float() * x.float() * (1 - 0.999))
            up = ((v32.view(torch.int32).long() + low) >> 20 << 20).int().view(torch.float32)
            first = (8 * v[i].exponents.int() + 8 - 255).clamp_min(0) + 1 << 20
            lowest = first.view(torch.float32).repeat_interleave(128)[:x.numel()]
            up = torch.where(v32 > 0, torch.maximum(up, lowest), up)
            assert torch.equal(optim.state8_values([v[i]])[0], up)


def test_nothing_but_its_group_is_lost_to_a_value_that_is_not_finite():
    p, g = model(5, [(400,)])
    m, v = zeros(p, 8)
    g[0][130], g[0][300] = float("nan"), float("inf")
    optim.adamw_step(p, g, m, v, torch.zeros((), dtype=torch.int64), 1e-3)
    for x in optim.state8_values([m[0], v[0]]):
        assert bool(x[128:384].isnan().all()) and bool(x[:128].isfinite().all()) and bool(x[384:].isfinite().all())
    assert p[0].isfinite().logical_not().nonzero().flatten().tolist() == [130, 300]


@pytest.mark.parametrize("clip", [None, 0.05])
def test_class_agrees_with_torch(clip):
    torch.manual_seed(0)
    a = torch.nn.Sequential(torch.nn.Linear(7, 20), torch.nn.ELU(), torch.nn.Linear(20, 3))
    b = copy.deepcopy(a)
    groups = lambda net: [dict(params=list(net[0].parameters()), lr=1e-2), dict(params=list(net[2].parameters()), weight_decay=0.0)]
    mine = optim.AdamW(groups(a), lr=3e-3, weight_decay=0.1, max_grad_norm=clip)
    other = torch.optim.AdamW(groups(b), lr=3e-3, weight_decay=0.1)
    x = torch.randn(30, 7)
    for _ in range(10):
        for net, opt in ((a, mine), (b, other)):
            opt.zero_grad()
            net(x).square().sum().backward()
            if clip is not None and opt is other:
                torch.nn.utils.clip_grad_norm_(net.parameters(), clip)
            opt.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.allclose(p, q, rtol=1e-4, atol=1e-6)


@pytest.mark.parametrize("bits,dtype", [(32, torch.bfloat16), (8, torch.float32), (8, torch.bfloat16)])
def test_class_goes_on_from_a_state_dict(bits, dtype):
    p, g = model(6, [(150,), (3, 4)], dtype)
    runs = []
    for again in (False, True):
        params = [torch.nn.Parameter(x.clone()) for x in p]
        opt = optim.AdamW(params, lr=1e-2, bits=bits, max_grad_norm=1.0)
        for k in range(4):
            if again and k == 2:
                saved, opt = opt.state_dict(), optim.AdamW(params, lr=1.0, bits=bits, max_grad_norm=1.0)
                opt.load_state_dict(copy.deepcopy(saved))
            for x, y in zip(params, g):
                x.grad = y * (k + 1)
            assert opt.step(lambda: 5.0) == 5.0
        runs.append([x.detach() for x in params] + [t for x in params for t in opt.state[x].values()])
        assert int(opt.param_groups[0]["step"]) == 4
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(*runs))


@pytest.mark.parametrize("kind", [torch.optim.Adam, torch.optim.AdamW])
def test_class_goes_on_from_torch(kind):
    p, g = model(8, [(150,), (3, 4)])
    results = []
    for switch in (False, True):
        params = [torch.nn.Parameter(x.clone()) for x in p]
        opt = kind(params, lr=1e-2, weight_decay=0.0)
        for k in range(6):
            if switch and k == 3:
                saved, opt = opt.state_dict(), optim.AdamW(params, bits=8)
                opt.load_state_dict(saved)
            for x, y in zip(params, g):
                x.grad = y * (k + 1)
            opt.step()
        results.append([x.detach() for x in params])
    assert int(opt.param_groups[0]["step"]) == 6 and opt.param_groups[0]["bits"] == 32
    for a, b in zip(*results):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)


def test_parameters_without_gradients():
    params = [torch.nn.Parameter(torch.ones(3)), torch.nn.Parameter(torch.ones(3))]
    opt = optim.AdamW(params, lr=0.1)
    opt.step()
    params[0].grad = torch.ones(3)
    opt.step()
    assert bool((params[0] < 1).all()) and torch.equal(params[1].detach(), torch.ones(3)) and params[1] not in opt.state


def test_refusals():
    p, g = model(7, [(10,), (4, 5)])
    m, v = zeros(p, 32)
    m8, v8 = zeros(p, 8)
    one = torch.zeros((), dtype=torch.int64)
    fine = dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, step=one, lr=1e-3)
    both = torch.zeros(15)
    bad = [
        dict(params=[]), dict(grads=g[:1]), dict(params=[x.double() for x in p]), dict(params=[p[0], p[1].t()]),
        dict(grads=[g[0], g[1][:2]]), dict(grads=[g[0].bfloat16(), g[1]]), dict(exp_avgs=[m[0], m[1].double()]),
        dict(exp_avgs=m8), dict(exp_avgs=[m8[0], m[1]], exp_avg_sqs=v8), dict(exp_avgs=v8, exp_avg_sqs=v8),
        dict(exp_avgs=m8, exp_avg_sqs=[v8[0], optim.State8(v8[1].codes, torch.zeros(2, dtype=torch.uint8))]),
        dict(params=[p[0], p[0]], grads=[g[0], g[0]], exp_avgs=[m[0], m[0].clone()], exp_avg_sqs=[v[0], v[0].clone()]),
        dict(params=[both[:10], both[5:]], grads=[g[0], g[0]], exp_avgs=[m[0], m[0].clone()],
             exp_avg_sqs=[v[0], v[0].clone()]),
        dict(exp_avg_sqs=m), dict(grads=[p[0], g[1]]), dict(step=0), dict(step=torch.zeros(())), dict(step=torch.zeros(2, dtype=torch.int64)),
        dict(lr=torch.zeros(2)), dict(betas=(0.9, 1.0)), dict(eps=-1.0), dict(weight_decay=float("nan")), dict(max_norm=-1.0),
        dict(max_norm=float("nan")),
    ]
    for i, change in enumerate(bad):
        with pytest.raises(RuntimeError):
            optim.adamw_step(**{**fine, **change})
            pytest.fail(f"case {i} was accepted")
    optim.adamw_step(**fine)
    with pytest.raises(RuntimeError):
        optim.state8_values([optim.State8(torch.zeros(4, dtype=torch.int16), torch.zeros(1, dtype=torch.uint8))])
    assert optim.state8_values([]) == []
    for wrong in (dict(bits=16), dict(max_grad_norm=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **wrong)


def test_packed_arguments_have_the_sizes_of_the_c_structs(tmp_path):
    got = offsets(tmp_path, "duck_adamw_tensor", ("param", "exp_avg_sq", "exp_avg_sq_exponents", "n", "type", "place"))
    assert got == [0, 24, 40, 48, 56, 60, optim._TENSOR.size]
    got = offsets(tmp_path, "duck_adamw", ("step", "sums", "rate_value", "max_norm", "sum_count", "bits"))
    assert got == [0, 16, 24, 64, 72, 76, optim._OPTIONS.size]
