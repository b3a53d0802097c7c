"""GPU: the optimizer's kernels (duck_gym_b200/optim.py) against float64
restatements (tests/gated_math.py) and, for codes, bit for bit against the plain
form on the CPU, whose own tests are in test_optim.py."""

import copy
import math

import pytest
import torch

import gated_math
from duck_gym_b200 import optim

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def model(seed, sizes, dtype=torch.float32):
    """Parameters, gradients and float32 moments of a run that has gone on for a while."""
    g = gen(seed)
    draw = lambda n, scale: scale * torch.randn(n, generator=g) * torch.exp(torch.randn(n, generator=g))
    return ([(0.1 * torch.randn(n, generator=g)).to(dtype) for n in sizes], [draw(n, 0.01).to(dtype) for n in sizes],
            [draw(n, 0.003) for n in sizes], [draw(n, 0.01).square() for n in sizes])


def eight(ms, vs):
    out = [[], []]
    for signed, xs, to in ((True, ms, out[0]), (False, vs, out[1])):
        for x in xs:
            to.append(optim.state8_zeros(x, signed))
            optim._encode(x, to[-1], torch.tensor(1 << 19))
    return out


def put(x):
    return type(x)(*map(put, x)) if isinstance(x, optim.State8) else [put(t) for t in x] if isinstance(x, list) else x.cuda()


def copied(x):
    return type(x)(*map(copied, x)) if isinstance(x, optim.State8) else [copied(t) for t in x] if isinstance(x, list) else x.clone()


def counter(n):
    return torch.full((), n, dtype=torch.int64)


SIZES = [[1], [14], [128], [129], [5000], [2048, 2049, 0, 4096], [61 * 512, 512, 3, 127, 100001], [0, 0]]


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_step_in_32_bits(sizes, dtype, max_norm):
    p, g, m, v = model(sum(sizes), sizes, dtype)
    lr, wd, betas, eps = 3e-3, 0.1, (0.9, 0.99), 1e-7
    clip = 1.0 if max_norm is None else min(1.0, max_norm / (math.sqrt(sum(float(x.double().square().sum()) for x in g)) + 1e-6))
    dev, step = put([p, g, m, v]), counter(7).cuda()
    optim.adamw_step(*dev, step, lr, betas, eps, wd, max_norm)
    assert int(step) == 8
    for (pd, gd, md, vd), (a, x, b, c) in zip(zip(*dev), zip(p, g, m, v)):
        assert torch.equal(gd.cpu(), x)
        pw, mw, vw = gated_math.adamw(a, x, b, c, 8, lr, betas, eps, wd, clip)
        # m: terms of both signs, each rounded three times, and their sum.
        assert bool(((md.cpu().double() - mw).abs() <= 4 * 2.0 ** -24 * (b.double().abs() + x.double().abs())).all())
        assert bool(((vd.cpu().double() - vw).abs() <= 6 * 2.0 ** -24 * vw).all())
        # The step itself: m's error over sqrt(v) (both at least (1 - beta) of the same gradient), and approximations of 2^-20.
        step_size = lr / (1 - betas[0] ** 8) / ((vw / (1 - betas[1] ** 8)).sqrt() + eps)
        slack = step_size * (4 * 2.0 ** -24 * (b.double().abs() + x.double().abs()) + 2.0 ** -19 * mw.abs())
        slack = slack + 4 * 2.0 ** -24 * a.double().abs()
        if dtype == torch.bfloat16:   # up or down by less than a place
            slack = slack + 2.0 ** -7 * pw.abs()
        assert bool(((pd.cpu().double() - pw).abs() <= slack + 1e-30).all())


@pytest.mark.parametrize("max_norm", [None, 0.5])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", SIZES)
def test_step_in_8_bits(sizes, dtype, max_norm):
    """Codes and exponents are those of the plain form, bit for bit, step after step."""
    p, g, m, v = model(sum(sizes) + 1, sizes, dtype)
    m, v = eight(m, v)
    dev, step, here = put([p, g, m, v]), counter(0).cuda(), counter(0)
    for t in range(3):
        old = copied(p)
        optim.adamw_step(*dev, step, 3e-3, max_norm=max_norm, weight_decay=0.1)
        optim.adamw_step(p, g, m, v, here, 3e-3, max_norm=max_norm, weight_decay=0.1)
        for (pd, _, md, vd), (a, x, b, c), was in zip(zip(*dev), zip(p, g, m, v), old):
            for got, want in zip((*md, *vd), (*b, *c)):
                assert got.dtype == want.dtype and torch.equal(got.cpu(), want)
            # The parameter: two roundings of 2^-24 of its old and its new value on either side, and the step itself, whose
            # root and quotient are approximated to 2^-21 each (moments of different seeds: a step may be a thousand times
            # lr).  Where bfloat16 is rounded by the same random bits, one place where they decide otherwise.
            a, was = a.float(), was.float()
            slack = 2.0 ** -22 * (a.abs() + was.abs()) + 2.0 ** -19 * (a - was).abs()
            slack = slack + (2.0 ** -7 * a.abs() if dtype == torch.bfloat16 else 0)
            assert bool(((pd.cpu().float() - a).abs() <= slack + 1e-12).all())
            pd.copy_(a.to(dtype))   # differences do not add up
    assert int(step) == 3
    for got, want in zip(optim.state8_values(dev[2] + dev[3]), m + v):
        assert torch.equal(got.cpu().double(), gated_math.code_values(*want))


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_types_and_places(bits):
    """More than a launch's arguments hold, float32 and bfloat16 ones, on every boundary; the same as each by itself."""
    sizes = [1 + (37 * i) % 700 for i in range(1000)]
    p, g, m, v = model(3, sizes)
    for i in range(0, 1000, 3):
        p[i], g[i] = p[i].bfloat16(), g[i].bfloat16()
    shift = lambda x, k: torch.cat((x.new_zeros(k), x)).cuda()[k:]
    m, v = eight(m, v) if bits == 8 else (m, v)
    move = lambda s, k: optim.State8(shift(s.codes, k), shift(s.exponents, k)) if bits == 8 else shift(s, k)
    dev = [[shift(x, i % 4) for i, x in enumerate(p)], [shift(x, i % 3) for i, x in enumerate(g)],
           [move(x, i % 5) for i, x in enumerate(m)], [move(x, i % 2) for i, x in enumerate(v)]]
    apart = put([p, g, m, v])
    step = counter(4).cuda()
    optim.adamw_step(*dev, step, 1e-2, max_norm=0.7)
    assert int(step) == 5
    again = put([p, g, m, v])
    optim.adamw_step(*again, counter(4).cuda(), 1e-2, max_norm=0.7)
    flat = lambda x: [t for s in x for t in (flat(s) if isinstance(s, (list, tuple)) else [s])]
    assert all(torch.equal(a, b) for a, b in zip(flat(dev), flat(again)))   # whatever the boundaries
    here = counter(4)
    optim.adamw_step(p, g, m, v, here, 1e-2, max_norm=0.7)
    del apart
    for a, b in zip(flat(dev[2:]), flat([m, v])):
        assert torch.equal(a.cpu(), b) if bits == 8 else torch.allclose(a.cpu(), b, rtol=1e-6, atol=1e-12)
    for a, b in zip(dev[0], p):
        assert bool(((a.cpu().float() - b.float()).abs() <= 2.0 ** -7 * b.float().abs() + 1e-7).all()) and a.dtype == b.dtype
        assert a.dtype != torch.float32 or torch.allclose(a.cpu(), b, rtol=1e-6, atol=1e-7)


def test_values_that_are_not_finite():
    p, g, m, v = model(5, [400, 400])
    m, v = eight(m, v)
    g[0][130], g[0][300], g[0][301] = float("nan"), float("inf"), 3e19   # the last one's square is infinite
    dev = put([p, g, m, v])
    optim.adamw_step(*dev, counter(3).cuda(), 1e-3)
    mm, vv = (optim.state8_values(s) for s in dev[2:])
    assert bool(mm[0][128:384].isnan().all()) and bool(vv[0][128:384].isnan().all())
    for x in (mm[0], vv[0]):
        assert bool(x[:128].isfinite().all()) and bool(x[384:].isfinite().all())
    assert bool(mm[1].isfinite().all()) and bool(dev[0][1].isfinite().all())
    assert dev[0][0].isfinite().logical_not().nonzero().flatten().tolist() == [130, 300]
    # Clipped by a norm that is not a number: everything is one, as with torch's.
    dev = put([p, g, *eight(*model(5, [400, 400])[2:])])
    optim.adamw_step(*dev, counter(3).cuda(), 1e-3, max_norm=1.0)
    assert bool(dev[0][1].isnan().all())
    # Nothing at all: zero gradients and moments leave the parameters.
    zero = torch.zeros(300, device="cuda")
    state = [optim.state8_zeros(zero, True)], [optim.state8_zeros(zero, False)]
    at = torch.ones(300, device="cuda")
    optim.adamw_step([at], [zero], *state, counter(0).cuda(), 1.0, max_norm=0.0)
    assert bool((at == 1).all()) and bool((state[1][0].codes == 0).all())


def test_bfloat16_parameters_are_rounded_without_bias():
    n = 1 << 20
    p, g = torch.ones(n, dtype=torch.bfloat16, device="cuda"), torch.ones(n, dtype=torch.bfloat16, device="cuda")
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    optim.adamw_step([p], [g], [m], [v], counter(0).cuda(), 1e-3)
    # 1 - 0.001 is 0.256 of the way to the next number below, 1 - 2^-8: the mean's deviation is 2^-8 sqrt(0.19 / n).
    assert sorted(p.float().unique().tolist()) == [1 - 2.0 ** -8, 1.0]
    assert abs(float(p.double().mean()) - 0.999) <= 5 * 2.0 ** -8 * math.sqrt(0.2 / n) + 1e-7


def test_more_values_than_32_bits_count():
    n = (1 << 31) + 200
    p = torch.ones(n, dtype=torch.bfloat16, device="cuda")
    g = torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    m, v = [optim.state8_zeros(p, True)], [optim.state8_zeros(p, False)]
    g[-1] = 2.0
    optim.adamw_step([p], [g], m, v, counter(0).cuda(), 0.5, max_norm=1e6)
    assert bool((p[-300:].float() == 0.5).all()) and bool((p[:300].float() == 0.5).all())   # a first step is lr, whatever g
    tail = optim.State8(m[0].codes[-200:].clone(), m[0].exponents[-2:].clone())
    got, = optim.state8_values([tail])
    assert abs(float(got[-1]) / 0.2 - 1) <= 0.126 and bool(((got[:-1] / 0.05 - 1).abs() <= 0.126).all())
    assert int((v[0].codes == 0).sum()) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_streams_graphs_and_the_same_bits(bits):
    p, g, m, v = model(9, [5000, 61, 300])
    m, v = eight(m, v) if bits == 8 else (m, v)
    start = put([p, g, m, v])
    rate = torch.full((), 1e-2, device="cuda")
    flat = lambda x: [t for s in x for t in (flat(s) if isinstance(s, (list, tuple)) else [s])]

    def steps(state, count, n):
        for _ in range(n):
            optim.adamw_step(*state, count, rate, max_norm=0.3, weight_decay=0.01)

    want, count = copied(start), counter(0).cuda()
    steps(want, count, 3)
    other, side = copied(start), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        steps(other, counter(0).cuda(), 3)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(flat(want), flat(other)))
    state, count = copied(start), counter(0).cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        steps(state, count, 1)
    assert int(count) == 0
    for _ in range(3):
        graph.replay()
    assert int(count) == 3 and all(torch.equal(a, b) for a, b in zip(flat(want), flat(state)))
    rate.fill_(0.0)   # a schedule on the device is seen by the graph
    before = [t.clone() for t in state[0]]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(before, state[0])) and int(count) == 4


def test_class_on_the_gpu():
    torch.manual_seed(0)
    a = torch.nn.Sequential(torch.nn.Linear(61, 200), torch.nn.ELU(), torch.nn.Linear(200, 3)).cuda()
    b, c = copy.deepcopy(a), copy.deepcopy(a)
    nets = [(a, optim.AdamW(a.parameters(), lr=3e-3, weight_decay=0.1, max_grad_norm=0.5)),
            (b, torch.optim.AdamW(b.parameters(), lr=3e-3, weight_decay=0.1)),
            (c, optim.AdamW([dict(params=[p]) for p in c.parameters()], lr=3e-3, weight_decay=0.1, max_grad_norm=0.5))]
    x = torch.randn(300, 61, device="cuda")
    for _ in range(10):
        for net, opt in nets:
            opt.zero_grad()
            net(x).square().mean().backward()
            if net is b:
                torch.nn.utils.clip_grad_norm_(net.parameters(), 0.5)
            opt.step()
    for p, q, r in zip(a.parameters(), b.parameters(), c.parameters()):
        assert torch.allclose(p, q, rtol=1e-4, atol=1e-6) and torch.allclose(p, r, rtol=1e-5, atol=1e-7)


@pytest.mark.parametrize("bits", [32, 8])
def test_class_goes_on_from_a_state_dict(bits):
    p, g, _, _ = model(6, [1500, 12], torch.bfloat16)
    runs = []
    for again in (False, True):
        params = [torch.nn.Parameter(x.cuda()) for x in p]
        opt = optim.AdamW(params, lr=1e-2, bits=bits, max_grad_norm=1.0)
        for k in range(4):
            if again and k == 2:
                saved, opt = opt.state_dict(), optim.AdamW(params, lr=1.0, bits=bits, max_grad_norm=1.0)
                on_host = torch.utils._pytree.tree_map(lambda t: t.cpu() if torch.is_tensor(t) else t, saved)
                opt.load_state_dict(on_host)
            for x, y in zip(params, g):
                x.grad = y.cuda() * (k + 1)
            opt.step()
        runs.append([x.detach() for x in params] + [t for x in params for t in opt.state[x].values()])
    assert all(a.dtype == b.dtype and torch.equal(a, b) for a, b in zip(*runs))


def test_a_step_is_seen_by_autograd():
    p, m, v = (torch.ones(40, device="cuda") for _ in range(3))
    p.requires_grad_()
    y = (p * p).sum()
    optim.adamw_step([p], [torch.ones(40, device="cuda")], [m], [v], counter(0).cuda(), 0.1)
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_refusals_on_the_gpu():
    import ctypes

    from duck_gym_b200.cuda_batch import library

    p, g, m, v = put(list(model(7, [10, 200])))
    one = counter(0).cuda()
    fine = dict(params=p, grads=g, exp_avgs=m, exp_avg_sqs=v, step=one, lr=1e-3)
    half = [x.half() for x in p]
    bad = [dict(params=half, grads=half), dict(grads=[x.cpu() for x in g]), dict(exp_avgs=[x.cpu() for x in m]),
           dict(step=counter(0)), dict(params=[p[0].cpu(), p[1]]), dict(lr=torch.zeros((), dtype=torch.int64, device="cuda"))]
    for i, change in enumerate(bad):
        with pytest.raises(RuntimeError):
            optim.adamw_step(**{**fine, **change})
            pytest.fail(f"case {i} was accepted")
    lib = library()
    row = [p[0].data_ptr(), g[0].data_ptr(), m[0].data_ptr(), v[0].data_ptr(), 0, 0, 10, 0, 0]
    options = [one.data_ptr(), 0, 0, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 0, 32]
    change = lambda x, i, y: x[:i] + [y] + x[i + 1:]
    for r, o in ((change(row, 0, 0), options), (change(row, 3, 0), options), (change(row, 6, -1), options),
                 (change(row, 7, 2), options), (change(row, 8, -1), options), (row, change(options, 0, 0)),
                 (row, change(options, 0, one.data_ptr() + 4)), (row, change(options, 4, 1.0)), (row, change(options, 6, float("nan"))),
                 (row, change(options, 9, 1)), (row, change(options, 9, 593)), (row, change(options, 10, 16)),
                 (row, change(options, 10, 8)), (row, change(options, 3, float("inf")))):
        assert lib.duck_adamw_step(optim._TENSOR.pack(*r), 1, optim._OPTIONS.pack(*o), None) != 0
    assert lib.duck_adamw_step(None, 1, optim._OPTIONS.pack(*options), None) != 0
    assert lib.duck_adamw_step(optim._TENSOR.pack(*row), 1, None, None) != 0
    count = ctypes.c_int()
    assert lib.duck_gradient_squares(optim._TENSOR.pack(*change(row, 1, 0)), 1, 0, one.data_ptr(), ctypes.byref(count), None) != 0
    assert lib.duck_gradient_squares(optim._TENSOR.pack(*row), 1, 593, one.data_ptr(), ctypes.byref(count), None) != 0
    assert lib.duck_gradient_squares(optim._TENSOR.pack(*row), 1, 0, None, ctypes.byref(count), None) != 0
    assert lib.duck_moment_values(optim._TENSOR.pack(*row), 1, None) != 0
    assert int(one) == 0
