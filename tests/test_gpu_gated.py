"""GPU: the gated operators' kernels (duck_gym_b200/memory.py) against float64
restatements (tests/gated_math.py), at the sizes, masks, strides and values where
they can go wrong, and their refusals."""

import pytest
import torch

import gated_math
import memory_math as ref
from duck_gym_b200 import memory

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


# ------------------------------------------------------------ gated recurrence
# A bfloat16 gate's exponential and quotient are off by some 2^-20 each; states and
# sums are float32, so that only the results' own rounding is left.
def rounded(dtype, T):
    return ref.bound(dtype, T) + ref.bound(torch.float32, T)


def rollout(seed, T, E, N, dtype, resets=0.05):
    g = gen(seed)
    gates = (normal(g, T, E, N) + 2 * torch.rand(N, generator=g)).to(dtype)
    values, dout = normal(g, T, E, N, dtype=dtype), normal(g, T, E, N, dtype=dtype)
    return gates, values, normal(g, E, N), torch.rand(T, E, generator=g) < resets, dout, normal(g, E, N)


def check(gates, values, state, resets, dout, dlast, devices=None):
    """Outputs and gradients of one call; returns them."""
    put = lambda t: None if t is None else t.cuda()
    dev = [put(t) for t in (gates, values, state)] if devices is None else devices
    for t in dev:
        if t is not None:
            t.requires_grad_()
    out, last = memory.gated_recurrence(*dev, put(resets), final_state=dlast is not None)
    assert out.dtype == gates.dtype and out.is_contiguous() and (last is None) == (dlast is None)
    leaves = [t for t in dev if t is not None]
    outs = [o for o, d in ((out, dout), (last, dlast)) if d is not None]
    grads = torch.autograd.grad(outs, leaves, [put(d) for d in (dout, dlast) if d is not None])
    want = gated_math.recurrence(gates, values, state, resets, dout, dlast)
    T, dtype = gates.shape[0], gates.dtype
    for got, exact in zip((out, *grads[:2]), (want[0], *want[2:4])):
        assert got.dtype == dtype and ref.error(got, exact) <= rounded(dtype, T)
    wide = rounded(torch.float32, T) if dtype == torch.float32 else 1e-5
    if last is not None:
        assert ref.error(last, want[1]) <= wide
    if state is not None:
        assert ref.error(grads[2], want[4]) <= wide
    return [out, *grads] + ([] if last is None else [last])


# Chunks of 8 and 16 steps, one to four channels at once (four from 148 x 2048 channels on), steps that are split.
SIZES = [(1, 1, 1), (2, 3, 5), (8, 1, 2), (9, 2, 6), (15, 2, 7), (16, 4, 8), (17, 1, 61), (24, 33, 64), (33, 5, 130),
         (127, 2, 24), (128, 2, 24), (129, 3, 61), (1000, 1, 8), (4099, 1, 3), (700, 9, 256), (19, 1200, 256), (5, 9999, 31)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,N", SIZES)
def test_recurrence(T, E, N, dtype):
    case = rollout(T * 1009 + N, T, E, N, dtype)
    first = check(*case)
    again = check(*case)
    assert all(torch.equal(a, b) for a, b in zip(first, again))   # bit for bit
    gates, values, state, resets, _, _ = case
    with torch.no_grad():   # nothing is kept then
        out, last = memory.gated_recurrence(gates.cuda(), values.cuda(), state.cuda(), resets.cuda())
    assert torch.equal(out, first[0]) and torch.equal(last, first[-1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [5, 300])
def test_recurrence_without_state_resets_or_some_gradients(T, dtype):
    gates, values, state, resets, dout, dlast = rollout(T, T, 3, 20, dtype)
    check(gates, values, None, None, dout, None)
    check(gates, values, None, resets, dout, dlast)
    check(gates, values, state, None, None, dlast)
    check(gates, values, state, resets.to(torch.uint8) * 3, dout, None)
    check(gates, values, state, torch.ones_like(resets), dout, dlast)   # an episode at every step: no state is left
    resets = torch.zeros_like(resets)
    resets[T // 2] = True
    check(gates, values, state, resets, dout, dlast)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,N", [(20, 4, 32), (200, 3, 30), (130, 2, 7)])
def test_recurrence_strides(T, E, N, dtype):
    gates, values, state, resets, dout, dlast = rollout(T, T, E, N, dtype)
    both = torch.cat((gates, values), -1).cuda()
    halves = [both[..., :N].detach(), both[..., N:].detach()]   # of one projection
    check(gates, values, state, resets, dout, dlast, [*halves, state.cuda()])
    turned = [t.transpose(0, 1).contiguous().cuda().transpose(0, 1).detach() for t in (gates, values)]
    check(gates, values, state, resets, dout, dlast, [*turned, state.cuda()])
    odd = torch.empty(T * E * N + 1, dtype=dtype, device="cuda")[1:].view(T, E, N)
    odd.copy_(gates)
    check(gates, values, state, resets, dout, dlast, [odd.detach(), values.cuda(), state.cuda()])
    one = gates[:1].expand(T, E, N)   # one gate for all steps: strides of zero
    check(one, values, state, resets, dout, dlast, [gates[:1].cuda().expand(T, E, N).detach(), values.cuda(), state.cuda()])
    columns = values.permute(2, 0, 1).contiguous().cuda().permute(1, 2, 0).detach()   # the last axis is not dense
    check(gates, values, state, resets, dout, dlast, [gates.cuda(), columns, state.cuda()])
    shifted = torch.empty(E * N + 1, device="cuda")[1:].view(E, N)
    shifted.copy_(state)
    check(gates, values, state, resets, dout, dlast, [gates.cuda(), values.cuda(), shifted.detach()])
    # The gradient of a sum has strides of zero.
    leaf = gates.cuda().requires_grad_()
    out, _ = memory.gated_recurrence(leaf, values.cuda(), state.cuda(), resets.cuda())
    out.float().sum().backward()
    want = gated_math.recurrence(gates, values, state, resets, torch.ones(T, E, N))
    assert ref.error(leaf.grad, want[2]) <= rounded(dtype, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [40, 400])
def test_recurrence_reset_drops_what_is_not_finite(T, dtype):
    gates, values, state, resets, dout, dlast = rollout(T, T, 2, 4, dtype, resets=0.0)
    state[0, 1], values[5, 0, 0], gates[6, 0, 2] = float("inf"), float("nan"), float("nan")
    dout[T - 5, 0, 0], dlast[0, 1] = float("nan"), float("inf")
    resets[T // 2, 0] = True
    leaves = [t.cuda().requires_grad_() for t in (gates, values, state)]
    out, last = memory.gated_recurrence(*leaves, resets.cuda())
    grads = torch.autograd.grad((out, last), leaves, (dout.cuda(), dlast.cuda()))
    assert bool(out[T // 2:].isfinite().all()) and bool(last.isfinite().all())
    assert not bool(out[T // 2 - 1, 0, :3].isfinite().any()) and bool(out[:, 1].isfinite().all())
    # What later steps give back does not pass the reset either; a gate's gradient has the state before it as a factor.
    assert bool(grads[1][8:T // 2].isfinite().all()) and bool(grads[0][8:T // 2, 0, 3].isfinite().all())
    assert bool(grads[0][:, 1].isfinite().all()) and bool(grads[1][:, 1].isfinite().all())
    assert bool(grads[2][1].isfinite().all()) and bool(grads[2][0, 0].isfinite())


@pytest.mark.parametrize("dtype", TYPES)
def test_recurrence_gates_at_the_ends(dtype):
    """Gates that hold the state for good, or replace it, at infinity too."""
    inf = float("inf")
    gates = torch.tensor([300.0, -300.0, inf, -inf, 60.0, -60.0, 0.0, 15.0]).to(dtype).expand(200, 1, 8).contiguous()
    _, values, state, resets, dout, dlast = rollout(3, 200, 1, 8, dtype, resets=0.0)
    out = check(gates, values, state, resets, dout, dlast)[0].cpu()
    assert torch.equal(out[:, 0, 2].float(), state[0, 2].to(dtype).float().expand(200))
    assert torch.equal(out[:, 0, 3], values[:, 0, 3])


def test_recurrence_empty():
    state = torch.randn(2, 3, device="cuda", requires_grad=True)
    x = torch.zeros(0, 2, 3, device="cuda", requires_grad=True)
    out, last = memory.gated_recurrence(x, x, state)
    assert out.shape == (0, 2, 3) and torch.equal(last, state) and last.data_ptr() != state.data_ptr()
    d, = torch.autograd.grad(last, state, torch.ones_like(last))
    assert torch.equal(d, torch.ones_like(d))
    assert float(memory.gated_recurrence(x.detach(), x.detach())[1].abs().sum()) == 0.0
    for shape in ((4, 0, 3), (4, 2, 0)):
        y = torch.zeros(shape, device="cuda", requires_grad=True)
        out, last = memory.gated_recurrence(y, y)
        assert out.shape == shape and last.shape == shape[1:]
        torch.autograd.grad(out.sum(), y)
    assert memory.gated_recurrence_step(y[0].detach(), y[0].detach(), torch.zeros(2, 0, device="cuda")).shape == (2, 0)


def test_recurrence_of_many_values():
    """Offsets beyond 2^31 elements."""
    T, E, N = 9, 65536, 4096
    gates = torch.zeros(T, E, N, dtype=torch.bfloat16, device="cuda")
    values = torch.empty(T, E, N, dtype=torch.bfloat16, device="cuda").normal_()
    resets = torch.zeros(T, E, dtype=torch.bool, device="cuda")
    resets[4, E - 1] = True
    values.requires_grad_()
    out, last = memory.gated_recurrence(gates, values, None, resets)
    want = gated_math.recurrence(torch.zeros(T, 1, N), values[:, E - 1:].detach().cpu(), None, resets[:, E - 1:].cpu())
    assert ref.error(out[:, E - 1:], want[0]) <= rounded(torch.bfloat16, T) and ref.error(last[E - 1:], want[1]) <= 1e-5
    dout = torch.ones((), dtype=torch.bfloat16, device="cuda").expand(T, E, N)
    dv, = torch.autograd.grad(out, values, dout)
    want = gated_math.recurrence(torch.zeros(T, 1, N), values[:, E - 1:].detach().cpu(), None, resets[:, E - 1:].cpu(),
                                 torch.ones(T, 1, N))
    assert ref.error(dv[:, E - 1:], want[3]) <= rounded(torch.bfloat16, T)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,N", [(1, 1), (3, 5), (16, 64), (301, 61), (4096, 256)])
def test_recurrence_step(E, N, dtype):
    gates, values, state, resets, _, _ = rollout(E + N, 3, E, N, dtype, resets=0.3)
    state[0, 0], resets[0, 0] = float("nan"), True
    moving = state.cuda()
    odd = torch.empty(E * N + 1, device="cuda")[1:].view(E, N)   # a state on a 4-byte boundary
    odd.copy_(state)
    wide = torch.cat((gates, values), -1).cuda()
    before = moving._version
    for t in range(3):
        want, last = gated_math.recurrence(gates[t:t + 1], values[t:t + 1], moving.cpu(), resets[t:t + 1])
        out = memory.gated_recurrence_step(gates[t].cuda(), values[t].cuda(), moving, resets[t].cuda())
        other = memory.gated_recurrence_step(wide[t, :, :N], wide[t, :, N:], odd, resets[t].cuda())
        assert out.dtype == dtype and ref.error(out, want[0]) <= rounded(dtype, 1)
        assert ref.error(moving, last) <= 1e-5 and torch.equal(out, other) and torch.equal(moving, odd)
    assert moving._version == before + 3
    memory.gated_recurrence_step(gates[0].cuda(), values[0].cuda(), moving)


def test_recurrence_and_a_step_on_its_state():
    gates, values, state, resets, dout, _ = rollout(1, 24, 2, 8, torch.float32)
    leaves, moving = [t.cuda().requires_grad_() for t in (gates, values)], state.cuda()
    out, _ = memory.gated_recurrence(*leaves, moving)
    memory.gated_recurrence_step(gates[0].cuda(), values[0].cuda(), moving)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(out, leaves, dout.cuda())


def test_recurrence_refuses_second_and_forward_mode_derivatives():
    from torch.autograd import forward_ad

    x, state = torch.randn(4, 3, 8, device="cuda"), torch.randn(3, 8, device="cuda")
    leaf = x.clone().requires_grad_()
    d, = torch.autograd.grad(memory.gated_recurrence(leaf, x)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: memory.gated_recurrence(dual, x), lambda: memory.gated_recurrence(x, dual),
                             lambda: memory.gated_recurrence_step(dual[0], x[0], state)):
                    with pytest.raises(RuntimeError):
                        call()


@pytest.mark.parametrize("T", [24, 600])
def test_recurrence_on_another_stream_and_in_a_graph(T):
    case = [t.cuda() for t in rollout(T, T, 4, 64, torch.bfloat16)]
    gates, values, state, resets, dout, dlast = case

    def everything():
        leaves = [t.detach().requires_grad_() for t in (gates, values, state)]
        out, last = memory.gated_recurrence(*leaves, resets)
        moving = state.clone()
        step = memory.gated_recurrence_step(gates[0], values[0], moving, resets[0])
        return [out, last, *torch.autograd.grad((out, last), leaves, (dout, dlast)), step, moving]

    want = everything()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything()
    for t in captured:
        t.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, captured))


def test_recurrence_refusals_on_the_gpu():
    from duck_gym_b200.cuda_batch import library

    x, state = torch.zeros(4, 2, 8, device="cuda"), torch.zeros(2, 8, device="cuda")
    bad = [lambda: memory.gated_recurrence(x.half(), x.half()), lambda: memory.gated_recurrence(x.double(), x.double()),
           lambda: memory.gated_recurrence(x, x.cpu()), lambda: memory.gated_recurrence(x, x, state.cpu()),
           lambda: memory.gated_recurrence(x, x, state.bfloat16()),
           lambda: memory.gated_recurrence(x, x, state, torch.zeros(4, 2, dtype=torch.bool)),
           lambda: memory.gated_recurrence_step(x[0], x[0], torch.zeros(8, 2, device="cuda").t())]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    lib, p = library(), x.data_ptr()
    pack = lambda pointers, T, E, N, kind: memory._RECURRENCE.pack(*pointers, *(E * N, N) * 3, T, E, N, kind)
    fine = [p, p, p, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0]
    for pointers, sizes in (([0] + fine[1:], (4, 2, 8, 0)), (fine[:2] + [0] + fine[3:], (4, 2, 8, 0)), (fine, (4, 2, 8, 2)),
                            (fine, (-1, 2, 8, 0)), (fine, (2**31 - 1, 2, 8, 0)), (fine, (4, 65536, 65536, 0)),
                            (fine, (1000, 2, 8, 0)),                                 # steps that are split need scratch
                            (fine[:4] + [p + 4] + fine[5:], (4, 2, 8, 0))):          # a state off its boundary
        assert lib.duck_gated_recurrence_forward(pack(pointers, *sizes), None) != 0
    assert lib.duck_gated_recurrence_backward(pack(fine, 4, 2, 8, 0), None) != 0
    assert lib.duck_gated_recurrence_backward(pack([p, p, 0, 0, 0, 0, p, 0, p, p, 0, 0, p], 40, 2, 8, 0), None) != 0   # saved
    assert lib.duck_gated_recurrence_step(pack(fine, 1, 2, 8, 0), None) != 0   # state_out
    for entry in (lib.duck_gated_recurrence_forward, lib.duck_gated_recurrence_backward, lib.duck_gated_recurrence_step):
        assert entry(None, None) != 0
    assert b"Invalid" in lib.duck_last_error()


# ---------------------------------------------------------------- gated linear
# bfloat16: h and the biases' gradients have one rounding (2^-8 at most); dx and the weights' gradients are sums of
# products with da or du, rounded once, and are rounded themselves: two, which add in the mean square (memory_math.bound).
# The hardware's exponential and quotient leave 2^-20.
def layer(seed, rows, D, F, dtype, bias=True):
    g = gen(seed)
    x, wg, wu = normal(g, rows, D), normal(g, F, D) / D ** 0.5, normal(g, F, D) / D ** 0.5
    bg, bu, dh = 0.3 * normal(g, F), 0.3 * normal(g, F), normal(g, rows, F)
    x, wg, wu, bg, bu, dh = (t.to(dtype) for t in (x, wg, wu, bg, bu, dh))
    return [x, wg, wu, bg if bias else None, bu if bias else None, dh]


def check_layer(case, activation, devices=None, dh=None):
    x, wg, wu, bg, bu, _ = case
    dev = [None if t is None else t.cuda() for t in case[:5]] if devices is None else devices
    leaves = [t.requires_grad_() for t in dev if t is not None]
    h = memory.gated_linear(*dev, activation=activation)
    dtype, (rows, D), F = x.dtype, x.shape, wg.shape[0]
    assert h.dtype == dtype and h.shape == (rows, F) and h.is_contiguous()
    grads = torch.autograd.grad(h, leaves, case[5].cuda() if dh is None else dh)
    want = gated_math.linear(*case[:5], activation, case[5])
    terms = (D, 2 * F + D, rows + D, rows + D, rows + D, rows + D)
    for i, (got, exact) in enumerate(zip((h, *grads), want)):
        assert got.dtype == dtype and got.shape == exact.shape
        two = 2 if i in (1, 2, 3) else 1
        assert ref.error(got, exact) <= ref.bound(dtype, terms[i], two) + ref.bound(torch.float32, terms[i]), i
    return [h, *grads]


# Tiles of 128 rows, 64 steps, 32 to 128 features; widths off every boundary; rows that are split for the weights.
LAYERS = [(1, 1, 1), (1, 64, 64), (2, 8, 5), (3, 16, 8), (40, 8, 24), (16, 256, 512), (127, 61, 33), (128, 64, 128), (129, 72, 130), (300, 61, 301),
          (513, 200, 96), (2000, 96, 264), (2501, 130, 40), (4096, 256, 512), (19000, 128, 128), (1025, 520, 1030), (64, 1024, 2048)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,D,F", LAYERS)
def test_linear(rows, D, F, dtype):
    case = layer(rows + D + F, rows, D, F, dtype)
    activation = ["silu", "gelu", "sigmoid"][rows % 3]
    first, again = check_layer(case, activation), check_layer(case, activation)
    assert all(torch.equal(a, b) for a, b in zip(first, again))   # bit for bit
    with torch.no_grad():
        assert torch.equal(memory.gated_linear(*[t.cuda() for t in case[:5]], activation=activation), first[0])
    check_layer(layer(rows + 1, rows, D, F, dtype, bias=False), "silu")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
def test_linear_partial_gradients(activation, dtype):
    case = layer(5, 200, 64, 72, dtype)
    want = check_layer(case, activation)
    for which in ((0,), (1,), (2,), (3,), (4,), (0, 3), (1, 2)):
        dev = [t.cuda().requires_grad_(i in which) for i, t in enumerate(case[:5])]
        h = memory.gated_linear(*dev, activation=activation)
        grads = torch.autograd.grad(h, [dev[i] for i in which], case[5].cuda())
        for i, got in zip(which, grads):
            assert torch.equal(got, want[1 + i])
    frozen = [t.cuda() for t in case[:5]]
    assert not memory.gated_linear(*frozen, activation=activation).requires_grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,F", [(64, 96), (61, 35)])
def test_linear_strides(D, F, dtype):
    case = layer(D, 150, D, F, dtype)
    dev = lambda: [t.cuda() for t in case[:5]]
    x, wg, wu, bg, bu, dh = case
    wide = torch.empty(150, D + 11, dtype=dtype, device="cuda")
    wide[:, 3:3 + D] = x.cuda()
    check_layer(case, "silu", [wide[:, 3:3 + D].detach(), *dev()[1:]])
    apart = torch.empty(300, D + (-D % 8), dtype=dtype, device="cuda")[::2, :D]
    apart.copy_(x)
    check_layer(case, "silu", [apart.detach(), *dev()[1:]])
    check_layer(case, "silu", [x.t().contiguous().cuda().t().detach(), *dev()[1:]])
    both = torch.cat((wg, wu)).cuda()   # of one parameter
    check_layer(case, "silu", [dev()[0], both[:F].detach(), both[F:].detach(), *dev()[3:]])
    turned = [w.t().contiguous().cuda().t().detach() for w in (wg, wu)]
    check_layer(case, "silu", [dev()[0], *turned, *dev()[3:]])
    odd = [torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape) for t in case[:5]]
    for a, b in zip(odd, case):
        a.copy_(b)
    check_layer(case, "silu", [t.detach() for t in odd])
    same = case[:]
    same[0], same[5] = x[:1].expand(150, D), dh[:1].expand(150, F)   # rows and their gradients with strides of zero
    check_layer(same, "gelu", [x[:1].cuda().expand(150, D).detach(), *dev()[1:]], dh[:1].cuda().expand(150, F))
    loose = torch.empty(150, F + 3, dtype=dtype, device="cuda")[:, 1:1 + F]
    loose.copy_(dh)
    check_layer(case, "silu", None, loose)
    window = torch.empty(150 * 8 + D, dtype=dtype, device="cuda").normal_().as_strided((150, D), (8, 1))   # rows that overlap
    over = [window.cpu(), *case[1:]]
    check_layer(over, "silu", [window.detach(), *dev()[1:]])
    ones = case[:5] + [torch.ones(150, F, dtype=dtype)]
    check_layer(ones, "silu", None, torch.ones((), dtype=dtype, device="cuda").expand(150, F))


def test_linear_shapes():
    x, wg, wu, bg, bu, dh = [t.cuda() for t in layer(6, 24, 16, 40, torch.bfloat16)]
    h = memory.gated_linear(x, wg, wu, bg, bu)
    leaf = x.view(2, 3, 4, 16).detach().requires_grad_()
    out = memory.gated_linear(leaf, wg, wu, bg, bu)
    assert out.shape == (2, 3, 4, 40) and torch.equal(out.view(24, 40), h)
    d, = torch.autograd.grad(out, leaf, dh.view(2, 3, 4, 40))
    flat = x.detach().requires_grad_()
    assert torch.equal(d.view(24, 16), torch.autograd.grad(memory.gated_linear(flat, wg, wu, bg, bu), flat, dh)[0])
    assert memory.gated_linear(x[0], wg, wu).shape == (40,)
    for dtype in TYPES:
        leaves = [t.to(dtype).detach().requires_grad_() for t in (x[:0], wg, wu, bg, bu)]
        out = memory.gated_linear(*leaves)
        grads = torch.autograd.grad(out, leaves, torch.zeros_like(out))
        assert out.shape == (0, 40) and grads[0].shape == (0, 16) and all(float(g.abs().sum()) == 0.0 for g in grads)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert memory.gated_linear(x.float(), wg.float(), wu.float()).dtype == torch.float32


@pytest.mark.parametrize("dtype", TYPES)
def test_linear_values_that_are_not_finite(dtype):
    """They stay in their row of h and dx, and in their feature's gradients."""
    case = layer(7, 200, 64, 96, dtype)
    x, wg, wu, bg, bu, dh = case
    x[3, 5], x[150, 0], dh[40, 7] = float("nan"), float("inf"), float("inf")
    leaves = [t.cuda().requires_grad_() for t in case[:5]]
    h = memory.gated_linear(*leaves)
    assert sorted(h.isfinite().logical_not().any(1).nonzero().flatten().tolist()) == [3, 150]
    dx, dwg, _, dbg, _ = torch.autograd.grad(h, leaves, dh.cuda())
    assert sorted(dx.isfinite().logical_not().any(1).nonzero().flatten().tolist()) == [3, 40, 150]
    wide = torch.zeros(200, 96, dtype=dtype, device="cuda")
    bias = bg.cuda()
    bias[95] = float("inf")   # rows and features behind the last ones stay apart
    case = layer(8, 130, 64, 96, dtype)
    leaves = [t.cuda().requires_grad_() for t in case[:3]] + [bias.requires_grad_(), bu.cuda().requires_grad_()]
    h = memory.gated_linear(*leaves)
    assert bool(h[:, :95].isfinite().all()) and not bool(h[:, 95].isfinite().any())
    grads = torch.autograd.grad(h, leaves, wide[:130])
    assert bool(grads[1][:95].isfinite().all()) and bool(grads[3][:95].isfinite().all())


def test_linear_large_projections():
    """Activations far from zero: exponentials that overflow leave no NaN."""
    for activation in ("silu", "gelu", "sigmoid"):
        for dtype in TYPES:
            case = layer(9, 64, 32, 16, dtype)
            case[1] = (case[1].float() * 300).to(dtype)
            check_layer(case, activation)


def test_linear_of_many_values():
    """Offsets beyond 2^31 elements, of h and of x."""
    rows, D, F = (1 << 21) + 70, 64, 1032
    x = torch.empty(rows, D, dtype=torch.bfloat16, device="cuda").normal_()
    case = layer(10, 8, D, F, torch.bfloat16)
    weights = [t.cuda() for t in case[1:5]]
    with torch.no_grad():
        h = memory.gated_linear(x, *weights)
    want = gated_math.linear(x[-70:].cpu(), *case[1:5], "silu")
    assert ref.error(h[-70:], want) <= ref.bound(torch.bfloat16, D) + ref.bound(torch.float32, D)
    del h
    leaf = x[:, :8].contiguous().requires_grad_()
    small = [t[:, :8].contiguous() for t in weights[:2]]
    dh = torch.empty(rows, F, dtype=torch.bfloat16, device="cuda").normal_()
    dx, = torch.autograd.grad(memory.gated_linear(leaf, *small), leaf, dh)
    want = gated_math.linear(leaf[-70:].detach().cpu(), *[t.cpu() for t in small], None, None, "silu", dh[-70:].cpu())
    assert ref.error(dx[-70:], want[1]) <= ref.bound(torch.bfloat16, 2 * F, 2) + ref.bound(torch.float32, 2 * F)


def test_linear_refuses_second_and_forward_mode_derivatives():
    from torch.autograd import forward_ad

    x, wg, wu, *_ = [t.cuda() for t in layer(11, 8, 16, 24, torch.float32)]
    leaf = x.clone().requires_grad_()
    d, = torch.autograd.grad(memory.gated_linear(leaf, wg, wu).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(wg, torch.ones_like(wg))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                memory.gated_linear(x, dual, wu)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows", [16, 3000])
def test_linear_on_another_stream_and_in_a_graph(rows, dtype):
    case = [t.cuda() for t in layer(12, rows, 64, 128, dtype)]

    def everything():
        leaves = [t.detach().requires_grad_() for t in case[:5]]
        h = memory.gated_linear(*leaves)
        return [h, *torch.autograd.grad(h, leaves, case[5])]

    want = everything()
    side, third = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (side, third):   # at the same time
        s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything()
    with torch.cuda.stream(third):
        another = everything()
    for s in (side, third):
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, another))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = everything()
    for t in captured:
        t.detach().zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, captured))


def test_linear_as_the_first_call_of_a_thread():
    """No other call has made the device's context that thread's before."""
    import threading

    x, wg, wu, *_ = [t.cuda() for t in layer(14, 40, 64, 64, torch.bfloat16)]
    with torch.no_grad():
        want, got = memory.gated_linear(x, wg, wu), []

        def run():
            with torch.no_grad():
                try:
                    got.append(memory.gated_linear(x, wg, wu))
                except RuntimeError as e:
                    got.append(e)

        thread = threading.Thread(target=run)
        thread.start()
        thread.join()
    assert torch.is_tensor(got[0]), got[0]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want)


def test_linear_refusals_on_the_gpu():
    from duck_gym_b200.cuda_batch import library

    x, wg, wu, bg, bu, dh = [t.cuda() for t in layer(13, 16, 16, 24, torch.float32)]
    for call in (lambda: memory.gated_linear(x.half(), wg.half(), wu.half()), lambda: memory.gated_linear(x, wg.cpu(), wu),
                 lambda: memory.gated_linear(x.double(), wg.double(), wu.double()), lambda: memory.gated_linear(x, wg, wu, bg.cpu(), bu)):
        with pytest.raises(RuntimeError):
            call()
    lib, p = library(), x.data_ptr()
    fine = dict(x=p, w_gate=p, w_up=p, b_gate=0, b_up=0, h=p, dh=p, dx=p, dw_gate=p, dw_up=p, db_gate=p, db_up=p, kept=p,
                scratch=p, rows=16, x_stride=16, dh_stride=24, D=16, F=24, activation=0, type=0)
    pack = lambda **change: memory._GATED.pack(*{**fine, **change}.values())
    for change in (dict(x=0), dict(w_gate=0), dict(h=0), dict(b_gate=p), dict(D=0), dict(F=-1), dict(rows=-1), dict(rows=1 << 31),
                   dict(activation=3), dict(type=2), dict(type=1, D=12, kept=0), dict(h=p + 4), dict(type=1, x=p + 2),
                   dict(type=1, x_stride=15), dict(type=1, x_stride=20)):
        assert lib.duck_gated_linear_forward(pack(**change), None) != 0, change
    for change in (dict(dh=0), dict(scratch=0), dict(kept=0), dict(dw_up=0), dict(db_gate=0), dict(dx=p + 4), dict(type=1, w_up=p + 2),
                   dict(type=1, D=12, kept=0)):
        assert lib.duck_gated_linear_backward(pack(**change), None) != 0, change
    assert lib.duck_gated_linear_forward(None, None) != 0 and lib.duck_gated_linear_backward(None, None) != 0
    assert b"Invalid" in lib.duck_last_error()
