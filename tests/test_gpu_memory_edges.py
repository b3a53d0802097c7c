"""GPU: the memory operators' kernels where autograd, states in place and values
that are not finite meet, and the precision of states and outputs."""

import pytest
import torch

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


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [24, 150])
def test_a_step_on_the_first_state_is_seen_by_the_backward_pass(T, dtype):
    g = gen(T)
    E, H, D = 2, 2, 32
    q, k, v, do = (normal(g, T, E, H, D, dtype=dtype) for _ in range(4))
    S, decay = normal(g, E, H, D, D), torch.tensor([0.9, 0.95])
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    step = [t[0].detach() for t in leaves]
    state = S.cuda()
    o, _ = memory.linear_attention(*leaves, decay.cuda(), state)
    memory.linear_attention_step(*step, decay.cuda(), state)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(o, leaves, do.cuda())
    # On a copy of the state, and before a rollout, a step is in nobody's way.
    state = S.cuda()
    o, _ = memory.linear_attention(*leaves, decay.cuda(), state)
    memory.linear_attention_step(*step, decay.cuda(), state.clone())
    grads = torch.autograd.grad(o, leaves, do.cuda())
    want = ref.attention(q, k, v, decay, S, None, D ** -0.5, do)
    for got, exact in zip(grads, want[2:5]):
        assert ref.error(got, exact) <= ref.bound(dtype, (T + 8) * 2 * D, 4)
    memory.linear_attention_step(*step, decay.cuda(), state)
    o, _ = memory.linear_attention(*leaves, decay.cuda(), state)
    torch.autograd.grad(o, leaves, do.cuda())
    with torch.inference_mode():
        memory.linear_attention_step(*step, decay.cuda(), torch.zeros_like(state))


def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad

    decay = torch.tensor([0.9, 0.95], device="cuda")
    x = torch.randn(4, 3, 2, 8, device="cuda")
    weight, state = torch.ones(8, device="cuda"), torch.randn(3, 2, 8, 8, device="cuda")
    calls = [(memory.layer_norm, x), (lambda w: memory.layer_norm(x, w), weight),
             (lambda q: memory.linear_attention(q, x, x, decay)[0], x),
             (lambda v: memory.linear_attention(x, x, v, decay)[1], x),
             (lambda S: memory.linear_attention(x, x, x, decay, S)[0], state)]
    for f, at in calls:
        want = f(at)
        with forward_ad.dual_level():
            assert torch.equal(f(at), want)   # no tangent, nothing to refuse
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError):
                    f(forward_ad.make_dual(at, torch.ones_like(at)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (at,), (torch.ones_like(at),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: f(t).sum())(at)


def test_checkpointed_mlp_backward_inside_autocast():
    g = gen(2)
    sizes = (61, 200, 96, 14)
    w = [(normal(g, o, i) / i ** 0.5).cuda().requires_grad_() for i, o in zip(sizes, sizes[1:])]
    b = [(0.1 * normal(g, o)).cuda().requires_grad_() for o in sizes[1:]]
    x, dy = normal(g, 300, 61).cuda().requires_grad_(), normal(g, 300, 14).cuda()
    want = torch.autograd.grad(memory.checkpointed_mlp(x, w, b), [x, *w, *b], dy)
    y = memory.checkpointed_mlp(x, w, b)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        got = torch.autograd.grad(y, [x, *w, *b], dy)
    for a, c in zip(got, want):
        assert a.dtype == torch.float32 and ref.error(a, c) <= ref.bound(torch.float32, 300)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [304, 300, 7])   # rows of whole 16-byte pieces and others
def test_the_bounded_derivative_is_that_of_an_elu(n, dtype):
    g = gen(n)
    x = normal(g, 50, n) * 3 - 4
    x[:, ::60] = 4 + 9 * torch.rand(50, 1, generator=g)
    x[:, 1::7] = -30.0
    x[0, 1], x[1, 1] = float("nan"), float("inf")
    x = x.to(dtype).cuda()
    y, kept = memory.elu_checkpoint(x)
    dy = normal(g, 50, n, dtype=dtype).cuda()
    plain, back = memory.elu_restore(dy, kept)
    dx, same = memory.elu_restore(dy, kept, bounded=True)
    stood = kept.codes.float() * kept.scales.repeat_interleave(128, 1)[:, :n]
    assert bool((stood < -1).any()) and torch.equal(back[2:], same[2:])
    slope = torch.where(stood > 0, 1.0, stood.clamp_min(-1) + 1)
    assert torch.equal(dx[2:], (dy.float() * slope)[2:].to(dtype))
    assert torch.equal(dx[stood >= -1], plain[stood >= -1]) and float((dx[2:] * dy[2:]).min()) >= 0.0
    assert bool(dx[:2, :min(n, 128)].isnan().all())   # what is not finite stays visible
    only, nothing = memory.elu_restore(dy, kept, restore=False, bounded=True)
    assert nothing is None and torch.equal(only[2:], dx[2:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 1), (20, 28), (32, 32), (40, 9), (100, 128), (128, 66)])
def test_infinity_beside_head_sizes_that_are_padded(Dk, Dv, dtype):
    """Of operands without a negative number an infinity makes infinities, and no NaN."""
    T, E, H = 45, 2, 2
    g = gen(Dk * 131 + Dv)
    q, k, v, do = (normal(g, T, E, H, D, dtype=dtype).abs() + 0.1 for D in (Dk, Dk, Dv, Dv))
    S, decay = normal(g, E, H, Dk, Dv).abs(), torch.tensor([0.5, 0.9])
    r = torch.zeros(T, E, dtype=torch.bool)
    r[30] = True
    v[7, 0, 0, Dv // 2] = do[20, 1, 0, 0] = float("inf")
    q[21, 0, 1, Dk - 1] = k[40, 1, 1, 0] = float("inf")
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, S)]
    o, last = memory.linear_attention(*leaves[:3], decay.cuda(), leaves[3], r.cuda())
    dlast = torch.ones_like(last)
    grads = torch.autograd.grad([o, last], leaves, [do.cuda(), dlast])
    want = ref.attention(q, k, v, decay, S, r, Dk ** -0.5, do, dlast.cpu())
    for i, (got, exact) in enumerate(zip((o, last, *grads), want)):
        got = got.cpu().double()
        assert not bool(exact.isnan().any()) and bool(exact.isinf().any())
        assert torch.equal(got.isinf(), exact.isinf()) and not bool(got.isnan().any()), i
        fine = exact.isfinite()
        terms = (T + 8) * (Dk + Dv)
        assert ref.error(got[fine], exact[fine]) <= (ref.bound(dtype, terms, 4) if i not in (1, 5) else 1e-5)


# A state from bfloat16 operands: each operand with its decay is the sum of three bfloat16 numbers (2^-24 of it is
# left), sums are float32 (2^-24 of the state for each product that it still remembers, at random: some 60 of 16 steps
# at 1000 steps), and a power of the decay is as exact as the logarithm in its exponent (2^-24 ln(1 / fading)).  All
# of it stays below 1.5e-6; two numbers an operand leave 2^-17 of it in the mean, 2.1e-6 to 2.4e-6 in the state.
WHOLE_STATE = 1.5e-6


@pytest.mark.parametrize("D", [16, 64, 128])
@pytest.mark.parametrize("T,quiet", [(104, 40), (192, 128), (1000, 300), (2000, 500), (24, 0), (1000, 0)])
@pytest.mark.parametrize("decay", [0.9, 0.97, 0.99])
def test_states_are_whole_where_later_steps_add_nothing(D, T, quiet, decay):
    """The last steps of the rollout for its last state, the first ones for the gradient of its first state."""
    g = gen(T + quiet + D)
    E = 1 if T > 1000 else 2   # the long ones are split over the steps
    q, k, v, do = (normal(g, T, E, 1, D, dtype=torch.bfloat16) for _ in range(4))
    k[T - quiet:], q[:quiet] = 0.0, 0.0
    decay = torch.tensor([decay])
    leaves = [t.cuda() for t in (q, k, v)]
    S = torch.zeros(E, 1, D, D, device="cuda", requires_grad=True)
    o, last = memory.linear_attention(*leaves, decay.cuda(), S)
    dS, = torch.autograd.grad(o, S, do.cuda())
    want = ref.attention(q, k, v, decay, torch.zeros(E, 1, D, D), None, D ** -0.5, do)
    assert ref.error(last, want[1]) <= WHOLE_STATE
    assert ref.error(dS, want[5]) <= WHOLE_STATE


@pytest.mark.parametrize("T,D,decay", [(48, 64, 0.97), (1000, 64, 0.996), (1000, 128, 0.99), (2000, 32, 0.996)])
def test_outputs_have_two_roundings(T, D, decay):
    """An output or gradient in bfloat16 is rounded once itself, and on its way each term once: a decayed score, or the
    state's copy.  A rounding to 8 bits of a normal value is 1.66e-3 in the mean square (2^-7 / sqrt(12) over values
    between 1 and 2 and their multiples), two are 2.35e-3; a third, an operand of the state rounded too, would make
    2.87e-3 where the state carries most of it."""
    g = gen(T + D)
    q, k, v, do = (normal(g, T, 4, 1, D, dtype=torch.bfloat16) for _ in range(4))
    S, dlast, decay = 3 * normal(g, 4, 1, D, D), 3 * normal(g, 4, 1, D, D), torch.tensor([decay])
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    for final in (False, True):
        o, last = memory.linear_attention(*leaves, decay.cuda(), S.cuda(), None, None, final)
        grads = torch.autograd.grad([o, last] if final else [o], leaves,
                                    [do.cuda(), dlast.cuda()] if final else [do.cuda()])
        want = ref.attention(q, k, v, decay, S, None, D ** -0.5, do, dlast if final else None)
        for got, exact in zip((o, *grads), (want[0], *want[2:5])):
            assert ref.error(got, exact) <= 2.6e-3


def test_tangents_are_refused_by_calls_without_gradients():
    from torch.autograd import forward_ad

    decay, x = torch.tensor([0.9, 0.95], device="cuda"), torch.randn(3, 2, 8, device="cuda")
    state = torch.randn(3, 2, 8, 8, device="cuda")
    y, kept = memory.elu_checkpoint(x)
    calls = [(lambda q: memory.linear_attention_step(q, x, x, decay, state.clone()), x),
             (lambda S: memory.linear_attention_step(x, x, x, decay, S.clone()), state),
             (lambda t: memory.elu_checkpoint(t)[0], x), (lambda t: memory.elu_restore(t, kept)[0], y),
             (lambda s: memory.elu_restore(y, memory.Checkpoint8(kept.codes, s))[0], kept.scales)]
    for f, at in calls:
        want = f(at)
        with forward_ad.dual_level():
            assert torch.equal(f(at), want)
            with pytest.raises(RuntimeError):
                f(forward_ad.make_dual(at, torch.ones_like(at)))
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (at,), (torch.ones_like(at),))
