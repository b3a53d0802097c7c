"""CPU: what the memory operators (duck_gym_b200/memory.py) have to refuse or
keep where autograd, autocast and states in place meet."""

import pytest
import torch

from duck_gym_b200 import memory


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def heads(g, *shape, count=3):
    return [torch.randn(*shape, generator=g) for _ in range(count)]


def test_step_refuses_a_state_that_requires_a_gradient():
    g = gen(0)
    q, k, v = heads(g, 3, 2, 4)
    decay = torch.tensor([0.7, 0.9])
    state = torch.randn(3, 2, 4, 4, generator=g, requires_grad=True)
    with pytest.raises(RuntimeError):
        memory.linear_attention_step(q, k, v, decay, state)
    with torch.no_grad():
        memory.linear_attention_step(q, k, v, decay, state)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checkpointed_mlp_backward_inside_autocast(dtype):
    g = gen(1)
    sizes = (7, 40, 30, 3)
    w = [(torch.randn(o, i, generator=g) / i ** 0.5).to(dtype) for i, o in zip(sizes, sizes[1:])]
    b = [(0.1 * torch.randn(o, generator=g)).to(dtype) for o in sizes[1:]]
    leaves = [t.requires_grad_() for t in (torch.randn(50, 7, generator=g).to(dtype), *w, *b)]
    dy = torch.randn(50, 3, generator=g).to(dtype)
    run = lambda: memory.checkpointed_mlp(leaves[0], leaves[1:4], leaves[4:])
    want = torch.autograd.grad(run(), leaves, dy)
    y = run()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(got, want))   # the very products of the pass outside


def test_attention_backward_inside_autocast():
    g = gen(2)
    leaves = [t.requires_grad_() for t in (*heads(g, 9, 2, 2, 8), torch.randn(2, 2, 8, 8, generator=g))]
    decay, do = torch.tensor([0.5, 0.9]), torch.randn(9, 2, 2, 8, generator=g)
    run = lambda: memory.linear_attention(*leaves[:3], decay, leaves[3])[0]
    want = torch.autograd.grad(run(), leaves, do)
    out = run()
    with torch.autocast("cpu", dtype=torch.bfloat16):
        got = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(a, c) for a, c in zip(got, want))


def test_no_steps_give_a_state_of_its_own():
    S = torch.randn(2, 1, 4, 4, generator=gen(3))
    q = torch.zeros(0, 2, 1, 4)
    _, last = memory.linear_attention(q, q, q, torch.tensor([0.9]), S)
    assert torch.equal(last, S)
    last.zero_()   # as a control step would
    assert bool(S.abs().sum() > 0)


def saturated(g):
    """Rows whose groups have a largest value of 12, 5 or 40 and many units that are saturated, or nearly."""
    x = torch.randn(3, 300, generator=g) * 3 - 4
    x[:, ::60] = torch.tensor([12.0, 5.0, 40.0])[:, None]
    x[:, 1::7] = -30.0
    return x


def test_the_bounded_derivative_is_that_of_an_elu():
    x = saturated(gen(4))
    y, kept = memory.elu_checkpoint(x)
    ones = torch.ones_like(x)
    plain, back = memory.elu_restore(ones, kept)
    dx, same = memory.elu_restore(ones, kept, bounded=True)
    assert bool((back < -1).any()) and torch.equal(back, same)
    assert float(dx.min()) >= 0.0 and float(dx.max()) <= 1.0
    assert torch.equal(dx, plain.clamp_min(0))
    exact = torch.where(x > 0, 1.0, x.double().exp())
    step = kept.scales.double().repeat_interleave(128, 1)[:, :300]
    # Half a step, and a step where the kept value of a small positive one is zero or the other way round.
    assert bool(((dx - exact).abs() <= 0.501 * step).all())
    # What is not finite stays visible.
    y, kept = memory.elu_checkpoint(torch.full((1, 4), float("nan")))
    assert bool(memory.elu_restore(torch.ones(1, 4), kept, bounded=True)[0].isnan().all())


def test_checkpointed_mlp_sends_nothing_back_through_saturated_units_that_are_kept_below():
    g = gen(5)
    bias = torch.full((64,), -20.0)
    bias[0] = 12.0
    first, second = 0.1 * torch.randn(64, 6, generator=g), torch.randn(3, 64, generator=g)
    leaves = [t.requires_grad_() for t in (torch.randn(40, 6, generator=g), first, second, bias, torch.zeros(3))]
    dz = torch.randn(40, 3, generator=g)
    grads = torch.autograd.grad(memory.checkpointed_mlp(leaves[0], leaves[1:3], leaves[3:]), leaves, dz)
    x, w, v, b, _ = (t.detach().double() for t in leaves)
    _, kept = memory.elu_checkpoint(torch.addmm(leaves[3], leaves[0], first.t()))
    stood = kept.codes.double() * kept.scales.double()
    assert bool((stood < -1).any())
    slope = torch.where(stood > 0, 1.0, (stood + 1).clamp_min(0))
    dy = (dz.double() @ v) * slope
    # float32 sums of 40 and of 64 terms.
    for got, want in zip((grads[0], grads[1], grads[3]), (dy @ w, dy.t() @ x, dy.sum(0))):
        assert float((got.double() - want).norm() / want.norm()) <= 4 * (64 ** 0.5 + 8) * 2.0 ** -24


@pytest.mark.parametrize("kind", [0, 1])
def test_more_steps_than_are_counted_in_32_bits_are_refused(kind):
    """Their segments end past 2^31, where the count of steps would turn negative."""
    for T in (2 ** 31 - 1, 2 ** 31 - 2 ** 24):
        with pytest.raises(RuntimeError, match="steps"):
            memory._workspace(T, 1, 1, 1, 1, kind)
    assert memory._workspace(2 ** 31 - 2 ** 24 - 1, 1, 1, 1, 1, kind)[0] > 0


@pytest.mark.skipif(torch.cuda.is_available(), reason="calls with host addresses, which only a refusal keeps from a GPU")
def test_statistics_at_an_odd_place_are_refused():
    from duck_gym_b200.cuda_batch import library

    lib = library()
    p = torch.zeros(64).data_ptr()
    assert lib.duck_layer_norm_forward(p, None, None, p, p + 4, 4, 8, 8, 1e-5, 0, None) == 1   # DUCK_EINVAL
    assert b"aligned" in lib.duck_last_error()
    assert lib.duck_layer_norm_backward(p, p, None, p + 4, p, None, None, None, 4, 8, 8, 8, 0, None) == 1
    assert b"aligned" in lib.duck_last_error()


def test_memory_ppo_says_that_its_update_is_not_captured():
    import warnings

    from duck_gym_b200.memory_policy import MemoryPPO, MemoryPPOConfig
    from test_memory_policy import RecallEnv

    small = dict(bf16=False, width=16, heads=2, head_size=8, hidden=24, steps_per_env=4)
    assert not MemoryPPOConfig().graph_update
    with pytest.warns(UserWarning, match="graph_update"):
        MemoryPPO(RecallEnv(8), MemoryPPOConfig(**small, graph_update=True), device="cpu")
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        MemoryPPO(RecallEnv(8), MemoryPPOConfig(**small), device="cpu")
