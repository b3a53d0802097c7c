"""CPU: the memory operators (duck_gym_b200/memory.py) in their plain torch form
against float64 restatements, their gradients against differences, and their
refusals."""

import pytest
import torch

import memory_math as ref
from duck_gym_b200 import memory


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


@pytest.mark.parametrize("T,E,H,Dk,Dv", [(0, 2, 1, 4, 4), (1, 1, 1, 1, 1), (9, 3, 2, 5, 7), (24, 2, 3, 8, 8)])
def test_attention_matches_restatement(T, E, H, Dk, Dv):
    g = gen(T)
    q, k = (torch.randn(T, E, H, Dk, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    v = torch.randn(T, E, H, Dv, generator=g, dtype=torch.float64, requires_grad=True)
    S = torch.randn(E, H, Dk, Dv, generator=g, dtype=torch.float64, requires_grad=True)
    decay, r = torch.rand(H, generator=g, dtype=torch.float64), torch.rand(T, E, generator=g) < 0.2
    o, last = memory.linear_attention(q, k, v, decay, S, r)
    do, dlast = torch.randn(o.shape, generator=g).double(), torch.randn(last.shape, generator=g).double()
    want = ref.attention(q.detach(), k.detach(), v.detach(), decay, S.detach(), r, Dk ** -0.5, do, dlast)
    got = [o, last]
    if T:
        got += torch.autograd.grad([o, last], [q, k, v, S], [do, dlast])
    for a, b in zip(got, want):
        assert ref.error(a, b) <= 1e-12


def test_attention_gradient_by_differences():
    g = gen(1)
    q, k, v = (torch.randn(7, 2, 2, 3, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(3))
    S = torch.randn(2, 2, 3, 3, generator=g, dtype=torch.float64, requires_grad=True)
    decay, r = torch.tensor([0.5, 0.9], dtype=torch.float64), torch.rand(7, 2, generator=g) < 0.2
    assert torch.autograd.gradcheck(lambda *x: memory.linear_attention(*x[:3], decay, x[3], r), (q, k, v, S))


def test_step_is_the_rollout_one_step_at_a_time():
    g = gen(2)
    q, k, v = (torch.randn(6, 3, 2, 4, generator=g) for _ in range(3))
    S, decay = torch.randn(3, 2, 4, 4, generator=g), torch.tensor([0.7, 0.95])
    r = torch.rand(6, 3, generator=g) < 0.3
    o, last = memory.linear_attention(q, k, v, decay, S, r)
    state = S.clone()
    for t in range(6):
        assert torch.equal(memory.linear_attention_step(q[t], k[t], v[t], decay, state, r[t]), o[t])
    assert torch.equal(state, last)


def test_an_earlier_episode_does_not_reach_the_next():
    g = gen(3)
    q, k, v = (torch.randn(6, 1, 1, 4, generator=g) for _ in range(3))
    v[1, 0, 0, 2] = float("nan")
    r = torch.zeros(6, 1, dtype=torch.bool)
    r[3] = True
    S = torch.full((1, 1, 4, 4), float("inf"))
    o, last = memory.linear_attention(q, k, v, torch.tensor([0.9]), S, r)
    assert bool(o[3:].isfinite().all()) and bool(last.isfinite().all()) and not bool(o[1].isfinite().all())


@pytest.mark.parametrize("n", [1, 61, 128, 129, 300])
def test_checkpoint_matches_restatement(n):
    g = gen(n)
    x, dy = 2 * torch.randn(9, n, generator=g), torch.randn(9, n, generator=g)
    x[0] = 0.0
    y, kept = memory.elu_checkpoint(x)
    codes, scales = ref.kept(y)
    assert torch.equal(kept.codes, codes) and torch.equal(kept.scales, scales)
    dx, back = memory.elu_restore(dy, kept)
    stood = codes.double() * scales.double().repeat_interleave(128, 1)[:, :n]
    assert ref.error(back, stood) <= ref.bound(torch.float32, 1)
    assert ref.error(dx, dy.double() * torch.where(stood > 0, torch.ones_like(stood), 1 + stood)) <= ref.bound(
        torch.float32, 1)


def test_checkpoint_of_values_that_are_not_finite():
    x = torch.randn(4, 256, generator=gen(4))
    x[0, 5], x[1, 130] = float("inf"), float("nan")
    y, kept = memory.elu_checkpoint(x)
    _, back = memory.elu_restore(torch.ones_like(y), kept)
    assert bool(back[0, :128].isnan().all()) and bool(back[1, 128:].isnan().all())
    assert bool(back[0, 128:].isfinite().all()) and bool(back[1, :128].isfinite().all())
    assert bool(back[2:].isfinite().all())


def test_checkpointed_mlp_gradients():
    g = gen(5)
    sizes = (7, 40, 30, 3)
    w = [torch.randn(o, i, generator=g) / i ** 0.5 for i, o in zip(sizes, sizes[1:])]
    b = [0.1 * torch.randn(o, generator=g) for o in sizes[1:]]
    leaves = [t.requires_grad_() for t in (torch.randn(50, 7, generator=g), *w, *b)]
    y = memory.checkpointed_mlp(leaves[0], leaves[1:4], leaves[4:])
    z = leaves[0]
    for i in range(3):
        z = torch.nn.functional.linear(z, leaves[1 + i], leaves[4 + i])
        z = torch.nn.functional.elu(z) if i < 2 else z
    assert ref.error(y, z) <= ref.bound(torch.float32, 40)
    dy = torch.randn(50, 3, generator=g)
    got, want = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(z, leaves, dy)
    # Kept to half of max |y| / 127: some 0.7 % a layer in the mean square.
    for a, c in zip(got, want):
        assert ref.error(a, c) <= 0.02


def test_checkpointed_mlp_under_autocast_and_its_second_derivative():
    g = gen(7)
    w, b = [torch.randn(6, 5, generator=g, requires_grad=True)], [torch.zeros(6, requires_grad=True)]
    x = torch.randn(4, 5, generator=g, requires_grad=True)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        y = memory.checkpointed_mlp(x, w, b)
    assert y.dtype == torch.float32
    dx, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):   # there is no second one
        torch.autograd.grad(dx.sum(), w)


def test_refusals():
    x, decay = torch.zeros(4, 2, 1, 8), torch.ones(1)
    state = torch.zeros(2, 1, 8, 8)
    bad = [
        lambda: memory.linear_attention(x, x[:3], x, decay),
        lambda: memory.linear_attention(x, x, x[:, :1], decay),
        lambda: memory.linear_attention(x[0], x[0], x[0], decay),
        lambda: memory.linear_attention(x, x, x.double(), decay),
        lambda: memory.linear_attention(x, x, x, torch.ones(2)),
        lambda: memory.linear_attention(x, x, x, decay.clone().requires_grad_()),
        lambda: memory.linear_attention(x, x, x, decay, state[:1]),
        lambda: memory.linear_attention(x, x, x, decay, state.double()),
        lambda: memory.linear_attention(x, x, x, decay, state, torch.zeros(4, 1, dtype=torch.bool)),
        lambda: memory.linear_attention(x, x, x, decay, state, torch.zeros(4, 2)),
        lambda: memory.linear_attention(torch.zeros(2, 2, 1, 129), torch.zeros(2, 2, 1, 129), x[:2], decay),
        lambda: memory.linear_attention(x[..., :0], x[..., :0], x, decay),
        lambda: memory.linear_attention_step(x, x, x, decay, state),
        lambda: memory.linear_attention_step(x[0], x[0], x[0], decay, state[:, :, :4]),
        lambda: memory.layer_norm(torch.zeros(3, 0)),
        lambda: memory.layer_norm(torch.zeros(3, 4), torch.ones(5)),
        lambda: memory.elu_checkpoint(torch.zeros(3, 0)),
        lambda: memory.elu_restore(torch.zeros(3, 4), memory.Checkpoint8(torch.zeros(3, 5, dtype=torch.int8),
                                                                         torch.zeros(3, 1))),
        lambda: memory.elu_restore(torch.zeros(3, 4), memory.Checkpoint8(torch.zeros(3, 4, dtype=torch.int8),
                                                                         torch.zeros(3, 2))),
        lambda: memory.checkpointed_mlp(torch.zeros(3, 4), [torch.zeros(2, 4, dtype=torch.float64)], [torch.zeros(2)]),
        lambda: memory.checkpointed_mlp(torch.zeros(3, 4), [], []),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"case {i} was accepted")


def test_layer_norm_on_the_cpu():
    g = gen(6)
    x, w, b = torch.randn(5, 3, 20, generator=g), torch.rand(20, generator=g), torch.rand(20, generator=g)
    assert ref.error(memory.layer_norm(x, w, b), ref.layer_norm(x, w, b, 1e-5)) <= ref.bound(torch.float32, 20)


def test_packed_arguments_have_the_size_of_the_c_struct(tmp_path):
    """The struct that the binding packs by hand against the C compiler's."""
    import subprocess
    from pathlib import Path

    fields = ("q", "resets", "state_out", "scratch", "q_stride", "dout_stride", "T", "type", "scale")
    lines = "".join(f'printf("%zu ", offsetof(duck_attention, {f}));' for f in fields)
    (tmp_path / "s.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "duck_b200.h"\n'
                                  f'int main(void){{{lines} printf("%zu", sizeof(duck_attention)); return 0;}}')
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-I", str(include), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = [int(w) for w in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()]
    assert got == [0, 40, 56, 120, 128, 200, 224, 244, 248, memory._ATTENTION.size]
