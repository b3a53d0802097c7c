"""CPU: the gated operators of duck_gym_b200/memory.py against float64
restatements (tests/gated_math.py) and differences, and their refusals."""

import subprocess
from pathlib import Path

import pytest
import torch

import gated_math
import memory_math as ref
from duck_gym_b200 import memory


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def rollout(seed, T, E, N, dtype=torch.float32, resets=0.2):
    g = gen(seed)
    gates, values, dout = (torch.randn(T, E, N, generator=g).to(dtype) for _ in range(3))
    return (gates + 1, values, torch.randn(E, N, generator=g), torch.rand(T, E, generator=g) < resets, dout,
            torch.randn(E, N, generator=g))


@pytest.mark.parametrize("T,E,N", [(1, 1, 1), (7, 3, 5), (40, 2, 4)])
def test_recurrence_matches_restatement(T, E, N):
    gates, values, state, resets, dout, dlast = rollout(T + 1, T, E, N)
    leaves = [t.requires_grad_() for t in (gates, values, state)]
    out, last = memory.gated_recurrence(*leaves, resets)
    grads = torch.autograd.grad((out, last), leaves, (dout, dlast))
    want = gated_math.recurrence(gates.detach(), values.detach(), state.detach(), resets, dout, dlast)
    for got, exact in zip((out, last, *grads), want):
        assert ref.error(got, exact) <= ref.bound(torch.float32, T + 1)
    empty, last = memory.gated_recurrence(gates[:0].detach(), values[:0].detach(), state)
    assert empty.shape == (0, E, N) and torch.equal(last, state) and last is not state


def test_recurrence_gradients_are_those_of_differences():
    gates, values, state, resets, _, _ = rollout(5, 6, 2, 3)
    args = [t.double().requires_grad_() for t in (gates, values, state)]
    assert torch.autograd.gradcheck(lambda g, c, h: memory.gated_recurrence(g, c, h, resets), args)


def test_recurrence_steps_agree_with_the_rollout():
    gates, values, state, resets, _, _ = rollout(6, 9, 3, 4)
    out, last = memory.gated_recurrence(gates, values, state, resets)
    moving = state.clone()
    for t in range(9):
        assert torch.equal(memory.gated_recurrence_step(gates[t], values[t], moving, resets[t]), out[t])
    assert torch.equal(moving, last)
    none, nothing = memory.gated_recurrence(gates, values, final_state=False)
    assert nothing is None and torch.equal(none, memory.gated_recurrence(gates, values, torch.zeros_like(state))[0])


def test_recurrence_reset_drops_what_is_not_finite():
    gates, values, state, resets, dout, _ = rollout(7, 6, 1, 2, resets=0.0)
    values[1, 0, 0], state[0, 1], dout[4, 0, 0] = float("nan"), float("inf"), float("nan")
    resets[3] = True
    leaves = [t.requires_grad_() for t in (gates, values)]
    out, last = memory.gated_recurrence(*leaves, state, resets)
    assert bool(out[3:].isfinite().all()) and bool(last.isfinite().all()) and not bool(out[2].isfinite().any())


def test_recurrence_refusals():
    x, state = torch.zeros(4, 2, 3), torch.zeros(2, 3)
    bad = [
        lambda: memory.gated_recurrence(x, x[:3]),
        lambda: memory.gated_recurrence(x, x.double()),
        lambda: memory.gated_recurrence(x[0], x[0]),
        lambda: memory.gated_recurrence(x.long(), x.long()),
        lambda: memory.gated_recurrence(x, x, state[:1]),
        lambda: memory.gated_recurrence(x, x, state.double()),
        lambda: memory.gated_recurrence(x, x, state, torch.zeros(4, 3, dtype=torch.bool)),
        lambda: memory.gated_recurrence(x, x, state, torch.zeros(4, 2)),
        lambda: memory.gated_recurrence_step(x, x, state),
        lambda: memory.gated_recurrence_step(x[0], x[0], None),
        lambda: memory.gated_recurrence_step(x[0], x[0], state.clone().requires_grad_()),
        lambda: memory.gated_recurrence_step(x[0], x[0], state, torch.zeros(3, dtype=torch.bool)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"case {i} was accepted")


def offsets(tmp_path, struct, fields):
    """Places of a C struct's fields and its size, by the C compiler."""
    lines = "".join(f'printf("%zu ", offsetof({struct}, {f}));' for f in fields)
    (tmp_path / "s.c").write_text('#include <stdio.h>\n#include <stddef.h>\n#include "duck_b200.h"\n'
                                  f'int main(void){{{lines} printf("%zu", sizeof({struct})); return 0;}}')
    include = Path(__file__).resolve().parents[1] / "include"
    subprocess.run(["gcc", "-I", str(include), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    return [int(w) for w in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True).stdout.split()]


def test_packed_recurrence_has_the_size_of_the_c_struct(tmp_path):
    got = offsets(tmp_path, "duck_recurrence", ("gates", "resets", "state_out", "dgates", "scratch", "gates_stride",
                                                "dout_stride", "T", "type"))
    assert got == [0, 24, 40, 64, 96, 104, 136, 152, 164, memory._RECURRENCE.size]


# ---------------------------------------------------------------- gated linear
def layer(seed, rows, D, F, dtype=torch.float32, bias=True):
    g = gen(seed)
    x, wg, wu = (torch.randn(s, generator=g) for s in ((rows, D), (F, D), (F, D)))
    bg, bu, dh = (torch.randn(s, generator=g) for s in ((F,), (F,), (rows, F)))
    x, wg, wu, bg, bu, dh = (t.to(dtype) for t in (x, wg / D ** 0.5, wu / D ** 0.5, 0.3 * bg, 0.3 * bu, dh))
    return x, wg, wu, bg if bias else None, bu if bias else None, dh


@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("bias", [True, False])
def test_linear_matches_restatement(activation, bias):
    case = layer(1, 20, 7, 11, bias=bias)
    leaves = [t.requires_grad_() for t in case[:5] if t is not None]
    h = memory.gated_linear(*case[:5], activation=activation)
    got = (h, *torch.autograd.grad(h, leaves, case[5]))
    want = gated_math.linear(*[None if t is None else t.detach() for t in case[:5]], activation, case[5])
    for a, b in zip(got, want):
        assert ref.error(a, b) <= ref.bound(torch.float32, 40)
    assert torch.autograd.gradcheck(lambda *t: memory.gated_linear(*t[:3], *(t[3:] or (None, None)), activation=activation),
                                    [t.detach()[:4].double().requires_grad_() if i == 0 else t.detach().double().requires_grad_()
                                     for i, t in enumerate(leaves)])


def test_linear_shapes_and_autocast():
    x, wg, wu, bg, bu, _ = layer(2, 24, 5, 6)
    h = memory.gated_linear(x, wg, wu, bg, bu)
    assert torch.equal(memory.gated_linear(x.view(2, 3, 4, 5), wg, wu, bg, bu).view(24, 6), h)
    assert memory.gated_linear(x[0], wg, wu).shape == (6,) and memory.gated_linear(x[:0], wg, wu).shape == (0, 6)
    with torch.autocast("cpu", dtype=torch.bfloat16):
        assert torch.equal(memory.gated_linear(x, wg, wu, bg, bu), h)


def test_linear_refusals():
    x, wg, wu, bg, bu, _ = layer(3, 4, 5, 6)
    bad = [
        lambda: memory.gated_linear(x, wg, wu[:5]), lambda: memory.gated_linear(x[:, :4], wg, wu),
        lambda: memory.gated_linear(x, wg, wu, bg), lambda: memory.gated_linear(x, wg, wu, bg, bu[:5]),
        lambda: memory.gated_linear(x, wg, wu.double()), lambda: memory.gated_linear(x, wg, wu, bg.double(), bu),
        lambda: memory.gated_linear(x, wg, wu, activation="relu"), lambda: memory.gated_linear(x, wg[:0], wu[:0]),
        lambda: memory.gated_linear(x[:, :0], wg[:, :0], wu[:, :0]), lambda: memory.gated_linear(x.long(), wg.long(), wu.long()),
        lambda: memory.gated_linear(torch.tensor(1.0), wg, wu), lambda: memory.gated_linear(x, wg[0], wu[0]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"case {i} was accepted")


def test_packed_layer_has_the_size_of_the_c_struct(tmp_path):
    got = offsets(tmp_path, "duck_gated", ("x", "h", "dw_gate", "db_gate", "kept", "scratch", "rows", "D", "F", "type"))
    assert got == [0, 40, 64, 80, 96, 104, 112, 136, 140, 148, memory._GATED.size]
