"""GPU: calls of the gated operators (duck_gym_b200/memory.py) at the edges of what
their documentation allows."""

import pytest
import torch

from duck_gym_b200 import memory

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("activation", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("up", [0.125, -3e37])
def test_linear_activations_over_the_whole_range(activation, dtype, up):
    """What far negative projections leave is zero, however large the numbers beside it."""
    a = [3.0, 0.0, -1.5, -60.0, -87.0, -88.0, -95.0, -200.0, -1e4, -1e30, -1e36, -3e38] + ([200.0, 1e36, 3e38] if up > 0 else [])
    a = torch.tensor(a).to(dtype)
    F = a.numel()
    x, w = torch.zeros(1, 8, dtype=dtype), [torch.zeros(F, 8, dtype=dtype) for _ in range(2)]
    x[0, 0], w[0][:, 0], w[1][:, 0] = 1, a, up
    biases = [torch.zeros(F, dtype=dtype, device="cuda", requires_grad=True) for _ in range(2)]
    h = memory.gated_linear(x.cuda(), w[0].cuda(), w[1].cuda(), *biases, activation=activation)
    got = (h[0], *torch.autograd.grad(h, biases, torch.full((1, F), 0.25, dtype=dtype, device="cuda")))
    A, u = a.double(), w[1][:, 0].double()
    s, rest = 1 / (1 + torch.exp(-A)), 1 / (1 + torch.exp(A))
    if activation == "gelu":
        s = torch.special.ndtr(A)
        y, slope = A * s, s + A * torch.exp(-A * A / 2) / (2 * torch.pi) ** 0.5
        # 1 + erf cancels: off by 2^-23 of 1, where it is not 0.
        lost = torch.where((A < 0) & (A > -20), 2.0 ** -23 * A.abs(), 0.0)
    else:
        y, slope = (A * s, s + A * s * rest) if activation == "silu" else (s, s * rest)
        # 1 / (1 + exp) may be flushed below the smallest normal number, 2^-126; times 100 at most.
        lost = torch.where(A > -100, 2.0 ** -119, 0.0)
    # Hardware's exponentials and quotients, with arguments of up to 128: 2^-18; the result's rounding; and denormals.
    relative = 2.0 ** -18 + (2.0 ** -8 if dtype == torch.bfloat16 else 0)
    for value, want, factor in zip(got, (y * u, 0.25 * u * slope, 0.25 * y), (u, u, torch.ones_like(u))):
        off = (value.detach().cpu().double() - want).abs()
        assert bool((off <= relative * want.abs() + lost * factor.abs() + 2.0 ** -124).all()), (off, want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [3, 300])
def test_recurrence_gates_over_the_whole_range(T, dtype):
    """What a far gate leaves of a state, or adds of a value, is nothing, however large they are."""
    gates = torch.tensor([-95.0, -200.0, -1e30, -3e38, float("-inf"), 110.0, 200.0, 3e38, float("inf")]).to(dtype).expand(T, 1, 9)
    values, state = torch.full((T, 1, 9), 0.5, dtype=dtype), torch.full((1, 9), 1e37)
    values[..., 5:], state[..., 5:] = 1e37, 0.5
    leaves = [t.contiguous().cuda().requires_grad_() for t in (gates, values, state)]
    out, last = memory.gated_recurrence(*leaves)
    # exp(-95) 1e37 is 0.05 of a half in the first step, which float32's gate keeps; bfloat16's is flushed.
    want = torch.full((T, 1, 9), 0.5)
    exact = want.clone()
    exact[0, 0, 0] = 0.5 + 1e37 * 5.521e-42
    got = out.detach().float().cpu()
    assert torch.equal(got[..., 1:], want[..., 1:]) and torch.equal(last.cpu()[..., 1:], want[0, :, 1:])
    assert bool(((got[..., 0] - 0.5).abs() <= 1.01 * (exact[..., 0] - 0.5)).all())
    step = state.cuda()
    assert torch.equal(memory.gated_recurrence_step(gates[0].cuda(), values[0].cuda(), step).float().cpu()[:, 1:], want[0, :, 1:])
    dg, dv, ds = torch.autograd.grad((out, last), leaves, (torch.full_like(out, 1e30), torch.zeros_like(last)))
    keep, replace = slice(5, 9), slice(1, 5)
    assert not bool(dg[..., 1:].any()) and not bool(ds[:, replace].any()) and not bool(dv[..., keep].any())
    assert torch.equal(dv[..., replace].float(), torch.full_like(dv[..., replace].float(), 1e30).to(dtype).float())


# Tiles of 64 rows and of 128, a last run that is whole, of one step and ragged.
@pytest.mark.parametrize("rows,D,F", [(70, 65536 + 37, 40), (33, 1025, 70), (5120, 8192, 256), (5200, 1024 + 17, 250), (64, 2048, 32)])
def test_linear_sums_of_many_steps_in_float32(rows, D, F):
    """A sum in one register is off by 2^-25 sqrt(D / 2) in the mean square, 5e-6 for 65536 values; in runs of 1024 by
    7e-7, their own sum by 2e-7: both projections, and the activation's few roundings, are within 2e-6."""
    g = torch.Generator("cuda")
    g.manual_seed(rows + D)
    x, wg, wu = (torch.randn(s, generator=g, device="cuda") for s in ((rows, D), (F, D), (F, D)))
    wg, wu = (w / D ** 0.5 for w in (wg, wu))
    bg, bu = (torch.randn(F, generator=g, device="cuda") for _ in range(2))
    leaves = [t.requires_grad_() for t in (wg, wu, bg, bu)]
    h = memory.gated_linear(x, *leaves)
    with torch.no_grad():
        assert torch.equal(memory.gated_linear(x, *leaves), h)
    a, u = (x.double() @ w.detach().double().t() + b.detach().double() for w, b in ((wg, bg), (wu, bu)))
    want = a * torch.sigmoid(a) * u
    assert float((h.detach() - want).norm() / want.norm()) <= 2e-6
    dh = torch.randn(rows, F, generator=g, device="cuda")
    db = torch.autograd.grad(h, leaves, dh)[3]
    exact = (dh.double() * a * torch.sigmoid(a)).sum(0)
    # Of the projection, and sums of `rows` values.
    assert float((db - exact).norm() / exact.norm()) <= 2e-6 + 4 * (rows ** 0.5 + 8) * 2.0 ** -24


def test_linear_long_sums_in_bfloat16():
    """Tensor cores cut sums off: one of 65536 products of one sign is too small by up to 6e-4, of 524288 by some 2e-3."""
    # Tiles enough that no split is needed for them: sums over rows, and over features.
    for rows, D, F in ((1 << 19, 64, 9472), (18944, 64, 1 << 18)):
        g = torch.Generator("cuda")
        g.manual_seed(rows)
        x = torch.rand(rows, D, generator=g, device="cuda").bfloat16().requires_grad_()
        w = (torch.rand(F, D, generator=g, device="cuda") / D).bfloat16().requires_grad_()
        none, forty = torch.zeros_like(w).detach(), torch.full((F,), 40.0, dtype=torch.bfloat16, device="cuda")
        # The gate is open: the gradient of u is dh, that of a zero.
        h = memory.gated_linear(x, none, w, forty, torch.zeros_like(forty), activation="sigmoid")
        dh = (0.5 + torch.rand(F, generator=g, device="cuda")).bfloat16()
        dx, dw = torch.autograd.grad(h, (x, w), dh.expand(rows, F))
        del h
        if rows > F:
            got, want = dw.double(), dh.double()[:, None] * x.detach().double().sum(0)
        else:
            got, want = dx[0].double(), dh.double() @ w.detach().double()
        # The mean of results that are each rounded by 1.7e-3 in the mean square, of 64 at least: 2.2e-4.
        assert abs(float((got / want - 1).mean())) <= 6e-4 + 2.2e-4


def test_linear_refuses_projections_of_long_sums_in_bfloat16():
    w = torch.zeros(2, (1 << 16) + 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(RuntimeError, match="65536"):
        memory.gated_linear(w, w, w)
    fine = w[:, :1 << 16].contiguous()
    assert memory.gated_linear(fine, fine, fine).shape == (2, 2)
    assert memory.gated_linear(w.float(), w.float(), w.float()).shape == (2, 2)


# One tile a block and many, steps that fit in the ring and do not, split sums, padded rows.
@pytest.mark.parametrize("rows,D,F", [(16, 256, 512), (300, 61, 301), (4096, 1024, 264), (40000, 64, 512)])
def test_linear_waits_that_run_out(rows, D, F):
    """A block that gives up ends, with its copies and products, and marks what it could not compute."""
    from duck_gym_b200.cuda_batch import library

    g = torch.Generator("cuda")
    g.manual_seed(rows)
    draw = lambda *s: torch.randn(s, generator=g, device="cuda").bfloat16()
    leaves = [t.requires_grad_() for t in (draw(rows, D), draw(F, D) / 16, draw(F, D) / 16, draw(F), draw(F))]
    dh = draw(rows, F)
    call = lambda: memory.gated_linear(*leaves)
    grads = lambda h: torch.autograd.grad(h, leaves, dh)

    def limited(f):
        torch.cuda.synchronize()
        assert library().duck_wait_limit(0) == 0
        try:
            return f()
        finally:
            torch.cuda.synchronize()
            assert library().duck_wait_limit(2 * 10**9) == 0

    def settled(f):
        """After one that did not; the first call may say so."""
        try:
            return f()
        except RuntimeError:
            return f()

    h = call()
    want = [h, *grads(h)]
    assert all(bool(t.isfinite().all()) for t in want)
    bad = limited(call)
    assert bool(bad.isnan().all())
    h = settled(call)
    bad = limited(lambda: grads(h))
    assert all(bool(t.isnan().all()) for t in bad)
    h = settled(call)
    assert all(torch.equal(a, b) for a, b in zip([h, *grads(h)], want))


def test_a_wait_limit_is_not_negative():
    from duck_gym_b200.cuda_batch import library

    assert library().duck_wait_limit(-1) != 0 and b"limit" in library().duck_last_error()


def test_linear_says_that_a_wait_ran_out():
    from duck_gym_b200.cuda_batch import library

    lib, w = library(), torch.ones(8, 16, dtype=torch.bfloat16, device="cuda")
    leaf = w.clone().requires_grad_()
    want = memory.gated_linear(leaf, w, w)

    def limited():
        lib.duck_wait_limit(0)
        try:
            with torch.no_grad():
                return memory.gated_linear(w, w, w)
        finally:
            lib.duck_wait_limit(2 * 10**9)
            torch.cuda.synchronize()

    assert lib.duck_wait_status() == 0
    for call in (lambda: memory.gated_linear(w, w, w), lambda: torch.autograd.grad(want, leaf, torch.ones_like(want), retain_graph=True)):
        assert bool(limited().isnan().all())
        with pytest.raises(RuntimeError, match="ran out"):
            call()
        call()   # once
    limited()
    # float32 layers do not wait; the status is there without a call, too.
    memory.gated_linear(w.float(), w.float(), w.float())
    assert lib.duck_wait_status() != 0 and b"ran out" in lib.duck_last_error() and lib.duck_wait_status() == 0
    assert torch.equal(memory.gated_linear(w, w, w), want)


def test_linear_whose_first_call_is_captured():
    """What a process needs once is made during a capture, too."""
    import subprocess
    import sys
    from pathlib import Path

    code = """
import torch
from duck_gym_b200 import memory
w = torch.ones(8, 16, dtype=torch.bfloat16, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    h = memory.gated_linear(w, w, w)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(h, memory.gated_linear(w, w, w)) and bool((h == 256).all()), h
"""
    run = subprocess.run([sys.executable, "-c", code], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stderr


@pytest.mark.parametrize("rows,D,F", [(16, 256, 512), (6000, 1024, 264)])
def test_linear_waits_that_may_run_out(rows, D, F):
    """With limits that are too short, a call's results are right, or the next call says that they are not."""
    from duck_gym_b200.cuda_batch import library

    lib, g = library(), torch.Generator("cuda")
    g.manual_seed(rows)
    x, wg, wu = (torch.randn(s, generator=g, device="cuda").bfloat16() / 4 for s in ((rows, D), (F, D), (F, D)))
    with torch.no_grad():
        want = memory.gated_linear(x, wg, wu)
        torch.cuda.synchronize()
        try:
            for k in range(40):
                assert lib.duck_wait_limit([1, 300, 1000, 3000][k % 4]) == 0
                h = memory.gated_linear(x, wg, wu)
                torch.cuda.synchronize()
                said = lib.duck_wait_status() != 0
                same = (h == want) | h.isnan()
                assert bool(same.all()) and said == bool(h.isnan().any())
        finally:
            lib.duck_wait_limit(2 * 10**9)
            torch.cuda.synchronize()
            lib.duck_wait_status()
        assert torch.equal(memory.gated_linear(x, wg, wu), want)
