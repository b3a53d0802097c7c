"""GPU: the memory operators' kernels (duck_gym_b200/memory.py) against float64
restatements (tests/memory_math.py), at the sizes, masks, strides and values
where they can go wrong, and their refusals."""

import pytest
import torch

import memory_math as ref
from duck_gym_b200 import memory

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16]
# States held in float32 from bfloat16 operands: an operand that carries a decay is kept as the sum of two
# bfloat16 numbers at least (2^-16 relative at most), and sums are float32.
STATE = 1e-5


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def normal(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype)


# ------------------------------------------------------------------ layer norm
NORM_SIZES = [(1, 1), (1, 7), (3, 8), (5, 61), (1000, 24), (17, 128), (33, 256), (301, 200), (9, 512), (4, 1000),
              (6, 1024), (3, 1025), (65, 1032), (2, 4096), (5, 5003), (3, 9000), (4099, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", NORM_SIZES)
def test_layer_norm(rows, n, dtype):
    g = gen(rows * 10007 + n)
    x = (normal(g, rows, n) * 2 + normal(g, rows, 1)).to(dtype)
    w, b, dy = 1 + 0.3 * normal(g, n), 0.3 * normal(g, n), normal(g, rows, n, dtype=dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    y = memory.layer_norm(*leaves, 1e-5)
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    want = ref.layer_norm(x, w, b, 1e-5, dy)
    assert y.dtype == dtype and [t.dtype for t in grads] == [dtype, torch.float32, torch.float32]
    # y and dx: one rounding to the type; the sums of the gradients are float32.
    for got, exact, terms in zip((y, *grads), want, (n, n, rows, rows)):
        held = dtype if got.dtype == dtype else torch.float32
        if n == 1 and got is grads[0]:
            assert float(got.abs().max()) == 0.0   # a single value is its own mean
        else:
            assert ref.error(got, exact) <= ref.bound(held, terms) + ref.bound(torch.float32, n)
    # Without gradients, and again: the same bits.
    with torch.no_grad():
        assert torch.equal(memory.layer_norm(*leaves, 1e-5), y)
    again = torch.autograd.grad(memory.layer_norm(*leaves, 1e-5), leaves, dy.cuda())
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_without_weight_or_bias_and_partial_gradients(dtype):
    g = gen(1)
    x, dy = normal(g, 37, 96, dtype=dtype), normal(g, 37, 96, dtype=dtype)
    w = 1 + 0.3 * normal(g, 96)
    xc = x.cuda().requires_grad_()
    y = memory.layer_norm(xc)
    dx, = torch.autograd.grad(y, xc, dy.cuda())
    want = ref.layer_norm(x, None, None, 1e-5, dy)
    assert ref.error(y, want[0]) <= ref.bound(dtype, 96) and ref.error(dx, want[1]) <= ref.bound(dtype, 96)
    wc = w.cuda().requires_grad_()
    dw, = torch.autograd.grad(memory.layer_norm(x.cuda(), wc), wc, dy.cuda())
    assert ref.error(dw, want[2]) <= ref.bound(torch.float32, 37) + ref.bound(torch.float32, 96)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [24, 61, 512, 1500])
def test_layer_norm_strides(n, dtype):
    g = gen(n)
    wide = normal(g, 40, n + 5, dtype=dtype)
    dy = normal(g, 20, n, dtype=dtype)
    w = 1 + 0.3 * normal(g, n)
    for view in (wide[:20, 3:n + 3], wide[::2, :n], wide[:1, :n].expand(20, n)):
        dev = wide.cuda().as_strided(view.size(), view.stride(), view.storage_offset())
        assert torch.equal(dev.cpu(), view)
        dev.requires_grad_()
        y = memory.layer_norm(dev, w.cuda())
        dx, = torch.autograd.grad(y, dev, dy.cuda())
        want = ref.layer_norm(view, w, None, 1e-5, dy)
        assert ref.error(y, want[0]) <= ref.bound(dtype, n) and ref.error(dx, want[1]) <= ref.bound(dtype, n)
    turned = normal(g, n, 20, dtype=dtype)
    y = memory.layer_norm(turned.cuda().t(), w.cuda())
    assert ref.error(y, ref.layer_norm(turned.t(), w, None, 1e-5)) <= ref.bound(dtype, n)
    # The gradient of a sum comes with strides of zero; more than two axes.
    x = normal(g, 4, 5, n, dtype=dtype)
    xc, wc = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    memory.layer_norm(xc, wc).float().sum().backward()
    want = ref.layer_norm(x.view(20, n), w, None, 1e-5, torch.ones(20, n))
    off = (xc.grad.cpu().double().view(20, n) - want[1]).abs().max()   # the exact gradient nearly cancels
    assert off <= ref.bound(dtype, n) * 4 and ref.error(wc.grad, want[2]) <= 1e-3


def test_layer_norm_values():
    # A constant row, a large level under a small spread, rows of infinity and NaN beside sound ones.
    x = normal(gen(3), 8, 200)
    x[0] = 3.0
    x[1] = 1e4 + x[1]
    x[2, 7], x[3, 9] = float("inf"), float("nan")
    y = memory.layer_norm(x.cuda()).cpu()
    assert torch.equal(y[0], torch.zeros(200))
    want = ref.layer_norm(x, None, None, 1e-5)
    # At 1e4 a float32 value is itself known to 2^-24 1e4 = 6e-4; the formula takes it as exact, the mean is rounded.
    assert ref.error(y[1], want[1]) <= 2e-3
    assert bool(y[2:4].isnan().all())
    assert ref.error(y[4:], want[4:]) <= ref.bound(torch.float32, 200)


def test_layer_norm_empty_and_long():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = memory.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y.sum(), (x, w))
    assert y.shape == (0, 16) and dx.shape == (0, 16) and torch.equal(dw, torch.zeros_like(w))
    # Offsets past 2^31 elements.
    rows, n = (1 << 22) + 3, 520
    x = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda").normal_()
    y = memory.layer_norm(x)
    tail = x[-5:].cpu()
    assert ref.error(y[-5:], ref.layer_norm(tail, None, None, 1e-5)) <= ref.bound(torch.bfloat16, n)


def test_layer_norm_differences():
    g = gen(5)
    x, w, b, dy = normal(g, 6, 50), 1 + 0.3 * normal(g, 50), normal(g, 50), normal(g, 6, 50)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(memory.layer_norm(*leaves), leaves, dy.cuda())
    for i, grad in enumerate(grads):
        d, h = normal(g, *leaves[i].shape).cuda(), 1e-2
        f = lambda s: float((memory.layer_norm(*[t + s * h * d if j == i else t for j, t in
                                                 enumerate(leaves)]).double().detach() * dy.cuda()).sum())
        slope = (f(1) - f(-1)) / (2 * h)
        # Central differences: h^2 times a third derivative of order 1, and 2^-24 sqrt(300) / h of rounding.
        assert abs(slope - float((grad * d).sum())) <= 2e-3 * float(grad.norm() * d.norm()) + 1e-3


# ------------------------------------------------------------ linear attention
def attention_case(seed, T, E, H, Dk, Dv, dtype, state=True, resets=0.1, decay=None):
    g = gen(seed)
    q, k, v = (normal(g, T, E, H, d, dtype=dtype) for d in (Dk, Dk, Dv))
    decay = 1 - torch.exp2(-1 - 5 * torch.rand(H, generator=g)) if decay is None else decay
    S = 2 * normal(g, E, H, Dk, Dv) if state else None
    r = torch.rand(T, E, generator=g) < resets if resets is not None else None
    do, dlast = normal(g, T, E, H, Dv, dtype=dtype), normal(g, E, H, Dk, Dv)
    return q, k, v, decay, S, r, do, dlast


def check_attention(case, dtype, final=True, scale=None, view=lambda t: t):
    q, k, v, decay, S, r, do, dlast = case
    scale_ = q.shape[-1] ** -0.5 if scale is None else scale
    leaves = [view(t.cuda()).requires_grad_() for t in (q, k, v)]
    Sc = None if S is None else S.cuda().requires_grad_()
    rc = None if r is None else r.cuda()
    o, last = memory.linear_attention(*leaves, decay.cuda(), Sc, rc, scale, final)
    outs, gos = [o], [do.cuda()]
    if final:
        outs.append(last)
        gos.append(dlast.cuda())
    wanted = leaves + ([] if Sc is None else [Sc])
    grads = torch.autograd.grad(outs, wanted, gos)
    want = ref.attention(q, k, v, decay, S, r, scale_, do, dlast if final else None)
    T = q.shape[0]
    terms = (T + 8) * (q.shape[3] + v.shape[3])
    # bfloat16: the output, a weight of the steps within a chunk, the state and a decayed operand are rounded once each.
    tol = ref.bound(dtype, terms, 4)
    assert ref.error(o, want[0]) <= tol
    if final:
        assert ref.error(last, want[1]) <= (STATE if dtype == torch.bfloat16 else ref.bound(dtype, terms))
    for got, exact in zip(grads[:3], want[2:5]):
        assert got.dtype == dtype and ref.error(got, exact) <= tol
    if Sc is not None:
        assert ref.error(grads[3], want[5]) <= (STATE if dtype == torch.bfloat16 else ref.bound(dtype, terms))
    with torch.no_grad():
        o2, last2 = memory.linear_attention(*leaves, decay.cuda(), Sc, rc, scale, final)
    assert ref.error(o2, want[0]) <= tol
    if final:
        assert ref.error(last2, want[1]) <= (STATE if dtype == torch.bfloat16 else ref.bound(dtype, terms))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 24, 31, 33, 48, 63, 64, 65, 128, 130, 200])
def test_attention_lengths(T, dtype):
    check_attention(attention_case(T, T, 3, 2, 64, 64, dtype), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("Dk,Dv", [(1, 1), (8, 8), (16, 24), (20, 28), (32, 32), (33, 7), (40, 64), (64, 16), (100, 72),
                                   (128, 128), (128, 8), (5, 128)])
def test_attention_head_sizes(Dk, Dv, dtype):
    for T in (20, 97):
        check_attention(attention_case(Dk * 131 + Dv, T, 2, 3, Dk, Dv, dtype), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("resets", [None, 0.0, 0.5, 1.0])
@pytest.mark.parametrize("final", [False, True])
def test_attention_options(dtype, state, resets, final):
    for T in (24, 150):
        check_attention(attention_case(7, T, 3, 2, 32, 32, dtype, state, resets), dtype, final,
                        0.7 if state else None)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_decays(dtype):
    # No memory, all of it, and powers that leave float32's range within a chunk.
    decay = torch.tensor([0.0, 1.0, 1e-3, 0.999])
    check_attention(attention_case(11, 150, 2, 4, 32, 32, dtype, resets=0.02, decay=decay), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,E,H,D", [(3000, 1, 2, 64), (1500, 2, 1, 128), (2500, 1, 1, 24), (129, 1, 1, 16), (700, 3, 5, 33)])
def test_attention_long(T, E, H, D, dtype):
    check_attention(attention_case(T, T, E, H, D, D, dtype, resets=0.005), dtype)
    check_attention(attention_case(T, T, E, H, D, D, dtype, state=False, resets=None), dtype, False)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [20, 64])
def test_attention_strides(D, dtype):
    T, E, H = 40, 3, 2
    case = attention_case(5, T, E, H, D, D, dtype)
    # Environment-major storage, one buffer of all three, heads broadcast from one.
    check_attention(case, dtype, view=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))
    check_attention(case, dtype, view=lambda t: torch.cat([t, t[..., :3]], -1)[..., :t.shape[-1]])
    check_attention(case, dtype, view=lambda t: t.transpose(2, 3).contiguous().transpose(2, 3))
    q, k, v, decay, S, r, do, dlast = case
    shared = k[:, :, :1].cuda().requires_grad_()
    o, _ = memory.linear_attention(q.cuda(), shared.expand(T, E, H, D), v.cuda(), decay.cuda(), S.cuda(), r.cuda())
    grad, = torch.autograd.grad(o, shared, do.cuda())
    want = ref.attention(q, k[:, :, :1].expand(T, E, H, D), v, decay, S, r, D ** -0.5, do)
    # The gradients of the heads are rounded before their sum, and the sum again.
    assert ref.error(grad, want[3].sum(2, keepdim=True)) <= ref.bound(dtype, 1000, 6)


def test_attention_of_many_heads_that_are_not_finite():
    T, E, H, D = 40, 250, 2, 16
    q, k, v, decay, S, _, do, _ = attention_case(37, T, E, H, D, D, torch.bfloat16, state=False)
    r = torch.zeros(T, E, dtype=torch.bool)
    r[20] = True
    want = ref.attention(q, k, v, decay, None, r, D ** -0.5, do)
    v = v.clone()
    v[3] = float("inf")
    leaves = [t.cuda().requires_grad_() for t in (q, k, v)]
    o, last = memory.linear_attention(*leaves, decay.cuda(), None, r.cuda())
    grads = torch.autograd.grad(o, leaves, do.cuda())
    tol = ref.bound(torch.bfloat16, 1000, 4)
    assert ref.error(o[:3], want[0][:3]) <= tol and ref.error(o[20:], want[0][20:]) <= tol
    assert ref.error(last, want[1]) <= STATE
    for got, exact in zip(grads, want[2:5]):
        assert ref.error(got[20:], exact[20:]) <= tol


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [24, 150, 900])
def test_attention_keeps_episodes_and_the_future_apart(T, dtype):
    """What an earlier episode or a later step holds, infinities and NaN
    included, reaches neither outputs nor gradients that do not depend on it."""
    bad, cut = T // 3, T // 2
    q, k, v, decay, S, _, do, dlast = attention_case(13, T, 2, 2, 32, 32, dtype)
    r = torch.zeros(T, 2, dtype=torch.bool)
    r[cut] = True
    want = ref.attention(q, k, v, decay, S, r, 32 ** -0.5, do, dlast)
    dirty_k, dirty_v, dirty_q, dirty_S = k.clone(), v.clone(), q.clone(), S.clone()
    dirty_v[bad, 0, 0, 3], dirty_k[bad, 0, 1, 4], dirty_q[bad, 0, 0, 5] = float("inf"), float("nan"), float("nan")
    dirty_S[1, 0, 0, 0] = float("inf")
    leaves = [t.cuda().requires_grad_() for t in (dirty_q, dirty_k, dirty_v)]
    o, last = memory.linear_attention(*leaves, decay.cuda(), dirty_S.cuda(), r.cuda())
    grads = torch.autograd.grad([o, last], leaves, [do.cuda(), dlast.cuda()])
    terms = (T + 8) * 64
    tol = ref.bound(dtype, terms, 4)
    # Environment 0: sound before the bad step and from the reset on.
    for part in (slice(0, bad), slice(cut, T)):
        assert ref.error(o[part, 0], want[0][part, 0]) <= tol
    assert not bool(o[bad, 0].isfinite().all())
    assert ref.error(last, want[1]) <= (STATE if dtype == torch.bfloat16 else ref.bound(dtype, terms))
    # dq sees the past, dk and dv the future up to the episode's end.
    assert ref.error(grads[0][:bad, 0], want[2][:bad, 0]) <= tol
    for got, exact in zip(grads, want[2:5]):
        assert ref.error(got[cut:, 0], exact[cut:, 0]) <= tol
    for got, exact in zip(grads[1:], want[3:5]):
        assert ref.error(got[bad + 1:cut, 0], exact[bad + 1:cut, 0]) <= tol
    # Environment 1: a state that is not finite ends at the reset.
    assert ref.error(o[cut:, 1], want[0][cut:, 1]) <= tol
    assert ref.error(o[:, 1, 1], want[0][:, 1, 1]) <= tol


@pytest.mark.parametrize("Dk,Dv", [(16, 16), (64, 64), (128, 128), (40, 64), (128, 24), (7, 100)])
def test_attention_keeps_apart_at_every_head_size(Dk, Dv):
    for T in (20, 70, 300):
        q, k, v, decay, S, _, do, dlast = attention_case(Dk + T, T, 3, 2, Dk, Dv, torch.bfloat16)
        cut = T // 2
        r = torch.zeros(T, 3, dtype=torch.bool)
        r[cut] = True
        want = ref.attention(q, k, v, decay, S, r, Dk ** -0.5, do, dlast)
        for name in range(4):   # in v, k, q, the gradient of the output, of environment 1 alone
            dirty = [t.clone() for t in (v, k, q, do)]
            dirty[name][cut - 2, 1] = float("nan")
            leaves = [t.cuda().requires_grad_() for t in (dirty[2], dirty[1], dirty[0])]
            state = S.cuda().requires_grad_()
            o, last = memory.linear_attention(*leaves, decay.cuda(), state, r.cuda())
            grads = torch.autograd.grad([o, last], [*leaves, state], [dirty[3].cuda(), dlast.cuda()])
            tol = ref.bound(torch.bfloat16, 1, 4)
            assert ref.error(last, want[1]) <= STATE
            for got, exact in zip((o, *grads[:3]), (want[0], *want[2:5])):
                assert ref.error(got[cut:], exact[cut:]) <= tol
                assert ref.error(got[:, ::2], exact[:, ::2]) <= tol
            assert ref.error(o[:cut - 2], want[0][:cut - 2]) <= tol
            assert ref.error(grads[0][:cut - 2], want[2][:cut - 2]) <= tol
            assert ref.error(grads[1][cut - 1:], want[3][cut - 1:]) <= tol
            assert ref.error(grads[3][::2], want[5][::2]) <= STATE


def test_attention_of_a_state_at_an_odd_place():
    T, E, H, D = 40, 2, 2, 32
    q, k, v, decay, S, r, do, _ = attention_case(3, T, E, H, D, D, torch.bfloat16)
    flat = torch.empty(S.numel() + 1, device="cuda")
    state = flat[1:].view(S.shape).copy_(S)
    want = ref.attention(q, k, v, decay, S, r, D ** -0.5)
    o, last = memory.linear_attention(q.cuda(), k.cuda(), v.cuda(), decay.cuda(), state, r.cuda())
    assert ref.error(o, want[0]) <= ref.bound(torch.bfloat16, 1, 4) and ref.error(last, want[1]) <= STATE
    first = ref.attention(q[:1], k[:1], v[:1], decay, S, r[:1], D ** -0.5)
    o = memory.linear_attention_step(q[0].cuda(), k[0].cuda(), v[0].cuda(), decay.cuda(), state, r[0].cuda())
    assert ref.error(o, first[0][0]) <= ref.bound(torch.bfloat16, 1) and ref.error(state, first[1]) <= 1e-6
    odd = torch.empty(q.numel() + 1, device="cuda", dtype=torch.bfloat16)[1:].view(q.shape).copy_(q)
    o2, _ = memory.linear_attention(odd, k.cuda(), v.cuda(), decay.cuda(), S.cuda(), r.cuda())
    assert ref.error(o2, want[0]) <= ref.bound(torch.bfloat16, 1, 4)


def test_attention_empty_and_far():
    decay = torch.tensor([0.9], device="cuda")
    S = torch.randn(2, 1, 8, 8, device="cuda", requires_grad=True)
    q = torch.zeros(0, 2, 1, 8, device="cuda", requires_grad=True)
    o, last = memory.linear_attention(q, q, q, decay, S)
    assert o.shape == (0, 2, 1, 8) and torch.equal(last, S)
    dS, = torch.autograd.grad(last.sum(), S)
    assert torch.equal(dS, torch.ones_like(S))
    assert torch.equal(memory.linear_attention(q.detach(), q.detach(), q.detach(), decay)[1], torch.zeros_like(S))
    q16 = q.detach().bfloat16()
    assert torch.equal(memory.linear_attention(q16, q16, q16, decay, S.detach())[1], S)
    none = torch.zeros(4, 0, 1, 8, device="cuda")
    assert memory.linear_attention(none, none, none, decay)[0].shape == (4, 0, 1, 8)
    # Offsets past 2^31 elements between steps.
    T, E, H, D = 10, 2, 1, 16
    case = attention_case(17, T, E, H, D, D, torch.bfloat16)
    far = torch.empty((1 << 31) + (1 << 28) + E * H * D, dtype=torch.bfloat16, device="cuda")
    place = lambda t: far.as_strided((T, E, H, D), (1 << 28, H * D, D, 1)).copy_(t)
    q, k, v, decay, S, r, do, dlast = case
    o, last = memory.linear_attention(place(q.cuda()), k.cuda(), v.cuda(), decay.cuda(), S.cuda(), r.cuda())
    want = ref.attention(q, k, v, decay, S, r, 0.25)
    assert ref.error(o, want[0]) <= ref.bound(torch.bfloat16, 100, 4) and ref.error(last, want[1]) <= STATE


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("E,H,Dk,Dv", [(1, 1, 1, 1), (5, 3, 20, 28), (16, 4, 64, 64), (700, 2, 32, 32), (3, 2, 128, 128),
                                       (4, 1, 100, 7), (9, 5, 16, 128)])
def test_attention_step(E, H, Dk, Dv, dtype):
    q, k, v, decay, S, r, _, _ = attention_case(E * 7 + Dk, 3, E, H, Dk, Dv, dtype, resets=0.3)
    state = S.cuda()
    outs = [memory.linear_attention_step(q[t].cuda(), k[t].cuda(), v[t].cuda(), decay.cuda(), state, r[t].cuda())
            for t in range(3)]
    want = ref.attention(q, k, v, decay, S, r, Dk ** -0.5)
    assert ref.error(torch.stack(outs), want[0]) <= ref.bound(dtype, Dk)
    assert ref.error(state, want[1]) <= ref.bound(torch.float32, 3)
    # Without resets, other strides, a scale.
    state = S.cuda()
    packed = torch.cat([q[0], k[0], v[0]], -1).cuda()
    o = memory.linear_attention_step(packed[..., :Dk], packed[..., Dk:2 * Dk], packed[..., 2 * Dk:], decay.cuda(), state,
                                     scale=0.5)
    want = ref.attention(q[:1], k[:1], v[:1], decay, S, None, 0.5)
    assert ref.error(o, want[0][0]) <= ref.bound(dtype, Dk) and ref.error(state, want[1]) <= ref.bound(torch.float32, 3)


def test_attention_step_clears_a_state_that_is_not_finite():
    S = torch.full((2, 1, 16, 16), float("nan"), device="cuda")
    q = torch.ones(2, 1, 16, device="cuda")
    o = memory.linear_attention_step(q, q, q, torch.tensor([0.5], device="cuda"), S,
                                     torch.tensor([True, False], device="cuda"), 1.0)
    assert torch.equal(S[0], torch.ones_like(S[0])) and bool(S[1].isnan().all())
    assert torch.equal(o[0], torch.full_like(o[0], 16.0))


def test_attention_step_far():
    # A state of more than 2^31 elements (8.6 GB), checked at its end.
    E, H, D = (1 << 17) + 1, 1, 128
    state = torch.ones(E, H, D, D, device="cuda")
    q = torch.ones(E, H, D, device="cuda", dtype=torch.bfloat16)
    o = memory.linear_attention_step(q, q, q, torch.tensor([0.5], device="cuda"), state, None, 1.0)
    assert torch.equal(state[-2:], torch.full_like(state[-2:], 1.5))
    assert torch.equal(o[-2:].float(), torch.full((2, H, D), 192.0, device="cuda"))


def test_attention_differences():
    T, E, H, D = 21, 2, 2, 12
    q, k, v, decay, S, r, do, dlast = attention_case(23, T, E, H, D, D, torch.float32)
    leaves = [t.cuda().requires_grad_() for t in (q, k, v, S)]
    run = lambda q, k, v, S: memory.linear_attention(q, k, v, decay.cuda(), S, r.cuda())
    value = lambda *x: sum(float((a.detach().double() * b.cuda()).sum()) for a, b in zip(run(*x), (do, dlast)))
    grads = torch.autograd.grad(run(*leaves), leaves, [do.cuda(), dlast.cuda()])
    g = gen(29)
    for i, grad in enumerate(grads):
        d, h = normal(g, *leaves[i].shape).cuda(), 0.25
        moved = lambda s: [t + s * h * d if j == i else t for j, t in enumerate(leaves)]
        # The output is linear in each operand: a difference has no error but float32's.
        slope = (value(*moved(1)) - value(*moved(-1))) / (2 * h)
        assert abs(slope - float((grad.double() * d).sum())) <= 1e-4 * float(grad.norm() * d.norm())


# ----------------------------------------------------------- 8-bit checkpoints
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 8), (5, 61), (7, 127), (4, 128), (6, 129), (9, 256), (33, 200), (2, 1000),
                                    (5, 512), (3, 4100), (129, 16)])
def test_checkpoint(rows, n, dtype):
    g = gen(rows * 31 + n)
    x, dy = (2 * normal(g, rows, n)).to(dtype), normal(g, rows, n, dtype=dtype)
    x[0, : n // 2] = 0.0
    y, kept = memory.elu_checkpoint(x.cuda())
    exact = torch.where(x > 0, x.double(), torch.expm1(x.double()))
    assert y.dtype == dtype and ref.error(y, exact) <= ref.bound(dtype, 1)
    codes, scales = ref.kept(y.cpu())
    assert torch.equal(kept.codes.cpu(), codes) and torch.equal(kept.scales.cpu(), scales)
    dx, back = memory.elu_restore(dy.cuda(), kept)
    stood = codes.double() * scales.double().repeat_interleave(128, 1)[:, :n]
    assert ref.error(back, stood) <= ref.bound(dtype, 1)
    want = dy.double() * torch.where(stood > 0, torch.ones_like(stood), 1 + stood)
    assert ref.error(dx, want) <= ref.bound(dtype, 1)
    # Half a step of a group's scale is the most that a kept value is off.
    assert bool(((stood - y.cpu().double()).abs() <= 0.501 * scales.double().repeat_interleave(128, 1)[:, :n]).all())
    only, nothing = memory.elu_restore(dy.cuda(), kept, restore=False)
    assert nothing is None and torch.equal(only, dx)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [256, 257])
def test_checkpoint_values(n, dtype):
    """A group of zeros, of denormals, with an infinity, with a NaN: the others
    of its row are not touched."""
    x = normal(gen(2), 6, n).to(dtype)
    x[0, :128], x[1, :128] = 0.0, 1e-39
    x[2, 5], x[3, 130], x[4, 7] = float("inf"), float("nan"), float("-inf")
    y, kept = memory.elu_checkpoint(x.cuda())
    dx, back = memory.elu_restore(torch.ones_like(y), kept)
    back, codes = back.cpu().float(), kept.codes.cpu()
    assert torch.equal(back[0, :128], torch.zeros(128)) and torch.equal(back[1, :128], torch.zeros(128))
    assert bool(back[2, :128].isnan().all()) and bool(back[2, 128:].isfinite().all())
    assert bool(back[3, 128:256].isnan().all()) and bool(back[3, :128].isfinite().all())
    assert bool(back[4].isfinite().all()) and float(y[4, 7]) == -1.0   # elu of minus infinity
    assert int(codes.min()) >= -127
    assert bool(dx[2, :128].isnan().all()) and bool(dx[5].isfinite().all())


def test_checkpoint_empty_strided_and_long():
    y, kept = memory.elu_checkpoint(torch.zeros(0, 40, device="cuda"))
    assert y.shape == (0, 40) and kept.scales.shape == (0, 1)
    assert memory.elu_restore(y, kept)[0].shape == (0, 40)
    x = normal(gen(4), 3, 5, 300)
    flat, _ = memory.elu_checkpoint(x.cuda())
    turned, kept = memory.elu_checkpoint(x.cuda().transpose(0, 1))
    assert torch.equal(turned.transpose(0, 1), flat) and kept.codes.shape == (5, 3, 300)
    dx, _ = memory.elu_restore(torch.ones(1, 1, 1, device="cuda").expand(5, 3, 300), kept)
    assert bool(dx.isfinite().all())
    rows, n = (1 << 22) + 3, 520
    x = torch.empty(rows, n, dtype=torch.bfloat16, device="cuda").normal_()
    y, kept = memory.elu_checkpoint(x)
    codes, scales = ref.kept(y[-3:].cpu())
    assert torch.equal(kept.codes[-3:].cpu(), codes) and torch.equal(kept.scales[-3:].cpu(), scales)
    del x
    dx, back = memory.elu_restore(y, kept)
    stood = codes.double() * scales.double().repeat_interleave(128, 1)[:, :n]
    assert ref.error(back[-3:], stood) <= ref.bound(torch.bfloat16, 1)


@pytest.mark.parametrize("dtype", TYPES)
def test_checkpointed_mlp(dtype):
    g = gen(6)
    sizes = (61, 200, 96, 14)
    x = normal(g, 300, sizes[0], dtype=dtype)
    w = [(normal(g, o, i) / i ** 0.5).to(dtype) for i, o in zip(sizes, sizes[1:])]
    b = [(0.1 * normal(g, o)).to(dtype) for o in sizes[1:]]
    dy = normal(g, 300, sizes[-1], dtype=dtype)
    leaves = [t.cuda().requires_grad_() for t in (x, *w, *b)]
    y = memory.checkpointed_mlp(leaves[0], leaves[1:4], leaves[4:])
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    exact = [t.double().requires_grad_() for t in (x, *w, *b)]
    z = exact[0]
    for i in range(3):
        z = z @ exact[1 + i].t() + exact[4 + i]
        z = torch.nn.functional.elu(z) if i < 2 else z
    want = torch.autograd.grad(z, exact, dy.double())
    assert ref.error(y, z) <= ref.bound(dtype, 400, 8)
    # A kept value is off by at most half of max |y| / 127 of its group, uniformly: max |y| 0.0023 in the mean square,
    # where max |y| is some 3 times the activations' own: 0.7 % a layer, two layers; bfloat16's roundings besides.
    for got, exact_ in zip(grads, want):
        assert ref.error(got, exact_) <= 0.02 + ref.bound(dtype, 400, 8)


# ------------------------------------------------ streams, graphs and refusals
def test_operators_on_another_stream_and_in_a_graph():
    g = gen(8)
    x, w = normal(g, 64, 256, dtype=torch.bfloat16).cuda(), torch.ones(256, device="cuda")
    case = attention_case(31, 30, 4, 2, 64, 64, torch.bfloat16)
    q, k, v, decay, S, r, do, _ = (t.cuda() for t in case)
    dy = torch.ones_like(x)

    def everything():
        xs, ws = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = memory.layer_norm(xs, ws)
        heads = [t.detach().requires_grad_() for t in (q, k, v)]
        o, last = memory.linear_attention(*heads, decay, S, r)
        z, kept = memory.elu_checkpoint(x)
        state = S.clone()
        step = memory.linear_attention_step(q[0], k[0], v[0], decay, state, r[0])
        return [y, *torch.autograd.grad(y, (xs, ws), dy), o, last, *torch.autograd.grad(o, heads, do), z,
                *memory.elu_restore(dy, kept), state, step]

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


def test_refusals_on_the_gpu():
    half = torch.zeros(4, 8, device="cuda", dtype=torch.float16)
    for call in (memory.layer_norm, memory.elu_checkpoint):
        with pytest.raises(RuntimeError):
            call(half)
        with pytest.raises(RuntimeError):
            call(half.double())
    x, decay = torch.zeros(4, 2, 1, 8, device="cuda"), torch.ones(1, device="cuda")
    state = torch.zeros(2, 1, 8, 8, device="cuda")
    with pytest.raises(RuntimeError):
        memory.linear_attention(x.half(), x.half(), x.half(), decay)
    with pytest.raises(RuntimeError):
        memory.linear_attention(x, x, x, decay.cpu())
    with pytest.raises(RuntimeError):
        memory.linear_attention(x, x, x, decay, state.cpu())
    with pytest.raises(RuntimeError):
        memory.linear_attention(x, x, x, decay, state.bfloat16())
    with pytest.raises(RuntimeError):
        memory.linear_attention_step(x[0], x[0], x[0], decay, state.transpose(2, 3))
    with pytest.raises(RuntimeError):
        memory.layer_norm(x, torch.ones(8))
    y, kept = memory.elu_checkpoint(x)
    with pytest.raises(RuntimeError):
        memory.elu_restore(y.cpu(), kept)


def test_c_entries_refuse():
    from duck_gym_b200.cuda_batch import library

    lib = library()
    x = torch.zeros(4, 8, device="cuda")
    p = x.data_ptr()
    assert lib.duck_layer_norm_forward(p, None, None, p, None, 4, 0, 8, 1e-5, 0, None) != 0
    assert lib.duck_layer_norm_forward(p, None, None, p, None, 4, 8, 8, 1e-5, 2, None) != 0
    assert lib.duck_layer_norm_forward(None, None, None, p, None, 4, 8, 8, 1e-5, 0, None) != 0
    assert lib.duck_layer_norm_forward(p, None, None, p, None, 4, 8, 8, float("nan"), 0, None) != 0
    assert lib.duck_layer_norm_backward(p, p, None, p, None, p, None, None, 4, 8, 8, 8, 0, None) != 0
    assert lib.duck_layer_norm_scratch(4, 0) == -1
    assert lib.duck_elu_checkpoint(p, p, None, p, 4, 8, 0, None) != 0
    assert lib.duck_elu_restore(p, p, p, None, p, -1, 8, 0, None) != 0
    q, decay = torch.zeros(4, 2, 1, 8, device="cuda"), torch.ones(1, device="cuda")
    state = torch.zeros(2, 1, 8, 8, device="cuda")
    for wrong in (dict(out=0), dict(out=p, state_in=state.data_ptr() + 4)):
        assert lib.duck_linear_attention_forward(memory._pack(q, q, q, decay, None, 1.0, **wrong), None) != 0
    assert lib.duck_linear_attention_backward(memory._pack(q, q, q, decay, None, 1.0, out=p), None) != 0
    wide = torch.zeros(1, 1, 1, 129, device="cuda")
    assert lib.duck_linear_attention_step(memory._pack(wide, wide, wide, decay, None, 1.0, out=p), None) != 0
    half = torch.zeros(4, 2, 1, 8, device="cuda", dtype=torch.bfloat16)
    assert lib.duck_linear_attention_forward(memory._pack(half, half, half, decay, None, 1.0, out=p), None) != 0   # scratch
    assert lib.duck_linear_attention_forward(None, None) != 0
    assert b"Invalid" in lib.duck_last_error()
