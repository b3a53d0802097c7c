"""Operators of a policy with memory: layer norm, linear attention with one
decay per head, a gated linear recurrence, a gated linear layer, and activations
kept in 8 bits for the backward pass.

    layer_norm(x, weight, bias, eps)                           -> y
    linear_attention(q, k, v, decay, state, resets, ...)       -> out, state
    linear_attention_step(q, k, v, decay, state, reset, ...)   -> out
    gated_recurrence(gates, values, state, resets, ...)        -> out, state
    gated_recurrence_step(gates, values, state, reset)         -> out
    gated_linear(x, w_gate, w_up, b_gate, b_up, activation)    -> h
    elu_checkpoint(x)                                          -> y, Checkpoint8
    elu_restore(dy, kept)                                      -> dx, y
    checkpointed_mlp(x, weights, biases)                       -> y

The reference has no counterpart: it trains rsl-rl's feed-forward actor-critic
(scripts/train_bam_native.py:14-140).  Rollouts are time-major, ``[T, E, ...]``,
as in ``ppo.Storage``.

CUDA tensors run the library's kernels on the current stream (float32 or
bfloat16 activations, no other type; there is no fallback), CPU tensors a plain
torch restatement.  Wrong devices, types or shapes raise ``RuntimeError``.  The
last axis of every operand has to be dense, otherwise a dense copy is made;
other strides are taken as they are.  The calls allocate only with torch, never
synchronise and can be captured in CUDA graphs.
"""

from __future__ import annotations

import ctypes
import functools
import struct
from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .cuda_batch import _raise, library

GROUP = 128      # values of a row that share one scale of a checkpoint
HEAD_MAX = 128   # largest head size of the linear attention
_TYPES = {torch.float32: 0, torch.bfloat16: 1}


# The stream and device that torch has current, without the objects around them:
# the public calls cost more than a launch.
_stream_of = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_current_device = getattr(torch._C, "_cuda_getDevice", None)


def _launch(entry, device, *args):
    """Calls a C entry on torch's current stream of `device`."""
    index = device.index
    if index == _current_device():
        status = entry(*args, _stream_of(index))
    else:
        with torch.cuda.device(device):
            status = entry(*args, _stream_of(index))
    if status:
        _raise(status)


def _once(backward):
    """A backward pass without a second one.  torch's once_differentiable does
    the bookkeeping for create_graph; it is left out where no graph is made."""
    twice = once_differentiable(backward)

    def run(ctx, *grads):
        return (twice if torch.is_grad_enabled() else backward)(ctx, *grads)

    return run


def _pointer(t):
    return None if t is None else t.data_ptr()


def _require(condition, message):
    if not condition:
        raise RuntimeError(message)


def _check_type(x, what):
    if x.is_cuda and x.dtype not in _TYPES:
        raise RuntimeError(f"{what}: CUDA activations are float32 or bfloat16, not {x.dtype}")


def _grad_needed(*tensors):
    """Whether a call goes through its autograd function: also wherever forward-mode
    derivatives are on, since that refuses an input with a tangent."""
    return forward_ad._current_level >= 0 or torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_tangents(*tensors):
    """For the calls without an autograd function: a tangent would be dropped."""
    if forward_ad._current_level >= 0:
        _require(all(forward_ad.unpack_dual(t).tangent is None for t in tensors),
                 "there are no forward-mode derivatives of this call")


# ------------------------------------------------------------------ layer norm
def _rows_of(x):
    """x as rows of its last axis, with a stride between them: a view where the
    layout allows one, else a dense copy."""
    n = x.shape[-1]
    if x.dim() != 2:
        x = x.reshape(-1, n)
    return x if x.stride(1) == 1 or n == 1 else x.contiguous()


def _dense_like(x):
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _norm_forward(x, weight, bias, eps, keep):
    rows = _rows_of(x)
    y = _dense_like(x)
    stats = torch.empty((rows.shape[0], 2), dtype=torch.float32, device=x.device) if keep else None
    _launch(library().duck_layer_norm_forward, x.device, rows.data_ptr(), _pointer(weight), _pointer(bias),
            y.data_ptr(), _pointer(stats), rows.shape[0], rows.shape[1], rows.stride(0), eps, _TYPES[x.dtype])
    return y, rows, stats


@functools.lru_cache(maxsize=1024)
def _norm_scratch(rows, n):
    return library().duck_layer_norm_scratch(rows, n)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, rows, stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, bias, stats)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, weight, bias, stats = ctx.saved_tensors
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        rows, n = x.shape
        dx = _dense_like(dy) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(bias) if need_b else None
        scratch = stats.new_empty(_norm_scratch(rows, n)) if need_w or need_b else None
        dy = _rows_of(dy)
        _launch(library().duck_layer_norm_backward, x.device, x.data_ptr(), dy.data_ptr(), _pointer(weight),
                stats.data_ptr(), _pointer(dx), _pointer(dw), _pointer(db), _pointer(scratch), rows, n, x.stride(0),
                dy.stride(0), _TYPES[x.dtype])
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x.

    ``weight`` and ``bias`` [n] are float32 on the GPU, whatever x's type (other
    types are converted, and their gradients converted back); the statistics
    and the sums of the gradients are float32, the result has x's type."""
    n = x.shape[-1] if x.dim() else 0
    _require(n > 0, "layer_norm: the last axis is empty")
    for t in (weight, bias):
        _require(t is None or (t.shape == (n,) and t.device == x.device), "layer_norm: invalid weight or bias")
    if not x.is_cuda:
        return F.layer_norm(x, (n,), weight, bias, eps)
    _check_type(x, "layer_norm")
    if weight is not None and (weight.dtype != torch.float32 or not weight.is_contiguous()):
        weight = weight.float().contiguous()
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_contiguous()):
        bias = bias.float().contiguous()
    if _grad_needed(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm_forward(x, weight, bias, eps, False)[0]


# ------------------------------------------------------------ linear attention
# struct duck_attention of include/duck_b200.h.
_ATTENTION = struct.Struct("@16P12q6if4x")


def _address(t):
    return 0 if t is None else t.data_ptr()


def _pack(q, k, v, decay, resets, scale, out=0, state_in=0, state_out=0, dout=None, dstate_out=0, dq=0, dk=0, dv=0,
          dstate_in=0, saved=0, scratch=0):
    T, E, H, Dk = q.shape
    return _ATTENTION.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out, decay.data_ptr(), 0 if resets is None else resets.data_ptr(),
        state_in, state_out, 0 if dout is None else dout.data_ptr(), dstate_out, dq, dk, dv, dstate_in, saved, scratch,
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *((0, 0, 0) if dout is None else dout.stride()[:3]),
        T, E, H, Dk, v.shape[3], _TYPES[q.dtype], scale)


def _dense_last(x):
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _aligned(state):
    """Dense and on a 16-byte boundary."""
    state = state.contiguous()
    return state if state.data_ptr() % 16 == 0 else state.clone()


@functools.lru_cache(maxsize=1024)
def _workspace(T, E, H, Dk, Dv, kind):
    """Bytes of scratch of a forward and of a backward call, and of what the
    first keeps for the second."""
    out = (ctypes.c_int64 * 3)()
    _raise(library().duck_linear_attention_sizes(
        _ATTENTION.pack(*(0,) * 16, *(0,) * 12, T, E, H, Dk, Dv, kind, 1.0), out))
    return tuple(out)


def _buffer(bytes_, device):
    return torch.empty(bytes_, dtype=torch.uint8, device=device) if bytes_ else None


def _attention_forward(q, k, v, decay, state, resets, scale, final_state, keep):
    T, E, H, Dk = q.shape
    Dv = v.shape[3]
    out = _dense_like(v)
    last = torch.empty((E, H, Dk, Dv), dtype=torch.float32, device=q.device) if final_state else None
    args = dict(out=out.data_ptr(), state_in=_address(state), state_out=_address(last))
    sizes = _workspace(T, E, H, Dk, Dv, _TYPES[q.dtype])
    scratch = _buffer(sizes[0], q.device)
    saved = _buffer(sizes[2], q.device) if keep else None
    _launch(library().duck_linear_attention_forward, q.device,
            _pack(q, k, v, decay, resets, scale, scratch=_address(scratch), saved=_address(saved), **args))
    return out, last, saved


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, decay, state, resets, scale, final_state):
        out, last, saved = _attention_forward(q, k, v, decay, state, resets, scale, final_state, True)
        ctx.save_for_backward(q, k, v, decay, state, resets, saved)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @_once
    def backward(ctx, dout, dlast):
        q, k, v, decay, state, resets, saved = ctx.saved_tensors
        if dout is None and dlast is None:
            return (None,) * 8
        T, E, H, Dk = q.shape
        Dv = v.shape[3]
        dout = q.new_zeros((T, E, H, Dv)) if dout is None else _dense_last(dout)
        dlast = None if dlast is None else _aligned(dlast)
        dq, dk, dv = _dense_like(q), _dense_like(k), _dense_like(v)
        dstate = torch.empty_like(state) if ctx.needs_input_grad[4] else None
        args = dict(state_in=_address(state), dout=dout, dstate_out=_address(dlast), dq=dq.data_ptr(),
                    dk=dk.data_ptr(), dv=dv.data_ptr(), dstate_in=_address(dstate), saved=_address(saved))
        scratch = _buffer(_workspace(T, E, H, Dk, Dv, _TYPES[q.dtype])[1], q.device)
        _launch(library().duck_linear_attention_backward, q.device,
                _pack(q, k, v, decay, resets, ctx.scale, scratch=_address(scratch), **args))
        return dq, dk, dv, None, dstate, None, None, None


@torch.autocast("cpu", enabled=False)
def _attention_plain(q, k, v, decay, state, resets, scale):
    """The recurrence step by step, in float32 or wider.  Element by element: the
    gradient of a matrix product would be rounded to fewer bits by a backward
    pass inside an autocast region."""
    dtype = q.dtype
    wide = torch.promote_types(dtype, torch.float32)
    T, E, H, Dk = q.shape
    q, k, v, decay = q.to(wide) * scale, k.to(wide), v.to(wide), decay.to(wide)[None, :, None, None]
    S = q.new_zeros(E, H, Dk, v.shape[3]) if state is None else state if T else state.clone()
    out = []
    for t in range(T):
        if resets is not None:
            S = torch.where(resets[t, :, None, None, None] != 0, torch.zeros_like(S), S)
        S = decay * S + k[t][..., :, None] * v[t][..., None, :]
        out.append((q[t][..., :, None] * S).sum(-2))
    out = torch.stack(out) if T else q.new_zeros(0, E, H, v.shape[3])
    return out.to(dtype), S


# The type of states and scores beside a type of activations.
_WIDE = {torch.float32: torch.float32, torch.bfloat16: torch.float32, torch.float16: torch.float32,
         torch.float64: torch.float64}


def _check_heads(q, k, v, decay, dims, what):
    qs, vs, dtype, device = q.shape, v.shape, q.dtype, q.device
    _require(len(qs) == len(vs) == dims and qs == k.shape and qs[:-1] == vs[:-1],
             "q and k have one shape, and v theirs but for its last axis")
    _require(dtype == k.dtype == v.dtype and device == k.device == v.device and dtype in _WIDE,
             "q, k and v have one floating type and device")
    _require(1 <= qs[-1] <= HEAD_MAX and 1 <= vs[-1] <= HEAD_MAX, "head sizes are 1 to 128")
    _check_type(q, what)
    _require(decay.shape == qs[-2:-1] and decay.device == device, "decay is [heads] on q's device")
    _require(not decay.requires_grad, "the decay is a constant of the layer, it has no gradient")


def _check_state(state, q, v):
    _require(state.shape == q.shape[-3:] + v.shape[-1:] and state.dtype == _WIDE[q.dtype] and state.device == q.device,
             "the state is float32 [environments, heads, Dk, Dv] on q's device")


def _mask(resets, shape, device):
    _require(resets.shape == shape and resets.device == device and resets.dtype in (torch.bool, torch.uint8),
             "resets are bool or uint8 [steps, environments] on q's device")
    return resets if resets.is_contiguous() else resets.contiguous()


def linear_attention(q, k, v, decay, state=None, resets=None, scale=None, final_state=True):
    """Linear attention over a rollout: ``(out, state)`` with

        S_t = f_t S_{t-1} + k_t v_t^T,   out_t = scale S_t^T q_t,

    f_t = decay[h], or 0 where ``resets[t, e]`` says that an episode begins.

    ``q`` and ``k`` [T, E, H, Dk], ``v`` [T, E, H, Dv] (T steps, E environments,
    H heads, head sizes up to 128); ``decay`` [H] in [0, 1], a constant of the
    layer; ``state`` [E, H, Dk, Dv] float32 before the first step (None: zero);
    ``scale`` is Dk ** -0.5 by default.  The state after the last step is
    returned where ``final_state`` is set, else None.  Gradients flow to q, k,
    v and the state.

    bfloat16 operands on the GPU: each term of an output or gradient is rounded to
    8 bits once on its way (a decayed score, or the state it is read from), and
    the result once more; the states themselves are float32.  Float32 operands
    are not rounded."""
    _check_heads(q, k, v, decay, 4, "linear_attention")
    if state is not None:
        _check_state(state, q, v)
    if resets is not None:
        resets = _mask(resets, q.shape[:2], q.device)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not q.is_cuda:
        out, last = _attention_plain(q, k, v, decay, state, resets, scale)
        return out, last if final_state else None
    q, k, v = _dense_last(q), _dense_last(k), _dense_last(v)
    if decay.dtype != torch.float32 or not decay.is_contiguous():
        decay = decay.float().contiguous()
    if state is not None:
        state = _aligned(state)
    if _grad_needed(q, k, v, state):
        return _LinearAttention.apply(q, k, v, decay, state, resets, scale, final_state)
    return _attention_forward(q, k, v, decay, state, resets, scale, final_state, False)[:2]


def linear_attention_step(q, k, v, decay, state, reset=None, scale=None):
    """One control step of ``linear_attention`` for every environment, without
    gradients: ``q`` and ``k`` [E, H, Dk], ``v`` [E, H, Dv], ``reset`` [E].
    ``state`` [E, H, Dk, Dv] float32 is updated in place; returns out
    [E, H, Dv].  A backward pass that still needs the state as it was raises, as
    after any operation in place (a replay of a CUDA graph is not seen)."""
    _check_heads(q, k, v, decay, 3, "linear_attention_step")
    _check_state(state, q, v)
    _require(not (state.requires_grad and torch.is_grad_enabled()),
             "the state is updated in place without gradients, it must not require one")
    if reset is not None:
        reset = _mask(reset, q.shape[:1], q.device)
    E, H, Dk = q.shape
    scale = Dk ** -0.5 if scale is None else float(scale)
    if not q.is_cuda:
        with torch.no_grad():
            out, last = _attention_plain(q[None], k[None], v[None], decay, state,
                                         None if reset is None else reset[None], scale)
            state.copy_(last)
        return out[0]
    _refuse_tangents(q, k, v, state)
    _require(state.is_contiguous(), "the state is updated in place and has to be contiguous")
    q, k, v = _dense_last(q), _dense_last(k), _dense_last(v)
    if decay.dtype != torch.float32 or not decay.is_contiguous():
        decay = decay.float().contiguous()
    qe, qh, _ = q.stride()
    ke, kh, _ = k.stride()
    ve, vh, Dv = *v.stride()[:2], v.shape[2]
    out = _dense_like(v)
    _launch(library().duck_linear_attention_step, q.device,
            _ATTENTION.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), decay.data_ptr(),
                            _address(reset), 0, state.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0,
                            0, qe, qh, 0, ke, kh, 0, ve, vh, 0, 0, 0, 1, E, H, Dk, Dv, _TYPES[q.dtype], scale))
    torch.autograd.graph.increment_version(state)   # autograd does not see a kernel's writes
    return out


# ------------------------------------------------------------ gated recurrence
# struct duck_recurrence of include/duck_b200.h.
_RECURRENCE = struct.Struct("@13P6q4i")


@functools.lru_cache(maxsize=1024)
def _recurrence_workspace(T, E, N, kind):
    """Bytes of scratch of a call, and of what a forward call keeps for the
    backward one."""
    out = (ctypes.c_int64 * 2)()
    _raise(library().duck_gated_recurrence_sizes(_RECURRENCE.pack(*(0,) * 13, *(0,) * 6, T, E, N, kind), out))
    return tuple(out)


def _recurrence_forward(gates, values, state, resets, final_state, keep):
    T, E, N = gates.shape
    kind = _TYPES[gates.dtype]
    out = _dense_like(gates)
    last = torch.empty((E, N), dtype=torch.float32, device=gates.device) if final_state else None
    sizes = _recurrence_workspace(T, E, N, kind)
    scratch = _buffer(sizes[0], gates.device)
    saved = _buffer(sizes[1], gates.device) if keep else None
    _launch(library().duck_gated_recurrence_forward, gates.device,
            _RECURRENCE.pack(gates.data_ptr(), values.data_ptr(), out.data_ptr(), _address(resets), _address(state),
                             _address(last), 0, 0, 0, 0, 0, _address(saved), _address(scratch),
                             *gates.stride()[:2], *values.stride()[:2], 0, 0, T, E, N, kind))
    return out, last, saved


class _GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, values, state, resets, final_state):
        out, last, saved = _recurrence_forward(gates, values, state, resets, final_state, True)
        ctx.save_for_backward(gates, values, state, resets, saved)
        ctx.set_materialize_grads(False)
        return out, last

    @staticmethod
    @_once
    def backward(ctx, dout, dlast):
        gates, values, state, resets, saved = ctx.saved_tensors
        if dout is None and dlast is None:
            return (None,) * 5
        T, E, N = gates.shape
        kind = _TYPES[gates.dtype]
        dout = gates.new_zeros((T, E, N)) if dout is None else _dense_last(dout)
        dlast = None if dlast is None else _aligned(dlast)
        dgates, dvalues = _dense_like(gates), _dense_like(values)
        dstate = torch.empty_like(state) if ctx.needs_input_grad[2] else None
        scratch = _buffer(_recurrence_workspace(T, E, N, kind)[0], gates.device)
        _launch(library().duck_gated_recurrence_backward, gates.device,
                _RECURRENCE.pack(gates.data_ptr(), values.data_ptr(), 0, _address(resets), _address(state), 0,
                                 dout.data_ptr(), _address(dlast), dgates.data_ptr(), dvalues.data_ptr(),
                                 _address(dstate), _address(saved), _address(scratch),
                                 *gates.stride()[:2], *values.stride()[:2], *dout.stride()[:2], T, E, N, kind))
        return dgates, dvalues, dstate, None, None


def _recurrence_plain(gates, values, state, resets):
    """The recurrence step by step, in float32 or wider."""
    dtype = gates.dtype
    wide = torch.promote_types(dtype, torch.float32)
    T, E, N = gates.shape
    gates, values = gates.to(wide), values.to(wide)
    h = gates.new_zeros(E, N) if state is None else state if T else state.clone()
    out = []
    for t in range(T):
        if resets is not None:
            h = torch.where(resets[t, :, None] != 0, torch.zeros_like(h), h)
        h = torch.sigmoid(gates[t]) * h + torch.sigmoid(-gates[t]) * values[t]
        out.append(h)
    out = torch.stack(out) if T else gates.new_zeros(0, E, N)
    return out.to(dtype), h


def _check_channels(gates, values, state, dims, what):
    _require(gates.dim() == dims and gates.shape == values.shape and gates.dtype == values.dtype
             and gates.device == values.device and gates.dtype in _WIDE,
             f"{what}: gates and values have one shape, floating type and device")
    _check_type(gates, what)
    _require(state is None or (state.shape == gates.shape[-2:] and state.dtype == _WIDE[gates.dtype]
                               and state.device == gates.device),
             f"{what}: the state is float32 [environments, channels] on the gates' device")


def gated_recurrence(gates, values, state=None, resets=None, final_state=True):
    """A gated linear recurrence over a rollout, channel by channel: ``(out, state)``
    with

        out_t = f_t out_{t-1} + (1 - f_t) values_t,   f_t = sigmoid(gates_t),

    out_{t-1} being zero where ``resets[t, e]`` says that an episode begins.

    ``gates`` and ``values`` [T, E, N] (T steps, E environments, N channels),
    ``state`` [E, N] float32 before the first step (None: zero).  The state after
    the last step is returned where ``final_state`` is set, else None.  Gradients
    flow to gates, values and the state.  States are float32; out has the gates'
    type, rounded once, and so have the gradients."""
    _check_channels(gates, values, state, 3, "gated_recurrence")
    if resets is not None:
        resets = _mask(resets, gates.shape[:2], gates.device)
    if not gates.is_cuda:
        out, last = _recurrence_plain(gates, values, state, resets)
        return out, last if final_state else None
    gates, values = _dense_last(gates), _dense_last(values)
    if state is not None:
        state = _aligned(state)
    if _grad_needed(gates, values, state):
        return _GatedRecurrence.apply(gates, values, state, resets, final_state)
    return _recurrence_forward(gates, values, state, resets, final_state, False)[:2]


def gated_recurrence_step(gates, values, state, reset=None):
    """One control step of ``gated_recurrence`` for every environment, without
    gradients: ``gates`` and ``values`` [E, N], ``reset`` [E].  ``state`` [E, N]
    float32 is updated in place; returns out [E, N].  A backward pass that still
    needs the state as it was raises, as after any operation in place (a replay of
    a CUDA graph is not seen)."""
    _require(state is not None, "gated_recurrence_step: there is no state")
    _check_channels(gates, values, state, 2, "gated_recurrence_step")
    _require(not (state.requires_grad and torch.is_grad_enabled()),
             "the state is updated in place without gradients, it must not require one")
    if reset is not None:
        reset = _mask(reset, gates.shape[:1], gates.device)
    if not gates.is_cuda:
        with torch.no_grad():
            out, last = _recurrence_plain(gates[None], values[None], state, None if reset is None else reset[None])
            state.copy_(last)
        return out[0]
    _refuse_tangents(gates, values, state)
    _require(state.is_contiguous(), "the state is updated in place and has to be contiguous")
    gates, values = _dense_last(gates), _dense_last(values)
    E, N = gates.shape
    out = _dense_like(gates)
    _launch(library().duck_gated_recurrence_step, gates.device,
            _RECURRENCE.pack(gates.data_ptr(), values.data_ptr(), out.data_ptr(), _address(reset), 0, state.data_ptr(),
                             0, 0, 0, 0, 0, 0, 0, 0, gates.stride(0), 0, values.stride(0), 0, 0, 1, E, N,
                             _TYPES[gates.dtype]))
    torch.autograd.graph.increment_version(state)   # autograd does not see a kernel's writes
    return out


# ---------------------------------------------------------------- gated linear
# struct duck_gated of include/duck_b200.h.
_GATED = struct.Struct("@14P3q4i")
ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}


@functools.lru_cache(maxsize=1024)
def _gated_workspace(rows, D, F, kind, input, weights, biases):
    """Bytes of scratch of a backward call with or without those gradients, and of
    what a forward call keeps for it."""
    out = (ctypes.c_int64 * 2)()
    pointers = [0] * 14
    pointers[7] = int(input)
    pointers[8] = pointers[9] = int(weights)
    pointers[10] = pointers[11] = int(biases)
    _raise(library().duck_gated_linear_sizes(_GATED.pack(*pointers, rows, 0, 0, D, F, 0, kind), out))
    return tuple(out)


def _gated_operand(t, strided):
    """Rows as the kernels take them: dense (`strided`: up to the distance of the
    rows); bfloat16 ones of whole 16-byte pieces on their boundaries, and apart (others
    are padded by the forward call)."""
    t = _rows_of(t) if strided else t.contiguous()
    if t.dtype is torch.bfloat16:
        n, stride = t.shape[1], t.stride(0)
        if n % 8 == 0 and (t.data_ptr() % 16 or stride % 8 or stride < n):
            t = t.clone(memory_format=torch.contiguous_format)
    return t


def _gated_forward(x, w_gate, w_up, b_gate, b_up, activation, keep):
    rows, D = x.shape
    F_ = w_gate.shape[0]
    kind = _TYPES[x.dtype]
    h = torch.empty((rows, F_), dtype=x.dtype, device=x.device)
    # float32: the projections, for a backward pass; bfloat16: padded operands, for a forward one too.
    needed = keep if kind == 0 else D % 8
    kept = _buffer(_gated_workspace(rows, D, F_, kind, False, False, False)[1], x.device) if needed else None
    _launch(library().duck_gated_linear_forward, x.device,
            _GATED.pack(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _address(b_gate), _address(b_up), h.data_ptr(),
                        0, 0, 0, 0, 0, 0, _address(kept), 0, rows, x.stride(0), 0, D, F_, activation, kind))
    return h, kept


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, b_gate, b_up, activation):
        ctx.shape = x.shape
        x, w_gate, w_up = _gated_operand(x, True), _gated_operand(w_gate, False), _gated_operand(w_up, False)
        h, kept = _gated_forward(x, w_gate, w_up, b_gate, b_up, activation, True)
        ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up, kept)
        ctx.activation = activation
        return h if len(ctx.shape) == 2 else h.view(ctx.shape[:-1] + (h.shape[1],))

    @staticmethod
    @_once
    def backward(ctx, dh):
        x, w_gate, w_up, b_gate, b_up, kept = ctx.saved_tensors
        needs = ctx.needs_input_grad
        weights, biases = needs[1] or needs[2], needs[3] or needs[4]
        rows, D = x.shape
        F_ = w_gate.shape[0]
        kind = _TYPES[x.dtype]
        dh = _rows_of(dh)
        empty = functools.partial(torch.empty, dtype=x.dtype, device=x.device)
        dx = empty((rows, D)) if needs[0] else None
        dw = (empty((F_, D)), empty((F_, D))) if weights else (None, None)
        db = (empty(F_), empty(F_)) if biases else (None, None)
        scratch = _buffer(_gated_workspace(rows, D, F_, kind, needs[0], weights, biases)[0], x.device)
        _launch(library().duck_gated_linear_backward, x.device,
                _GATED.pack(x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _address(b_gate), _address(b_up), 0,
                            dh.data_ptr(), _address(dx), _address(dw[0]), _address(dw[1]), _address(db[0]), _address(db[1]),
                            _address(kept), _address(scratch), rows, x.stride(0), dh.stride(0), D, F_, ctx.activation, kind))
        return dx if dx is None or len(ctx.shape) == 2 else dx.view(ctx.shape), *dw, *db, None


class _PlainLinear(torch.autograd.Function):
    """x w^T + b on the CPU, outside autocast regions in the backward pass too."""

    generate_vmap_rule = True

    @staticmethod
    def forward(x, w, b):
        return F.linear(x, w, b)

    @staticmethod
    def setup_context(ctx, inputs, output):
        x, w, _ = inputs
        ctx.save_for_backward(x, w)
        ctx.save_for_forward(x, w)

    @staticmethod
    @torch.autocast("cpu", enabled=False)
    def backward(ctx, dy):
        x, w = ctx.saved_tensors
        need_x, need_w, need_b = ctx.needs_input_grad
        return (_PlainLinear.apply(dy, w.t(), None) if need_x else None,
                _PlainLinear.apply(dy.t(), x.t(), None) if need_w else None, dy.sum(0) if need_b else None)

    @staticmethod
    @torch.autocast("cpu", enabled=False)
    def jvp(ctx, dx, dw, db):
        x, w = ctx.saved_tensors
        terms = [] if dx is None else [_PlainLinear.apply(dx, w, None)]
        terms += [] if dw is None else [_PlainLinear.apply(x, dw, None)]
        terms += [] if db is None else [db.expand(x.shape[0], -1)]
        return sum(terms[1:], terms[0])


@torch.autocast("cpu", enabled=False)
def _gated_plain(x, w_gate, w_up, b_gate, b_up, activation):
    """In float32 or wider, rounded once."""
    wide = torch.promote_types(x.dtype, torch.float32)
    to = lambda t: None if t is None else t.to(wide)
    rows = to(x).reshape(-1, x.shape[-1])
    a, u = _PlainLinear.apply(rows, to(w_gate), to(b_gate)), _PlainLinear.apply(rows, to(w_up), to(b_up))
    act = {"silu": F.silu, "gelu": F.gelu, "sigmoid": torch.sigmoid}[activation]
    return (act(a) * u).to(x.dtype).view(x.shape[:-1] + w_gate.shape[:1])


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """Two projections of the same rows, multiplied, one of them through an
    activation:

        act(x w_gate^T + b_gate) * (x w_up^T + b_up),   act: "silu", "gelu" (of erf) or "sigmoid"

    ``x`` [..., D], weights [F, D] (each up to 2^20; D up to 2^16 for bfloat16 on the
    GPU), biases [F] or none, all of one type; returns [..., F].  Gradients flow to
    all of them.  Sums are float32, and so are the two projections; the result is
    rounded once.  bfloat16 on the GPU: the backward pass needs only x and the weights
    (where D is no multiple of 8, their padded copies are kept beside them); gradients
    of the projections are rounded to 8 bits on their way to those of x and the
    weights.  A kernel whose waits run out, which takes a fault, leaves NaN, and the
    next call that finds it so raises."""
    _require(activation in ACTIVATIONS, f"gated_linear: the activation is one of {', '.join(ACTIVATIONS)}")
    _require(x.dim() > 0 and w_gate.dim() == 2 and w_gate.shape == w_up.shape and w_gate.shape[1] == x.shape[-1]
             and w_gate.numel() > 0, "gated_linear: weights are [F, D] for x [..., D]")
    _require((b_gate is None) == (b_up is None) and all(b is None or b.shape == w_gate.shape[:1] for b in (b_gate, b_up)),
             "gated_linear: biases are [F], both or neither")
    dtype, device = x.dtype, x.device
    _require(dtype in _WIDE and w_gate.dtype is dtype and w_up.dtype is dtype and w_gate.device == device == w_up.device
             and (b_gate is None or (b_gate.dtype is dtype and b_up.dtype is dtype and b_gate.device == device == b_up.device)),
             "gated_linear: one floating type and device for x, weights and biases")
    if not x.is_cuda:
        return _gated_plain(x, w_gate, w_up, b_gate, b_up, activation)
    _check_type(x, "gated_linear")
    if b_gate is not None:
        b_gate, b_up = b_gate.contiguous(), b_up.contiguous()
    if _grad_needed(x, w_gate, w_up, b_gate, b_up):
        return _GatedLinear.apply(x, w_gate, w_up, b_gate, b_up, ACTIVATIONS[activation])
    shape = x.shape
    x, w_gate, w_up = _gated_operand(x, True), _gated_operand(w_gate, False), _gated_operand(w_up, False)
    h, _ = _gated_forward(x, w_gate, w_up, b_gate, b_up, ACTIVATIONS[activation], False)
    return h if len(shape) == 2 else h.view(shape[:-1] + (h.shape[1],))


# ----------------------------------------------------------- 8-bit checkpoints
class Checkpoint8(NamedTuple):
    """An activation kept in 8 bits: ``codes`` int8 of its shape and ``scales``
    float32, one per group of 128 values of the last axis; it stands for
    codes * scales."""

    codes: torch.Tensor
    scales: torch.Tensor


def _keep_plain(y):
    n = y.shape[-1]
    groups = -(-n // GROUP)
    wide = F.pad(y.float(), (0, groups * GROUP - n)).unflatten(-1, (groups, GROUP))
    scales = wide.abs().amax(-1) * (1.0 / 127.0)
    scales = torch.where(scales < torch.finfo(torch.float32).tiny, torch.zeros_like(scales), scales)
    inverse = torch.where(scales == 0, torch.zeros_like(scales), torch.reciprocal(scales))
    codes = torch.nan_to_num(torch.round(wide * inverse[..., None])).to(torch.int8)
    return Checkpoint8(codes.flatten(-2)[..., :n].contiguous(), scales)


def _kept_plain(kept):
    n = kept.codes.shape[-1]
    return kept.codes.float() * kept.scales.repeat_interleave(GROUP, -1)[..., :n]


def elu_checkpoint(x):
    """``(elu(x), kept)``: the activation, and its 8-bit form for the backward
    pass (``elu_restore``).  Not differentiable by itself; ``checkpointed_mlp``
    is the differentiable use."""
    _require(x.dim() > 0 and x.shape[-1] > 0, "elu_checkpoint: the last axis is empty")
    _refuse_tangents(x)
    x = x.detach()
    if not x.is_cuda:
        y = F.elu(x)
        return y, _keep_plain(y)
    _check_type(x, "elu_checkpoint")
    x = x.contiguous()
    n = x.shape[-1]
    y = torch.empty_like(x)
    codes = torch.empty_like(x, dtype=torch.int8)
    scales = torch.empty(x.shape[:-1] + (-(-n // GROUP),), dtype=torch.float32, device=x.device)
    _launch(library().duck_elu_checkpoint, x.device, x.data_ptr(), y.data_ptr(), codes.data_ptr(), scales.data_ptr(),
            x.numel() // n, n, _TYPES[x.dtype])
    return y, Checkpoint8(codes, scales)


def elu_restore(dy, kept, restore=True, bounded=False):
    """``(dx, y)`` from the gradient of elu's output and its checkpoint:
    dx = dy (y > 0 ? 1 : 1 + y) and the kept output y in dy's type (None where
    ``restore`` is not set).  A saturated unit's kept output may lie below -1, by
    half a step of its group at most; with ``bounded`` it counts as -1 in dx, so that
    the derivative is in [0, 1] as that of elu is."""
    codes, scales = kept
    shape = codes.shape
    _require(dy.shape == shape and len(shape) and scales.shape == shape[:-1] + (-(-shape[-1] // GROUP),) and codes.dtype == torch.int8
             and scales.dtype == torch.float32 and dy.device == codes.device == scales.device,
             "elu_restore: the gradient and the checkpoint do not belong together")
    _refuse_tangents(dy, scales)
    dy = dy.detach()
    if not dy.is_cuda:
        y = _kept_plain(kept)
        below = torch.where(y < -1.0, -torch.ones_like(y), y) if bounded else y
        dx = (dy.float() * torch.where(y > 0, torch.ones_like(y), below + 1.0)).to(dy.dtype)
        return dx, y.to(dy.dtype) if restore else None
    _check_type(dy, "elu_restore")
    dy, codes, scales = dy.contiguous(), codes.contiguous(), scales.contiguous()
    n = dy.shape[-1]
    dx = torch.empty_like(dy)
    y = torch.empty_like(dy) if restore else None
    entry = library().duck_elu_restore_bounded if bounded else library().duck_elu_restore
    _launch(entry, dy.device, dy.data_ptr(), codes.data_ptr(), scales.data_ptr(), _pointer(y),
            dx.data_ptr(), dy.numel() // n, n, _TYPES[dy.dtype])
    return dx, y


class _CheckpointedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, layers, *parameters):
        weights, biases = parameters[:layers], parameters[layers:]
        keep = [x]
        for i, (w, b) in enumerate(zip(weights, biases)):
            x = torch.addmm(b, x, w.t())
            if i < layers - 1:
                x, kept = elu_checkpoint(x)
                keep += kept
        ctx.layers = layers
        ctx.save_for_backward(*keep, *weights)
        return x

    @staticmethod
    @_once
    def backward(ctx, dz):
        with torch.autocast(dz.device.type, enabled=False):   # as in the forward pass
            return _CheckpointedMLP._gradients(ctx, dz)

    @staticmethod
    def _gradients(ctx, dz):
        saved, n = ctx.saved_tensors, ctx.layers
        weights = saved[2 * n - 1:]
        dw, db, dx = [None] * n, [None] * n, None
        for i in reversed(range(n)):
            db[i] = dz.sum(0)
            if i == 0:
                y = saved[0]
                dx = dz @ weights[0] if ctx.needs_input_grad[0] else None
            else:
                dnext, y = elu_restore(dz @ weights[i], Checkpoint8(*saved[2 * i - 1:2 * i + 1]), bounded=True)
            dw[i] = dz.t() @ y
            if i:
                dz = dnext
        return (dx, None, *dw, *db)


def checkpointed_mlp(x, weights, biases):
    """Linear layers with ELU between them (as ``ppo.mlp``) on rows x [rows, n];
    each hidden activation is kept for the backward pass in 8 bits only: the
    derivative of ELU and the next layer's weight gradient come from there."""
    _require(x.dim() == 2 and len(weights) == len(biases) > 0, "checkpointed_mlp: rows, weights and biases")
    _require(all(t.dtype == x.dtype for t in (*weights, *biases)), "checkpointed_mlp: one type for x and parameters")
    with torch.autocast(x.device.type, enabled=False):   # products in x's type, in the backward pass too
        return _CheckpointedMLP.apply(x, len(weights), *weights, *biases)
