"""AdamW over all tensors of a model in one launch, with moments in 32 bits or in
8, and gradients clipped by their common norm on the way.

    adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, ...)
    state8_zeros(like, signed)                                   -> State8
    state8_values(states)                                        -> tensors
    AdamW(params, lr, ..., bits=8, max_grad_norm=1.0)            torch.optim.Optimizer

The reference trains with torch's Adam (scripts/train_bam_native.py:14-140), whose
formula this is; see ``ppo.PPOConfig.optimizer``.

CUDA tensors run the library's kernels on the current stream (float32 or bfloat16
parameters, no other type; there is no fallback), CPU tensors a plain torch
restatement of the same arithmetic.  Wrong devices, types or shapes raise
``RuntimeError``.  The calls allocate only with torch, never synchronise and can be
captured in CUDA graphs: the count of steps is a tensor on the device, and so can
the learning rate be.
"""

from __future__ import annotations

import bisect
import ctypes
import itertools
import math
import operator
import struct
from typing import NamedTuple

import torch

from .cuda_batch import library
from .memory import _launch

GROUP = 128          # values that share one exponent of a moment in 8 bits
SUMS = 592           # DUCK_GRADIENT_SUMS
_TYPES = {torch.float32: 0, torch.bfloat16: 1}
_TENSOR = struct.Struct("@6Pq2i")       # struct duck_adamw_tensor of include/duck_b200.h
_OPTIONS = struct.Struct("@3P6d2i")     # struct duck_adamw


class State8(NamedTuple):
    """A moment in 8 bits: ``codes`` of its tensor's shape, int8 for a first moment
    and uint8 for a second one, and ``exponents`` uint8, one per group of 128 values.
    A value's float32 has the leading 12 bits |code| + max(0, 8 exponent + 8 - most),
    most = 127 and 255; code 0 is zero, and exponent 255 makes a group's values NaN."""

    codes: torch.Tensor
    exponents: torch.Tensor


def _require(condition, message):
    if not condition:
        raise RuntimeError(message)


def _groups(t):
    return -(-t.numel() // GROUP)


def state8_zeros(like, signed):
    """The first (``signed``) or second moment of a tensor before any step."""
    return State8(torch.zeros(like.shape, dtype=torch.int8 if signed else torch.uint8, device=like.device),
                  torch.zeros(_groups(like), dtype=torch.uint8, device=like.device))


# The checks run before every step: maps over methods cost a third of loops.
def _pointers(ts):
    return list(map(torch.Tensor.data_ptr, ts))


def _numbers(ts):
    return list(map(torch.Tensor.numel, ts))


def _devices(ts):
    return set(map(torch.Tensor.get_device, ts))


_dtype, _layout = operator.attrgetter("dtype"), operator.attrgetter("layout")


def _dtypes(ts):
    return set(map(_dtype, ts))


def _dense(ts):
    return all(map(torch.Tensor.is_contiguous, ts))


def _alike(ts, others):
    return all(map(torch.Tensor.is_same_size, ts, others))


def _group_counts(numbers):
    return [(n + GROUP - 1) // GROUP for n in numbers]


def _check_states8(states, dtypes, what):
    """Codes and exponents of moments in 8 bits, and how many values they have."""
    codes, exponents = [s[0] for s in states], [s[1] for s in states]
    numbers = _numbers(codes)
    _require(_dtypes(codes) <= dtypes and _dtypes(exponents) == {torch.uint8} and _numbers(exponents) == _group_counts(numbers)
             and _dense(codes) and _dense(exponents),
             f"{what}: a moment in 8 bits is dense codes of its tensor's shape and one exponent for 128 of them")
    return codes, exponents, numbers


# ------------------------------------------------------------ plain restatement
def _mix(x):
    """The 32-bit finaliser of MurmurHash3, on int64."""
    x = (x ^ (x >> 16)) * 0x85EBCA6B & 0xFFFFFFFF
    x = (x ^ (x >> 13)) * 0xC2B2AE35 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _spread(per_group, n):
    return per_group.repeat_interleave(GROUP)[:n]


def _decode(codes, exponents):
    most, n = 127 if codes.dtype == torch.int8 else 255, codes.numel()
    c, e = codes.reshape(-1).int(), exponents.int()
    bits = torch.where(c == 0, 0, c.abs() + _spread((8 * e + (8 - most)).clamp_min(0), n)) << 20
    value = torch.where(_spread(e, n) == 255, math.nan, bits.view(torch.float32))
    return torch.where(c < 0, -value, value).view(codes.shape)


def _encode(x, state, noise):
    """Writes x to `state`, its low 20 bits rounded by `noise` in [0, 2^20)."""
    codes, exponents = state
    most, n = 127 if codes.dtype == torch.int8 else 255, x.numel()
    if n == 0:
        return
    bits = x.reshape(-1).view(torch.int32) & 0x7FFFFFFF
    padded = torch.nn.functional.pad(bits, (0, exponents.numel() * GROUP - n)).view(-1, GROUP)
    e = padded.amax(1) >> 23
    place = ((bits.clamp_max(0x7F800000) + noise.int()) >> 20).clamp_max(2039)
    place = place - _spread((8 * e + (8 - most)).clamp_min(0), n)
    place = place.clamp(0, 127) if most == 127 else torch.where(bits == 0, 0, place.clamp(1, 255))
    if most == 127:
        place = torch.where(x.reshape(-1).signbit(), -place, place)
    codes.copy_(place.view(codes.shape))
    exponents.copy_(e)


def _plain_tensor(place, p, g, m, v, count, clip, beta1, beta2, ahead, widen, shrink, eps):
    eight = not torch.is_tensor(m)
    m32, v32 = (_decode(*m), _decode(*v)) if eight else (m, v)
    g = g.float() if clip is None else g.float() * clip
    m32 = m32 * beta1 + g * (1.0 - beta1)
    v32 = v32 * beta2 + g * g * (1.0 - beta2)
    new = p.float() * shrink - ahead * (m32 / (v32.sqrt() * widen + eps))
    if eight or p.dtype == torch.bfloat16:
        key = _mix(torch.tensor((count + 0x9E3779B9 * (place + 1)) & 0xFFFFFFFF))
        noise = _mix(key ^ (torch.arange(p.numel()) & 0xFFFFFFFF))
    if p.dtype == torch.bfloat16:
        bits = new.reshape(-1).view(torch.int32)
        up = torch.where(new.reshape(-1).isfinite(), bits + (noise & 0xFFFF).int(), bits)
        new = torch.where(new.isfinite(), (up & -65536).view(torch.float32).view(p.shape), new)
    p.copy_(new)
    if eight:
        _encode(m32, m, (noise >> 20 << 8) + 128)
        _encode(v32, v, noise & 0xFFFFF)
    else:
        m.copy_(m32)
        v.copy_(v32)


def _plain(params, grads, ms, vs, places, step, lr, betas, eps, weight_decay, max_norm, total):
    step += 1
    count, rate = int(step), float(lr)
    clip = None
    if max_norm is not None:
        clip = (max_norm / (total.sqrt() + 1e-6)).clamp_max(1.0).float()
    scalars = (torch.tensor(x, dtype=torch.float64).float() for x in (
        rate / (1.0 - betas[0] ** count), (1.0 - betas[1] ** count) ** -0.5, 1.0 - rate * weight_decay))
    ahead, widen, shrink = scalars
    for place, *each in zip(places, params, grads, ms, vs):
        _plain_tensor(place, *each, count, clip, *betas, ahead, widen, shrink, eps)


# ----------------------------------------------------------------- entry points
def _check_apart(written, read, what):
    """Arrays, as (first bytes, bytes): none that is written overlaps another one."""
    starts, ends = [], []
    for first, size in written:
        starts += first
        ends += map(operator.add, first, size)
    starts.sort()
    ends.sort()   # disjoint spans end in the order that they begin in
    _require(all(map(operator.le, ends, starts[1:])), f"{what}: a tensor is there twice, or two of them overlap")
    first, size = read
    before = map(bisect.bisect_left, itertools.repeat(starts), map(operator.add, first, size))   # spans that begin before its end
    _require(all(not k or ends[k - 1] <= a for k, a in zip(before, first)), f"{what}: a gradient overlaps what is written")


def _checked(params, grads, exp_avgs, exp_avg_sqs, places):
    """Whether the moments of these lists have 8 bits, the tensors' device, their table,
    and dense gradients (which have to live until the launch)."""
    _require(len(params) == len(grads) == len(exp_avgs) == len(exp_avg_sqs) > 0,
             "adamw_step: one gradient and two moments for each of one or more parameters")
    eight = not torch.is_tensor(exp_avgs[0])
    kinds = {*map(type, exp_avgs), *map(type, exp_avg_sqs)}
    _require(all(issubclass(kind, torch.Tensor) != eight for kind in kinds), "adamw_step: all moments have 32 bits, or all have 8")
    dtypes = list(map(_dtype, params))
    kinds = list(map(_TYPES.get, dtypes))
    _require(None not in kinds and _dense(params), "adamw_step: parameters are dense float32 or bfloat16 tensors of one device")
    _require(set(map(_layout, grads)) == {torch.strided} and _alike(grads, params) and list(map(_dtype, grads)) == dtypes,
             "adamw_step: a gradient has its parameter's shape, type and device")
    if not _dense(grads):
        grads = [g.contiguous() for g in grads]
    numbers = _numbers(params)
    if eight:
        (ms, me, _), (vs, ve, _) = (_check_states8(exp_avgs, {torch.int8}, "adamw_step"),
                                    _check_states8(exp_avg_sqs, {torch.uint8}, "adamw_step"))
        _require(_alike(ms, params) and _alike(vs, params), "adamw_step: a moment has its parameter's shape")
        arrays = [*params, *grads, *ms, *vs, *me, *ve]
        me, ve, size = _pointers(me), _pointers(ve), numbers
    else:
        ms, vs, me, ve = exp_avgs, exp_avg_sqs, (0,) * len(params), (0,) * len(params)
        _require(_dtypes(ms) == _dtypes(vs) == {torch.float32} and _alike(ms, params) and _alike(vs, params) and _dense(ms)
                 and _dense(vs), "adamw_step: moments are dense float32 tensors of their parameters' shapes")
        arrays = [*params, *grads, *ms, *vs]
        size = [4 * n for n in numbers]
    _require(len(_devices(arrays)) == 1, "adamw_step: one device for parameters, gradients and moments")
    at, gat, mat, vat = _pointers(params), _pointers(grads), _pointers(ms), _pointers(vs)
    bytes_ = [n << (2 - kind) for n, kind in zip(numbers, kinds)]
    written = [(at, bytes_), (mat, size), (vat, size)]
    if eight:
        groups = _group_counts(numbers)
        written += [(me, groups), (ve, groups)]
    _check_apart(written, (gat, bytes_), "adamw_step")
    table = b"".join(map(_TENSOR.pack, at, gat, mat, vat, me, ve, numbers, kinds, places))
    return eight, params[0].device, table, grads


class _Norm:
    """The squares of gradients, summed over several lists of them."""

    def __init__(self, device):
        self.count = 0
        self.sums = (torch.empty(SUMS, dtype=torch.float64, device=device) if device.type == "cuda"
                     else torch.zeros((), dtype=torch.float64))

    def add(self, table, grads):
        if self.sums.dim() == 0:
            for g in grads:
                self.sums += g.double().square().sum()
            return
        count = ctypes.c_int()
        _launch(library().duck_gradient_squares, self.sums.device, table, len(grads), self.count, self.sums.data_ptr(),
                ctypes.byref(count))
        self.count = count.value
        if self.count == 0:   # only empty gradients: a norm of zero
            self.sums[:1].zero_()
            self.count = 1


def _step(params, grads, ms, vs, places, eight, device, table, step, lr, betas, eps, weight_decay, max_norm, norm):
    if device.type != "cuda":
        with torch.no_grad():
            return _plain(params, grads, ms, vs, places, step, lr, betas, eps, weight_decay, max_norm,
                          None if norm is None else norm.sums)
    on_device = torch.is_tensor(lr) and lr.is_cuda
    if on_device and lr.dtype != torch.float32:
        lr = lr.float()
    options = _OPTIONS.pack(step.data_ptr(), lr.data_ptr() if on_device else 0, norm.sums.data_ptr() if norm else 0,
                            0.0 if on_device else float(lr), *betas, eps, weight_decay, 0.0 if norm is None else max_norm,
                            norm.count if norm else 0, 8 if eight else 32)
    _launch(library().duck_adamw_step, device, table, len(grads), options)
    written = [*params, step]
    written += itertools.chain(*ms, *vs) if eight else (*ms, *vs)
    torch.autograd.graph.increment_version(written)   # autograd does not see a kernel's writes


def _check_options(step, lr, betas, eps, weight_decay, max_norm, device):
    _require(torch.is_tensor(step) and step.dtype == torch.int64 and step.numel() == 1 and step.device == device,
             "adamw_step: the count of steps is an int64 tensor of one value on the parameters' device")
    if torch.is_tensor(lr):
        _require(lr.numel() == 1 and lr.is_floating_point() and lr.device in (device, torch.device("cpu")),
                 "adamw_step: the learning rate is a number, or a floating tensor of one value")
    else:
        _require(math.isfinite(lr), "adamw_step: the learning rate is not finite")
    _require(len(betas) == 2 and all(0.0 <= b < 1.0 for b in betas) and (eps == 0.0 or 2.0 ** -126 <= eps < 2.0 ** 127)
             and 0.0 <= weight_decay < math.inf,
             "adamw_step: betas in [0, 1), eps 0 or a normal float32 number, weight decay of 0 or more")
    _require(max_norm is None or max_norm >= 0.0, "adamw_step: a norm of 0 or more")


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0,
               max_norm=None):
    """One AdamW step over lists of tensors, in place:

        m = beta1 m + (1 - beta1) g,   v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

    ``exp_avgs`` (m) and ``exp_avg_sqs`` (v) are float32 tensors, or all of them
    ``State8``; ``step`` is an int64 tensor, the steps done before (t - 1), and is
    counted up (not to be read on another stream meanwhile).  ``lr`` is a number or a
    tensor.  With ``max_norm`` g is the gradient times min(1, max_norm / (norm + 1e-6)),
    norm that of all gradients together; the gradients themselves stay as they are.

    bfloat16 parameters and codes are rounded up or down at random, by a hash of t, the
    tensor's place in the list and the value's place in the tensor: what a step adds is
    mostly less than half a place of theirs, and would be lost."""
    params, exp_avgs, exp_avg_sqs = list(params), list(exp_avgs), list(exp_avg_sqs)   # they may be iterators
    eight, device, table, grads = _checked(params, list(grads), exp_avgs, exp_avg_sqs, range(len(params)))
    _check_options(step, lr, betas, eps, weight_decay, max_norm, device)
    norm = None
    if max_norm is not None:
        norm = _Norm(device)
        norm.add(table, grads)
    _step(params, grads, exp_avgs, exp_avg_sqs, range(len(params)), eight, device, table, step, lr, betas, eps, weight_decay,
          max_norm, norm)


def state8_values(states):
    """The float32 tensors that moments in 8 bits stand for (on the GPU, parts of one
    buffer)."""
    states = list(states)
    if not states:
        return []
    codes, exponents, numbers = _check_states8(states, {torch.int8, torch.uint8}, "state8_values")
    _require(len(_devices([*codes, *exponents])) == 1, "state8_values: states of one device")
    device = codes[0].device
    if device.type != "cuda":
        return [_decode(*s) for s in states]
    # One allocation, each tensor on a 16-byte boundary.
    sizes = [part for n in numbers for part in (n, -n % 4)]
    values = torch.empty(sum(sizes), dtype=torch.float32, device=device).split(sizes)[::2]
    signed = [c.dtype is torch.int8 for c in codes]
    at, es = _pointers(codes), _pointers(exponents)
    either = lambda ps, which: [p if s == which else 0 for p, s in zip(ps, signed)]
    table = b"".join(map(_TENSOR.pack, _pointers(values), itertools.repeat(0), either(at, True), either(at, False),
                         either(es, True), either(es, False), numbers, itertools.repeat(0), itertools.repeat(0)))
    _launch(library().duck_moment_values, device, table, len(codes))
    return [v if c.dim() == 1 else v.view(c.shape) for v, c in zip(values, codes)]


def _check_loaded(group):
    """A group of a state dict: one of AdamW below, or of torch's without what would be lost."""
    if "bits" in group:
        return
    _require(group.keys() >= {"lr", "betas", "eps", "weight_decay", "amsgrad"},
             "AdamW: the state dict is not one of this class, nor of torch's Adam or AdamW")
    _require(not group["amsgrad"] and not group.get("maximize"), "AdamW: there is no amsgrad and no maximize")
    _require(group["weight_decay"] == 0 or group.get("decoupled_weight_decay"),
             "AdamW: the state dict's weight decay is, or may be, added to the gradient; decoupled_weight_decay=True in its "
             "groups says that it is not")


def _refuse_capture(device):
    """Where state is made: a replay would make it anew each time."""
    _require(device.type != "cuda" or not torch.cuda.is_current_stream_capturing(),
             "AdamW: a step that makes moments, or a count of steps, is not captured: step once, or prepare(), before the capture")


class AdamW(torch.optim.Optimizer):
    """``adamw_step`` as a torch optimizer.

    ``bits`` (32 or 8) of the moments; with ``max_grad_norm`` gradients are clipped by
    the norm of those of all groups, in the step itself (``.grad`` stays as it is).
    ``lr`` may be a tensor on the device that a schedule writes to.  A parameter without a
    gradient is left as it is, and so is its count of steps, as torch's.  The group's
    ``step`` counts for all parameters that have had a gradient in each of its steps; one
    that came later, or was left out of one, has a ``step`` in its own state, and a launch
    for those that share it.  A step that is captured in a CUDA graph follows one that was
    not, which made the moments, or ``prepare()``."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, bits=32, max_grad_norm=None):
        if bits not in (8, 32):
            raise ValueError("moments have 8 or 32 bits")
        if max_grad_norm is not None and not max_grad_norm >= 0.0:
            raise ValueError("invalid max_grad_norm")
        self.max_grad_norm = max_grad_norm
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, bits=bits))

    def _counts(self, group):
        """The group's parameters with gradients: lists of those that have the same steps
        behind them, each with that count, the parameters' states and their places."""
        params = [p for p in group["params"] if p.grad is not None]
        if not params:
            return []
        states = [self.state[p] for p in params]
        have = lambda name: map(dict.__contains__, states, itertools.repeat(name))
        if not all(have("exp_avg")):
            _refuse_capture(params[0].device)
            count = torch.zeros((), dtype=torch.int64, device=params[0].device)
            apart = any("exp_avg" in state and "step" not in state for state in map(self._known, group["params"]))
            for p, state in zip(params, states):
                if "exp_avg" not in state:
                    state.update(self._zeros(p, group["bits"]), **(dict(step=count) if apart else {}))
            if not apart:
                group["step"] = count
        behind = {}
        if len(params) < len(group["params"]):
            going = {state.get("step", group["step"]).data_ptr() for state in states}
            for p in group["params"]:
                state = self._known(p)
                if p.grad is None and "exp_avg" in state:
                    count = state.get("step", group["step"])
                    if count.data_ptr() in going:
                        _refuse_capture(count.device)
                        state["step"] = behind.setdefault(count.data_ptr(), count.clone())
        if not any(have("step")):
            return [(group["step"], params, states, range(len(params)))]
        lists = {}
        for place, (p, state) in enumerate(zip(params, states)):
            count = state.get("step", group["step"])
            for to, x in zip(lists.setdefault(count.data_ptr(), (count, [], [], []))[1:], (p, state, place)):
                to.append(x)
        return list(lists.values())

    def _known(self, p):
        return self.state[p] if p in self.state else {}

    @staticmethod
    def _zeros(p, bits):
        """A parameter's moments before any step."""
        if bits == 8:
            m, v = state8_zeros(p, True), state8_zeros(p, False)
            return dict(exp_avg=m.codes, exp_avg_exponents=m.exponents, exp_avg_sq=v.codes, exp_avg_sq_exponents=v.exponents)
        zeros = lambda: torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return dict(exp_avg=zeros(), exp_avg_sq=zeros())

    @staticmethod
    def _moments(states, bits):
        if bits == 8:
            return ([State8(state["exp_avg"], state["exp_avg_exponents"]) for state in states],
                    [State8(state["exp_avg_sq"], state["exp_avg_sq_exponents"]) for state in states])
        return [state["exp_avg"] for state in states], [state["exp_avg_sq"] for state in states]

    def prepare(self):
        """Makes the moments and counts that the next step with the present gradients
        needs, so that it can be captured."""
        for group in self.param_groups:
            self._counts(group)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        work, norms = [], {}
        for group in self.param_groups:
            for count, params, states, places in self._counts(group):
                ms, vs = self._moments(states, group["bits"])
                eight, device, table, grads = _checked(params, [p.grad for p in params], ms, vs, places)
                _check_options(count, group["lr"], group["betas"], group["eps"], group["weight_decay"],
                               self.max_grad_norm, device)
                if self.max_grad_norm is not None:
                    _require(not norms or device in norms, "AdamW: one device where gradients are clipped")
                    norms.setdefault(device, None)
                    norms[device] = norms[device] or _Norm(device)
                    norms[device].add(table, grads)
                work.append(((params, grads, ms, vs, places, eight, device, table, count), group))
        for tensors, group in work:
            _step(*tensors, group["lr"], group["betas"], group["eps"], group["weight_decay"], self.max_grad_norm,
                  norms.get(tensors[0][0].device))
        return loss

    @torch.no_grad()
    def load_state_dict(self, state_dict):
        """As torch's, but moments keep their types (torch would convert them to the
        parameters').  One of torch's own Adam or AdamW is taken too, unless it has maximize,
        amsgrad or a weight decay that is added to the gradient (Adam's; an older dict does not
        say whose it is), which raise: its moments become float32 whatever they were
        (bfloat16 parameters' are bfloat16), and the count that most parameters of a group
        have the group's."""
        for group in state_dict["param_groups"]:
            _check_loaded(group)
        theirs = {i for group in state_dict["param_groups"] if "bits" not in group for i in group["params"]}
        super().load_state_dict(state_dict)
        saved = [i for group in state_dict["param_groups"] for i in group["params"]]
        mine = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(saved, mine):
            for name, value in state_dict["state"].get(i, {}).items():
                if torch.is_tensor(value):
                    dtype = torch.float32 if i in theirs and name != "step" else value.dtype
                    self.state[p][name] = value.to(p.device, dtype, copy=True).contiguous()
        for group in self.param_groups:
            group.setdefault("bits", 32)
            own = [(state, int(state.pop("step"))) for state in map(self._known, group["params"]) if "step" in state]
            values = [n for _, n in own]
            if "step" not in group and not own:
                continue
            most = int(group["step"]) if "step" in group else max(values, key=values.count)
            counts = {n: torch.full((), n, dtype=torch.int64, device=group["params"][0].device) for n in (most, *values)}
            group["step"] = counts[most]
            for state, n in own:
                if n != most:
                    state["step"] = counts[n]
