"""Cases of the gated operators and of the optimizer that trains them: their
plain forms in elementary torch operations and the calls of
``duck_gym_b200.memory`` and ``duck_gym_b200.optim``.

Four kinds of case:

* ``linear``: a gated feed-forward layer, activation(x Wg' + bg) * (x Wu' + bu),
  forward alone or with its backward pass;
* ``scan``: a gated linear recurrence over a whole rollout,
  h = f h + (1 - f) c with f = sigmoid(gate), forward alone or with its backward
  pass;
* ``step``: the same recurrence for a single control step of every environment,
  state updated;
* ``adamw``: one AdamW step over all tensors of a model, with moments in 32 bits
  or in 8, gradients clipped by their common norm or not.

``own`` selects the framework's kernels; otherwise ``run`` is the plain form,
computed in 32 bits (a sum over a whole model's gradients in 64) and rounded once
at the end.

A moment kept in 8 bits has one exponent for 128 values, e = the largest exponent
field of their float32 forms; a code counts eighths of an octave from the float
whose leading 12 bits are max(0, 8 e + 8 - most), most = 255 for the second
moment (uint8) and 127 for the first (int8, with its sign).  A value's low 20 bits
are rounded up or down at random, by a hash of the step, the tensor's place in the
list and the value's place in the tensor.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
GROUP = 128   # values that share one exponent of a moment in 8 bits
BETAS, EPS = (0.9, 0.999), 1e-8


def listed():
    return [
        # One control step of the 16-env workload through the memory policy's MLP: latency.
        {"name": "linear step 16x256x512", "kind": "linear", "rows": 16, "D": 256, "F": 512, "type": "bf16",
         "activation": "silu", "bias": True, "train": False},
        # A PPO minibatch (24 steps x 4096 envs / 4) of that policy.
        {"name": "linear train 24576x256x512", "kind": "linear", "rows": 24576, "D": 256, "F": 512, "type": "bf16",
         "activation": "silu", "bias": True, "train": True},
        # Odd sizes in float32: the 61 actor observations into a hidden layer of no round width.
        {"name": "linear train 4999x61x301 fp32", "kind": "linear", "rows": 4999, "D": 61, "F": 301, "type": "fp32",
         "activation": "gelu", "bias": True, "train": True},
        # A wide feed-forward layer, as large models have it.
        {"name": "linear train 16384x1024x4096", "kind": "linear", "rows": 16384, "D": 1024, "F": 4096, "type": "bf16",
         "activation": "silu", "bias": False, "train": True},
        # One control step of 4096 envs.
        {"name": "step 4096x256", "kind": "step", "E": 4096, "N": 256, "type": "bf16"},
        # A PPO minibatch by envs: 24 steps of a quarter of 4096 envs, from the state that the rollout began with.
        {"name": "scan train 24x1024x256", "kind": "scan", "T": 24, "E": 1024, "N": 256, "type": "bf16", "train": True,
         "state": True, "final": False},
        # Whole logged episodes of 1000 steps (20 s at 50 Hz), trained from their start.
        {"name": "scan train 1000x256x256", "kind": "scan", "T": 1000, "E": 256, "N": 256, "type": "bf16", "train": True,
         "state": False, "final": False},
        # One long log read in before control goes on by single steps: few channels, a long axis.
        {"name": "scan replay 16384x1x1024", "kind": "scan", "T": 16384, "E": 1, "N": 1024, "type": "bf16", "train": False,
         "state": False, "final": True},
        # Odd sizes in float32, rows off every 16-byte boundary.
        {"name": "scan train 101x301x61 fp32", "kind": "scan", "T": 101, "E": 301, "N": 61, "type": "fp32", "train": True,
         "state": True, "final": True},
        # The actor-critic of the PPO, its gradients clipped: 17 small tensors, latency.
        {"name": "adamw policy", "kind": "adamw", "model": "policy", "tensors": 17, "values": 0, "type": "fp32", "bits": 32,
         "clip": True, "fresh": False},
        # A large model with moments in 8 bits.
        {"name": "adamw 16x4M 8-bit", "kind": "adamw", "model": "equal", "tensors": 16, "values": 1 << 22, "type": "fp32",
         "bits": 8, "clip": False, "fresh": False},
        # Odd sizes, bfloat16 parameters, moments in 8 bits from the first step on.
        {"name": "adamw ragged bf16 8-bit", "kind": "adamw", "model": "ragged", "tensors": 20, "values": 300007,
         "type": "bf16", "bits": 8, "clip": True, "fresh": True},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "scan", "scan", "scan", "step", "adamw", "adamw"])
    kind_type = rng.choice(["bf16", "bf16", "fp32"])
    if kind == "linear":
        D, F = _spread(rng, 32, 1024), _spread(rng, 64, 4096)
        if rng.random() < 0.6:   # mostly widths that rows of whole 16-byte pieces have
            D, F = (D + 7) // 8 * 8, (F + 7) // 8 * 8
        train = rng.random() < 0.7
        limit = 1 << (36 if kind_type == "bf16" else 32)
        rows = _spread(rng, 64 if train else 1, max(64, min(65536, limit // (D * F))))
        return {"kind": kind, "rows": rows, "D": D, "F": F, "type": kind_type,
                "activation": rng.choice(["silu", "silu", "gelu", "sigmoid"]), "bias": rng.random() < 0.5, "train": train}
    if kind == "adamw":
        model = rng.choice(["equal", "ragged"])
        tensors = rng.randint(1, 20)
        values = _spread(rng, 100, (1 << 26) // tensors)
        return {"kind": kind, "model": model, "tensors": tensors, "values": values, "type": kind_type,
                "bits": rng.choice([8, 8, 32]), "clip": rng.random() < 0.5, "fresh": rng.random() < 0.25}
    N = rng.choice([61, 64, 128, 200, 256, 256, 512, 1024])
    if kind == "step":
        return {"kind": kind, "E": _spread(rng, 1, 65536 * 64 // N), "N": N, "type": kind_type}
    T = _spread(rng, 1, 16384)
    E = _spread(rng, 1, max(1, min(4096, (1 << 26) // (T * N))))
    return {"kind": kind, "T": T, "E": E, "N": N, "type": kind_type, "train": rng.random() < 0.6,
            "state": rng.random() < 0.5, "final": rng.random() < 0.5}


def _shapes(case):
    if case["model"] == "policy":
        layers = [(512, 61), (512,), (256, 512), (256,), (128, 256), (128,)]
        return layers + [(14, 128), (14,)] + layers + [(1, 128), (1,)] + [(14,)]
    if case["model"] == "equal":
        return [(case["values"],)] * case["tensors"]
    return [(max(1, int(case["values"] / (1.0 + 1.7 * i))),) for i in range(case["tensors"])]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    s = dict(case)
    if case["kind"] == "linear":
        rows, D, F, train = case["rows"], case["D"], case["F"], case["train"]
        # Normed activations, weights of a linear layer after a while.
        s["x"] = normal(rows, D).to(dtype).requires_grad_(train)
        for name in ("gate", "up"):
            s["w_" + name] = (normal(F, D) * D ** -0.5).to(dtype).requires_grad_(train)
            s["b_" + name] = (0.1 * normal(F)).to(dtype).requires_grad_(train) if case["bias"] else None
        s["dh"] = normal(rows, F).to(dtype) if train else None
        return s
    if case["kind"] == "adamw":
        shapes = _shapes(case)
        sizes = [normal(1).abs() + 0.1 for _ in shapes]   # each tensor's gradients have a size of their own
        s["params"] = [(0.05 * normal(*shape)).to(dtype) for shape in shapes]
        s["grads"] = [(1e-3 * size * normal(*shape) * torch.exp(normal(*shape))).to(dtype) for size, shape in zip(sizes, shapes)]
        seen = 0.0 if case["fresh"] else 1.0
        m = [3e-4 * seen * size * normal(*shape) for size, shape in zip(sizes, shapes)]
        v = [1e-6 * seen * (size * torch.exp(normal(*shape))).square() for size, shape in zip(sizes, shapes)]
        eight = case["bits"] == 8
        half = torch.tensor(1 << 19, device="cuda")
        s["m"] = [_encode(x, 127, half) for x in m] if eight else m
        s["v"] = [_encode(x, 255, half) for x in v] if eight else v
        s["step"] = torch.full((), 0 if case["fresh"] else 1000, dtype=torch.int64, device="cuda")
        s["lr"] = torch.full((), 3e-4, device="cuda")   # on the device, as an adaptive schedule has it
        s["weight_decay"] = 0.01
        s["max_norm"] = 1.0 if case["clip"] else None
        return s
    E, N, train = case["E"], case["N"], bool(case.get("train"))
    lead = (E,) if case["kind"] == "step" else (case["T"], E)
    # Channels that remember between some two and some hundred steps.
    level = torch.linspace(0.0, 4.5, N, device="cuda")
    s["gates"] = (level + normal(*lead, N)).to(dtype).requires_grad_(train)
    s["values"] = normal(*lead, N).to(dtype).requires_grad_(train)
    # Episodes end after some 100 steps.
    s["resets"] = torch.rand(lead, generator=g, device="cuda") < 0.01
    # States of environments that have run for a while.
    s["memory"] = 0.5 * normal(E, N) if case.get("state", True) else None
    s["dout"] = normal(*lead, N).to(dtype) if train else None
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from duck_gym_b200 import memory, optim

    if s["kind"] == "linear":
        h = memory.gated_linear(s["x"], s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], activation=s["activation"])
        if not s["train"]:
            return {"h": h}
        names = ["x", "w_gate", "w_up"] + (["b_gate", "b_up"] if s["bias"] else [])
        grads = torch.autograd.grad(h, [s[name] for name in names], s["dh"])
        return {"h": h, **{"d" + name: grad for name, grad in zip(names, grads)}}
    if s["kind"] == "adamw":
        # Parameters and moments are updated in place, as in training: the next pass goes on from them.
        optim.adamw_step(s["params"], s["grads"], s["m"], s["v"], s["step"], s["lr"], betas=BETAS, eps=EPS,
                         weight_decay=s["weight_decay"], max_norm=s["max_norm"])
        if s["bits"] == 32:
            return {"p": s["params"], "m": s["m"], "v": s["v"]}
        return {"p": s["params"], "m": optim.state8_values(s["m"]), "v": optim.state8_values(s["v"])}
    if s["kind"] == "step":
        # The state is updated in place, as in a rollout.
        out = memory.gated_recurrence_step(s["gates"], s["values"], s["memory"], s["resets"])
        return {"out": out, "state": s["memory"]}
    h, final = memory.gated_recurrence(s["gates"], s["values"], s["memory"], s["resets"], final_state=s["final"])
    out = {"out": h}
    if s["final"]:
        out["state"] = final
    if s["train"]:
        out["dgates"], out["dvalues"] = torch.autograd.grad(h, (s["gates"], s["values"]), s["dout"])
    return out


def _run_plain(s):
    with torch.no_grad():
        return {"linear": _plain_linear, "scan": _plain_scan, "step": _plain_step, "adamw": _plain_adamw}[s["kind"]](s)


def _plain_linear(s):
    dtype = s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    a, u = x @ wg.t(), x @ wu.t()
    if s["bias"]:
        a, u = a + s["b_gate"].float(), u + s["b_up"].float()
    # The activation and its derivative.
    if s["activation"] == "gelu":
        below = 0.5 * (1.0 + torch.erf(a * 0.5 ** 0.5))
        y, slope = a * below, below + a * torch.exp(-0.5 * a * a) * (2.0 * math.pi) ** -0.5
    else:
        f = torch.sigmoid(a)
        y, slope = (a * f, f + a * f * (1.0 - f)) if s["activation"] == "silu" else (f, f * (1.0 - f))
    out = {"h": (y * u).to(dtype)}
    if s["train"]:
        dh = s["dh"].float()
        da, du = dh * u * slope, dh * y
        out["dx"] = (da @ wg + du @ wu).to(dtype)
        out["dw_gate"], out["dw_up"] = (da.t() @ x).to(dtype), (du.t() @ x).to(dtype)
        if s["bias"]:
            out["db_gate"], out["db_up"] = da.sum(0).to(dtype), du.sum(0).to(dtype)
    return out


def _scan(f, b):
    """h[t] = f[t] h[t - 1] + b[t] from h[-1] = 0: pairs of steps joined to one,
    the odd steps from the scan over these, the even ones from them."""
    T = f.shape[0]
    if T == 1:
        return b
    odd = _scan(f[1::2] * f[:-1:2], f[1::2] * b[:-1:2] + b[1::2])
    h = torch.empty_like(b)
    h[1::2] = odd
    h[0] = b[0]
    h[2::2] = f[2::2] * odd[:(T - 1) // 2] + b[2::2]
    return h


def _plain_scan(s):
    dtype = s["gates"].dtype
    gates, c = s["gates"].float(), s["values"].float()
    f, rest = torch.sigmoid(gates), torch.sigmoid(-gates)
    kept = torch.where(s["resets"][..., None], 0.0, f)   # of the state before the step
    b = rest * c
    if s["memory"] is not None:
        b[0] += kept[0] * s["memory"]
    h = _scan(kept, b)
    out = {"out": h.to(dtype)}
    if s["final"]:
        out["state"] = h[-1].clone()
    if s["train"]:
        # dh[t] = dout[t] + kept[t + 1] dh[t + 1]: the same scan, backwards.
        later = torch.cat([kept[1:], torch.zeros_like(kept[:1])])
        dh = _scan(later.flip(0), s["dout"].float().flip(0)).flip(0)
        first = torch.zeros_like(h[:1]) if s["memory"] is None else s["memory"][None]
        before = torch.where(s["resets"][..., None], 0.0, torch.cat([first, h[:-1]]))
        out["dgates"] = (dh * (before - c) * (f * rest)).to(dtype)
        out["dvalues"] = (dh * rest).to(dtype)
    return out


def _plain_step(s):
    gates, state = s["gates"].float(), s["memory"]   # updated in place
    state.masked_fill_(s["resets"][:, None], 0.0)
    state.mul_(torch.sigmoid(gates)).add_(torch.sigmoid(-gates) * s["values"].float())
    return {"out": state.to(s["gates"].dtype), "state": state}


def _mix(x):
    """The 32-bit finaliser of MurmurHash3, on int64."""
    x = (x ^ (x >> 16)) * 0x85EBCA6B & 0xFFFFFFFF
    x = (x ^ (x >> 13)) * 0xC2B2AE35 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _encode(x, most, noise):
    """Codes and exponents of float32 values; noise in [0, 2^20)."""
    n = x.numel()
    groups = (n + GROUP - 1) // GROUP
    bits = x.reshape(-1).abs().view(torch.int32)
    padded = torch.zeros(groups * GROUP, dtype=torch.int32, device=x.device)
    padded[:n] = bits
    exponents = (padded.view(groups, GROUP) >> 23).amax(1)
    low = (8 * exponents + (8 - most)).clamp_min(0).repeat_interleave(GROUP)[:n]
    codes = ((bits + noise.int()) >> 20).clamp_max(2039) - low
    if most == 127:
        codes = codes.clamp(0, 127).int() * torch.where(x.reshape(-1) < 0, -1, 1)
        return codes.to(torch.int8).view(x.shape), exponents.to(torch.uint8)
    codes = torch.where(bits == 0, 0, codes.clamp(1, 255))
    return codes.to(torch.uint8).view(x.shape), exponents.to(torch.uint8)


def _decode(codes, exponents):
    most = 127 if codes.dtype == torch.int8 else 255
    c = codes.reshape(-1).int()
    low = (8 * exponents.int() + (8 - most)).clamp_min(0).repeat_interleave(GROUP)[:c.numel()]
    value = torch.where(c == 0, 0, (c.abs() + low) << 20).view(torch.float32)
    return torch.where(c < 0, -value, value).view(codes.shape)


def _plain_adamw(s):
    s["step"] += 1
    t = s["step"]
    coef = None
    if s["max_norm"] is not None:
        total = torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
        coef = (s["max_norm"] / (total + 1e-6)).clamp_max(1.0).float()
    beta1, beta2 = BETAS
    rate = s["lr"].double()
    ahead = (rate / (1.0 - torch.pow(torch.tensor(beta1, dtype=torch.float64, device=t.device), t))).float()
    widen = (1.0 - torch.pow(torch.tensor(beta2, dtype=torch.float64, device=t.device), t)).rsqrt().float()
    shrink = (1.0 - rate * s["weight_decay"]).float()
    new = [_plain_tensor(i, *each, t, coef, beta1, beta2, ahead, widen, shrink)
           for i, each in enumerate(zip(s["params"], s["grads"], s["m"], s["v"]))]
    return {"p": s["params"], "m": [m for m, _ in new], "v": [v for _, v in new]}


def _plain_tensor(i, p, g, m, v, t, coef, beta1, beta2, ahead, widen, shrink):
    """One tensor's step; returns its moments as values."""
    kept = None if torch.is_tensor(m) else (m, v)
    old_m, old_v = (m, v) if kept is None else (_decode(*m), _decode(*v))
    g = g.float()
    g = g if coef is None else g * coef
    new_m = old_m * beta1 + g * (1.0 - beta1)
    new_v = old_v * beta2 + g * g * (1.0 - beta2)
    new_p = p.float() * shrink - ahead * (new_m / (new_v.sqrt() * widen + EPS))
    noise = None
    if kept is not None or p.dtype == torch.bfloat16:
        key = _mix((t + 0x9E3779B9 * (i + 1)) & 0xFFFFFFFF)
        noise = _mix(key ^ (torch.arange(p.numel(), device=p.device) & 0xFFFFFFFF))
    if p.dtype == torch.bfloat16:
        # Rounded up or down at random: most updates are less than half a step of the type.
        bits = new_p.view(torch.int32) + (noise & 0xFFFF).int().view(p.shape)
        new_p = (bits & -65536).view(torch.float32)
    p.copy_(new_p)
    if kept is None:
        m.copy_(new_m)
        v.copy_(new_v)
        return m, v
    new = _encode(new_m, 127, (noise >> 20 << 8) + 128), _encode(new_v, 255, noise & 0xFFFFF)
    _ = [a.copy_(b) for old, fresh in zip(kept, new) for a, b in zip(old, fresh)]
    return _decode(*new[0]), _decode(*new[1])


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["kind"] == "linear":
        rows, D, F = case["rows"], case["D"], case["F"]
        weights = 2 * F * D + (2 * F if case["bias"] else 0)
        # Forward: x and the weights in, h out; backward: x, the weights and dh in, dx and the weights' gradients out.
        if not case["train"]:
            return {"bytes": size * (rows * (D + F) + weights), "flops": 4 * rows * D * F}
        return {"bytes": size * (rows * (3 * D + 2 * F) + 3 * weights), "flops": 12 * rows * D * F}
    if case["kind"] == "adamw":
        values = sum(math.prod(shape) for shape in _shapes(case))
        moment = 4 if case["bits"] == 32 else 1 + 1 / GROUP
        # Parameter and moments in and out, the gradient in, once more where its norm comes first; moments in 8 bits as values.
        total = values * (2 * size + 4 * moment + size * (2 if case["clip"] else 1) + (0 if case["bits"] == 32 else 8))
        return {"bytes": total, "flops": 16 * values}
    if case["kind"] == "step":
        values = case["E"] * case["N"]
        return {"bytes": values * (3 * size + 8) + case["E"], "flops": 8 * values}
    values, states = case["T"] * case["E"] * case["N"], case["E"] * case["N"]
    total = 3 * values * size + case["T"] * case["E"] + 4 * states * (int(case["state"]) + int(case["final"]))
    if not case["train"]:
        return {"bytes": total, "flops": 8 * values}
    # Backward: gates, values and the output's gradient in, two gradients out.
    return {"bytes": total + 5 * values * size + case["T"] * case["E"] + 4 * states * int(case["state"]), "flops": 24 * values}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["kind"] == "adamw":
            return _exact_adamw(s)
        d = {name: x.detach().double() if torch.is_tensor(x) and x.is_floating_point() else x for name, x in s.items()}
        return {"linear": _exact_linear, "scan": _exact_scan, "step": _exact_step}[case["kind"]](d)


def _exact_linear(d):
    lines = lambda w, b: torch.einsum("rd,fd->rf", d["x"], w) + (0.0 if b is None else b)
    a, u = lines(d["w_gate"], d["b_gate"]), lines(d["w_up"], d["b_up"])
    normal = torch.distributions.Normal(torch.zeros((), dtype=torch.float64, device="cuda"), 1.0, validate_args=False)
    kind = d["activation"]
    share = normal.cdf(a) if kind == "gelu" else 1.0 / (1.0 + torch.exp(-a))
    y = share if kind == "sigmoid" else a * share
    out = {"h": y * u}
    if d["train"]:
        dshare = normal.log_prob(a).exp() if kind == "gelu" else share - share.square()
        slope = dshare if kind == "sigmoid" else torch.addcmul(share, a, dshare)
        da, du = d["dh"] * u * slope, d["dh"] * y
        out["dx"] = torch.einsum("rf,fd->rd", da, d["w_gate"]) + torch.einsum("rf,fd->rd", du, d["w_up"])
        out["dw_gate"], out["dw_up"] = torch.einsum("rf,rd->fd", da, d["x"]), torch.einsum("rf,rd->fd", du, d["x"])
        if d["bias"]:
            ones = da.new_ones(da.shape[0])
            out["db_gate"], out["db_up"] = ones @ da, ones @ du
    return out


def _exact_step(d):
    f = 1.0 / (1.0 + torch.exp(-d["gates"]))
    before = d["memory"] * (~d["resets"]).double()[:, None]
    state = torch.lerp(d["values"], before, f)
    return {"out": state, "state": state}


def _exact_scan(d):
    """The recurrence step by step, and its transpose backwards."""
    gates, c, alive = d["gates"], d["values"], (~d["resets"]).double()[..., None]
    f = 1.0 / (1.0 + torch.exp(-gates))
    state = torch.zeros_like(c[0]) if d["memory"] is None else d["memory"]
    h, before = torch.empty_like(c), torch.empty_like(c)
    for t in range(d["T"]):
        before[t] = state * alive[t]
        state = torch.lerp(c[t], before[t], f[t])
        h[t] = state
    out = {"out": h}
    if d["final"]:
        out["state"] = state
    if d["train"]:
        out["dgates"], out["dvalues"] = torch.empty_like(c), torch.empty_like(c)
        back = torch.zeros_like(c[0])
        for t in reversed(range(d["T"])):
            back = back + d["dout"][t]
            out["dvalues"][t] = back - back * f[t]
            out["dgates"][t] = back * (before[t] - c[t]) * (f[t] - f[t] ** 2)
            back = back * f[t] * alive[t]
    return out


def _exact_adamw(s):
    """Moments in 8 bits: which of two codes a value gets is decided by float32's
    last bit now and then, so that there is no such value for them."""
    t, (beta1, beta2) = int(s["step"]) + 1, BETAS
    clip = 1.0
    if s["max_norm"] is not None:
        clip = min(1.0, s["max_norm"] / (math.sqrt(sum(float(g.double().norm()) ** 2 for g in s["grads"])) + 1e-6))
    rate = float(s["lr"])
    out = {"p": [], "m": [], "v": []}
    for p, g, m, v in zip(s["params"], s["grads"], s["m"], s["v"]):
        eight = not torch.is_tensor(m)
        m, v = (_exact_moment(m, 127), _exact_moment(v, 255)) if eight else (m.double(), v.double())
        g = g.double() * clip
        m, v = torch.lerp(g, m, beta1), torch.lerp(g ** 2, v, beta2)
        best = m / (1.0 - beta1 ** t) / ((v / (1.0 - beta2 ** t)).sqrt() + EPS)
        out["p"].append(p.double() - rate * (best + s["weight_decay"] * p.double()))
        out["m"].append(None if eight else m)
        out["v"].append(None if eight else v)
    return out


def _exact_moment(kept, most):
    """A code's value: 2^octaves (1 + eighths / 8), read from the count of eighths."""
    codes, exponents = kept[0].reshape(-1).double(), kept[1].double()
    low = (8.0 * exponents + 8.0 - most).clamp_min(0.0)
    place = codes.abs() + low[torch.arange(codes.numel(), device=codes.device) // GROUP]
    octave = torch.floor(place / 8.0)
    value = torch.where(octave > 0, torch.exp2(octave - 127.0) * (1.0 + (place - 8.0 * octave) / 8.0),
                        place * 2.0 ** -129)
    return (torch.sign(codes) * value).view(kept[0].shape)
