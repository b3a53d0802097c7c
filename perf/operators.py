"""Cases of the memory policy's operators: their plain forms in elementary
torch operations and the calls of ``duck_gym_b200.memory``.

Four kinds of case:

* ``norm``: layer norm over the last axis, forward alone or with its backward
  pass (gradients of the input, the weight and the bias);
* ``memory``: linear attention with one decay per head over a whole rollout
  (chunked form), forward alone or with its backward pass;
* ``step``: the same recurrence for a single control step of every
  environment, state updated (recurrent form);
* ``checkpoint``: ELU whose output is kept in 8 bits, and the backward pass
  that reads it.

``own`` selects the framework's kernels; otherwise ``run`` is the plain form,
computed in 32 bits and rounded once at the end.
"""

import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5
GROUP = 128   # values that share one scale of an 8-bit checkpoint
CHUNK = 64    # steps per chunk of the plain form of linear attention


def listed():
    return [
        # One control step of the 16-env workload through a 128-wide norm: latency.
        {"name": "norm step 16x128", "kind": "norm", "rows": 16, "n": 128, "type": "bf16", "train": False},
        # Odd sizes: the 61 actor observations normalised without a hidden layer, float32, rows not 16-byte aligned.
        {"name": "norm train 4999x61 fp32", "kind": "norm", "rows": 4999, "n": 61, "type": "fp32", "train": True},
        # A PPO minibatch (24 steps x 4096 envs / 4) through a 256-wide norm.
        {"name": "norm train 24576x256", "kind": "norm", "rows": 24576, "n": 256, "type": "bf16", "train": True},
        # The same minibatch of 65536 envs through the 512-wide first hidden layer.
        {"name": "norm train 393216x512", "kind": "norm", "rows": 393216, "n": 512, "type": "bf16", "train": True},
        # One control step of 16 envs: latency of the recurrent form.
        {"name": "step 16 envs", "kind": "step", "E": 16, "H": 4, "Dk": 64, "Dv": 64, "type": "bf16"},
        # One control step of 4096 envs: 268 MB of state read and written.
        {"name": "step 4096 envs", "kind": "step", "E": 4096, "H": 4, "Dk": 64, "Dv": 64, "type": "bf16"},
        # A PPO minibatch by envs: 24 steps of a quarter of 4096 envs, from the state that the rollout began with.
        {"name": "memory train 24x1024", "kind": "memory", "T": 24, "E": 1024, "H": 4, "Dk": 64, "Dv": 64, "type": "bf16",
         "train": True, "state": True, "final": False},
        # Odd sizes in float32: head sizes that are no multiple of 8, a length that ends inside a chunk.
        {"name": "memory train 101x301 fp32", "kind": "memory", "T": 101, "E": 301, "H": 3, "Dk": 20, "Dv": 28,
         "type": "fp32", "train": True, "state": True, "final": True},
        # Whole logged episodes of 1000 steps (20 s at 50 Hz), trained from their start.
        {"name": "memory train 1000x256", "kind": "memory", "T": 1000, "E": 256, "H": 4, "Dk": 64, "Dv": 64, "type": "bf16",
         "train": True, "state": False, "final": False},
        # One long log read in before control goes on by single steps: few rows, a long axis.
        {"name": "memory replay 16384x1", "kind": "memory", "T": 16384, "E": 1, "H": 8, "Dk": 128, "Dv": 128, "type": "bf16",
         "train": False, "state": False, "final": True},
        # The 512-wide hidden layer of a PPO minibatch, kept in 8 bits for the backward pass.
        {"name": "checkpoint 24576x512", "kind": "checkpoint", "rows": 24576, "n": 512, "type": "bf16"},
        # Odd sizes: a width that ends one value into its second group, float32.
        {"name": "checkpoint 4999x129 fp32", "kind": "checkpoint", "rows": 4999, "n": 129, "type": "fp32"},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "memory", "memory", "memory", "step", "checkpoint"])
    kind_type = rng.choice(["bf16", "bf16", "fp32"])
    if kind in ("norm", "checkpoint"):
        n = _spread(rng, 8, 4096) if kind == "norm" else _spread(rng, 16, 2048)
        rows = _spread(rng, 1, max(1, min(393216, (1 << 26) // n)))
        case = {"kind": kind, "rows": rows, "n": n, "type": kind_type}
        return {**case, "train": rng.random() < 0.7} if kind == "norm" else case
    H = rng.choice([1, 2, 3, 4, 8])
    size = rng.choice([16, 20, 32, 64, 64, 128])
    Dk, Dv = size, rng.choice([size, size, 24, 40])
    if kind == "step":
        E = _spread(rng, 1, max(1, min(16384, (1 << 26) // (H * Dk * Dv))))
        return {"kind": kind, "E": E, "H": H, "Dk": Dk, "Dv": Dv, "type": kind_type}
    T = _spread(rng, 1, 8192)
    E = _spread(rng, 1, max(1, min(2048, (1 << 24) // (T * H * max(Dk, Dv)))))
    return {"kind": kind, "T": T, "E": E, "H": H, "Dk": Dk, "Dv": Dv, "type": kind_type, "train": rng.random() < 0.6,
            "state": rng.random() < 0.5, "final": rng.random() < 0.5}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    dtype = TYPES[case["type"]]
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")
    s = dict(case)
    if case["kind"] == "norm":
        rows, n = case["rows"], case["n"]
        # Hidden activations: a level and a spread of each row's own.
        x = normal(rows, n) * (0.5 + normal(rows, 1).abs()) + normal(rows, 1)
        s["x"] = x.to(dtype).requires_grad_(case["train"])
        s["weight"] = (1.0 + 0.1 * normal(n)).requires_grad_(case["train"])
        s["bias"] = (0.1 * normal(n)).requires_grad_(case["train"])
        s["dy"] = normal(rows, n).to(dtype)
        return s
    if case["kind"] == "checkpoint":
        s["x"] = (1.5 * normal(case["rows"], case["n"])).to(dtype)
        s["dy"] = normal(case["rows"], case["n"]).to(dtype)
        return s
    E, H, Dk, Dv = (case[k] for k in ("E", "H", "Dk", "Dv"))
    lead = (E,) if case["kind"] == "step" else (case["T"], E)
    for name, width in (("q", Dk), ("k", Dk), ("v", Dv)):
        s[name] = normal(*lead, H, width).to(dtype).requires_grad_(bool(case.get("train")))
    # Memories of about 4 to 250 steps, one per head.
    s["decay"] = 1.0 - torch.exp2(-torch.linspace(2.0, 8.0, H, device="cuda"))
    # Episodes end after some 100 steps.
    s["resets"] = torch.rand(lead, generator=g, device="cuda") < 0.01
    # States of environments that have run for a while.
    s["memory"] = 3.0 * normal(E, H, Dk, Dv) if case.get("state", True) else None
    if case.get("train"):
        s["do"] = normal(*lead, H, Dv).to(dtype)
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    from duck_gym_b200 import memory

    if s["kind"] == "norm":
        y = memory.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        if not s["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    if s["kind"] == "checkpoint":
        y, kept = memory.elu_checkpoint(s["x"])
        dx, restored = memory.elu_restore(s["dy"], kept)
        return {"y": y, "restored": restored, "dx": dx}
    if s["kind"] == "step":
        # The state is updated in place, as in a rollout: the next pass goes on from it.
        o = memory.linear_attention_step(s["q"], s["k"], s["v"], s["decay"], s["memory"], s["resets"])
        return {"o": o, "state": s["memory"]}
    o, final = memory.linear_attention(s["q"], s["k"], s["v"], s["decay"], s["memory"], s["resets"],
                                       final_state=s["final"])
    out = {"o": o}
    if s["final"]:
        out["state"] = final
    if s["train"]:
        out["dq"], out["dk"], out["dv"] = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
    return out


def _run_plain(s):
    if s["kind"] == "norm":
        return _plain_norm(s)
    if s["kind"] == "checkpoint":
        return _plain_checkpoint(s)
    if s["kind"] == "step":
        return _plain_step(s)
    if not s["train"]:
        with torch.no_grad():
            return _plain_memory(s, s["q"].float(), s["k"].float(), s["v"].float())
    leaves = [s[name].detach().float().requires_grad_() for name in ("q", "k", "v")]
    out = _plain_memory(s, *leaves)
    grads = torch.autograd.grad(out["o"], leaves, s["do"])
    out = {name: x.detach() for name, x in out.items()}
    out["dq"], out["dk"], out["dv"] = (d.to(s["q"].dtype) for d in grads)
    return out


def _plain_norm(s):
    x, w, dtype = s["x"].detach().float(), s["weight"].detach(), s["x"].dtype
    centred = x - x.mean(1, keepdim=True)
    rstd = torch.rsqrt((centred * centred).mean(1, keepdim=True) + EPS)
    unit = centred * rstd
    out = {"y": (unit * w + s["bias"].detach()).to(dtype)}
    if s["train"]:
        dy = s["dy"].float()
        g = dy * w
        dx = rstd * (g - g.mean(1, keepdim=True) - unit * (g * unit).mean(1, keepdim=True))
        out.update(dx=dx.to(dtype), dweight=(dy * unit).sum(0), dbias=dy.sum(0))
    return out


def _plain_checkpoint(s):
    x, dtype = s["x"], s["x"].dtype
    rows, n = x.shape
    groups = (n + GROUP - 1) // GROUP
    xf = x.float()
    y = torch.where(xf > 0, xf, torch.expm1(xf)).to(dtype)
    padded = torch.zeros(rows, groups * GROUP, device=x.device)
    padded[:, :n] = y
    padded = padded.view(rows, groups, GROUP)
    scale = padded.abs().amax(2, keepdim=True) * (1.0 / 127.0)
    inverse = torch.where(scale > 0, torch.reciprocal(scale), torch.zeros_like(scale))
    codes = torch.round(padded * inverse).to(torch.int8)
    restored = (codes.float() * scale).view(rows, -1)[:, :n]
    dx = s["dy"].float() * torch.where(restored > 0, torch.ones_like(restored), restored + 1.0)
    return {"y": y, "restored": restored.to(dtype), "dx": dx.to(dtype)}


def _plain_step(s):
    q, k, v = s["q"].float() * s["Dk"] ** -0.5, s["k"].float(), s["v"].float()
    state = s["memory"]                       # updated in place
    state.masked_fill_(s["resets"][:, None, None, None], 0.0)
    state.mul_(s["decay"][None, :, None, None]).addcmul_(k[..., :, None], v[..., None, :])
    o = (q[..., None, :] @ state)[..., 0, :]
    return {"o": o.to(s["q"].dtype), "state": state}


def _plain_memory(s, q, k, v):
    """Chunks of CHUNK steps: products within a chunk, and with the state that
    each chunk starts from, which a product over chunks gives.  ``part`` numbers
    the episodes of an env: only steps of one part see one another."""
    T, E, H, Dk, Dv, C = s["T"], s["E"], s["H"], s["Dk"], s["Dv"], min(CHUNK, s["T"])
    N = (T + C - 1) // C
    resets = s["resets"]
    pad = N * C - T
    if pad:
        q, k, v = (torch.cat([x, x.new_zeros(pad, *x.shape[1:])]) for x in (q, k, v))
        resets = torch.cat([resets, resets.new_zeros(pad, E)])
    heads = lambda x: x.view(N, C, E, H, -1).permute(2, 3, 0, 1, 4)   # [E, H, N, C, D]
    q, k, v = heads(q) * Dk ** -0.5, heads(k), heads(v)
    log_decay = torch.log(s["decay"])[None, :, None, None]
    part = resets.cumsum(0).t().reshape(E, 1, N, C)
    steps = torch.arange(C, device=q.device)
    gap = (steps[:, None] - steps[None, :]).float()
    same = (part[..., :, None] == part[..., None, :]) & (gap >= 0)
    within = torch.where(same, torch.exp(gap.clamp_min(0) * log_decay[..., None]), 0.0)
    o = ((q @ k.transpose(-1, -2)) * within) @ v
    # What each chunk adds to the state at its end, and the chunks before it.
    last = part[..., -1:]
    to_end = torch.where(part == last, torch.exp((C - 1 - steps).float() * log_decay), 0.0)
    added = ((k * to_end[..., None]).transpose(-1, -2) @ v).reshape(E, H, N, Dk * Dv)
    first = torch.zeros(E, H, 1, Dk * Dv, device=q.device) if s["memory"] is None else s["memory"].reshape(E, H, 1, -1)
    added = torch.cat([first, added], 2)                                # what is in the state before chunk 0, 1, ...
    ends = torch.cat([torch.zeros_like(last[:, :, :1, 0]), last[..., 0]], 2)   # [E, 1, N + 1]
    chunks = torch.arange(N + 1, device=q.device)
    away = (chunks[:, None] - chunks[None, :]).float()
    joined = (ends[..., :, None] == ends[..., None, :]) & (away >= 0)
    weights = torch.where(joined, torch.exp(C * away.clamp_min(0) * log_decay), 0.0)
    states = (weights @ added).reshape(E, H, N + 1, Dk, Dv)
    from_start = torch.where(part == ends[..., :-1, None], torch.exp((steps + 1).float() * log_decay), 0.0)
    o = o + (q * from_start[..., None]) @ states[:, :, :-1]
    o = o.permute(2, 3, 0, 1, 4).reshape(N * C, E, H, Dv)[:T].to(s["q"].dtype)
    out = {"o": o}
    if s["final"]:
        # The padding steps after the last one only decay the state.
        left = torch.exp(-pad * log_decay)
        out["state"] = (states[:, :, -1] * left).contiguous()
    return out


def work(case):
    size = 2 if case["type"] == "bf16" else 4
    if case["kind"] == "norm":
        values = case["rows"] * case["n"]
        if not case["train"]:
            return {"bytes": 2 * values * size + 8 * case["n"], "flops": 8 * values}
        # Forward: x in, y out; backward: x and dy in, dx out; a mean and a deviation per row between them.
        return {"bytes": 5 * values * size + 16 * case["rows"] + 24 * case["n"], "flops": 20 * values}
    if case["kind"] == "checkpoint":
        values = case["rows"] * case["n"]
        kept = values + 4 * case["rows"] * ((case["n"] + GROUP - 1) // GROUP)
        # x in, y and the checkpoint out; dy and the checkpoint in, dx and the restored y out.
        return {"bytes": 5 * values * size + 2 * kept, "flops": 12 * values}
    E, H, Dk, Dv = (case[k] for k in ("E", "H", "Dk", "Dv"))
    state = 4 * E * H * Dk * Dv
    if case["kind"] == "step":
        return {"bytes": 2 * state + E * H * (2 * Dk + 2 * Dv) * size + E, "flops": 5 * E * H * Dk * Dv}
    rows = case["T"] * E * H
    total = rows * (2 * Dk + 2 * Dv) * size + case["T"] * E
    flops = 4 * rows * Dk * Dv
    if case["train"]:
        # Backward: q, k, v and the output's gradient in, three gradients out.
        total += rows * (4 * Dk + 3 * Dv) * size + case["T"] * E + (state if case["state"] else 0)
        flops += 10 * rows * Dk * Dv
    total += (state if case["state"] else 0) + (state if case["final"] else 0)
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        d = {name: x.detach().double() if torch.is_tensor(x) and x.is_floating_point() else x for name, x in s.items()}
        if case["kind"] == "norm":
            return _exact_norm(d)
        if case["kind"] == "checkpoint":
            return _exact_checkpoint(d, TYPES[case["type"]])
        return _exact_step(d) if case["kind"] == "step" else _exact_memory(d)


def _exact_norm(d):
    x, w = d["x"], d["weight"]
    deviation = ((x * x).mean(1) - x.mean(1) ** 2 + EPS).sqrt()[:, None]
    unit = (x - x.mean(1)[:, None]) / deviation
    out = {"y": torch.addcmul(d["bias"], unit, w)}
    if d["train"]:
        n, h = x.shape[1], d["dy"] * w
        dx = (n * h - h.sum(1)[:, None] - unit * (h * unit).sum(1)[:, None]) / (n * deviation)
        out.update(dx=dx, dweight=torch.einsum("rn,rn->n", d["dy"], unit),
                   dbias=d["dy"].new_ones(x.shape[0]) @ d["dy"])
    return out


def _exact_checkpoint(d, dtype):
    """The codes are those of the output as it is stored.  In float32 the last
    bit of the exponential decides which of two codes a value near their middle
    gets, so that there is no such value for what the codes stand for."""
    x = d["x"]
    y = x.clamp_min(0) + torch.expm1(x.clamp_max(0))
    if dtype == torch.float32:
        return {"y": y, "restored": None, "dx": None}
    stored = y.to(dtype).double()
    restored = torch.empty_like(y)
    for at in range(0, x.shape[1], GROUP):
        part = stored[:, at:at + GROUP]
        unit = part.abs().max(1, keepdim=True).values / 127.0
        restored[:, at:at + GROUP] = (part / unit.clamp_min(1e-300)).round() * unit
    return {"y": y, "restored": restored, "dx": d["dy"] * (1.0 + restored.clamp_max(0))}


def _exact_step(d):
    alive = d["decay"].expand(d["E"], -1) * (~d["resets"]).double()[:, None]
    state = torch.einsum("eh,ehij->ehij", alive, d["memory"]) + torch.einsum("ehi,ehj->ehij", d["k"], d["v"])
    return {"o": torch.einsum("ehi,ehij->ehj", d["q"], state) / math.sqrt(d["Dk"]), "state": state}


def _exact_memory(d):
    """The recurrence step by step, and its transpose backwards."""
    T, E, H, Dk, Dv = (d[k] for k in ("T", "E", "H", "Dk", "Dv"))
    scale = 1.0 / math.sqrt(Dk)
    kept = d["decay"][None, None, :] * (~d["resets"]).double()[:, :, None]     # [T, E, H]
    kept = kept[..., None, None]
    state = torch.zeros(E, H, Dk, Dv, dtype=torch.float64, device="cuda") if d["memory"] is None else d["memory"].clone()
    o = torch.empty_like(d["v"])
    dq = torch.empty_like(d["q"]) if d["train"] else None
    for t in range(T):
        state.mul_(kept[t]).add_(d["k"][t][..., :, None] * d["v"][t][..., None, :])
        o[t] = (d["q"][t][..., None, :] @ state)[..., 0, :] * scale
        if d["train"]:
            dq[t] = (state @ d["do"][t][..., :, None])[..., 0] * scale
    out = {"o": o}
    if d["final"]:
        out["state"] = state
    if d["train"]:
        dk, dv = torch.empty_like(d["k"]), torch.empty_like(d["v"])
        back = torch.zeros(E, H, Dk, Dv, dtype=torch.float64, device="cuda")
        for t in reversed(range(T)):
            back.add_(d["q"][t][..., :, None] * d["do"][t][..., None, :], alpha=scale)
            dk[t] = (back @ d["v"][t][..., :, None])[..., 0]
            dv[t] = (d["k"][t][..., None, :] @ back)[..., 0, :]
            back.mul_(kept[t])
        out.update(dq=dq, dk=dk, dv=dv)
    return out
