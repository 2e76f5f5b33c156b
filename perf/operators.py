"""Work of the recurrent block's operators: the gated linear recurrence, group normalisation with an activation
over channels-last tensors, and dropout from the counter-based generator, each forwards and backwards.

`run` computes them in elementary torch operations, or (where `own` is true) with the calls of the C ABI in
include/homura_nn.h that a user of homura_amd.capi makes."""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
DEVICE = "cuda:0"


# ---- the cases ---------------------------------------------------------------------------------------------------

def listed():
    return [
        # One token for each of 64 sequences of a served model: the smallest call, where latency counts.
        {"name": "recurrence_step", "op": "recurrence", "form": "sigmoid", "dtype": "bf16", "B": 64, "T": 1, "C": 4096,
         "ragged": False},
        # A prompt batch of the size of the framework's own activation tensors.
        {"name": "recurrence_prompt", "op": "recurrence", "form": "factor", "dtype": "bf16", "B": 8, "T": 2048, "C": 4096,
         "ragged": False},
        # Two long documents of different lengths in f32, with a number of channels no vector divides.
        {"name": "recurrence_long_odd", "op": "recurrence", "form": "sigmoid", "dtype": "f32", "B": 2, "T": 16411, "C": 1003,
         "ragged": True},
        # The gradient of a training step over medium sequences.
        {"name": "recurrence_gradient", "op": "recurrence_backward", "form": "sigmoid", "dtype": "bf16", "B": 4, "T": 4096,
         "C": 2048, "ragged": False},
        # Every head of every token normalised by itself, after the recurrence.
        {"name": "norm_heads", "op": "norm", "act": "silu", "dtype": "bf16", "N": 16384, "S": 1, "C": 4096, "G": 32},
        # Its gradient.
        {"name": "norm_heads_gradient", "op": "norm_backward", "act": "silu", "dtype": "f16", "N": 8192, "S": 1, "C": 4096,
         "G": 64},
        # Feature maps of 64 x 64 positions, ten channels a group.
        {"name": "norm_maps", "op": "norm", "act": "silu", "dtype": "bf16", "N": 16, "S": 4096, "C": 320, "G": 32},
        # The gradient over fewer, larger maps in f32.
        {"name": "norm_maps_gradient", "op": "norm_backward", "act": "gelu_tanh", "dtype": "f32", "N": 4, "S": 9216, "C": 512,
         "G": 32},
        # A residual branch's end: dropout and the residual's addition over a whole activation tensor.
        {"name": "dropout_residual", "op": "dropout", "dtype": "bf16", "n": 8 * 2048 * 4096, "p": 0.1, "residual": True},
        # The gradient through a dropout of one in two, of an odd number of f32 elements.
        {"name": "dropout_gradient", "op": "dropout", "dtype": "f32", "n": 33333331, "p": 0.5, "residual": False},
        # A small layer's activations: latency again.
        {"name": "dropout_small", "op": "dropout", "dtype": "f16", "n": 32 * 1000, "p": 0.25, "residual": False},
    ]


def _spread(rng, low, high):
    """A whole number between the two, spread over its logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    op = rng.choice(["recurrence", "recurrence", "recurrence_backward", "norm", "norm", "norm_backward", "dropout"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op.startswith("recurrence"):
        C = rng.choice([8, 64, 1]) * _spread(rng, 1, 64) if rng.random() < 0.7 else _spread(rng, 1, 4099)
        most = 33_000_000 if op == "recurrence" else 16_000_000  # elements
        T = 1 if op == "recurrence" and rng.random() < 0.2 else _spread(rng, 2, min(16384, most // C))
        B = _spread(rng, 1, max(1, min(256, most // (T * C))))
        return {"op": op, "form": rng.choice(["factor", "sigmoid"]), "dtype": dtype, "B": B, "T": T, "C": C,
                "ragged": T > 1 and rng.random() < 0.5}
    if op.startswith("norm"):
        G = rng.choice([1, 2, 8, 12, 32, 64])
        C = G * (rng.choice([8, 16, 32, 64, 128]) if rng.random() < 0.6 else _spread(rng, 1, 130))
        S = 1 if rng.random() < 0.5 else _spread(rng, 2, min(16384, 24_000_000 // C))
        N = _spread(rng, 1, max(1, min(16384, 24_000_000 // (S * C))))
        return {"op": op, "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), "dtype": dtype, "N": N, "S": S,
                "C": C, "G": G}
    return {"op": op, "dtype": dtype, "n": _spread(rng, 64, 30_000_000), "p": rng.choice([0.05, 0.1, 0.25, 0.5, 0.9]),
            "residual": rng.random() < 0.5}


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op.startswith("recurrence"):
        B, T, C = case["B"], case["T"], case["C"]
        steps = sum(_lengths(B, T)) if case["ragged"] else B * T  # padding is written, not read
        if op == "recurrence":
            return {"bytes": size * C * (2 * steps + B * T) + 8 * B * C, "flops": (2 if case["form"] == "factor" else 8) * steps * C}
        reads = 3 if case["form"] == "factor" else 4
        return {"bytes": size * C * (reads * steps + 2 * B * T) + 12 * B * C, "flops": (5 if case["form"] == "factor" else 14) * steps * C}
    if op.startswith("norm"):
        n = case["N"] * case["S"] * case["C"]
        stats = 8 * case["N"] * case["G"]
        if op == "norm":
            return {"bytes": size * 2 * n + stats + 2 * size * case["C"], "flops": 12 * n}
        return {"bytes": size * 3 * n + stats + 4 * size * case["C"], "flops": 30 * n}
    return {"bytes": size * case["n"] * (3 if case["residual"] else 2), "flops": (3 if case["residual"] else 2) * case["n"]}


def _lengths(B, T):
    """The lengths of a padded batch: from the whole length down to about half of it, none of them in step with a tile."""
    return [max(1, T - (b * T) // (2 * B) - (b % 3)) for b in range(B)]


# ---- inputs ------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed * 2654435761 % (1 << 62))
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, mean=0.0, std=1.0):
        return torch.randn(*shape, device=DEVICE, generator=g) * std + mean

    s = {"case": dict(case)}
    op = case["op"]
    if op.startswith("recurrence"):
        B, T, C = case["B"], case["T"], case["C"]
        if case["form"] == "factor":
            gate = torch.sigmoid(normal(B, T, C, mean=3.0, std=1.5))
            # Documents that begin inside the batch: every channel forgets.
            gate = gate * (torch.rand(B, T, 1, device=DEVICE, generator=g) > 1 / 997)
        else:
            gate = normal(B, T, C, mean=3.0, std=2.0)
        s["gate"] = gate.to(dtype)
        s["input"] = normal(B, T, C).to(dtype)
        s["initial"] = normal(B, C)
        order = torch.randperm(B, device=DEVICE, generator=g)
        s["lengths"] = torch.tensor(_lengths(B, T), device=DEVICE, dtype=torch.int32)[order] if case["ragged"] else None
        del gate
        if op == "recurrence":
            s["out"] = torch.empty(B, T, C, device=DEVICE, dtype=dtype)
            s["last"] = torch.empty(B, C, device=DEVICE)
        else:
            s["out"] = _recurrence(s)["out"]
            s["grad"] = normal(B, T, C, std=0.1).to(dtype)
            s["grad_last"] = normal(B, C, std=0.1)
            s["d_gate"] = torch.empty(B, T, C, device=DEVICE, dtype=dtype)
            s["d_input"] = torch.empty(B, T, C, device=DEVICE, dtype=dtype)
            s["d_initial"] = torch.empty(B, C, device=DEVICE)
    elif op.startswith("norm"):
        N, S, C, G = (case[k] for k in "NSCG")
        # Channels with means and scales of their own, as activations have.
        x = normal(N, S, C) * normal(C, mean=1.0, std=0.3) + normal(C, std=0.5)
        s["x"] = x.to(dtype)
        s["weight"] = normal(C, mean=1.0, std=0.2).to(dtype)
        s["bias"] = normal(C, std=0.2).to(dtype)
        s["eps"] = 1e-5
        if op == "norm":
            s["out"] = torch.empty(N, S, C, device=DEVICE, dtype=dtype)
            s["mean"] = torch.empty(N, G, device=DEVICE)
            s["rstd"] = torch.empty(N, G, device=DEVICE)
        else:
            s["mean"], s["rstd"] = _statistics(s["x"].view(N, S, G, C // G).float(), s["eps"])
            s["grad"] = normal(N, S, C).to(dtype)
            s["d_x"] = torch.empty(N, S, C, device=DEVICE, dtype=dtype)
            s["d_weight"] = torch.empty(C, device=DEVICE, dtype=dtype)
            s["d_bias"] = torch.empty(C, device=DEVICE, dtype=dtype)
    else:
        s["x"] = normal(case["n"]).to(dtype)
        s["residual"] = normal(case["n"]).to(dtype) if case["residual"] else None
        s["out"] = torch.empty(case["n"], device=DEVICE, dtype=dtype)
        # A generator that a long run has taken to where the counter's low word wraps.
        s["seed"], s["offset"] = 67280421310721 + seed, (1 << 32) - 1000 + 977 * seed
    if own:
        _plan(s)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------

def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1 with h before the first step zero, by doubling: after a pass of
    `step`, (a, b) at t stand for the 2 * step steps that end there."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], a[:, step:] * b[:, :-step] + b[:, step:]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _inside(s):
    """[B, T, 1]: which steps lie inside their sequence."""
    T = s["case"]["T"]
    return (torch.arange(T, device=DEVICE)[None, :] < s["lengths"][:, None].long())[..., None]


def _recurrence(s):
    gate, x = s["gate"].float(), s["input"].float()
    if s["case"]["form"] == "factor":
        a, b = gate, x
    else:
        a = 1 / (1 + torch.exp(-gate))
        b = x * (1 / (1 + torch.exp(gate)))
    if s["lengths"] is not None:
        inside = _inside(s)
        a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
    b = torch.cat([b[:, :1] + a[:, :1] * s["initial"][:, None], b[:, 1:]], 1)
    h = _scan(a, b)
    last = h[:, -1].clone()
    if s["lengths"] is not None:
        h = torch.where(inside, h, 0.0)
    return {"out": h.to(s["gate"].dtype), "last": last}


def _recurrence_backward(s):
    gate, dh = s["gate"].float(), s["grad"].float()
    before = torch.cat([s["initial"][:, None], s["out"][:, :-1].float()], 1)  # the state that each step starts from
    a = gate if s["case"]["form"] == "factor" else 1 / (1 + torch.exp(-gate))
    b = a * dh
    if s["lengths"] is not None:
        inside = _inside(s)
        a, b = torch.where(inside, a, 1.0), torch.where(inside, b, 0.0)
    # e_t = a_t (dh_t + e_{t+1}) is what step t hands back to the one before it.
    e = torch.cat([b[:, :-1], b[:, -1:] + a[:, -1:] * s["grad_last"][:, None]], 1)
    e = _scan(a.flip(1), e.flip(1)).flip(1)
    g = dh + torch.cat([e[:, 1:], s["grad_last"][:, None]], 1)
    if s["case"]["form"] == "factor":
        d_gate, d_input = g * before, g
    else:
        rest = 1 / (1 + torch.exp(gate))
        d_gate, d_input = g * (before - s["input"].float()) * a * rest, g * rest
    if s["lengths"] is not None:
        d_gate, d_input = torch.where(inside, d_gate, 0.0), torch.where(inside, d_input, 0.0)
    return {"d_gate": d_gate.to(s["gate"].dtype), "d_input": d_input.to(s["gate"].dtype), "d_initial": e[:, 0].clone()}


def _statistics(x, eps):
    mean = x.mean((1, 3))
    centred = x - mean[:, None, :, None]
    return mean, 1 / torch.sqrt((centred * centred).mean((1, 3)) + eps)


_ROOT2, _ROOT2PI, _INNER = 2.0 ** 0.5, 0.7978845608028654, 0.044715


def _activate(z, act):
    if act == "relu":
        return torch.where(z < 0, 0.0, z)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z / _ROOT2))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(_ROOT2PI * (z + _INNER * z * z * z)))
    return z


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        q = 1 / (1 + torch.exp(-z))
        return q * (1 + z * (1 - q))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z / _ROOT2)) + z * torch.exp(-0.5 * z * z) * (_ROOT2PI / 2)
    if act == "gelu_tanh":
        t = torch.tanh(_ROOT2PI * (z + _INNER * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * _ROOT2PI * (1 + 3 * _INNER * z * z)
    return torch.ones_like(z)


def _norm(s):
    N, S, C, G = (s["case"][k] for k in "NSCG")
    x = s["x"].view(N, S, G, C // G).float()
    mean, rstd = _statistics(x, s["eps"])
    hat = (x - mean[:, None, :, None]) * rstd[:, None, :, None]
    z = hat * s["weight"].float().view(G, -1) + s["bias"].float().view(G, -1)
    return {"out": _activate(z, s["case"]["act"]).to(s["x"].dtype).view(N, S, C), "mean": mean, "rstd": rstd}


def _norm_backward(s):
    N, S, C, G = (s["case"][k] for k in "NSCG")
    x, dy = s["x"].view(N, S, G, C // G).float(), s["grad"].view(N, S, G, C // G).float()
    rstd, w = s["rstd"][:, None, :, None], s["weight"].float().view(G, -1)
    hat = (x - s["mean"][:, None, :, None]) * rstd
    dz = dy * _slope(hat * w + s["bias"].float().view(G, -1), s["case"]["act"])
    d_bias, d_weight = dz.sum((0, 1)).view(C), (dz * hat).sum((0, 1)).view(C)
    dz = dz * w
    d_x = rstd * (dz - dz.mean((1, 3), keepdim=True) - hat * (dz * hat).mean((1, 3), keepdim=True))
    dtype = s["x"].dtype
    return {"d_x": d_x.to(dtype).view(N, S, C), "d_weight": d_weight.to(dtype), "d_bias": d_bias.to(dtype)}


def _dropout(s):
    n, p = s["case"]["n"], s["case"]["p"]
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=DEVICE) + s["offset"]
    c0, c1, c2, c3 = block & low, block >> 32, torch.zeros_like(block), torch.zeros_like(block)
    k0, k1 = s["seed"] & low, s["seed"] >> 32
    for _ in range(10):
        # Products wrap at 64 bits; their two halves are read off the pattern.
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    keep = torch.stack([c0, c1, c2, c3], 1).view(-1)[:n] >= round(p * 2.0 ** 32)
    y = torch.where(keep, s["x"].float() * (1 / (1 - p)), 0.0)
    if s["residual"] is not None:
        y = s["residual"].float() + y
    return y.to(s["x"].dtype)


_PLAIN = {"recurrence": _recurrence, "recurrence_backward": _recurrence_backward, "norm": _norm, "norm_backward": _norm_backward,
          "dropout": _dropout}


# ---- the framework's calls -------------------------------------------------------------------------------------------

_context = None


def _plan(s):
    """What a program that makes these calls keeps beside its tensors: the context, their descriptions, a workspace."""
    global _context
    from ctypes import byref, c_int64
    from homura_amd import capi
    if _context is None:
        _context = capi.Context(0)
    code = {torch.bfloat16: capi.BF16, torch.float16: capi.F16, torch.float32: capi.F32, torch.int32: capi.I32}
    s["call"], s["ctx"] = capi.nn, _context.handle
    d = s["descs"] = {k: byref(capi.make_desc(t.data_ptr(), code[t.dtype], t.shape, t.stride()))
                      for k, t in s.items() if isinstance(t, torch.Tensor)}
    for k in ("lengths", "residual"):
        d.setdefault(k, None)
    need, case = c_int64(0), s["case"]
    if case["op"].startswith("recurrence"):
        s["code"] = {"factor": capi.GATE_FACTOR, "sigmoid": capi.GATE_SIGMOID}[case["form"]]
        capi.check_nn(capi.nn.hmn_recurrence_workspace(d["gate"], byref(need)))
    elif case["op"].startswith("norm"):
        s["code"] = capi.ACTIVATION[case["act"]]
        capi.check_nn(capi.nn.hmn_group_norm_workspace(d["x"], case["G"], case["op"] == "norm_backward", byref(need)))
    s["workspace"] = torch.empty(max(1, need.value), device=DEVICE, dtype=torch.uint8)
    s["room"] = (s["workspace"].data_ptr(), need.value)
    s["check"] = capi.check_nn
    torch.cuda.synchronize()  # the context has a stream of its own


def _own_recurrence(s):
    d = s["descs"]
    s["check"](s["call"].hmn_recurrence(s["ctx"], s["code"], d["out"], d["last"], d["gate"], d["input"], d["initial"], d["lengths"],
                                        *s["room"]))
    return {"out": s["out"], "last": s["last"]}


def _own_recurrence_backward(s):
    d = s["descs"]
    s["check"](s["call"].hmn_recurrence_backward(s["ctx"], s["code"], d["d_gate"], d["d_input"], d["d_initial"], d["grad"],
                                                 d["grad_last"], d["gate"], d["input"], d["out"], d["initial"], d["lengths"],
                                                 *s["room"]))
    return {"d_gate": s["d_gate"], "d_input": s["d_input"], "d_initial": s["d_initial"]}


def _own_norm(s):
    d = s["descs"]
    s["check"](s["call"].hmn_group_norm(s["ctx"], d["out"], d["mean"], d["rstd"], d["x"], d["weight"], d["bias"], s["case"]["G"],
                                        s["eps"], s["code"], *s["room"]))
    return {"out": s["out"], "mean": s["mean"], "rstd": s["rstd"]}


def _own_norm_backward(s):
    d = s["descs"]
    s["check"](s["call"].hmn_group_norm_backward(s["ctx"], d["d_x"], d["d_weight"], d["d_bias"], d["grad"], d["x"], d["mean"],
                                                 d["rstd"], d["weight"], d["bias"], s["case"]["G"], s["code"], *s["room"]))
    return {"d_x": s["d_x"], "d_weight": s["d_weight"], "d_bias": s["d_bias"]}


def _own_dropout(s):
    d = s["descs"]
    s["check"](s["call"].hmn_dropout(s["ctx"], d["out"], d["x"], d["residual"], s["case"]["p"], s["seed"], s["offset"], None))
    return s["out"]


_OWN = {"recurrence": _own_recurrence, "recurrence_backward": _own_recurrence_backward, "norm": _own_norm,
        "norm_backward": _own_norm_backward, "dropout": _own_dropout}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: t.double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for k, t in s.items()}
    op = case["op"]
    if op == "dropout":
        return _exact_dropout(wide)
    return {"recurrence": _exact_recurrence, "recurrence_backward": _exact_recurrence_backward, "norm": _exact_norm,
            "norm_backward": _exact_norm_backward}[op](wide)


def _exact_recurrence(s):
    """Step by step, as the recurrence is written."""
    T, sigmoid = s["case"]["T"], s["case"]["form"] == "sigmoid"
    lengths = torch.full((s["case"]["B"],), T, device=DEVICE) if s["lengths"] is None else s["lengths"]
    h, out = s["initial"], torch.zeros_like(s["input"])
    for t in range(T):
        a, x = s["gate"][:, t], s["input"][:, t]
        if sigmoid:
            a = torch.sigmoid(a)
            x = (1 - a) * x
        going = (t < lengths)[:, None]
        h = torch.where(going, a * h + x, h)
        out[:, t] = torch.where(going, h, 0.0)
    return {"out": out, "last": h}


def _exact_recurrence_backward(s):
    """The chain rule, from the last step to the first."""
    T, sigmoid = s["case"]["T"], s["case"]["form"] == "sigmoid"
    lengths = torch.full((s["case"]["B"],), T, device=DEVICE) if s["lengths"] is None else s["lengths"]
    d_h = s["grad_last"]
    d_gate, d_input = torch.zeros_like(s["gate"]), torch.zeros_like(s["gate"])
    for t in range(T - 1, -1, -1):
        a, x = s["gate"][:, t], s["input"][:, t]
        before = s["out"][:, t - 1] if t else s["initial"]
        going = (t < lengths)[:, None]
        g = torch.where(going, d_h + s["grad"][:, t], 0.0)
        if sigmoid:
            a = torch.sigmoid(a)
            d_input[:, t] = (1 - a) * g
            d_gate[:, t] = g * (before - x) * a * (1 - a)
        else:
            d_input[:, t] = g
            d_gate[:, t] = g * before
        d_h = torch.where(going, a * g, d_h)
    return {"d_gate": d_gate, "d_input": d_input, "d_initial": d_h}


def _exact_normalised(s):
    N, S, C, G = (s["case"][k] for k in "NSCG")
    rows = s["x"].reshape(N, S, G, C // G).transpose(1, 2).reshape(N * G, -1)
    return rows, lambda r: r.reshape(N, G, S, C // G).transpose(1, 2).reshape(N, S, C)


def _exact_norm(s):
    rows, back = _exact_normalised(s)
    mean = rows.mean(1, keepdim=True)
    rstd = (rows.var(1, unbiased=False, keepdim=True) + s["eps"]).rsqrt()
    z = back((rows - mean) * rstd) * s["weight"] + s["bias"]
    shape = (s["case"]["N"], s["case"]["G"])
    act = {"none": lambda z: z, "relu": torch.relu, "silu": lambda z: z * torch.sigmoid(z),
           "gelu": lambda z: z * (0.5 * torch.erfc(-z * 0.5 ** 0.5)),
           "gelu_tanh": lambda z: z * torch.sigmoid(2 * _ROOT2PI * (z + 0.044715 * z ** 3))}[s["case"]["act"]]
    return {"out": act(z), "mean": mean.view(shape), "rstd": rstd.view(shape)}


def _exact_norm_backward(s):
    N, S, C, G = (s["case"][k] for k in "NSCG")
    rows, back = _exact_normalised(s)
    hat = back((rows - s["mean"].view(-1, 1)) * s["rstd"].view(-1, 1))
    z = hat * s["weight"] + s["bias"]
    if s["case"]["act"] == "silu":
        q = torch.sigmoid(z)
        slope = q + z * q * (1 - q)
    elif s["case"]["act"] == "gelu":
        slope = 0.5 * torch.erfc(-z * 0.5 ** 0.5) + z * torch.exp(-z * z / 2) / 6.283185307179586 ** 0.5
    elif s["case"]["act"] == "gelu_tanh":
        q = torch.sigmoid(2 * _ROOT2PI * (z + 0.044715 * z ** 3))
        slope = q + z * q * (1 - q) * 2 * _ROOT2PI * (1 + 3 * 0.044715 * z ** 2)
    else:
        slope = (z > 0).double() if s["case"]["act"] == "relu" else torch.ones_like(z)
    dz = s["grad"] * slope
    by_group = lambda v: (v.view(N, S, G, -1).sum((1, 3)) / (S * (C // G))).repeat_interleave(C // G, 1)[:, None]  # noqa: E731
    wdz = dz * s["weight"]
    d_x = s["rstd"].repeat_interleave(C // G, 1)[:, None] * (wdz - by_group(wdz) - hat * by_group(wdz * hat))
    return {"d_x": d_x, "d_weight": (dz * hat).sum((0, 1)), "d_bias": dz.sum((0, 1))}


def _exact_dropout(s):
    """The generator with its 32-bit products taken apart into 16-bit limbs, every step below 2^63."""
    n, p, mask = s["case"]["n"], s["case"]["p"], (1 << 32) - 1

    def product(m, c):
        low, high = m * (c & 0xFFFF), m * (c >> 16)  # below 2^48 each
        carry = (low >> 16) + high
        return carry >> 16, ((carry & 0xFFFF) << 16) | (low & 0xFFFF)

    at = s["offset"] + torch.arange(-(-n // 4), device=DEVICE)
    words = [torch.remainder(at, 1 << 32), torch.div(at, 1 << 32, rounding_mode="floor"), at * 0, at * 0]
    for i in range(10):
        key = [((s["seed"] & mask) + i * 0x9E3779B9) & mask, ((s["seed"] >> 32) + i * 0xBB67AE85) & mask]
        (h0, l0), (h1, l1) = product(0xD2511F53, words[0]), product(0xCD9E8D57, words[2])
        words = [h1 ^ words[1] ^ key[0], l1, h0 ^ words[3] ^ key[1], l0]
    uniform = torch.stack(words, 1).flatten()[:n].double() / 2.0 ** 32
    y = (uniform >= round(p * 2.0 ** 32) / 2.0 ** 32).double() * s["x"] / (1 - p)
    return y if s["residual"] is None else y + s["residual"]
