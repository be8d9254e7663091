"""The language-model operators of this framework as cases that can be timed and compared.

Three operators make one recurrent block: a gated linear recurrence over time (swiftrt_b200.gated_recurrence and its
backward), a gated Dense layer (swiftrt_b200.GatedDense: forward, forward that keeps, backward) and products with 4-bit
weights (swiftrt_b200.matmul_int4, and GatedDense over two such weights).

`run` computes a case in its plain form -- elementary torch operations in 32 bits, rounded once at the end -- or, where
`own` is true, through the framework's entry points.  `exact` gives the definition in 64 bits, step by step.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
CHUNK = 64          # steps between two kept states of the recurrence


# ------------------------------------------------------------------------------------------------ cases
def _recurrence(name, B, T, D, dtype="bf16", gate_in=False, gate_out=True, initial=True, ragged=False, keep=False, backward=False):
    c = {"op": "recurrence", "B": B, "T": T, "D": D, "dtype": dtype, "gate_in": gate_in, "gate_out": gate_out, "initial": initial,
         "ragged": ragged, "keep": keep, "backward": backward}
    return {"name": name, **c} if name else c


def _gated(name, M, K, H, dtype="bf16", act="silu", bias=False, mode="forward"):
    c = {"op": "gated", "M": M, "K": K, "H": H, "dtype": dtype, "act": act, "bias": bias, "mode": mode}
    return {"name": name, **c} if name else c


def _int4(name, M, K, N, G=128, dtype="bf16", zeros=False, act="identity", bias=False, gated=False):
    c = {"op": "int4", "M": M, "K": K, "N": N, "G": G, "dtype": dtype, "zeros": zeros, "act": act, "bias": bias, "gated": gated}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one generated token for each of 16 requests: the state of every channel moves one step
        _recurrence("recurrence_token", 16, 1, 2048),
        # the prompt of a single request, of odd length: all parallelism has to come from channels and time
        _recurrence("recurrence_prompt", 1, 8191, 4096),
        # forward of a training step over a padded batch, with the states that the backward pass needs
        _recurrence("recurrence_train", 8, 2048, 4096, ragged=True, keep=True),
        # Float32 with separate input gates, no output gate and a channel count that nothing divides
        _recurrence("recurrence_fp32_odd", 3, 1025, 1001, dtype="fp32", gate_in=True, gate_out=False),
        # backward of the training step
        _recurrence("recurrence_grad", 8, 2048, 4096, keep=True, backward=True),
        # backward with every gate in fp16 over short padded sequences
        _recurrence("recurrence_grad_ragged", 5, 777, 1530, dtype="fp16", gate_in=True, ragged=True, keep=True, backward=True),
        # one token through both projections: bound by reading the weights
        _gated("gated_token", 1, 4096, 16384),
        # forward of a training step, keeping what the backward pass needs
        _gated("gated_train", 4096, 4096, 16384, mode="keep"),
        # backward of a training step with biases and ragged sizes
        _gated("gated_grad", 3999, 4096, 8200, bias=True, mode="backward"),
        # one token through a 4-bit layer
        _int4("int4_token", 1, 4096, 16384),
        # a small serving batch in fp16 with zero points, short groups and sizes off every tile
        _int4("int4_batch_odd", 17, 4104, 1001, G=32, dtype="fp16", zeros=True, act="gelu", bias=True),
        # four tokens through a gated block held in 4 bits
        _int4("int4_gated_tokens", 4, 4096, 16384, act="silu", gated=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("recurrence", "recurrence", "gated", "gated", "int4"))
    if op == "recurrence":
        backward = rng.random() < 0.4
        B, D = _log(rng, 1, 16), _log(rng, 64, 4096)
        T = _log(rng, 1, 8192)
        while B * T * D > 8 * 2048 * 4096:
            T = max(1, T // 2)
        return _recurrence(None, B, T, D, rng.choice(("bf16", "bf16", "fp16", "fp32")), rng.random() < 0.4, rng.random() < 0.6,
                           rng.random() < 0.7, rng.random() < 0.5, backward or rng.random() < 0.3, backward)
    if op == "gated":
        mode = rng.choice(("forward", "forward", "keep", "backward"))
        # rows of whole 16-byte units, as a model's widths are; any number of tokens
        M, K, H = _log(rng, 1, 4096), 8 * _log(rng, 32, 512), 8 * _log(rng, 32, 2048)
        if mode == "backward":
            M, H = max(2, M // 2), min(H, 8192)
        return _gated(None, M, K, H, rng.choice(("bf16", "bf16", "fp16")), rng.choice(("silu", "gelu", "geluTanh", "sigmoid", "relu")),
                      rng.random() < 0.5, mode)
    return _int4(None, _log(rng, 1, 48), _log(rng, 64, 8192), _log(rng, 64, 16384), rng.choice((32, 64, 128)), rng.choice(("bf16", "fp16")),
                 rng.random() < 0.5, rng.choice(("identity", "relu", "silu")), rng.random() < 0.5, rng.random() < 0.3)


def work(case):
    c, e = case, SIZE[case["dtype"]]
    if c["op"] == "recurrence":
        n, bd = c["B"] * c["T"] * c["D"], c["B"] * c["D"]
        inputs = 2 + c["gate_in"] + c["gate_out"]
        kept = 4 * c["B"] * -(-c["T"] // CHUNK) * c["D"] if c["keep"] else 0
        if c["backward"]:
            return {"bytes": n * e * (2 * inputs + 1) + kept + 8 * bd, "flops": n * (24 + 8 * (inputs - 2))}
        return {"bytes": n * e * (inputs + 1) + kept + 4 * bd * (1 + c["initial"]), "flops": n * (8 + 5 * (inputs - 2))}
    if c["op"] == "gated":
        x, w, h = c["M"] * c["K"], c["K"] * c["H"], c["M"] * c["H"]
        if c["mode"] == "backward":
            return {"bytes": e * (2 * x + 4 * w + 3 * h + 2 * c["H"] * c["bias"]), "flops": 8 * c["M"] * c["K"] * c["H"]}
        return {"bytes": e * (x + 2 * w + h * (3 if c["mode"] == "keep" else 1) + 2 * c["H"] * c["bias"]), "flops": 4 * c["M"] * c["K"] * c["H"]}
    two = 2 if c["gated"] else 1
    groups = -(-c["K"] // c["G"])
    weight = 4 * -(-c["K"] // 8) * c["N"] + groups * c["N"] * (e + c["zeros"])
    return {"bytes": two * (weight + e * c["N"] * c["bias"]) + e * c["M"] * (c["K"] + c["N"]), "flops": 2 * two * c["M"] * c["K"] * c["N"]}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, mean=0.0, dtype=dt):
        return (torch.randn(shape, generator=g, device=DEVICE) * scale + mean).to(dtype)

    s = {"case": case}
    if case["op"] == "recurrence":
        B, T, D = case["B"], case["T"], case["D"]
        s["update"] = normal(B, T, D)
        s["forget"] = normal(B, T, D, scale=1.5, mean=2.5)          # memories from a few to hundreds of steps
        s["input"] = normal(B, T, D) if case["gate_in"] else None
        s["output"] = normal(B, T, D) if case["gate_out"] else None
        s["initial"] = normal(B, D, dtype=torch.float32) if case["initial"] else None
        s["lengths"] = None
        if case["ragged"]:
            n = torch.randint(0, T + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32)
            n[0] = T
            s["lengths"] = n
        if case["backward"]:
            s["out_grad"] = normal(B, T, D)
            s["last_grad"] = normal(B, D, dtype=torch.float32)
            s["states"] = _plain_states(*_plain_gates(s), s["initial"])[1]
    elif case["op"] == "gated":
        M, K, H = case["M"], case["K"], case["H"]
        s["x"] = normal(M, K)
        s["w_gate"], s["w_up"] = normal(K, H, scale=K ** -0.5), normal(K, H, scale=K ** -0.5)
        s["b_gate"], s["b_up"] = (normal(H, scale=0.5), normal(H, scale=0.5)) if case["bias"] else (None, None)
        if case["mode"] == "backward":
            s["gate"], s["up"], s["out_grad"] = normal(M, H), normal(M, H), normal(M, H)
    else:
        M, K, N, G = case["M"], case["K"], case["N"], case["G"]
        s["x"] = normal(M, K)
        s["w"] = []
        for _ in range(2 if case["gated"] else 1):
            packed = torch.randint(-2 ** 31, 2 ** 31, (-(-K // 8), N), generator=g, device=DEVICE, dtype=torch.int64).to(torch.int32)
            # a normal weight of variance 1 / K spans about six deviations over the sixteen values of its group
            scales = ((0.5 + torch.rand((-(-K // G), N), generator=g, device=DEVICE)) * (0.4 * K ** -0.5)).to(dt)
            zeros = torch.randint(5, 11, (-(-K // G), N), generator=g, device=DEVICE, dtype=torch.int32).to(torch.uint8) if case["zeros"] else None
            bias = normal(N, scale=0.5) if case["bias"] else None
            s["w"].append((packed, scales, zeros, bias))
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _act(name, z):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    if name == "relu":
        return torch.where(z >= 0, z, torch.zeros_like(z))
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if name == "geluTanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    return z


def _act_slope(name, z):
    if name == "silu":
        s = torch.sigmoid(z)
        return s * (1 + z * (1 - s))
    if name == "sigmoid":
        s = torch.sigmoid(z)
        return s * (1 - s)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    if name == "geluTanh":
        a = (2 / math.pi) ** 0.5
        t = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * a * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _live(s):
    """[B, T, 1] of 1 where a step belongs to its sequence, or None."""
    if s["lengths"] is None:
        return None
    T = s["update"].shape[1]
    return (torch.arange(T, device=DEVICE)[None, :] < s["lengths"][:, None])[:, :, None]


def _plain_gates(s):
    """(f, i x) of every step in 32 bits; a step behind its sequence keeps the state."""
    a, x, live = s["forget"].float(), s["update"].float(), _live(s)
    f = torch.sigmoid(a)
    b = (torch.sigmoid(-a) if s["input"] is None else torch.sigmoid(s["input"].float())) * x
    if live is not None:
        f, b = torch.where(live, f, torch.ones_like(f)), torch.where(live, b, torch.zeros_like(b))
    return f, b


def _scan(f, b):
    """c_t = f_t c_{t-1} + b_t along dim 1 with c_{-1} = 0, by doubling spans: (products of f, c)."""
    T, span = f.shape[1], 1
    while span < T:
        b = torch.cat((b[:, :span], f[:, span:] * b[:, :-span] + b[:, span:]), 1)
        f = torch.cat((f[:, :span], f[:, span:] * f[:, :-span]), 1)
        span *= 2
    return f, b


def _plain_states(f, b, initial):
    """Every c_t, and the kept c before steps 0, CHUNK, 2 CHUNK, ..."""
    first = torch.zeros_like(f[:, 0]) if initial is None else initial
    p, c = _scan(f, b)
    c = c + p * first[:, None]
    return c, torch.cat((first[:, None], c[:, CHUNK - 1:-1:CHUNK]), 1).contiguous()


def _plain_recurrence(s):
    case, dt, live = s["case"], s["update"].dtype, _live(s)
    f, b = _plain_gates(s)
    c, states = _plain_states(f, b, s["initial"])
    if not case["backward"]:
        y = c if s["output"] is None else c * torch.sigmoid(s["output"].float())
        y = y if live is None else torch.where(live, y, torch.zeros_like(y))
        out = {"hidden": y.to(dt), "last": c[:, -1].contiguous()}
        return {**out, "states": states} if case["keep"] else out
    x, dy = s["update"].float(), s["out_grad"].float()
    dy = dy if live is None else torch.where(live, dy, torch.zeros_like(dy))
    o = None if s["output"] is None else torch.sigmoid(s["output"].float())
    # dc_t = p_t + f_{t+1} dc_{t+1}: the scan from the other end, with f moved by one step; behind a sequence f is 1 and p is 0
    p = dy if o is None else dy * o
    p = torch.cat((p[:, :-1], p[:, -1:] + s["last_grad"][:, None]), 1)
    dc = _scan(torch.cat((torch.ones_like(f[:, :1]), f[:, 1:].flip(1)), 1), p.flip(1))[1].flip(1)
    before = torch.cat((states[:, :1], c[:, :-1]), 1)
    nf = torch.sigmoid(-s["forget"].float())
    zero = (lambda v: v.to(dt)) if live is None else (lambda v: torch.where(live, v, torch.zeros_like(v)).to(dt))
    out = {"initial": (f[:, 0] * dc[:, 0]).contiguous()}
    if s["input"] is None:
        out["update"], out["forget"] = zero(dc * nf), zero(dc * (before - x) * f * nf)
    else:
        i = torch.sigmoid(s["input"].float())
        out["update"], out["forget"] = zero(dc * i), zero(dc * before * f * nf)
        out["input"] = zero(dc * x * i * torch.sigmoid(-s["input"].float()))
    if o is not None:
        out["output"] = zero(dy * c * o * torch.sigmoid(-s["output"].float()))
    return out


def _plain_gated(s):
    case, dt = s["case"], s["x"].dtype
    x, wg, wu = s["x"].float(), s["w_gate"].float(), s["w_up"].float()
    if case["mode"] == "backward":
        g, u, dy = s["gate"].float(), s["up"].float(), s["out_grad"].float()
        dg, du = dy * u * _act_slope(case["act"], g), dy * _act(case["act"], g)
        out = {"x": (dg @ wg.t() + du @ wu.t()).to(dt), "w_gate": (x.t() @ dg).to(dt), "w_up": (x.t() @ du).to(dt)}
        if case["bias"]:
            out["b_gate"], out["b_up"] = dg.double().sum(0).to(dt), du.double().sum(0).to(dt)
        return out
    g, u = x @ wg, x @ wu
    if case["bias"]:
        g, u = g + s["b_gate"].float(), u + s["b_up"].float()
    y = (_act(case["act"], g) * u).to(dt)
    return {"y": y, "gate": g.to(dt), "up": u.to(dt)} if case["mode"] == "keep" else y


def _plain_weight(packed, scales, zeros, K, G):
    shifts = torch.arange(0, 32, 4, device=DEVICE, dtype=torch.int32)
    q = ((packed[:, None, :] >> shifts[None, :, None]) & 15).reshape(-1, packed.shape[1])[:K].float()
    group = torch.arange(K, device=DEVICE) // G
    z = 8.0 if zeros is None else zeros.float()[group]
    return (q - z) * scales.float()[group]


def _plain_int4(s):
    case, x = s["case"], s["x"].float()
    z = [x @ _plain_weight(p, sc, ze, case["K"], case["G"]) + (0 if b is None else b.float()) for p, sc, ze, b in s["w"]]
    y = _act(case["act"], z[0])
    return (y * z[1] if case["gated"] else y).to(s["x"].dtype)


# ------------------------------------------------------------------------------------------------ one pass
def _own(s):
    import swiftrt_b200 as srt
    case = s["case"]
    if case["op"] == "recurrence":
        if not case["backward"]:
            out = srt.gated_recurrence(s["update"], s["forget"], s["input"], s["output"], s["initial"], s["lengths"], keep=case["keep"])
            return dict(zip(("hidden", "last", "states"), out))
        out = srt.gated_recurrence_backward(s["out_grad"], s["update"], s["forget"], s["input"], s["output"], s["states"], s["lengths"],
                                            last_grad=s["last_grad"])
        return {k: v for k, v in zip(("update", "forget", "input", "output", "initial"), out) if v is not None}
    layer = s.get("layer")
    if case["op"] == "gated":
        if layer is None:
            layer = s["layer"] = srt.GatedDense(s["w_gate"], s["w_up"], s["b_gate"], s["b_up"], srt.ActivationType[case["act"]])
        if case["mode"] == "forward":
            return layer(s["x"])
        if case["mode"] == "keep":
            y, (gate, up) = layer.forward_keep(s["x"])
            return {"y": y, "gate": gate, "up": up}
        out = layer.backward(s["x"], (s["gate"], s["up"]), s["out_grad"])
        return {k: v for k, v in zip(("x", "w_gate", "w_up", "b_gate", "b_up"), out) if v is not None}
    if layer is None:
        w = [srt.Int4Weight(p, sc, ze, case["G"], case["K"]) for p, sc, ze, _ in s["w"]]
        b = [t[3] for t in s["w"]]
        act = srt.ActivationType[case["act"]]
        layer = s["layer"] = srt.GatedDense(w[0], w[1], b[0], b[1], act) if case["gated"] else srt.Dense(w[0], b[0], act)
    return layer(s["x"])


def run(state):
    if own:
        return _own(state)
    return {"recurrence": _plain_recurrence, "gated": _plain_gated, "int4": _plain_int4}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _logistic(z):
    return 1 / (1 + torch.exp(-z))


def _exact_act(name, z):
    """(value, derivative)"""
    if name == "silu":
        e = _logistic(z)
        return z * e, e + z * e * (1 - e)
    if name == "sigmoid":
        e = _logistic(z)
        return e, e * (1 - e)
    if name == "relu":
        return z.clamp_min(0), (z > 0).double()
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * phi, phi + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "geluTanh":
        a, c = math.sqrt(2 / math.pi), 0.044715
        e = _logistic(2 * a * (z + c * z ** 3))          # (1 + tanh v) / 2 = logistic(2 v)
        return z * e, e + z * e * (1 - e) * 2 * a * (1 + 3 * c * z * z)
    return z, torch.ones_like(z)


def _exact_recurrence(s):
    case = s["case"]
    B, T, D = case["B"], case["T"], case["D"]
    if 8 * B * T * D * 9 > 60e9 or T > 20000:
        return None
    n = torch.full((B,), T, device=DEVICE) if s["lengths"] is None else s["lengths"].long()
    c = torch.zeros(B, D, dtype=torch.float64, device=DEVICE) if s["initial"] is None else s["initial"].double()
    x = s["update"].double()
    f = _logistic(s["forget"].double())
    i = 1 - f if s["input"] is None else _logistic(s["input"].double())
    o = torch.ones((), dtype=torch.float64, device=DEVICE).expand(B, T, D) if s["output"] is None else _logistic(s["output"].double())
    trace = torch.empty(B, T + 1, D, dtype=torch.float64, device=DEVICE)
    trace[:, 0] = c
    for t in range(T):
        c = torch.where((t < n)[:, None], f[:, t] * c + i[:, t] * x[:, t], c)
        trace[:, t + 1] = c
    on = (torch.arange(T, device=DEVICE)[None] < n[:, None])[:, :, None].double()
    if not case["backward"]:
        out = {"hidden": trace[:, 1:] * o * on, "last": c}
        if case["keep"]:
            out["states"] = trace[:, :T:CHUNK]
        return out
    dy = s["out_grad"].double() * on
    dc_all, e = torch.empty_like(x), s["last_grad"].double()
    for t in range(T - 1, -1, -1):
        now = (t < n)[:, None]
        dc = dy[:, t] * o[:, t] + e
        dc_all[:, t] = torch.where(now, dc, torch.zeros_like(dc))
        e = torch.where(now, dc * f[:, t], e)
    before, after = trace[:, :-1], trace[:, 1:]
    out = {"initial": e, "update": dc_all * i}
    if s["input"] is None:
        out["forget"] = dc_all * (before - x) * f * (1 - f)
    else:
        out["forget"], out["input"] = dc_all * before * f * (1 - f), dc_all * x * i * (1 - i)
    if s["output"] is not None:
        out["output"] = dy * after * o * (1 - o)
    return out


def _exact_gated(s):
    case = s["case"]
    x, wg, wu = s["x"].double(), s["w_gate"].double(), s["w_up"].double()
    if case["mode"] == "backward":
        a, slope = _exact_act(case["act"], s["gate"].double())
        dy = s["out_grad"].double()
        du = dy * a
        dg = dy * s["up"].double() * slope
        out = {"x": torch.mm(dg, wg.t()).addmm_(du, wu.t()), "w_gate": torch.mm(x.t(), dg), "w_up": torch.mm(x.t(), du)}
        if case["bias"]:
            out["b_gate"], out["b_up"] = dg.sum(0), du.sum(0)
        return out
    g, u = torch.mm(x, wg), torch.mm(x, wu)
    if case["bias"]:
        g += s["b_gate"].double()
        u += s["b_up"].double()
    y = _exact_act(case["act"], g)[0] * u
    return {"y": y, "gate": g, "up": u} if case["mode"] == "keep" else y


def _exact_int4(s):
    case, x = s["case"], s["x"].double()
    K, G = case["K"], case["G"]
    z = []
    for packed, scales, zeros, bias in s["w"]:
        acc = torch.zeros(case["M"], case["N"], dtype=torch.float64, device=DEVICE)
        words = packed.long()
        for r in range(8):                                   # rows r, r + 8, r + 16, ... of the weight
            rows = torch.arange(r, K, 8, device=DEVICE)
            q = (words[: rows.numel()] // 16 ** r) % 16 if r else words[: rows.numel()] % 16
            q = q.double() - (8 if zeros is None else zeros.double()[rows // G])
            acc += x[:, rows] @ (q * scales.double()[rows // G])
        z.append(acc if bias is None else acc + bias.double())
    y = _exact_act(case["act"], z[0])[0]
    return y * z[1] if case["gated"] else y


def exact(case, seed):
    s = prepare(case, seed)
    return {"recurrence": _exact_recurrence, "gated": _exact_gated, "int4": _exact_int4}[case["op"]](s)
