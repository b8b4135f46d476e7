"""Operators of a gated recurrent token mixer and of its training with activations kept in 8 bits, as timed cases.

Four operators of one block, whose gates come from the tokens alone and whose training keeps codes in place of activations:

``scan``     the gated linear recurrence over prompts, over single tokens, and with its gradients
``keep``     an activation as 8-bit codes with a power of two for each 32 elements of a row, and the values that these stand for
``product``  the product of an activated gate with its partner, forward and backward; the backward pass starts from kept codes
``weights``  the gradient of a weight from the gradient of its products and the kept codes of its input

``listed()`` names fixed cases, ``draw()`` gives further ones of the same ranges.  With ``own`` false the operators run as
elementary torch operations in 32 bits, with ``own`` true through the public entry points of this framework.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 32   # elements of a row that share a power of two
LOWEST = {torch.float32: -126, torch.bfloat16: -126, torch.float16: -24}   # least exponents of kept codes


def listed():
    return [
        # one token for each of sixteen streams: latency
        dict(name="scan_token", kind="scan_step", batch=16, width=1024, input=False, activation="none", type="bf16"),
        # a batch of prompts
        dict(name="scan_prompt", kind="scan", batch=8, tokens=4096, width=2048, input=False, activation="none", ragged=False, state=False, type="bf16"),
        # one long recording continued from a state: the axis of time has to be split
        dict(name="scan_long", kind="scan", batch=1, tokens=65536, width=512, input=False, activation="none", ragged=False, state=True, type="fp16"),
        # a training step over full sequences
        dict(name="scan_train", kind="scan_train", batch=8, tokens=2048, width=2048, input=False, activation="none", ragged=False, state=False, type="bf16"),
        # a training step in full precision over utterances of several lengths, with a gate of its own for what comes in, a width that nothing divides
        dict(name="scan_train_ragged", kind="scan_train", batch=6, tokens=1000, width=1001, input=True, activation="tanh", ragged=True, state=True, type="fp32"),
        # an activation of a batch of sequences, kept for the backward pass, and what the backward pass reads of it
        dict(name="keep_batch", kind="keep", rows=16384, width=4096, type="bf16"),
        # a few rows of a width that no group divides, in full precision
        dict(name="keep_ragged", kind="keep", rows=333, width=1001, type="fp32"),
        # the hidden half of a block over a batch of sequences
        dict(name="product_train", kind="product", rows=16384, width=4096, activation="silu", type="bf16"),
        # the same over a few sequences, in full precision, rows and width that nothing divides
        dict(name="product_train_ragged", kind="product", rows=1203, width=1001, activation="gelu", type="fp32"),
        # the gradient of a projection over a batch of sequences
        dict(name="weights_train", kind="weights", tokens=16384, inner=4096, outer=4096, type="bf16", out="bf16"),
        # a small weight over a long batch: the axis of the tokens has to be split; the gradient goes to weights in full precision
        dict(name="weights_long", kind="weights", tokens=65536, inner=512, outer=512, type="fp16", out="fp32"),
        # full precision and sizes that no tile divides
        dict(name="weights_ragged", kind="weights", tokens=1000, inner=777, outer=1100, type="fp32", out="fp32"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _width(rng, low, high):
    """A width: two of three are multiples of 64, as networks mostly have them, the others any number."""
    n = _log(rng, low, high)
    return n if rng.random() < 1 / 3 else min(high, max(64, (n + 32) // 64 * 64))


def draw(rng):
    kind = rng.choice(("scan_step", "scan", "scan", "scan_train", "scan_train", "keep", "product", "weights", "weights"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if kind.startswith("scan"):
        width = _width(rng, 64, 4096)
        case = dict(kind=kind, width=width, input=rng.random() < 0.4, activation=rng.choice(("none", "none", "tanh")), type=dtype)
        if kind == "scan_step":
            return dict(case, batch=_log(rng, 1, 256))
        most = (1 << 24) if kind == "scan_train" else (1 << 25)
        tokens = _log(rng, 1, min(65536, most // width))
        return dict(case, batch=_log(rng, 1, max(1, min(64, most // (tokens * width)))), tokens=tokens, ragged=rng.random() < 0.4, state=rng.random() < 0.5)
    if kind == "weights":
        inner, outer = _width(rng, 64, 8192), _width(rng, 64, 8192)
        tokens = _log(rng, 1, max(1, min(65536, (1 << 37) // (inner * outer * (4 if dtype == "fp32" else 1)))))
        return dict(kind=kind, tokens=tokens, inner=inner, outer=outer, type=dtype, out=rng.choice((dtype, "fp32")))
    width = _width(rng, 64, 8192)
    rows = _log(rng, 1, min(16384, (32 << 20) // width))
    case = dict(kind=kind, rows=rows, width=width, type=dtype)
    return case if kind == "keep" else dict(case, activation=rng.choice(("none", "relu", "silu", "gelu")))


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    s = dict(case=case)
    if kind.startswith("scan"):
        B, T, D = case["batch"], case.get("tokens", 1), case["width"]
        # one projection's result, split into the gates and the values
        joint = torch.randn((B, T, D * (3 if case["input"] else 2)), generator=g, device=DEVICE)
        # memories of two tokens to some hundred, spread over the channels
        joint[..., :D] += torch.linspace(0, 6, D, device=DEVICE)
        parts = joint.to(dtype).split(D, dim=-1)
        s["forget"], s["value"], s["input"] = parts[0], parts[1], parts[2] if case["input"] else None
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32) if case.get("ragged") else None
        s["state"] = _normal(g, (B, D), torch.float32) if kind == "scan_step" or case["state"] else None
        if kind == "scan_step":
            for n in ("forget", "value", "input"):
                s[n] = None if s[n] is None else s[n][:, 0]
            s["new_state"] = torch.empty_like(s["state"])
        if kind == "scan_train":
            s["dout"] = _normal(g, (B, T, D), dtype)
            s["dfinal"] = _normal(g, (B, D), torch.float32) if case["state"] else None
            for n in ("forget", "value", "input", "state"):
                if s[n] is not None:
                    s[n] = s[n].detach().requires_grad_()
        return s
    # activations: some channels are larger than the others
    width = case["inner"] if kind == "weights" else case["width"]
    rows = case["tokens"] if kind == "weights" else case["rows"]
    spread = 1.0 + 8.0 * (torch.rand(width, generator=g, device=DEVICE) < 0.01)
    x = (torch.randn((rows, width), generator=g, device=DEVICE) * spread).to(dtype)
    if kind == "keep":
        s["x"] = x
    elif kind == "product":
        # gate and partner are the halves of one projection's result
        joint = torch.cat([x, _normal(g, (rows, width), dtype)], dim=1)
        s["gate"], s["up"] = (t.detach().requires_grad_() for t in joint.split(width, dim=1))
        s["dy"] = _normal(g, (rows, width), dtype)
    else:
        codes, s["exponents"] = _plain_keep(x.float(), LOWEST[dtype])
        # rows of codes start at multiples of 16 bytes, as the framework lays them out
        held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device=DEVICE)
        held[:, :width] = codes
        s["codes"] = held[:, :width]
        s["dy"] = _normal(g, (rows, case["outer"]), dtype)
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------

def _plain_scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1 from zero, and the products of a up to t: spans of twice the tokens each time."""
    a, b = a.clone(), b.clone()
    span = 1
    while span < a.shape[1]:
        b[:, span:] = b[:, span:] + a[:, span:] * b[:, :-span]
        a[:, span:] = a[:, span:] * a[:, :-span]
        span *= 2
    return a, b


def _plain_sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _plain_gates(s, step=False):
    """f, z and c of h = f h + z c, and who is a token."""
    forget, value = s["forget"].detach().float(), s["value"].detach().float()
    f = _plain_sigmoid(forget)
    z = _plain_sigmoid(-forget) if s["input"] is None else _plain_sigmoid(s["input"].detach().float())
    c = torch.tanh(value) if s["case"]["activation"] == "tanh" else value
    if step:
        return f, z, c, None
    T = f.shape[1]
    live = None
    if s["lengths"] is not None:
        live = (torch.arange(T, device=f.device)[None] < s["lengths"][:, None])[..., None]
        f, z, c = torch.where(live, f, 1.0), torch.where(live, z, 0.0), torch.where(live, c, 0.0)
    return f, z, c, live


def _plain_sequence(s):
    f, z, c, live = _plain_gates(s)
    a, h = _plain_scan(f, z * c)
    if s["state"] is not None:
        h = h + a * s["state"].detach()[:, None]
    return f, z, c, live, h


def _masked(x, live):
    return x if live is None else torch.where(live, x, 0.0)


def _plain_scan_train(s, dtype):
    f, z, c, live, h = _plain_sequence(s)
    start = torch.zeros_like(h[:, 0]) if s["state"] is None else s["state"].detach()
    before = torch.cat([start[:, None], h[:, :-1]], dim=1)
    dout = _masked(s["dout"].float(), live)
    # the gradient of h_t: what its output gives and what h_{t+1} hands back
    if s["dfinal"] is not None:
        dout = torch.cat([dout[:, :-1], dout[:, -1:] + s["dfinal"][:, None]], dim=1)
    later = torch.cat([torch.zeros_like(f[:, :1]), f[:, 1:].flip(1)], dim=1)
    _, g = _plain_scan(later, dout.flip(1))
    g = g.flip(1)
    held = before - c if s["input"] is None else before
    result = dict(out=_masked(h, live).to(dtype), final=h[:, -1].clone())
    result["dforget"] = _masked(g * held * f * _plain_sigmoid(-s["forget"].detach().float()), live).to(dtype)
    slope = 1 - c * c if s["case"]["activation"] == "tanh" else 1.0
    result["dvalue"] = _masked(g * z * slope, live).to(dtype)
    if s["input"] is not None:
        result["dinput"] = _masked(g * c * z * _plain_sigmoid(-s["input"].detach().float()), live).to(dtype)
    if s["state"] is not None:
        result["dstate"] = f[:, 0] * g[:, 0]
    return result


def _plain_keep(x, lowest):
    """Codes and exponents of rows: the least power of two with which a group's largest magnitude is at most 127."""
    rows, width = x.shape
    groups = -(-width // GROUP)
    held = torch.zeros(rows, groups * GROUP, device=x.device)
    held[:, :width] = x
    held = held.view(rows, groups, GROUP)
    mantissa, exponent = torch.frexp(held.abs().amax(dim=2))
    exponent = torch.where(mantissa == 0, torch.full_like(exponent, lowest), exponent - 7 + (mantissa > 127 / 128).int()).clamp(min=lowest)
    # two factors: the power of a tiny group's exponent is beyond 32 bits
    half = torch.div(-exponent, 2, rounding_mode="floor")
    scaled = torch.ldexp(torch.ldexp(held, half[..., None]), (-exponent - half)[..., None])
    return torch.round(scaled).to(torch.int8).view(rows, -1)[:, :width], exponent.to(torch.int8)


def _plain_values(codes, exponents):
    powers = torch.ldexp(torch.ones_like(exponents, dtype=torch.float32), exponents.int())
    return codes.float() * powers.repeat_interleave(GROUP, dim=1)[:, :codes.shape[1]]


def _plain_activation(x, name):
    """The activation and its slope."""
    if name == "relu":
        return torch.clamp(x, min=0), (x > 0).float()
    if name == "silu":
        s = _plain_sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(x * math.sqrt(0.5)))
        return x * p, p + x * torch.exp(-0.5 * x * x) / math.sqrt(2 * math.pi)
    return x, torch.ones_like(x)


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    dtype = TYPES[case["type"]]
    if kind == "scan_step":
        f, z, c, _ = _plain_gates(s, step=True)
        h = f * s["state"] + z * c
        return dict(out=h.to(dtype), state=h)
    if kind == "scan":
        *_, live, h = _plain_sequence(s)
        return dict(out=_masked(h, live).to(dtype), state=h[:, -1].clone())
    if kind == "scan_train":
        return _plain_scan_train(s, dtype)
    if kind == "keep":
        return _plain_values(*_plain_keep(s["x"].float(), LOWEST[dtype])).to(dtype)
    if kind == "product":
        gate, up, dy = s["gate"].detach().float(), s["up"].detach().float(), s["dy"].float()
        y = _plain_activation(gate, case["activation"])[0] * up
        kept_gate, kept_up = (_plain_values(*_plain_keep(t, LOWEST[dtype])) for t in (gate, up))
        value, slope = _plain_activation(kept_gate, case["activation"])
        return dict(y=y.to(dtype), dgate=(dy * kept_up * slope).to(dtype), dup=(dy * value).to(dtype))
    return (s["dy"].float().T @ _plain_values(s["codes"], s["exponents"])).to(TYPES[case["out"]])


# ---- the framework's operators ----------------------------------------------------------------------------------------------

def _run_own(s):
    from rx_met_b200 import gated_recurrence, kept_codes
    case, kind = s["case"], s["case"]["kind"]
    dtype = TYPES[case["type"]]
    if kind == "scan_step":
        out = gated_recurrence.gated_recurrence_step(s["forget"], s["value"], s["state"], input=s["input"], activation=case["activation"],
                                                     new_state=s["new_state"])
        return dict(out=out, state=s["new_state"])
    if kind == "keep":
        return kept_codes.values(kept_codes.keep(s["x"]))
    if kind == "product":
        y = kept_codes.gated_product(s["gate"], s["up"], activation=case["activation"])
        dgate, dup = torch.autograd.grad(y, [s["gate"], s["up"]], s["dy"])
        return dict(y=y.detach(), dgate=dgate, dup=dup)
    if kind == "weights":
        return kept_codes.weight_gradient(s["dy"], kept_codes.KeptCodes(s["codes"], s["exponents"], dtype), dtype=TYPES[case["out"]])
    out, final = gated_recurrence.gated_recurrence(s["forget"], s["value"], input=s["input"], activation=case["activation"], state=s["state"],
                                                   lengths=s["lengths"])
    if kind == "scan":
        return dict(out=out, state=final)
    names = [n for n in ("forget", "value", "input", "state") if s[n] is not None]
    ends, given = ([out], [s["dout"]]) if s["dfinal"] is None else ([out, final], [s["dout"], s["dfinal"]])
    grads = torch.autograd.grad(ends, [s[n] for n in names], given)
    return dict(dict(out=out.detach(), final=final.detach()), **{"d" + n: d for n, d in zip(names, grads)})


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    kind, size = case["kind"], 4 if case["type"] == "fp32" else 2
    if kind == "keep":      # x in, codes and exponents and the values out
        n = case["rows"] * case["width"]
        return {"bytes": n * (2 * size + 1) + case["rows"] * -(-case["width"] // GROUP), "flops": 5 * n}
    if kind == "product":   # gate, up and dy in, y and two gradients out
        n = case["rows"] * case["width"]
        return {"bytes": n * 6 * size, "flops": 20 * n}
    if kind == "weights":
        M, K, N = case["tokens"], case["inner"], case["outer"]
        return {"bytes": M * N * size + M * K + M * -(-K // GROUP) + N * K * (4 if case["out"] == "fp32" else 2), "flops": 2 * M * N * K}
    inputs = 3 if case["input"] else 2
    n = case["batch"] * case.get("tokens", 1) * case["width"]
    state = 4 * case["batch"] * case["width"]
    if kind == "scan_step":
        return {"bytes": n * (inputs + 1) * size + 2 * state, "flops": 12 * n}
    if kind == "scan":
        return {"bytes": n * (inputs + 1) * size + state * (2 if case["state"] else 1), "flops": 12 * n}
    # the gates, the values and dout in, out and the gradients out
    return {"bytes": n * 2 * (inputs + 1) * size + state * (4 if case["state"] else 1), "flops": 32 * n}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def _exact_scan(s):
    """Token by token, and the gradients from the last token to the first."""
    case = s["case"]
    step, own_gate, squash = case["kind"] == "scan_step", s["input"] is not None, case["activation"] == "tanh"

    def wide(name):
        t = s[name].detach().double()
        return t[:, None] if step else t

    f = torch.sigmoid(wide("forget"))
    z = torch.sigmoid(wide("input")) if own_gate else torch.sigmoid(-wide("forget"))
    v = wide("value")
    c = v.tanh() if squash else v
    B, T, D = f.shape
    h = torch.zeros(B, D, dtype=torch.float64, device=f.device) if s["state"] is None else s["state"].detach().double()
    lengths = s.get("lengths")
    counts = torch.full((B,), T, device=f.device) if lengths is None else lengths
    train = case["kind"] == "scan_train"
    out = torch.zeros_like(f)
    before = torch.zeros_like(f) if train else None
    added = z * c
    for t in range(T):
        if train:
            before[:, t] = h
        new = torch.addcmul(added[:, t], f[:, t], h)
        h = new if lengths is None else torch.where((t < counts)[:, None], new, h)
        out[:, t] = h
    live = (torch.arange(T, device=f.device)[None] < counts[:, None])[..., None]
    out = out * live
    if not train:
        return dict(out=out[:, 0] if step else out, state=h)
    G = torch.zeros_like(f)
    R = torch.zeros_like(h) if s["dfinal"] is None else s["dfinal"].double()
    dout = s["dout"].double()
    for t in reversed(range(T)):
        g = R + dout[:, t]
        if lengths is None:
            G[:, t], R = g, f[:, t] * g
        else:
            here = (t < counts)[:, None]
            G[:, t] = torch.where(here, g, 0.0)
            R = torch.where(here, f[:, t] * g, R)
    result = dict(out=out, final=h)
    fall = torch.sigmoid(-wide("forget"))
    result["dforget"] = G * f * fall * (before if own_gate else before - c)
    result["dvalue"] = G * z * (1 - c ** 2) if squash else G * z
    if own_gate:
        result["dinput"] = G * c * z * torch.sigmoid(-wide("input"))
    if s["state"] is not None:
        result["dstate"] = R
    return result


def _exact_kept(x, lowest):
    """The nearest multiples of a power of two, 127 of which reach a group's largest magnitude."""
    x = x.double()
    width = x.shape[1]
    parts = torch.nn.functional.pad(x, (0, -width % GROUP)).unflatten(1, (-1, GROUP))
    largest = parts.abs().amax(dim=2, keepdim=True)
    exponent = torch.frexp(largest).exponent - 8   # too low by one or two
    for _ in range(2):
        exponent = torch.where(largest > 127 * torch.ldexp(torch.ones_like(largest), exponent), exponent + 1, exponent)
    power = torch.ldexp(torch.ones_like(largest), exponent.clamp(min=lowest))
    return (torch.round(parts / power) * power).flatten(1)[:, :width]


def exact(case, seed):
    s = prepare(case, seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    if kind.startswith("scan"):
        return _exact_scan(s)
    if kind == "keep":
        return _exact_kept(s["x"], LOWEST[dtype])
    if kind == "weights":
        scales = torch.exp2(s["exponents"].double())
        index = torch.arange(case["inner"], device=scales.device) // GROUP
        return torch.einsum("mn,mk->nk", s["dy"].double(), s["codes"].double() * scales[:, index])
    gate, up, dy = s["gate"].detach().double(), s["up"].detach().double(), s["dy"].double()
    curves = {"none": (lambda v: v, lambda v: torch.ones_like(v)),
              "relu": (torch.relu, lambda v: (v > 0).double()),
              "silu": (lambda v: v * torch.sigmoid(v), lambda v: torch.sigmoid(v) + v * torch.sigmoid(v) * torch.sigmoid(-v)),
              "gelu": (lambda v: v * 0.5 * torch.special.erfc(-v / math.sqrt(2)),
                       lambda v: 0.5 * torch.special.erfc(-v / math.sqrt(2)) + v * torch.exp(-v ** 2 / 2) / math.sqrt(2 * math.pi))}
    value, slope = curves[case["activation"]]
    kept_gate, kept_up = _exact_kept(gate, LOWEST[dtype]), _exact_kept(up, LOWEST[dtype])
    return dict(y=value(gate) * up, dgate=dy * kept_up * slope(kept_gate), dup=dy * value(kept_gate))
