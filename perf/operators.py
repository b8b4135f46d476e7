"""Operators of a decaying recurrent token mixer, as timed cases.

Three operators that a streaming model calls one after another in every block:

``norm``    the residual stream's addition and its root-mean-square norm; for serving with 8-bit codes and a scale for each
            row, for training with the gradients
``linear``  the product of such codes with 8-bit weights, with bias, activation and residual in its epilogue
``attend``  linear attention with a fixed decay for each head: prompts, single tokens, and the gradients

``listed()`` names fixed cases, ``draw()`` gives further ones of the same ranges.  With ``own`` false the operators run as
elementary torch operations in 32 bits, with ``own`` true through the public entry points of this framework.
"""
import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64   # tokens of a chunk of the plain linear attention


def listed():
    return [
        # one token of one stream between two projections: latency
        dict(name="norm_token", kind="norm_codes", rows=1, width=1024, type="bf16"),
        # the tokens of a batch of prompts in front of the block's first projection
        dict(name="norm_prompt", kind="norm_codes", rows=8192, width=4096, type="bf16"),
        # a training step's norm, forward and backward, in the mixed precision of the model
        dict(name="norm_train", kind="norm_train", rows=16384, width=2048, type="bf16"),
        # the same in full precision at a width and a number of rows that nothing divides
        dict(name="norm_train_ragged", kind="norm_train", rows=5003, width=1001, type="fp32"),
        # one token through an expanding projection: the weights are read once for it
        dict(name="linear_token", kind="linear", rows=1, inner=1024, outer=4096, activation="silu", bias=True, residual=False, type="bf16"),
        # tokens of a few short prompts, sizes that no tile divides, result in full precision for what follows on the host
        dict(name="linear_ragged", kind="linear", rows=777, inner=1000, outer=1100, activation="gelu", bias=True, residual=False, type="fp32"),
        # a batch of prompts through a projection back onto the residual stream
        dict(name="linear_prompt", kind="linear", rows=8192, inner=4096, outer=4096, activation="none", bias=True, residual=True, type="bf16"),
        # one token for each of sixteen streams: the states are read and written once
        dict(name="attend_token", kind="attend_step", batch=16, heads=16, shared=1, key=128, value=128, type="bf16"),
        # a batch of prompts
        dict(name="attend_prompt", kind="attend", batch=8, tokens=4096, heads=16, shared=1, key=128, value=128, ragged=False, state=False, type="bf16"),
        # one long recording continued from a state, few heads: the axis of time has to be split
        dict(name="attend_long", kind="attend", batch=1, tokens=16384, heads=8, shared=1, key=64, value=64, ragged=False, state=True, type="fp16"),
        # a training step over full sequences
        dict(name="attend_train", kind="attend_train", batch=8, tokens=2048, heads=16, shared=1, key=64, value=64, ragged=False, state=False, type="bf16"),
        # a training step over utterances of several lengths that goes on from a state, keys and values shared by four heads each
        dict(name="attend_train_shared", kind="attend_train", batch=6, tokens=1000, heads=8, shared=4, key=96, value=64, ragged=True, state=True, type="fp16"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def _width(rng, low, high):
    """A width: two of three are multiples of 64, as networks mostly have them, the others any number."""
    n = _log(rng, low, high)
    return n if rng.random() < 1 / 3 else min(high, max(64, (n + 32) // 64 * 64))


def draw(rng):
    kind = rng.choice(("norm_codes", "norm_train", "linear", "linear", "attend_step", "attend", "attend_train"))
    if kind in ("norm_codes", "norm_train"):
        width = _width(rng, 64, 8192)
        rows = _log(rng, 1, min(16384, (32 << 20) // width))
        return dict(kind=kind, rows=rows, width=width, type=rng.choice(("bf16", "fp16") if kind == "norm_codes" else ("bf16", "fp16", "fp32")))
    if kind == "linear":
        inner, outer = _width(rng, 64, 8192), _width(rng, 64, 8192)
        rows = _log(rng, 1, min(8192, (8192 * 4096 * 4096) // (inner * outer)))
        return dict(kind=kind, rows=rows, inner=inner, outer=outer, activation=rng.choice(("none", "relu", "silu", "gelu")),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5, type=rng.choice(("bf16", "bf16", "fp16", "fp32")))
    heads = rng.choice((1, 2, 4, 6, 8, 12, 16))
    shared = rng.choice([n for n in (1, 1, 2, 4) if heads % n == 0])
    key, value = rng.choice(((64, 64), (128, 128), (128, 128), (128, 64), (96, 64), (80, 80), (40, 72)))
    if kind == "attend_step":
        return dict(kind=kind, batch=_log(rng, 1, 256), heads=heads, shared=shared, key=key, value=value, type=rng.choice(("bf16", "fp16", "fp32")))
    tokens = _log(rng, 2, 16384)
    most = 8 * 4096 * 16 * 128 // 2 // (3 if kind == "attend_train" else 1)
    batch = _log(rng, 1, max(1, min(64, most // (tokens * heads * max(key, value)))))
    return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, shared=shared, key=key, value=value, ragged=rng.random() < 0.4,
                state=rng.random() < 0.5, type=rng.choice(("bf16", "bf16", "fp16")))


# ---- inputs -----------------------------------------------------------------------------------------------------------

def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(dtype)


def _coded(values):
    """8-bit codes of the rows of `values` and a scale for each; rows start at multiples of 16 bytes, as the framework lays them out."""
    scale = values.abs().amax(dim=1) / 127
    codes = torch.round(values / scale[:, None]).to(torch.int8)
    rows, width = values.shape
    held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device=values.device)
    held[:, :width] = codes
    return held[:, :width], scale


def prepare(case, seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case["type"]]
    s = dict(case=case)
    if kind in ("norm_codes", "norm_train"):
        shape = (case["rows"], case["width"])
        # a residual stream has some channels that are larger than the others
        spread = 1.0 + 8.0 * (torch.rand(case["width"], generator=g, device=DEVICE) < 0.01)
        s["x"] = _normal(g, shape, dtype)
        s["residual"] = (_normal(g, shape, torch.float32, 2.0) * spread).to(dtype)
        s["weight"] = 1 + _normal(g, (case["width"],), torch.float32, 0.1)
        if kind == "norm_train":
            s["dy"], s["dtotal"] = _normal(g, shape, dtype), _normal(g, shape, dtype)
            for name in ("x", "residual", "weight"):
                s[name].requires_grad_()
    elif kind == "linear":
        M, K, N = case["rows"], case["inner"], case["outer"]
        s["codes"], s["scale"] = _coded(_normal(g, (M, K), torch.float32))
        s["weight"], s["weight_scale"] = _coded(_normal(g, (N, K), torch.float32, K ** -0.5))
        s["bias"] = _normal(g, (N,), torch.float32, 0.1) if case["bias"] else None
        s["residual"] = _normal(g, (M, N), dtype) if case["residual"] else None
    else:
        B, H, Hk, Dk, Dv = case["batch"], case["heads"], case["heads"] // case["shared"], case["key"], case["value"]
        T = case.get("tokens", 1)
        # one projection's result, split into queries, keys and values
        joint = _normal(g, (B, T, H * Dk + Hk * (Dk + Dv)), dtype)
        q, k, v = joint.split([H * Dk, Hk * Dk, Hk * Dv], dim=-1)
        s["q"], s["k"], s["v"] = q.view(B, T, H, Dk), k.view(B, T, Hk, Dk), v.view(B, T, Hk, Dv)
        # memories of two tokens to some hundred, spread over the heads
        s["log_decay"] = torch.log1p(-torch.exp2(-torch.linspace(1, 9, H, device=DEVICE)))
        s["lengths"] = torch.randint(0, T + 1, (B,), generator=g, device=DEVICE, dtype=torch.int32) if case.get("ragged") else None
        s["state"] = _normal(g, (B, H, Dk, Dv), torch.float32) if kind == "attend_step" or case["state"] else None
        if kind == "attend_step":
            s["q"], s["k"], s["v"] = s["q"][:, 0], s["k"][:, 0], s["v"][:, 0]
            s["new_state"] = torch.empty_like(s["state"])
        if kind == "attend_train":
            s["dout"] = _normal(g, (B, T, H, Dv), dtype)
            s["dstate"] = _normal(g, (B, H, Dk, Dv), torch.float32) if case["state"] else None
            for name in ("q", "k", "v", "state"):
                if s[name] is not None:
                    s[name] = s[name].detach().requires_grad_()
    return s


# ---- plain forms --------------------------------------------------------------------------------------------------------

def _plain_norm(x, residual, weight):
    total = x + residual
    return total * torch.rsqrt(total.square().mean(dim=-1, keepdim=True) + EPS) * weight, total


def _plain_activation(x, name):
    if name == "relu":
        return torch.clamp(x, min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    return x


def _plain_attend(q, k, v, log_decay, state, lengths):
    """Chunks of tokens: inside a chunk a masked product, between chunks the states, all chunks at once."""
    B, T, H, Dk = q.shape
    Dv = v.shape[-1]
    k, v = k.repeat_interleave(H // k.shape[2], dim=2), v.repeat_interleave(H // v.shape[2], dim=2)
    N = -(-T // CHUNK)
    t = torch.arange(N * CHUNK, device=q.device)
    real = t[None] < (torch.full((B,), T, device=q.device) if lengths is None else lengths)[:, None]     # [B, N CHUNK]
    seen = real.cumsum(dim=1).float()                                                                  # tokens up to here, itself too
    pad = N * CHUNK - T

    def chunks(x):   # [B, H, N, CHUNK, D]
        x = torch.nn.functional.pad(x, (0, 0, 0, 0, 0, pad))
        x = torch.where(real[:, :, None, None], x, torch.zeros_like(x))
        return x.view(B, N, CHUNK, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v = chunks(q) * Dk ** -0.5, chunks(k), chunks(v)
    g = log_decay[None, :, None, None]
    at = seen.view(B, 1, N, CHUNK)
    before = torch.cat([torch.zeros_like(at[:, :, :1, 0]), at[:, :, :, -1]], dim=2)                       # [B, 1, N + 1] tokens before a chunk
    inside = torch.exp(g[..., None] * (at[..., :, None] - at[..., None, :]).clamp(min=0))               # [B, H, N, CHUNK, CHUNK]
    inside = torch.where((t[:CHUNK, None] >= t[None, :CHUNK]), inside, torch.zeros_like(inside))
    out = ((q @ k.transpose(-1, -2)) * inside) @ v
    weights = torch.exp(g * (before[:, :, 1:, None] - at))                                              # to the chunk's end
    added = (k * weights[..., None]).transpose(-1, -2) @ v                                              # [B, H, N, Dk, Dv]
    reach = torch.exp(g * (before[..., :, None] - before[..., None, 1:]).clamp(min=0))                  # [B, H, N + 1, N]
    c = torch.arange(N + 1, device=q.device)
    reach = torch.where(c[:, None] > c[None, :N], reach, torch.zeros_like(reach))
    states = (reach @ added.reshape(B, H, N, Dk * Dv)).view(B, H, N + 1, Dk, Dv)
    if state is not None:
        states = states + torch.exp(g * before[..., None])[..., None] * state[:, :, None]
    out = out + torch.exp(g * (at - before[:, :, :-1, None]))[..., None] * (q @ states[:, :, :-1])
    out = out.permute(0, 2, 3, 1, 4).reshape(B, N * CHUNK, H, Dv)[:, :T]
    return out, states[:, :, -1]


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    dtype = TYPES[case["type"]]
    if kind == "norm_codes":
        y, total = _plain_norm(s["x"].float(), s["residual"].float(), s["weight"])
        scale = y.abs().amax(dim=1) / 127
        codes = torch.where(scale[:, None] > 0, torch.round(y / scale[:, None]), torch.zeros_like(y))
        return dict(values=(codes * scale[:, None]).to(dtype), scale=scale, total=total.to(dtype))
    if kind == "norm_train":
        leaves = [s[n].detach().float().requires_grad_() for n in ("x", "residual", "weight")]
        y, total = _plain_norm(*leaves)
        dx, dresidual, dweight = torch.autograd.grad([y, total], leaves, [s["dy"].float(), s["dtotal"].float()])
        return dict(y=y.detach().to(dtype), total=total.detach().to(dtype), dx=dx.to(dtype), dresidual=dresidual.to(dtype), dweight=dweight)
    if kind == "linear":
        y = (s["codes"].float() @ s["weight"].float().T) * s["scale"][:, None] * s["weight_scale"]
        if s["bias"] is not None:
            y = y + s["bias"]
        y = _plain_activation(y, case["activation"])
        if s["residual"] is not None:
            y = y + s["residual"].float()
        return y.to(dtype)
    if kind == "attend_step":
        q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
        k, v = k.repeat_interleave(case["shared"], dim=1), v.repeat_interleave(case["shared"], dim=1)
        state = torch.exp(s["log_decay"])[:, None, None] * s["state"] + k[..., :, None] * v[..., None, :]
        out = (q[..., None, :] @ state)[..., 0, :] * case["key"] ** -0.5
        return dict(out=out.to(dtype), state=state)
    if kind == "attend":
        out, state = _plain_attend(s["q"].float(), s["k"].float(), s["v"].float(), s["log_decay"], s["state"], s["lengths"])
        return dict(out=out.to(dtype), state=state)
    names = ["q", "k", "v"] + (["state"] if s["state"] is not None else [])
    leaves = {n: s[n].detach().float().requires_grad_() for n in names}
    out, state = _plain_attend(leaves["q"], leaves["k"], leaves["v"], s["log_decay"], leaves.get("state"), s["lengths"])
    ends, given = ([out], [s["dout"].float()]) if s["dstate"] is None else ([out, state], [s["dout"].float(), s["dstate"]])
    grads = torch.autograd.grad(ends, list(leaves.values()), given)
    result = {"d" + n: d if n == "state" else d.to(dtype) for n, d in zip(names, grads)}
    return dict(result, out=out.detach().to(dtype), final=state.detach())


# ---- the framework's operators ----------------------------------------------------------------------------------------------

def _run_own(s):
    from rx_met_b200 import coded_linear, decayed_attention, rms_norm
    case, kind = s["case"], s["case"]["kind"]
    dtype = TYPES[case["type"]]
    if kind == "norm_codes":
        codes, scale, total = rms_norm.add_rms_norm_codes(s["x"], s["weight"], s["residual"], EPS)
        values = torch.mul(codes, scale[:, None], out=torch.empty_like(total))   # what the codes stand for
        return dict(values=values, scale=scale, total=total)
    if kind == "norm_train":
        leaves = [s[n] for n in ("x", "residual", "weight")]
        y, total = rms_norm.add_rms_norm(s["x"], s["weight"], s["residual"], EPS)
        dx, dresidual, dweight = torch.autograd.grad([y, total], leaves, [s["dy"], s["dtotal"]])
        return dict(y=y.detach(), total=total.detach(), dx=dx, dresidual=dresidual, dweight=dweight)
    if kind == "linear":
        return coded_linear.coded_linear(s["codes"], s["scale"], coded_linear.CodedWeight(s["weight"], s["weight_scale"]), bias=s["bias"],
                                         activation=case["activation"], residual=s["residual"], dtype=dtype)
    if kind == "attend_step":
        out = decayed_attention.decayed_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], new_state=s["new_state"])
        return dict(out=out, state=s["new_state"])
    if kind == "attend":
        out, state = decayed_attention.decayed_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], lengths=s["lengths"])
        return dict(out=out, state=state)
    names = ["q", "k", "v"] + (["state"] if s["state"] is not None else [])
    out, state = decayed_attention.decayed_attention(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], lengths=s["lengths"])
    ends, given = ([out], [s["dout"]]) if s["dstate"] is None else ([out, state], [s["dout"], s["dstate"]])
    grads = torch.autograd.grad(ends, [s[n] for n in names], given)
    return dict({"d" + n: d for n, d in zip(names, grads)}, out=out.detach(), final=state.detach())


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------

def work(case):
    kind, size = case["kind"], 4 if case["type"] == "fp32" else 2
    if kind == "norm_codes":   # x and residual in, the sum and the codes out
        n = case["rows"] * case["width"]
        return {"bytes": n * (3 * size + 1) + 4 * case["rows"] + 4 * case["width"], "flops": 7 * n}
    if kind == "norm_train":   # x, residual, dy, dtotal in, y, total, dx (the gradient of both) out
        n = case["rows"] * case["width"]
        return {"bytes": n * 7 * size + 8 * case["width"], "flops": 16 * n}
    if kind == "linear":
        M, K, N = case["rows"], case["inner"], case["outer"]
        return {"bytes": M * K + N * K + M * N * size * (2 if case["residual"] else 1) + 4 * (M + N * (2 if case["bias"] else 1)),
                "flops": 2 * M * N * K}
    B, H, Hk, Dk, Dv = case["batch"], case["heads"], case["heads"] // case["shared"], case["key"], case["value"]
    rows = B * case.get("tokens", 1)
    inputs, out, state = rows * (H * Dk + Hk * (Dk + Dv)) * size, rows * H * Dv * size, B * H * Dk * Dv * 4
    if kind == "attend_step":
        return {"bytes": inputs + out + 2 * state, "flops": 4 * rows * H * Dk * Dv}
    if kind == "attend":       # the state's update and the query's product with it
        return {"bytes": inputs + out + state * (2 if case["state"] else 1), "flops": 4 * rows * H * Dk * Dv}
    # and for the gradients the state's gradient, and a product each for q, k and v
    return {"bytes": 2 * (inputs + out) + state * (4 if case["state"] else 1), "flops": 12 * rows * H * Dk * Dv}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------------

def _exact_attend(s):
    """Token by token: S = decay S + k v', out = q S; the gradients by the same recurrence from the last token to the first."""
    step = s["case"]["kind"] == "attend_step"
    q, k, v = ((s[n].detach()[:, None] if step else s[n].detach()).double() for n in ("q", "k", "v"))
    B, T, H, Dk = q.shape
    Dv, share = v.shape[-1], H // k.shape[2]
    head = torch.arange(H, device=q.device) // share
    k, v = k[:, :, head], v[:, :, head]
    scale = 1 / math.sqrt(Dk)
    decay = torch.exp(s["log_decay"].double())[None, :, None, None]
    S = torch.zeros(B, H, Dk, Dv, dtype=torch.float64, device=q.device) if s["state"] is None else s["state"].detach().double()
    lengths = s.get("lengths")
    train = s["case"]["kind"] == "attend_train"
    out, dq = torch.zeros(B, T, H, Dv, dtype=torch.float64, device=q.device), torch.zeros_like(q)
    dout = s["dout"].double() if train else None
    for t in range(T):
        new = decay * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        live = None if lengths is None else (t < lengths)[:, None, None, None]
        S = new if live is None else torch.where(live, new, S)
        o = torch.einsum("bhk,bhkv->bhv", q[:, t], S) * scale
        out[:, t] = o if live is None else o * live[..., 0]
        if train:
            d = torch.einsum("bhv,bhkv->bhk", dout[:, t], S) * scale
            dq[:, t] = d if live is None else d * live[..., 0]
    if not train:
        return dict(out=out[:, 0] if step else out, state=S)
    G = torch.zeros_like(S) if s["dstate"] is None else s["dstate"].double()
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    for t in reversed(range(T)):
        new = G + q[:, t, :, :, None] * dout[:, t, :, None, :] * scale
        a, b = torch.einsum("bhkv,bhv->bhk", new, v[:, t]), torch.einsum("bhkv,bhk->bhv", new, k[:, t])
        live = None if lengths is None else (t < lengths)[:, None, None, None]
        dk[:, t], dv[:, t] = (a, b) if live is None else (a * live[..., 0], b * live[..., 0])
        G = decay * new if live is None else torch.where(live, decay * new, G)
    grouped = lambda d: d.view(B, T, H // share, share, -1).sum(dim=3)  # noqa: E731
    result = dict(out=out, final=S, dq=dq, dk=grouped(dk), dv=grouped(dv))
    return dict(result, dstate=G) if s["state"] is not None else result


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "linear":
        y = torch.einsum("mk,nk->mn", s["codes"].double(), s["weight"].double())
        y = y * (s["scale"].double()[:, None] * s["weight_scale"].double()[None])
        y = y if s["bias"] is None else y + s["bias"].double()
        if case["activation"] == "relu":
            y = torch.relu(y)
        elif case["activation"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["activation"] == "gelu":
            y = y * 0.5 * torch.special.erfc(-y / math.sqrt(2))
        return y if s["residual"] is None else s["residual"].double() + y
    if kind.startswith("norm"):
        total = s["x"].detach().double() + s["residual"].detach().double()
        weight = s["weight"].detach().double()
        rms = torch.sqrt((total ** 2).sum(dim=1, keepdim=True) / case["width"] + EPS)
        unit = total / rms
        y = unit * weight
        if kind == "norm_codes":
            scale = y.abs().max(dim=1).values / 127
            return dict(values=torch.round(y / scale[:, None]) * scale[:, None], scale=scale, total=total)
        dy, dtotal = s["dy"].double(), s["dtotal"].double()
        dunit = dy * weight
        dx = dtotal + (dunit - unit * (dunit * unit).sum(dim=1, keepdim=True) / case["width"]) / rms
        return dict(y=y, total=total, dx=dx, dresidual=dx, dweight=(dy * unit).sum(dim=0))
    return _exact_attend(s)
