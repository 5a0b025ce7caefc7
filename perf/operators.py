"""Linear attention with a decay for each head, and the norms around its block, as measurable cases.

``run`` computes them in their plain form, in elementary torch operations and 32 bits, or (``own``) through the public API
(``nebula_b200.api``).  Inputs are seeded synthetic tensors with the value ranges of a trained block: unit-variance queries
and values, keys of unit length, log decays between those of heads that remember a few tokens and heads that remember
thousands.
"""
import math
import random

import torch

own = False

CHUNK = 64
_handle = []


def listed():
    return [
        # a server's prefill of a batch of prompts, one decay per token and head
        {"name": "prompt_8x4096_h16_d128", "kind": "prompt", "batch": 8, "tokens": 4096, "heads": 16, "key_heads": 16, "key_dim": 128,
         "value_dim": 128, "dtype": "bf16", "decay": "token", "packed": False, "resets": False, "initial": False},
        # one long document and few heads (a shard of a model): little work side by side, a long axis; fixed decays
        {"name": "prompt_1x32768_h8_d128", "kind": "prompt", "batch": 1, "tokens": 32768, "heads": 8, "key_heads": 8, "key_dim": 128,
         "value_dim": 128, "dtype": "bf16", "decay": "head", "packed": False, "resets": False, "initial": False},
        # continuous batching: prompts of very different lengths packed one behind the other, some empty, that carry on from
        # a pool of states; heads share their queries and keys; document boundaries inside a prompt
        {"name": "prompt_packed_24x1999_h12k4_d64x128", "kind": "prompt", "batch": 24, "tokens": 1999, "heads": 12, "key_heads": 4,
         "key_dim": 64, "value_dim": 128, "dtype": "bf16", "decay": "token", "packed": True, "resets": True, "initial": True},
        # the same layer in fp32, the type of the framework's other layers
        {"name": "prompt_f32_4x1023_h8_d64", "kind": "prompt", "batch": 4, "tokens": 1023, "heads": 8, "key_heads": 8, "key_dim": 64,
         "value_dim": 64, "dtype": "f32", "decay": "token", "packed": False, "resets": False, "initial": True},
        # a short prompt of a small model with odd sizes
        {"name": "prompt_2x37_h3_d40x72", "kind": "prompt", "batch": 2, "tokens": 37, "heads": 3, "key_heads": 3, "key_dim": 40,
         "value_dim": 72, "dtype": "bf16", "decay": "token", "packed": False, "resets": False, "initial": True},
        # one token of one sequence: latency
        {"name": "step_1_h8_d64", "kind": "step", "batch": 1, "heads": 8, "key_heads": 8, "key_dim": 64, "value_dim": 64, "dtype": "bf16",
         "decay": "token"},
        # a token for each sequence of an ordinary server batch
        {"name": "step_64_h16_d128", "kind": "step", "batch": 64, "heads": 16, "key_heads": 16, "key_dim": 128, "value_dim": 128,
         "dtype": "bf16", "decay": "token"},
        # a large batch off the powers of two, fp32, fixed decays, shared keys
        {"name": "step_f32_333_h12k3_d64x96", "kind": "step", "batch": 333, "heads": 12, "key_heads": 3, "key_dim": 64, "value_dim": 96,
         "dtype": "f32", "decay": "head"},
        # the norms between two blocks for a single token
        {"name": "norms_1x4096", "kind": "norm", "rows": 1, "width": 4096, "groups": 1, "norm": "rms", "gate": "none", "residual": True,
         "next": "rms", "dtype": "bf16"},
        # the same for a prompt batch: post-norm, residual scale, residual sum, the next block's pre-norm
        {"name": "norms_8192x4096", "kind": "norm", "rows": 8192, "width": 4096, "groups": 1, "norm": "rms", "gate": "none", "residual": True,
         "next": "rms", "dtype": "bf16"},
        # the norm of each head behind the attention, with its gate
        {"name": "head_norm_gate_16384x16x128", "kind": "norm", "rows": 16384, "width": 2048, "groups": 16, "norm": "rms", "gate": "silu",
         "residual": False, "next": "none", "dtype": "bf16"},
        # fp32, mean and variance, odd sizes, everything at once
        {"name": "norms_f32_1001x1000", "kind": "norm", "rows": 1001, "width": 1000, "groups": 4, "norm": "layer", "gate": "sigmoid",
         "residual": True, "next": "layer", "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _divisors(n):
    return [d for d in range(1, n + 1) if n % d == 0]


def draw(rng):
    dtype = "bf16" if rng.random() < 0.7 else "f32"
    kind = rng.choice(["prompt", "prompt", "step", "norm"])
    if kind == "norm":
        rows, groups = _log(rng, 1, 16384), rng.choice([1, 1, 1, 4, 8, 16])
        width = groups * max(1, _log(rng, 64, 8192) // groups)
        if rng.random() < 0.6:
            width = groups * 8 * max(1, width // (8 * groups))
        rows = max(1, min(rows, (1 << 25) // width // (2 if dtype == "f32" else 1)))
        return {"kind": kind, "rows": rows, "width": width, "groups": groups, "norm": rng.choice(["rms", "rms", "layer"]),
                "gate": rng.choice(["none", "silu", "sigmoid"]), "residual": rng.random() < 0.7, "next": rng.choice(["none", "rms", "layer"]),
                "dtype": dtype}
    heads = rng.randint(1, 24)
    dims = [16, 32, 48, 64, 64, 80, 96, 128, 128, 128] + [rng.randint(9, 128)]
    key_dim = rng.choice(dims)
    case = {"kind": kind, "heads": heads, "key_heads": heads if rng.random() < 0.6 else rng.choice(_divisors(heads)), "key_dim": key_dim,
            "value_dim": key_dim if rng.random() < 0.6 else rng.choice(dims), "dtype": dtype, "decay": "token" if rng.random() < 0.7 else "head"}
    if kind == "step":
        most = (64 * 16 * 128 * 128) // (heads * case["key_dim"] * case["value_dim"])
        return dict(case, batch=max(1, min(_log(rng, 1, 512), most)))
    tokens = _log(rng, 1, 16384)
    most = (8 * 4096 * 16 * 256) // (heads * (case["key_dim"] + case["value_dim"]) * tokens * (4 if dtype == "f32" else 1))
    packed = rng.random() < 0.4
    return dict(case, batch=max(1, min(_log(rng, 1, 32), most)), tokens=tokens, packed=packed, resets=rng.random() < 0.3,
                initial=rng.random() < 0.5)


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """Tokens of each sequence: the same ones for every seed, in an order of its own."""
    B, T = case["batch"], case["tokens"]
    if not case["packed"]:
        return [T] * B
    n = [int(T * (i / max(1, B - 1)) ** 2) for i in range(B)]      # 0, ..., T: many short ones, few long ones
    n[-1] = T
    return n


_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}


def _normal(g, dtype, *shape):
    return torch.randn(*shape, device="cuda", dtype=torch.float32, generator=g).to(dtype)


def _log_decay(case, g, *lead):
    """A head's time constant lies between a few tokens and some thousands; a token's own decay varies around it."""
    H = case["heads"]
    rate = torch.exp(torch.linspace(math.log(0.5), math.log(5e-4), H, device="cuda")) if H > 1 else torch.full((1,), 0.05, device="cuda")
    if case["decay"] == "head":
        return -rate * (0.8 + 0.4 * torch.rand(H, device="cuda", generator=g))
    return -rate * 2 * torch.rand(*lead, H, device="cuda", generator=g)


def _keys(g, case, *lead):
    k = torch.randn(*lead, case["key_heads"], case["key_dim"], device="cuda", generator=g)
    return (k / k.norm(dim=-1, keepdim=True)).to(_TYPE[case["dtype"]])


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = _TYPE[case["dtype"]]
    s = {"case": case}
    if case["kind"] == "norm":
        R, W = case["rows"], case["width"]
        s["x"] = _normal(g, t, R, W) * 2
        s["weight"] = 1 + 0.2 * _normal(g, torch.float32, W)
        s["bias"] = 0.1 * _normal(g, torch.float32, W) if case["norm"] == "layer" else None
        s["gate"] = _normal(g, t, R, W) if case["gate"] != "none" else None
        s["residual"] = _normal(g, t, R, W) * 3 if case["residual"] else None
        s["channel_scale"] = 0.5 + 0.1 * _normal(g, torch.float32, W) if case["residual"] else None
        s["next_weight"] = 1 + 0.2 * _normal(g, torch.float32, W) if case["next"] != "none" else None
        s["next_bias"] = 0.1 * _normal(g, torch.float32, W) if case["next"] == "layer" else None
        return s
    B, H, K, dk, dv = case["batch"], case["heads"], case["key_heads"], case["key_dim"], case["value_dim"]
    if case["kind"] == "step":
        s["q"], s["k"], s["v"] = _normal(g, t, B, K, dk), _keys(g, case, B), _normal(g, t, B, H, dv)
        s["log_decay"] = _log_decay(case, g, B)
        s["state"] = _normal(g, torch.float32, B, H, dk, dv)
        s["slots"] = torch.randperm(B, device="cuda", generator=g).int()
        return s
    n = _lengths(case)
    random.Random(seed).shuffle(n)
    s["lengths"] = n
    if case["packed"]:
        lead = (sum(n),)
        s["offsets"] = torch.tensor([sum(n[:i]) for i in range(B + 1)], dtype=torch.int32, device="cuda")
        s["slots"] = torch.randperm(B, device="cuda", generator=g).int()
    else:
        lead = (B, case["tokens"])
        s["offsets"] = s["slots"] = None
    s["q"], s["k"], s["v"] = _normal(g, t, *lead, K, dk), _keys(g, case, *lead), _normal(g, t, *lead, H, dv)
    s["log_decay"] = _log_decay(case, g, *lead)
    if case["resets"] and case["decay"] == "token":
        s["log_decay"][torch.rand(*lead, device="cuda", generator=g) < 1 / 300] = -math.inf
    s["state"] = _normal(g, torch.float32, B, H, dk, dv) if case["initial"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = case
    if own:
        from nebula_b200 import api
        if not _handle:
            _handle.append(api.Handle(0, "tf32x3"))
        if c["kind"] == "norm":
            s["handle"] = _handle[0]
        else:
            s["layer"] = api.LinearAttention(_handle[0], c["batch"], c.get("tokens", 1), c["heads"], c["key_dim"], c["value_dim"],
                                             key_heads=c["key_heads"], dtype=c["dtype"], scale=c["key_dim"] ** -0.5)
            s["layer"].prepare()
    if c["kind"] != "norm":
        s["out"] = torch.empty_like(s["v"])
        s["new_state"] = torch.empty(c["batch"], c["heads"], c["key_dim"], c["value_dim"], device="cuda")
    return s


# ------------------------------------------------------------- plain forms
def _norm_plain(x, mode, groups, weight, bias):
    R, W = x.shape
    x = x.view(R, groups, W // groups)
    if mode == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6)
    x = x.view(R, W) * weight
    return x if bias is None else x + bias


def _norms(s):
    c, t = s["case"], s["x"].dtype
    u = _norm_plain(s["x"].float(), c["norm"], c["groups"], s["weight"], s["bias"])
    if s["gate"] is not None:
        z = s["gate"].float()
        u = u * (torch.sigmoid(z) if c["gate"] == "sigmoid" else z * torch.sigmoid(z))
    if s["residual"] is not None:
        u = s["residual"].float() + 0.5 * s["channel_scale"] * u
    if c["next"] == "none":
        return {"sum": u.to(t)}
    return {"sum": u.to(t), "y": _norm_plain(u, c["next"], 1, s["next_weight"], s["next_bias"]).to(t)}


def _between(g):
    """exp of the sum of g over (j, i] for i >= j, else 0, by partial sums of their own for every j: [..., C] -> [..., C, C]."""
    C = g.shape[-1]
    at = torch.arange(C, device=g.device)
    later = at[:, None] > at[None, :]
    sums = torch.where(later, g[..., :, None], g.new_zeros(())).cumsum(-2)
    return torch.where(later | (at[:, None] == at[None, :]), torch.exp(sums), g.new_zeros(()))


def _steps(s):
    c = s["case"]
    r = c["heads"] // c["key_heads"]
    q, k = (s[n].float().repeat_interleave(r, dim=1) for n in ("q", "k"))
    at = s["slots"].long()
    decay = torch.exp(s["log_decay"]).expand(c["batch"], c["heads"])
    new = decay[:, :, None, None] * s["state"][at] + k[..., :, None] * s["v"].float()[..., None, :]
    o = c["key_dim"] ** -0.5 * torch.matmul(q[..., None, :], new)[..., 0, :]
    return {"out": o.to(s["v"].dtype), "state": torch.empty_like(new).index_copy_(0, at, new)}


def _prompts(s):
    c, (B, T, H) = s["case"], (s["case"]["batch"], s["case"]["tokens"], s["case"]["heads"])
    r, dk, dv = H // c["key_heads"], c["key_dim"], c["value_dim"]
    N = -(-T // CHUNK)
    q, k, v, g = s["q"], s["k"], s["v"], s["log_decay"]
    g = g.expand(*v.shape[:-1])
    if s["offsets"] is not None:
        off = s["offsets"].long()
        rows = off[:-1, None] + torch.arange(T, device="cuda")
        there = rows < off[1:, None]
        rows = rows.clamp(max=v.shape[0] - 1)
        q, k, v, g = q[rows], k[rows] * there[..., None, None], v[rows], torch.where(there[..., None], g[rows], 0.0)

    def chunks(x):      # [B, T, heads, d] -> [B, H, N, CHUNK, d]
        x = torch.nn.functional.pad(x.float(), (0, 0, 0, 0, 0, N * CHUNK - T))
        return x.view(B, N, CHUNK, x.shape[2], x.shape[3]).permute(0, 3, 1, 2, 4)

    q, k = (chunks(x).repeat_interleave(r, dim=1) for x in (q, k))
    v, g = chunks(v), chunks(g[..., None])[..., 0]
    L = _between(g)                                                     # [B, H, N, C, C]
    first = torch.exp(g.cumsum(-1))                                     # the decay from a chunk's start to each position
    o = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * L, v)
    own_states = torch.matmul((k * L[..., -1, :, None]).transpose(-1, -2), v)
    S0 = torch.zeros(B, H, dk, dv, device="cuda") if s["state"] is None else s["state"]
    at = None if s["slots"] is None else s["slots"].long()
    if at is not None:
        S0 = S0[at]
    across = _between(torch.nn.functional.pad(g.sum(-1), (1, 0)))       # [B, H, N + 1, N + 1]: S_0, then each chunk's own
    states = torch.matmul(across, torch.cat([S0[:, :, None], own_states], 2).reshape(B, H, N + 1, dk * dv)).view(B, H, N + 1, dk, dv)
    o = dk ** -0.5 * (o + first[..., None] * torch.matmul(q, states[:, :, :N]))
    o = o.permute(0, 2, 3, 1, 4).reshape(B, N * CHUNK, H, dv)[:, :T].to(s["v"].dtype)
    new = states[:, :, N]
    if s["offsets"] is not None:
        o = torch.zeros_like(s["v"]).index_put_((rows[there],), o[there])
    if at is not None:
        new = torch.empty_like(new).index_copy_(0, at, new)
    return {"out": o, "state": new}


def run(s):
    c = s["case"]
    if not own:
        return {"prompt": _prompts, "step": _steps, "norm": _norms}[c["kind"]](s)
    if c["kind"] == "norm":
        total, y = s["handle"].norm_gate_residual(
            s["x"], s["weight"], bias=s["bias"], norm=c["norm"], groups=c["groups"], eps=1e-6, gate=s["gate"], gate_act=c["gate"],
            residual=s["residual"], scale=0.5 if c["residual"] else 1.0, channel_scale=s["channel_scale"], next_norm=c["next"],
            next_weight=s["next_weight"], next_bias=s["next_bias"])
        return {"sum": total} if y is None else {"sum": total, "y": y}
    if c["kind"] == "step":
        s["layer"].step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], state_out=s["new_state"], slots=s["slots"], out=s["out"])
    else:
        s["layer"].forward(s["q"], s["k"], s["v"], s["log_decay"], state=s["state"], state_out=s["new_state"], offsets=s["offsets"],
                           slots=s["slots"], out=s["out"])
    return {"out": s["out"], "state": s["new_state"]}


# ------------------------------------------------------ the work, and 64 bits
def work(case):
    c = case
    size = 2 if c["dtype"] == "bf16" else 4
    if c["kind"] == "norm":
        n = c["rows"] * c["width"]
        tensors = 2 + (c["gate"] != "none") + c["residual"] + (c["next"] != "none")
        return {"bytes": n * size * tensors, "flops": n * (5 + 2 * (c["gate"] != "none") + 2 * c["residual"] + 5 * (c["next"] != "none"))}
    H, dk, dv = c["heads"], c["key_dim"], c["value_dim"]
    tokens = c["batch"] if c["kind"] == "step" else sum(_lengths(c))
    states = 2 if c["kind"] == "step" or c["initial"] else 1
    b = tokens * size * (2 * c["key_heads"] * dk + 2 * H * dv) + 4 * H * (tokens if c["decay"] == "token" else 1)
    return {"bytes": b + states * 4 * c["batch"] * H * dk * dv, "flops": 4 * dk * dv * H * tokens}


def _exact_norm(x, mode, groups, weight, bias):
    parts = x.reshape(x.shape[0] * groups, -1)
    mean = parts.mean(1, keepdim=True) if mode == "layer" else torch.zeros_like(parts[:, :1])
    power = ((parts - mean) ** 2).mean(1, keepdim=True)
    out = ((parts - mean) / torch.sqrt(power + 1e-6)).reshape(x.shape) * weight.double()
    return out if bias is None else out + bias.double()


def exact(case, seed):
    s, c = _inputs(case, seed), case
    if c["kind"] == "norm":
        u = _exact_norm(s["x"].double(), c["norm"], c["groups"], s["weight"], s["bias"])
        if c["gate"] != "none":
            z = s["gate"].double()
            u = u / (1 + torch.exp(-z)) * (z if c["gate"] == "silu" else 1)
        if c["residual"]:
            u = s["residual"].double() + 0.5 * s["channel_scale"].double() * u
        return {"sum": u} if c["next"] == "none" else {"sum": u, "y": _exact_norm(u, c["next"], 1, s["next_weight"], s["next_bias"])}
    B, H, dk, dv = c["batch"], c["heads"], c["key_dim"], c["value_dim"]
    head = torch.arange(H, device="cuda") // (H // c["key_heads"])
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device="cuda")
    order = s["slots"].long() if s["slots"] is not None else torch.arange(B, device="cuda")
    S = s["state"].double()[order] if s["state"] is not None else torch.zeros(B, H, dk, dv, dtype=torch.float64, device="cuda")
    n = [1] * B if c["kind"] == "step" else s["lengths"]
    start = [sum(n[:i]) for i in range(B)]
    flat = {name: s[name].reshape(-1, *s[name].shape[-2:]) for name in ("q", "k", "v")}
    g = torch.exp(s["log_decay"].double().reshape(-1, H))
    by_length = sorted(range(B), key=lambda b: -n[b])
    S = S[by_length]
    start = torch.tensor([start[b] for b in by_length], device="cuda")
    flat_out = out.view(-1, H, dv)
    for t in range(max(n)):        # token by token, over the sequences that are still running
        live = sum(x > t for x in n)
        at = start[:live] + t
        q, k = (flat[name][at][:, head].double() for name in ("q", "k"))
        decay = g[at] if c["decay"] == "token" else g.expand(live, H)
        S[:live] = decay[..., None, None] * S[:live] + k[..., :, None] * flat["v"][at].double()[..., None, :]
        flat_out[at] = dk ** -0.5 * (q[..., :, None] * S[:live]).sum(-2)
    new = torch.empty_like(S)
    new[order[by_length]] = S
    return {"out": out, "state": new}
