"""The attention-block operators over voxel tokens, as cases to be timed and compared.

Four operators, in the order in which a transformer block over the rows of a SparseTensor uses them:

- ``linear``: y = act(x @ w^T + bias) + residual
- ``rope``: rotary positions over the voxel axes x, y, z
- ``qk_norm_rope``: RMS norm of every head of q and k with its own gains, and the rotation, in one pass
- ``attention``: softmax(q k^T * scale) v inside each sequence of a ragged batch

``run`` computes them with elementary torch operations in 32 bits, or, where ``own`` is set, through t2sc.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6
THETA = 10000.0


def _t2sc():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trellis2-mojo_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import t2sc
    return t2sc


# ---- cases ----

def listed():
    return [
        # the modulation vector of one shape: a single row against a weight that is only streamed
        {"name": "linear one row", "op": "linear", "rows": 1, "ci": 1536, "co": 9216, "act": "silu", "bias": True,
         "residual": False, "dtype": "bf16"},
        # packed q, k, v of a 32^3 stage's tokens
        {"name": "linear qkv 1941", "op": "linear", "rows": 1941, "ci": 1536, "co": 4608, "act": "none", "bias": True,
         "residual": False, "dtype": "bf16"},
        # the feed-forward's first product over the cascade's tokens
        {"name": "linear gelu 23024", "op": "linear", "rows": 23024, "ci": 1536, "co": 6144, "act": "gelu",
         "bias": True, "residual": False, "dtype": "bf16"},
        # the feed-forward's second product with the block's residual, at the token budget, odd row count
        {"name": "linear residual 49151 f16", "op": "linear", "rows": 49151, "ci": 4096, "co": 1024, "act": "none",
         "bias": True, "residual": True, "dtype": "f16"},
        # queries of a small stage: launch latency counts
        {"name": "rope 509", "op": "rope", "rows": 509, "heads": 12, "dim": 128, "layout": "pairs", "dtype": "bf16"},
        # every token of the budget, rotated in f32
        {"name": "rope 49152 f32", "op": "rope", "rows": 49152, "heads": 16, "dim": 64, "layout": "halves",
         "dtype": "f32"},
        # q and k slices of a packed projection, 32^3 stage
        {"name": "qk norm rope 1941", "op": "qk_norm_rope", "rows": 1941, "heads": 12, "dim": 128, "layout": "pairs",
         "packed": True, "dtype": "bf16"},
        # an odd row count above the token budget, separate q and k
        {"name": "qk norm rope 100003 f16", "op": "qk_norm_rope", "rows": 100003, "heads": 16, "dim": 64,
         "layout": "pairs", "packed": False, "dtype": "f16"},
        # one pooling query over every voxel token: reads k and v once
        {"name": "attention 1 x 49152", "op": "attention", "q": "1", "kv": "49152", "heads": 16, "dim": 64,
         "packed": False, "dtype": "bf16"},
        # self-attention of two shapes of a 32^3 stage, ragged
        {"name": "attention 1203+738", "op": "attention", "q": "1203,738", "kv": "1203,738", "heads": 12, "dim": 128,
         "packed": True, "dtype": "bf16"},
        # self-attention over the cascade's tokens
        {"name": "attention 23024", "op": "attention", "q": "23024", "kv": "23024", "heads": 12, "dim": 128,
         "packed": True, "dtype": "bf16"},
        # cross-attention of two shapes' tokens to their image tokens
        {"name": "attention cross f16", "op": "attention", "q": "12011,9877", "kv": "1029,1029", "heads": 16,
         "dim": 64, "packed": False, "dtype": "f16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "rope", "qk_norm_rope", "attention"])
    if op == "linear":
        rows, ci, co = _log(rng, 1, 60000), 8 * _log(rng, 8, 768), 8 * _log(rng, 1, 1152)
        if rng.random() < 0.2:
            co += rng.randint(1, 7)
        while rows * ci * co > 23024 * 1536 * 6144:
            rows = rows // 2 + 1
        return {"op": op, "rows": rows, "ci": ci, "co": co, "act": rng.choice(["none", "silu", "gelu"]),
                "bias": rng.random() < 0.7, "residual": rng.random() < 0.5, "dtype": rng.choice(["bf16", "f16"])}
    heads, dim = rng.randint(1, 24), rng.choice([32, 64, 64, 80, 96, 128, 128])
    if op in ("rope", "qk_norm_rope"):
        case = {"op": op, "rows": _log(rng, 1, 100000), "heads": heads, "dim": dim,
                "layout": rng.choice(["pairs", "halves"]), "dtype": rng.choice(["bf16", "f16", "f32"])}
        if op == "qk_norm_rope":
            case["packed"] = rng.random() < 0.5
        return case
    batch = rng.choice([1, 1, 2, 3, 5])
    same = rng.random() < 0.5
    q = [_log(rng, 1, 12000) for _ in range(batch)]
    kv = list(q) if same else [rng.choice([0, 1]) if rng.random() < 0.1 else _log(rng, 1, 30000) for _ in range(batch)]
    # the plain form pads a batch to its longest sequences
    while heads * dim * batch * max(q) * max(kv) > 12 * 128 * 23024 * 23024 // 4 or heads * batch * max(q) * max(kv) > 3 << 30:
        q = [n // 2 + 1 for n in q]
        kv = list(q) if same else [n // 2 for n in kv]
    return {"op": op, "q": ",".join(map(str, q)), "kv": ",".join(map(str, kv)), "heads": heads, "dim": dim,
            "packed": same and rng.random() < 0.5, "dtype": rng.choice(["bf16", "f16"])}


def _lens(text):
    return [int(n) for n in text.split(",")]


def work(case):
    s = SIZES[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["rows"], case["ci"], case["co"]
        return {"bytes": s * (m * k + n * k + m * n * (2 if case["residual"] else 1)) + (4 * n if case["bias"] else 0),
                "flops": 2 * m * n * k}
    values = case["heads"] * case["dim"]
    if case["op"] == "rope":
        return {"bytes": case["rows"] * (2 * values * s + 12), "flops": 3 * case["rows"] * values}
    if case["op"] == "qk_norm_rope":
        return {"bytes": case["rows"] * (4 * values * s + 12) + 8 * values, "flops": 14 * case["rows"] * values}
    q, kv = _lens(case["q"]), _lens(case["kv"])
    return {"bytes": 2 * values * s * (sum(q) + sum(kv)), "flops": 4 * values * sum(a * b for a, b in zip(q, kv))}


# ---- inputs ----

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)

    s = {"case": case}
    if case["op"] == "linear":
        m, k, n = case["rows"], case["ci"], case["co"]
        s["x"], s["w"] = normal(m, k), normal(n, k, std=k ** -0.5)
        s["bias"] = normal(n, std=0.1, dtype=torch.float32) if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
        s["act"] = None if case["act"] == "none" else case["act"]
    elif case["op"] in ("rope", "qk_norm_rope"):
        m, h, d = case["rows"], case["heads"], case["dim"]
        s["coords"] = torch.randint(0, 1024, (m, 4), generator=g, device="cuda", dtype=torch.int32)
        s["coords"][:, 0] = 0
        if case["op"] == "rope":
            s["x"] = normal(m, h, d)
        else:
            if case["packed"]:
                qkv = normal(m, 3, h, d, std=0.7)
                s["q"], s["k"] = qkv[:, 0], qkv[:, 1]
            else:
                s["q"], s["k"] = normal(m, h, d, std=0.7), normal(m, h, d, std=1.8)
            s["gq"] = 1 + normal(h, d, std=0.2, dtype=torch.float32)
            s["gk"] = 1 + normal(h, d, std=0.2, dtype=torch.float32)
        # angles of an axis fall geometrically over its pairs; pairs that no axis takes are not rotated
        n = d // 2 // 3
        s["freqs"] = THETA ** (-torch.arange(n, device="cuda", dtype=torch.float64) / n)
        if own:
            t2sc = _t2sc()
            s["ctx"] = t2sc.Context.default(0)
            s["ctx"].use_torch_stream()
            s["rope"] = t2sc.RotaryPositionEmbedder(d, theta=THETA, layout=case["layout"], ctx=s["ctx"])
    else:
        q, kv = _lens(case["q"]), _lens(case["kv"])
        h, d = case["heads"], case["dim"]
        if case["packed"]:
            qkv = normal(sum(q), 3, h, d, std=1.2)
            s["q"], s["k"], s["v"] = qkv[:, 0], qkv[:, 1], qkv[:, 2]
        else:
            s["q"], s["k"], s["v"] = normal(sum(q), h, d, std=1.2), normal(sum(kv), h, d, std=1.2), normal(sum(kv), h, d)
        s["scale"] = d ** -0.5
        if own:
            t2sc = _t2sc()
            s["ctx"] = t2sc.Context.default(0)
            s["ctx"].use_torch_stream()
            s["layout"] = t2sc.SequenceLayout(q, kv, ctx=s["ctx"])
        else:
            s["rows"], s["q_at"], _ = _padded(q)
            _, s["kv_at"], s["kv_there"] = _padded(kv)
    if own and case["op"] == "linear":
        s["ctx"] = _t2sc().Context.default(0)
        s["ctx"].use_torch_stream()
    return s


def _padded(lens):
    """Where a ragged batch's rows stand in a padded one: (row -> place [sum], place -> row [B, L], which places hold a row [B, L])."""
    n = torch.tensor(lens, device="cuda")
    at = torch.arange(max(lens), device="cuda")
    there = at[None, :] < n[:, None]
    rows = (torch.cumsum(n, 0) - n)[:, None] + at[None, :]
    return there.reshape(-1).nonzero()[:, 0], torch.where(there, rows, 0), there


# ---- the operators ----

def run(s):
    op = s["case"]["op"]
    if op == "linear":
        return _linear(s)
    if op == "rope":
        return _rope(s)
    if op == "qk_norm_rope":
        return _qk_norm_rope(s)
    return _attention(s)


def _linear(s):
    if own:
        return _t2sc().dense_linear_device(s["x"], s["w"], s["bias"], activation=s["act"], residual=s["residual"],
                                           ctx=s["ctx"])
    y = s["x"].float() @ s["w"].float().T
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["act"] == "silu":
        y = y / (1 + torch.exp(-y))
    elif s["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(s["x"].dtype)


def _rotate(x, s):
    """x: f32 [rows, heads, dim]; the angles in 64 bits."""
    n, half = s["freqs"].numel(), x.shape[-1] // 2
    angle = (s["coords"][:, 1:].double()[:, :, None] * s["freqs"]).reshape(x.shape[0], 1, 3 * n)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    if s["case"]["layout"] == "pairs":
        a, b = x[..., 0:6 * n:2], x[..., 1:6 * n:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
        return torch.cat((turned, x[..., 6 * n:]), -1)
    a, b = x[..., :3 * n], x[..., half:half + 3 * n]
    return torch.cat((a * cos - b * sin, x[..., 3 * n:half], a * sin + b * cos, x[..., half + 3 * n:]), -1)


def _rope(s):
    if own:
        return s["rope"].forward_device(s["x"], s["coords"])
    return _rotate(s["x"].float(), s).to(s["x"].dtype)


def _norm(x, gain):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * gain


def _qk_norm_rope(s):
    if own:
        return _t2sc().qk_norm_rope_device(s["q"], s["k"], s["gq"], s["gk"], s["coords"], s["rope"], eps=EPS)
    dt = s["q"].dtype
    return _rotate(_norm(s["q"].float(), s["gq"]), s).to(dt), _rotate(_norm(s["k"].float(), s["gk"]), s).to(dt)


def _attention(s):
    if own:
        return s["layout"].attention_device(s["q"], s["k"], s["v"], scale=s["scale"])
    h, d = s["case"]["heads"], s["case"]["dim"]
    b, lq = s["q_at"].shape
    lk = s["kv_at"].shape[1]
    q = s["q"][s["q_at"]].float().transpose(1, 2) if lq else s["q"].float().reshape(b, h, 0, d)
    if lk == 0:
        return torch.zeros_like(s["q"], memory_format=torch.contiguous_format)
    there = s["kv_there"][:, None, :, None]
    k = s["k"][s["kv_at"]].float().transpose(1, 2)
    v = (s["v"][s["kv_at"]].float().transpose(1, 2) * there)
    p = (q @ k.transpose(-1, -2)).mul_(s["scale"])
    p.masked_fill_(~s["kv_there"][:, None, None, :], -math.inf)
    p.sub_(p.amax(-1, keepdim=True).clamp_(min=-3e38)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p @ v) / torch.where(total > 0, total, 1)
    return out.transpose(1, 2).reshape(b * lq, h, d)[s["rows"]].to(s["q"].dtype)


# ---- the same from the definitions, in 64 bits ----

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        # blocks of rows, so that a large case's f64 products stay small
        w, out = s["w"].double(), []
        for at in range(0, case["rows"], 8192):
            z = torch.nn.functional.linear(s["x"][at:at + 8192].double(), w,
                                           None if s["bias"] is None else s["bias"].double())
            if case["act"] == "silu":
                z = z * torch.sigmoid(z)
            elif case["act"] == "gelu":
                z = torch.nn.functional.gelu(z, approximate="tanh")
            if s["residual"] is not None:
                z = z + s["residual"][at:at + 8192].double()
            out.append(z)
        return torch.cat(out)
    if case["op"] in ("rope", "qk_norm_rope"):
        n, d = case["dim"] // 6, case["dim"]
        turn = torch.ones(case["rows"], d // 2, dtype=torch.complex128, device="cuda")
        for axis in range(3):
            for j in range(n):
                angle = s["coords"][:, 1 + axis].double() * math.exp(-math.log(THETA) * j / n)
                turn[:, axis * n + j] = torch.polar(torch.ones_like(angle), angle)

        def rotated(x):
            if case["layout"] == "pairs":
                z = torch.view_as_complex(x.reshape(*x.shape[:-1], d // 2, 2)) * turn[:, None]
                return torch.view_as_real(z).flatten(-2)
            z = torch.complex(x[..., :d // 2], x[..., d // 2:]) * turn[:, None]
            return torch.cat((z.real, z.imag), -1)

        if case["op"] == "rope":
            return rotated(s["x"].double())
        both = []
        for x, gain in ((s["q"], s["gq"]), (s["k"], s["gk"])):
            x = x.double()
            rms = torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / d + EPS)
            both.append(rotated(x / rms * gain.double()))
        return tuple(both)
    out, q0, k0 = [], 0, 0
    for a, b in zip(_lens(case["q"]), _lens(case["kv"])):
        o = torch.zeros(a, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for h in range(case["heads"] if b else 0):
            k, v = s["k"][k0:k0 + b, h].double(), s["v"][k0:k0 + b, h].double()
            for at in range(0, a, 8192):
                p = torch.softmax(s["q"][q0 + at:min(q0 + at + 8192, q0 + a), h].double() @ k.T * s["scale"], -1)
                o[at:at + 8192, h] = p @ v
        out.append(o)
        q0, k0 = q0 + a, k0 + b
    return torch.cat(out)
