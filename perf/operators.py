"""The learner's feed-forward operators as workloads: layer norm, counter-based dropout and the gated linear layer.

``run`` computes them in plain 32-bit torch operations, or (``own`` true) through ``gsc_amd.ops``.  The three make up
the residual feed-forward block of the actor and critic; the sizes are those of an acting batch (1 to a few hundred
rows), of a DDPG update (100 samples per environment step: 100 to 25,600 rows) and of wider networks.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------------------------
# cases

def _norm(name, rows, cols, dtype, train):
    return {"name": name, "op": "layer_norm", "rows": rows, "cols": cols, "dtype": dtype, "train": train}


def _drop(name, rows, cols, dtype, p, residual):
    return {"name": name, "op": "dropout", "rows": rows, "cols": cols, "dtype": dtype, "p": p, "residual": residual,
            "train": True}


def _gated(name, rows, d, f, dtype, act, train):
    return {"name": name, "op": "gated_linear", "rows": rows, "d": d, "f": f, "dtype": dtype, "act": act, "train": train}


def listed():
    return [
        # greedy action of one environment: one row of the actor's 256-wide hidden layer (latency)
        _norm("norm act 1x256 bf16", 1, 256, "bf16", False),
        # one update of 256 environments (100 samples each) through the 256-wide actor
        _norm("norm update 25600x256 bf16", 25600, 256, "bf16", True),
        # odd row count and row length, 32-bit learner
        _norm("norm odd 8191x1003 fp32", 8191, 1003, "fp32", True),
        # wide layer, bandwidth
        _norm("norm wide 16384x8192 bf16", 16384, 8192, "bf16", True),
        # the reference's update: 100 samples, 64-wide critic (latency)
        _drop("drop update 100x64 bf16", 100, 64, "bf16", 0.1, False),
        # residual branch of the 256-environment update
        _drop("drop update 25600x256 bf16", 25600, 256, "bf16", 0.1, True),
        # odd and large, 32-bit learner
        _drop("drop odd 25601x2047 fp32", 25601, 2047, "fp32", 0.35, False),
        # greedy action of one environment through a 4x wider gated layer (one row: reads the weights)
        _gated("gated act 1x256x1024 bf16", 1, 256, 1024, "bf16", "silu", False),
        # a few rows through a wide gated layer (bound by the weights)
        _gated("gated act 8x2048x8192 bf16", 8, 2048, 8192, "bf16", "gelu", False),
        # one update of 256 environments through a 4x wider gated layer
        _gated("gated update 25600x256x1024 bf16", 25600, 256, 1024, "bf16", "silu", True),
        # wide gated layer (matrix products)
        _gated("gated wide 8192x2048x8192 bf16", 8192, 2048, 8192, "bf16", "gelu", True),
        # odd sizes, 32-bit learner
        _gated("gated odd 2500x257x515 fp32", 2500, 257, 515, "fp32", "sigmoid", True),
    ]


def _log_int(rng, lo, hi):
    """A whole number in lo .. hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("layer_norm", "dropout", "gated_linear"))
    dtype = rng.choice(("bf16", "bf16", "fp32"))
    if op == "layer_norm":
        cols = _log_int(rng, 16, 16384)
        rows = _log_int(rng, 1, min(32768, 128 * 1024 * 1024 // (cols * (2 if dtype == "fp32" else 1))))
        case = _norm("", rows, cols, dtype, rng.random() < 0.75)
    elif op == "dropout":
        cols = _log_int(rng, 1, 8192)
        rows = _log_int(rng, 1, min(32768, 25601 * 2047 // cols))
        case = _drop("", rows, cols, dtype, round(rng.uniform(0.0, 0.9), 4), rng.random() < 0.5)
    else:
        act = rng.choice(("silu", "gelu", "sigmoid"))
        d, f = _log_int(rng, 16, 4096), _log_int(rng, 16, 8192)
        if rng.random() < 0.4:
            case = _gated("", _log_int(rng, 1, 512), d, f, dtype, act, False)
        else:
            most = 8192 * 2048 * 8192 // (16 if dtype == "fp32" else 1)
            case = _gated("", _log_int(rng, 32, max(32, min(25600, most // (d * f)))), d, f, dtype, act, True)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------------------
# inputs

def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(bound, *shape):
        return torch.rand(*shape, generator=g, device="cuda").mul_(2 * bound).sub_(bound)

    if case["op"] == "layer_norm":
        rows, cols = case["rows"], case["cols"]
        # pre-activations of a linear layer: a mean of its own and about unit spread per row; the weight and bias of a
        # layer under training are the learner's 32-bit masters
        s = {"x": (normal(rows, cols) + 0.5 * normal(rows, 1)).to(dtype), "w": 1 + 0.1 * normal(cols),
             "b": 0.1 * normal(cols)}
        leaves = ("x", "w", "b")
        if train:
            s["dy"] = (0.01 * normal(rows, cols)).to(dtype)
    elif case["op"] == "dropout":
        rows, cols = case["rows"], case["cols"]
        s = {"x": normal(rows, cols).to(dtype), "dy": (0.01 * normal(rows, cols)).to(dtype), "seed": 977 * int(seed) + 5,
             "offset": (1 << 33) + int(seed) % 1000}
        if case["residual"]:
            s["res"] = normal(rows, cols).to(dtype)
        leaves = ("x", "res")
    else:
        rows, d, f = case["rows"], case["d"], case["f"]
        # normalised activations; weights and bias drawn as a linear layer's are
        s = {"x": normal(rows, d).to(dtype), "w": uniform(1 / math.sqrt(d), 2 * f, d).to(dtype),
             "b": uniform(1 / math.sqrt(d), 2 * f).to(dtype)}
        leaves = ("x", "w", "b")
        if train:
            s["dh"] = (0.01 * normal(rows, f)).to(dtype)
    if train:
        for k in leaves:
            if k in s:
                s[k].requires_grad_(True)
    return {"case": case, **s}


# ---------------------------------------------------------------------------------------------------------------
# plain forms

def _plain_norm(s):
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    xf = x.float()
    centred = xf - xf.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    xh = centred * rstd
    y = (xh * w + b).to(x.dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return {"y": y, "dx": dx.to(x.dtype), "dw": (dy * xh).sum(0), "db": dy.sum(0)}


def _words(group, seed, offset, second):
    """Philox4x32-10 blocks of the groups: [groups, 4] 32-bit words held in 64."""
    low = 0xFFFFFFFF
    k0, k1 = seed & low, (seed >> 32) & low
    c0, c1 = group & low, group >> 32
    c2 = torch.full_like(group, offset & low)
    c3 = torch.full_like(group, (offset >> 32) | (second << 31))
    for _ in range(10):
        p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((p1 >> 32) & low) ^ c1 ^ k0, p1 & low, ((p0 >> 32) & low) ^ c3 ^ k1, p0 & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), -1)


def _plain_keep(n, p, seed, offset, device):
    """Which of n elements stay: a 32-bit uniform of each, 8 elements to a pair of blocks."""
    group = torch.arange(-(-n // 8), device=device)
    a, b = _words(group, seed, offset, 0), _words(group, seed, offset, 1)
    u = torch.stack((((a & 0xFFFF) << 16) | (b & 0xFFFF), ((a >> 16) << 16) | (b >> 16)), -1)
    return u.reshape(-1)[:n] >= min(round(p * 2.0 ** 32), 2 ** 32 - 1)


def _plain_dropout(s):
    x, p = s["x"].detach(), s["case"]["p"]
    keep = _plain_keep(x.numel(), p, s["seed"], s["offset"], x.device).view(x.shape)
    scale = 1.0 / (1.0 - p)
    zero = torch.zeros((), device=x.device)
    y = torch.where(keep, x.float() * scale, zero)
    out = {"dx": torch.where(keep, s["dy"].float() * scale, zero).to(x.dtype)}
    if "res" in s:
        y = y + s["res"].detach().float()
        out["dres"] = s["dy"]
    return {"y": y.to(x.dtype), **out}


def _plain_act(g, act):
    """act(g) and its derivative."""
    if act == "gelu":
        phi = 0.5 * (1 + torch.erf(g * math.sqrt(0.5)))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))
    sg = 1 / (1 + torch.exp(-g))
    if act == "sigmoid":
        return sg, sg * (1 - sg)
    return g * sg, sg * (1 + g * (1 - sg))


def _plain_gated(s):
    x, w, b = s["x"].detach(), s["w"].detach(), s["b"].detach()
    xf, wf, f = x.float(), w.float(), s["case"]["f"]
    gu = xf @ wf.t() + b.float()
    g, u = gu[:, :f], gu[:, f:]
    a, da = _plain_act(g, s["case"]["act"])
    h = (a * u).to(x.dtype)
    if not s["case"]["train"]:
        return {"h": h}
    dh = s["dh"].float()
    dgu = torch.cat((dh * u * da, dh * a), 1)
    return {"h": h, "dx": (dgu @ wf).to(x.dtype), "dw": (dgu.t() @ xf).to(w.dtype), "db": dgu.sum(0).to(b.dtype)}


# ---------------------------------------------------------------------------------------------------------------
# one pass

def _own(s):
    from gsc_amd import ops
    case = s["case"]
    if case["op"] == "layer_norm":
        y = ops.layer_norm(s["x"], s["w"], s["b"], EPS)
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if case["op"] == "dropout":
        y = ops.dropout(s["x"], case["p"], s["seed"], s["offset"], residual=s.get("res"))
        if "res" in s:
            dx, dres = torch.autograd.grad(y, (s["x"], s["res"]), s["dy"])
            return {"y": y, "dx": dx, "dres": dres}
        return {"y": y, "dx": torch.autograd.grad(y, s["x"], s["dy"])[0]}
    h = ops.gated_linear(s["x"], s["w"], s["b"], activation=case["act"])
    if not case["train"]:
        return {"h": h}
    dx, dw, db = torch.autograd.grad(h, (s["x"], s["w"], s["b"]), s["dh"])
    return {"h": h, "dx": dx, "dw": dw, "db": db}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return {"layer_norm": _plain_norm, "dropout": _plain_dropout, "gated_linear": _plain_gated}[state["case"]["op"]](state)


def work(case):
    es, train = (2 if case["dtype"] == "bf16" else 4), case["train"]
    if case["op"] == "layer_norm":
        n, c = case["rows"] * case["cols"], case["cols"]
        # x, y (and dy, dx); weight, bias (and their gradients) in 32 bits
        return {"bytes": n * es * (4 if train else 2) + 4 * c * (4 if train else 2), "flops": n * (20 if train else 8)}
    if case["op"] == "dropout":
        n = case["rows"] * case["cols"]
        return {"bytes": n * es * (5 if case["residual"] else 4), "flops": n * 4}
    m, d, f = case["rows"], case["d"], case["f"]
    once = m * d + 2 * f * d + 2 * f + m * f   # x, weight, bias, h: each again as a gradient in training
    return {"bytes": once * es * (2 if train else 1), "flops": m * d * f * (12 if train else 4)}


# ---------------------------------------------------------------------------------------------------------------
# 64 bits, from the definitions

def _exact_blocks(groups, seed, offset, top):
    """Philox4x32-10 in numpy: the four words of each group's block, in 32 bits."""
    m32, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    i = np.arange(groups, dtype=np.uint64)
    x = [i & m32, i >> sh, np.full(groups, offset & 0xFFFFFFFF, np.uint64),
         np.full(groups, (offset >> 32) + (top << 31), np.uint64)]
    for r in range(10):
        key = [np.uint64(((seed & 0xFFFFFFFF) + r * 0x9E3779B9) & 0xFFFFFFFF),
               np.uint64(((seed >> 32) + r * 0xBB67AE85) & 0xFFFFFFFF)]
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> sh) ^ x[1] ^ key[0], b & m32, (a >> sh) ^ x[3] ^ key[1], a & m32]
    return np.ascontiguousarray(np.stack(x, 1).astype("<u4"))


def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "dropout":
        n, p = case["rows"] * case["cols"], case["p"]
        groups = -(-n // 8)
        # little-endian halves of the blocks: element j of a group has half j of both
        hi = _exact_blocks(groups, s["seed"], s["offset"], 0).view("<u2").reshape(-1)[:n].astype(np.uint32)
        lo = _exact_blocks(groups, s["seed"], s["offset"], 1).view("<u2").reshape(-1)[:n]
        u = hi * np.uint32(65536) + lo
        kept = torch.from_numpy(u >= np.uint32(min(round(p * 2.0 ** 32), 2 ** 32 - 1))).to("cuda").view(case["rows"], -1)
        y = (wide["x"] / (1 - p)).masked_fill_(~kept, 0.0)
        out = {"dx": (wide["dy"] / (1 - p)).masked_fill_(~kept, 0.0)}
        if case["residual"]:
            y += wide["res"]
            out["dres"] = wide["dy"]
        return {"y": y, **out}
    for k in ("x", "w", "b"):
        wide[k].requires_grad_(case["train"])
    x, w, b = wide["x"], wide["w"], wide["b"]
    if case["op"] == "layer_norm":
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y, names = (x - mean) / (var + EPS) ** 0.5 * w + b, ("y", "dx", "dw", "db")
        dy = wide.get("dy")
    else:
        f = case["f"]
        g, u = x.matmul(w[:f].t()) + b[:f], x.matmul(w[f:].t()) + b[f:]
        a = {"silu": lambda t: t * torch.sigmoid(t), "sigmoid": torch.sigmoid,
             "gelu": lambda t: t * torch.special.ndtr(t)}[case["act"]](g)
        y, names = a * u, ("h", "dx", "dw", "db")
        dy = wide.get("dh")
    if not case["train"]:
        return {names[0]: y}
    return dict(zip(names, (y.detach(), *torch.autograd.grad(y, (x, w, b), dy))))
