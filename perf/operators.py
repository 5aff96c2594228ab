"""Cases that time the training and streaming operators of the engine.

Three operators around a temporal block: the gated linear recurrence over
time (with its backward pass and its single-step form), group norm with an
activation on channels-last tensors (with its backward pass), and dropout
from a counter-based generator, with the residual added (with its backward
pass).  `run` computes a case in its plain form (elementary torch operations)
or, with `own` true, through the engine's public calls; `exact` gives the
results from the definitions in 64 bits.
"""
import math

import numpy as np
import torch

own = False

_DEV = "cuda"
_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---------------------------------------------------------------------- cases
def _recurrence(name, layout, batch, length, width, form, dtype, train, ragged=False):
    return {"name": name, "op": "recurrence", "layout": layout, "batch": batch, "length": length, "width": width,
            "form": form, "dtype": dtype, "train": train, "ragged": ragged}


def _norm(name, samples, positions, channels, groups, act, dtype, train):
    return {"name": name, "op": "group_norm", "samples": samples, "positions": positions, "channels": channels,
            "groups": groups, "act": act, "dtype": dtype, "train": train}


def _dropout(name, rows, width, p, residual, dtype, train):
    return {"name": name, "op": "dropout", "rows": rows, "width": width, "p": p, "residual": residual,
            "dtype": dtype, "train": train}


def listed():
    return [
        # streaming: one new time plane of one sample (64 tokens of width 128) against the kept state
        {"name": "step_64x128", "op": "step", "rows": 64, "width": 128, "form": "leaky", "dtype": "fp32"},
        # the batch-512 model's chunk of 64 samples: 4 time planes of 64 x 1024 tokens, inference
        _recurrence("planes_4x65536x512", "planes", 65536, 4, 512, "leaky", "fp32", False),
        # training on long event streams: few sequences, the parallel work lies along time
        _recurrence("stream_4x32768x512", "sequence", 4, 32768, 512, "leaky", "bf16", True),
        # a padded batch of odd lengths (an empty one and one of a single step among them) and an odd width
        _recurrence("ragged_13x1021x197", "sequence", 13, 1021, 197, "gate", "fp16", True, True),
        # streaming: the three planes of one sample of the small model
        _norm("norm_3x64x128", 3, 64, 128, 8, "silu", "fp32", False),
        # a training batch of 256 samples of the small model, 3 planes each
        _norm("norm_768x64x128", 768, 64, 128, 8, "silu", "bf16", True),
        # the batch-512 model's chunk of 64 samples, 4 planes each, inference
        _norm("norm_256x1024x512", 256, 1024, 512, 32, "silu", "fp32", False),
        # few long samples with odd positions and odd groups
        _norm("norm_5x3001x330", 5, 3001, 330, 10, "none", "fp16", True),
        # training on long event streams: each sample far larger than one SM's memory
        _norm("norm_4x32768x512", 4, 32768, 512, 32, "silu", "bf16", True),
        # streaming sizes: the input of one sample's three planes
        _dropout("dropout_192x128", 192, 128, 0.1, False, "fp32", False),
        # the residual branch of the batch-512 model's chunk in training
        _dropout("dropout_262144x512", 262144, 512, 0.1, True, "bf16", True),
        # an odd number of elements
        _dropout("dropout_9973x331", 9973, 331, 0.25, True, "fp16", True),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    most = 1 << 25  # elements: below the largest listed cases of each operator
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    kind = rng.choice(["step", "recurrence", "recurrence", "recurrence", "group_norm", "group_norm", "group_norm",
                       "dropout", "dropout"])
    if kind == "step":
        return {"op": "step", "rows": _log_int(rng, 1, 8192), "width": _log_int(rng, 1, 2048),
                "form": rng.choice(["leaky", "gate"]), "dtype": dtype}
    if kind == "recurrence":
        layout = rng.choice(["planes", "sequence"])
        width = _log_int(rng, 1, 1536)
        if layout == "planes":
            length = _log_int(rng, 1, 64)
            batch = _log_int(rng, 1, max(1, min(65536, most // (length * width))))
        else:
            length = _log_int(rng, 1, 32768)
            batch = _log_int(rng, 1, max(1, min(512, most // (length * width))))
        c = _recurrence("", layout, batch, length, width, rng.choice(["leaky", "gate"]), dtype, rng.random() < 0.6,
                        rng.random() < 0.3)
    elif kind == "group_norm":
        groups = _log_int(rng, 1, 64)
        channels = groups * _log_int(rng, 1, 48)
        positions = _log_int(rng, 1, 32768)
        samples = _log_int(rng, 1, max(1, min(1024, most // (positions * channels))))
        c = _norm("", samples, positions, channels, groups, rng.choice(["none", "silu"]), dtype, rng.random() < 0.6)
    else:
        width = _log_int(rng, 1, 2048)
        rows = _log_int(rng, 1, most // width)
        c = _dropout("", rows, width, rng.choice([0.0, 0.05, 0.1, 0.5, round(rng.random(), 3)]), rng.random() < 0.7,
                     dtype, rng.random() < 0.6)
    del c["name"]
    return c


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "step":  # x, gate and the fp32 state in; the output and the new state out
        n = case["rows"] * case["width"]
        return {"bytes": n * (3 * size + 8), "flops": 6 * n}
    if case["op"] == "recurrence":  # x, gate, (grad of h) in; h, (grads of x and gate) out; states fp32
        n = case["batch"] * case["length"] * case["width"]
        state = case["batch"] * case["width"]
        if case["train"]:
            return {"bytes": 6 * n * size + 16 * state, "flops": 20 * n}
        return {"bytes": 3 * n * size + 8 * state, "flops": 7 * n}
    if case["op"] == "group_norm":  # x, (grad of y) in; y, (grad of x) out; fp32 affine parameters
        n = case["samples"] * case["positions"] * case["channels"]
        if case["train"]:
            return {"bytes": 4 * n * size + 16 * case["channels"], "flops": 40 * n}
        return {"bytes": 2 * n * size + 8 * case["channels"], "flops": 14 * n}
    n = case["rows"] * case["width"]  # x, (residual), (grad of y) in; y, (grad of x) out
    tensors = 2 + int(case["residual"]) + (2 if case["train"] else 0)
    return {"bytes": tensors * n * size, "flops": 4 * n}


# --------------------------------------------------------------------- inputs
def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=_DEV)


def _lengths(case, gen):
    """Valid steps of each sequence: an empty one and one of a single step first, the rest spread over the length."""
    b, n = case["batch"], case["length"]
    lens = torch.randint(0, n + 1, (b,), generator=gen, device=_DEV, dtype=torch.int32)
    lens[-1] = n
    if b > 2:
        lens[0], lens[1] = 0, 1
    return lens


def prepare(case, seed):
    gen = torch.Generator(device=_DEV).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] in ("step", "recurrence"):
        width = case["width"]
        if case["op"] == "step":
            lead, rows = (case["rows"],), case["rows"]
        else:
            rows = case["batch"]
            lead = (case["length"], rows) if case["layout"] == "planes" else (rows, case["length"])
        # slow and fast channels side by side: memories from a couple of steps to some hundred
        logit = _normal(gen, *lead, width) + 6.0 * torch.rand(width, generator=gen, device=_DEV)
        st["gate"] = (logit if case["form"] == "leaky" else torch.sigmoid(logit)).to(dtype)
        st["x"] = _normal(gen, *lead, width).to(dtype)
        st["state"] = _normal(gen, rows, width)
        if case["op"] == "recurrence":
            st["lengths"] = _lengths(case, gen) if case["ragged"] else None
            if case["train"]:
                st["gh"] = _normal(gen, *lead, width).to(dtype)
                st["glast"] = _normal(gen, rows, width)
                for k in ("x", "gate", "state"):
                    st[k].requires_grad_()
    elif case["op"] == "group_norm":
        shape = (case["samples"], case["positions"], case["channels"])
        scale = torch.rand(case["channels"], generator=gen, device=_DEV) + 0.5
        st["x"] = (_normal(gen, *shape) * scale + 0.5).to(dtype)
        st["weight"] = _normal(gen, case["channels"]) * 0.2 + 1.0
        st["bias"] = _normal(gen, case["channels"]) * 0.2
        if case["train"]:
            st["gy"] = _normal(gen, *shape).to(dtype)
            for k in ("x", "weight", "bias"):
                st[k].requires_grad_()
    else:
        shape = (case["rows"], case["width"])
        st["x"] = _normal(gen, *shape).to(dtype)
        st["residual"] = _normal(gen, *shape).to(dtype) if case["residual"] else None
        # (seed, offset) of the mask: the random numbers are a function of it
        st["key"] = torch.randint(0, 1 << 62, (2,), generator=gen, device=_DEV, dtype=torch.int64)
        if case["train"]:
            st["gy"] = _normal(gen, *shape).to(dtype)
            for k in ("x", "residual"):
                if st[k] is not None:
                    st[k].requires_grad_()
    return st


# ---------------------------------------------------------------- plain forms
def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dimension 1, h before the first step 0, by doubling."""
    step = 1
    while step < b.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _gates(case, gate):
    """(a, 1 - a) in 32 bits."""
    gate = gate.float()
    if case["form"] == "leaky":
        return 1.0 / (1.0 + torch.exp(-gate)), 1.0 / (1.0 + torch.exp(gate))
    return gate, None


def _plain_step(st):
    a, q = _gates(st["case"], st["gate"])
    x = st["x"].float()
    h = st["state"] + q * (x - st["state"]) if q is not None else a * st["state"] + x
    return [h.to(st["x"].dtype), h]


def _plain_recurrence(st):
    case = st["case"]
    planes = case["layout"] == "planes"

    def rows_first(t):
        return t.transpose(0, 1) if planes else t

    x, gate, h0 = rows_first(st["x"].detach().float()), rows_first(st["gate"].detach()), st["state"].detach()
    a, q = _gates(case, gate)
    b = x if q is None else q * x
    valid = None
    if st["lengths"] is not None:  # a step behind the end keeps the state
        valid = (torch.arange(case["length"], device=x.device) < st["lengths"].unsqueeze(1)).unsqueeze(2)
        a, b = torch.where(valid, a, 1.0), torch.where(valid, b, 0.0)
    b = torch.cat([b[:, :1] + a[:, :1] * h0.unsqueeze(1), b[:, 1:]], 1)
    h = _scan(a, b)
    last = h[:, -1].clone()
    out = h if valid is None else torch.where(valid, h, 0.0)
    outs = [rows_first(out).to(st["x"].dtype).contiguous(), last]
    if not case["train"]:
        return outs
    # g_t = dL/dh_t = gh_t + a_{t+1} g_{t+1}, the gradient of the last state entering behind the last step
    g = rows_first(st["gh"].float())
    if valid is not None:
        g = torch.where(valid, g, 0.0)
    g = torch.cat([g[:, :-1], g[:, -1:] + st["glast"].unsqueeze(1)], 1)
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scan(later.flip(1), g.flip(1)).flip(1)
    before = torch.cat([h0.unsqueeze(1), h[:, :-1]], 1)
    gx = g if q is None else q * g
    gg = g * before if q is None else g * (before - x) * a * q
    if valid is not None:
        gx, gg = torch.where(valid, gx, 0.0), torch.where(valid, gg, 0.0)
    return outs + [rows_first(gx).to(st["x"].dtype).contiguous(), rows_first(gg).to(st["x"].dtype).contiguous(),
                   a[:, 0] * g[:, 0]]


def _plain_group_norm(st):
    case = st["case"]
    s, p, c, groups = case["samples"], case["positions"], case["channels"], case["groups"]
    x = st["x"].detach().float().view(s, p, groups, c // groups)
    w = st["weight"].detach().view(groups, c // groups)
    b = st["bias"].detach().view(groups, c // groups)
    count = p * (c // groups)
    mean = x.sum((1, 3), keepdim=True) / count
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).sum((1, 3), keepdim=True) / count + 1e-5)
    xhat = xc * rstd
    z = xhat * w + b
    if case["act"] == "silu":
        sig = 1.0 / (1.0 + torch.exp(-z))
        y = z * sig
    else:
        y = z
    y = y.view(s, p, c).to(st["x"].dtype)
    if not case["train"]:
        return y
    dz = st["gy"].float().view(s, p, groups, c // groups)
    if case["act"] == "silu":
        dz = dz * (sig * (1.0 + z * (1.0 - sig)))
    gw = (dz * xhat).sum(1).sum(0).view(c)
    gb = dz.sum(1).sum(0).view(c)
    dn = dz * w
    m1 = dn.sum((1, 3), keepdim=True) / count
    m2 = (dn * xhat).sum((1, 3), keepdim=True) / count
    gx = rstd * (dn - m1 - xhat * m2)
    return [y, gx.view(s, p, c).to(st["x"].dtype), gw, gb]


_MASK32 = 0xFFFFFFFF


def _random_words(n, key):
    """n 32-bit words: word i is word i % 4 of Philox4x32 with 7 rounds (Salmon et al., 2011) at counter
    (i // 4, offset) under the key seed, (seed, offset) = key; 64-bit numbers enter as two 32-bit words, low first."""
    c0 = torch.arange((n + 3) // 4, device=key.device)
    c1 = c0 >> 32
    c0 = c0 & _MASK32
    c2 = (key[1] & _MASK32).expand_as(c0)
    c3 = ((key[1] >> 32) & _MASK32).expand_as(c0)
    k0, k1 = key[0] & _MASK32, (key[0] >> 32) & _MASK32
    for _ in range(7):
        # the 64-bit products wrap, their bits are those of the unsigned products
        m0, m1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((m1 >> 32) & _MASK32) ^ c1 ^ k0, m1 & _MASK32, ((m0 >> 32) & _MASK32) ^ c3 ^ k1, m0 & _MASK32
        k0, k1 = (k0 + 0x9E3779B9) & _MASK32, (k1 + 0xBB67AE85) & _MASK32
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _plain_dropout(st):
    case = st["case"]
    x = st["x"].detach()
    keep = (_random_words(x.numel(), st["key"]) >= int(math.floor(case["p"] * 2.0 ** 32 + 0.5))).view_as(x)
    scale = 1.0 / (1.0 - case["p"]) if case["p"] < 1.0 else 0.0
    y = torch.where(keep, x.float() * scale, 0.0)
    if case["residual"]:
        y = y + st["residual"].detach().float()
    y = y.to(x.dtype)
    if not case["train"]:
        return y
    gx = torch.where(keep, st["gy"].float() * scale, 0.0).to(x.dtype)
    return [y, gx, st["gy"]] if case["residual"] else [y, gx]


# --------------------------------------------------------------- engine calls
def _engine(st):
    from spikestack_lite_b200 import ops

    case = st["case"]
    if case["op"] == "step":
        with torch.no_grad():
            return list(ops.gated_recurrence_step(st["x"], st["gate"], st["state"], form=case["form"]))
    if case["op"] == "recurrence":
        dim = 0 if case["layout"] == "planes" else -2
        with torch.set_grad_enabled(case["train"]):
            h, last = ops.gated_recurrence(st["x"], st["gate"], st["state"], form=case["form"], dim=dim,
                                           lengths=st["lengths"])
        if not case["train"]:
            return [h, last]
        grads = torch.autograd.grad((h, last), (st["x"], st["gate"], st["state"]), (st["gh"], st["glast"]))
        return [h.detach(), last.detach(), *grads]
    if case["op"] == "group_norm":
        with torch.set_grad_enabled(case["train"]):
            y = ops.group_norm_act(st["x"], case["groups"], st["weight"], st["bias"], eps=1e-5, act=case["act"])
        if not case["train"]:
            return y
        return [y.detach(), *torch.autograd.grad(y, (st["x"], st["weight"], st["bias"]), st["gy"])]
    with torch.set_grad_enabled(case["train"]):
        y = ops.dropout(st["x"], case["p"], st["key"], residual=st["residual"])
    if not case["train"]:
        return y
    inputs = (st["x"], st["residual"]) if case["residual"] else (st["x"],)
    return [y.detach(), *torch.autograd.grad(y, inputs, st["gy"])]


def run(state):
    if own:
        return _engine(state)
    op = state["case"]["op"]
    if op == "step":
        return _plain_step(state)
    if op == "recurrence":
        return _plain_recurrence(state)
    if op == "group_norm":
        return _plain_group_norm(state)
    return _plain_dropout(state)


# ------------------------------------------------------------ 64-bit results
def _exact_recurrence(case, st):
    axis = 0 if case["layout"] == "planes" else 1
    xs = st["x"].detach().double().unbind(axis)
    gs = st["gate"].detach().double().unbind(axis)
    lens = st["lengths"]
    live = None if lens is None else lens.unsqueeze(1)
    leaky = case["form"] == "leaky"
    h = st["state"].detach().double()
    hs, outs, a_of = [h], [], []
    for t, (x, g) in enumerate(zip(xs, gs)):
        a = torch.sigmoid(g) if leaky else g
        new = a * h + (torch.sigmoid(-g) * x if leaky else x)
        out = new
        if live is not None:
            new = torch.where(live > t, new, h)
            out = torch.where(live > t, new, torch.zeros_like(new))
        h = new
        a_of.append(a)
        hs.append(h)
        outs.append(out)
    res = [torch.stack(outs, axis), h]
    if not case["train"]:
        return res
    back = st["glast"].double()
    gx, gg = [None] * len(xs), [None] * len(xs)
    ghs = st["gh"].unbind(axis)
    for t in range(len(xs) - 1, -1, -1):
        total = back + ghs[t].double()
        a = a_of[t]
        dx = total * torch.sigmoid(-gs[t]) if leaky else total
        dg = total * (hs[t] - xs[t]) * a * torch.sigmoid(-gs[t]) if leaky else total * hs[t]
        prev = total * a
        if live is not None:
            on = live > t
            dx, dg, prev = (torch.where(on, dx, torch.zeros_like(dx)), torch.where(on, dg, torch.zeros_like(dg)),
                            torch.where(on, prev, back))
        gx[t], gg[t], back = dx, dg, prev
    return res + [torch.stack(gx, axis), torch.stack(gg, axis), back]


def _exact_group_norm(case, st):
    x = st["x"].detach().double().requires_grad_(case["train"])
    w = st["weight"].detach().double().requires_grad_(case["train"])
    b = st["bias"].detach().double().requires_grad_(case["train"])
    s, p, c, g = case["samples"], case["positions"], case["channels"], case["groups"]
    by_group = x.reshape(s, p, g, c // g).transpose(1, 2).reshape(s, g, -1)
    var, mean = torch.var_mean(by_group, dim=2, correction=0, keepdim=True)
    n = ((by_group - mean) / torch.sqrt(var + 1e-5)).reshape(s, g, p, c // g).transpose(1, 2).reshape(s, p, c)
    y = n * w + b
    if case["act"] == "silu":
        y = y / (1.0 + torch.exp(-y))
    if not case["train"]:
        return y
    return [y.detach(), *torch.autograd.grad(y, (x, w, b), st["gy"].double())]


def _exact_mask(n, key, threshold):
    """The mask with unsigned 64-bit host arithmetic, a block of counters at a time."""
    seed, offset = (int(v) for v in key.cpu().numpy().astype(np.uint64))
    low, half = np.uint64(_MASK32), np.uint64(32)
    parts = []
    total = (n + 3) // 4
    for first in range(0, total, 1 << 20):
        i = np.arange(first, min(total, first + (1 << 20)), dtype=np.uint64)
        r = [i & low, i >> half, np.full_like(i, offset & _MASK32), np.full_like(i, offset >> 32)]
        key0, key1 = seed & _MASK32, seed >> 32
        for _ in range(7):
            even, odd = r[0] * np.uint64(0xD2511F53), r[2] * np.uint64(0xCD9E8D57)
            r = [(odd >> half) ^ r[1] ^ np.uint64(key0), odd & low, (even >> half) ^ r[3] ^ np.uint64(key1), even & low]
            key0, key1 = (key0 + 0x9E3779B9) & _MASK32, (key1 + 0xBB67AE85) & _MASK32
        parts.append(np.stack([w >= np.uint64(threshold) for w in r], 1).reshape(-1))
    return np.concatenate(parts)[:n]


def _exact_dropout(case, st):
    x = st["x"].detach().double()
    keep = torch.from_numpy(_exact_mask(x.numel(), st["key"], round(case["p"] * 4294967296.0))).to(x.device).view_as(x)
    factor = keep.double() / (1.0 - case["p"]) if case["p"] < 1.0 else torch.zeros_like(x)
    y = x * factor
    if case["residual"]:
        y = y + st["residual"].detach().double()
    if not case["train"]:
        return y
    gy = st["gy"].double()
    return [y, gy * factor, gy] if case["residual"] else [y, gy * factor]


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "step":
        g, h, x = st["gate"].double(), st["state"].double(), st["x"].double()
        new = torch.sigmoid(g) * h + torch.sigmoid(-g) * x if case["form"] == "leaky" else g * h + x
        return [new, new]
    if case["op"] == "recurrence":
        return _exact_recurrence(case, st)
    if case["op"] == "group_norm":
        return _exact_group_norm(case, st)
    return _exact_dropout(case, st)
