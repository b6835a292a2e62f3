"""Measured cases of the training and streaming operators: the gated scan, layer norm, dropout and the fused
dropout + residual + layer norm.

Each case runs either in a plain form (elementary torch operations in 32 bits, rounded once at an operator's end) or,
with ``own`` set, through the package's public calls.  The operators, element by element:

* gated scan over gate projections in the gate order i, f, g, o (an LSTM layer whose gates do not look back):
  c_t = sigmoid(f_t) c_{t-1} + sigmoid(i_t) tanh(g_t),  h_t = sigmoid(o_t) tanh(c_t); from a row's length on the state
  stands still and h is zero.
* layer norm over the last axis: y = (x - mean) / sqrt(var + eps) * weight + bias.
* dropout: element e of the flattened tensor is kept where word e % 4 of Philox4x32-10 (Salmon, Moraes, Dror, Shaw:
  "Parallel random numbers: as easy as 1, 2, 3", 2011) at counter (e // 4, offset) under key `seed` is at least
  floor(p * 2^32); what is kept is scaled by 1 / (1 - p), and an optional residual is added.
* the fused form: z = residual + dropout(x), stored in the residual's type; y = layer norm of the stored z.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-5


# ---- the cases -----------------------------------------------------------------------------------------------------
def listed():
    return [
        # One new time step for 16 streams of a deployed H = 512 layer: the smallest call, all latency.
        {"name": "scan_step_b16_h512", "op": "scan_step", "dtype": "bf16", "B": 16, "H": 512},
        # A training step at the repository's benchmark shape (batch 512, 1000 steps, H = 128, f16).
        {"name": "scan_train_b512_t1000", "op": "scan", "dtype": "f16", "B": 512, "T": 1000, "H": 128, "train": True,
         "lens": False},
        # Inference over variable lengths in [200, 1000], the repository's ragged workload, on 1024 rows.
        {"name": "scan_ragged_b1024_t1000", "op": "scan", "dtype": "bf16", "B": 1024, "T": 1000, "H": 128,
         "train": False, "lens": True},
        # One long recording read in at once: a single row, where only the time axis can be split.
        {"name": "scan_long_b1_t65536", "op": "scan", "dtype": "bf16", "B": 1, "T": 65536, "H": 512, "train": False,
         "lens": False},
        # Full-precision training on odd sizes: few rows, an odd time length, an odd hidden size.
        {"name": "scan_train_odd_f32", "op": "scan", "dtype": "f32", "B": 3, "T": 8191, "H": 255, "train": True,
         "lens": True},
        # Norm of one time step of 16 streams: latency.
        {"name": "ln_step_m16_n512", "op": "norm", "dtype": "bf16", "wdtype": "bf16", "M": 16, "N": 512, "pad": 0,
         "train": False},
        # Training step of a norm over a batch of sequences, weights kept in 32 bits.
        {"name": "ln_train_m65536_n1024", "op": "norm", "dtype": "bf16", "wdtype": "f32", "M": 65536, "N": 1024,
         "pad": 0, "train": True},
        # Odd width, rows that are a slice of a wider projection (so no row starts on a 16-byte boundary).
        {"name": "ln_train_odd_f32", "op": "norm", "dtype": "f32", "wdtype": "f32", "M": 4099, "N": 515, "pad": 514,
         "train": True},
        # The residual step between two layers of a training pass: 512 sequences of 256 steps, H = 512.
        {"name": "fused_train_m131072_n512", "op": "fused", "dtype": "bf16", "rdtype": "bf16", "wdtype": "f32",
         "M": 131072, "N": 512, "p": 0.1, "train": True},
        # The same step on a small batch with the residual stream kept in 32 bits.
        {"name": "fused_train_m1000_n128", "op": "fused", "dtype": "f16", "rdtype": "f32", "wdtype": "f32", "M": 1000,
         "N": 128, "p": 0.2, "train": True},
        # Inter-layer dropout (0.2, the repository's model default) on the benchmark shape's activations.
        {"name": "dropout_train_b512_t1000", "op": "dropout", "dtype": "f16", "n": 512 * 1000 * 128, "p": 0.2,
         "residual": False, "train": True},
        # A small odd-sized dropout with a residual, in 32 bits.
        {"name": "dropout_train_odd_f32", "op": "dropout", "dtype": "f32", "n": 5 * 999 * 127, "p": 0.2,
         "residual": True, "train": True},
    ]


def _spread(rng, low, high):
    """A whole number in [low, high], uniform over its logarithm, often odd; never 3072."""
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))
    v = min(high, max(low, v))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(["scan", "scan", "scan", "scan_step", "norm", "norm", "fused", "fused", "dropout"])
    dtype = rng.choice(["bf16", "f16", "f32"])
    if op == "scan_step":
        h = _spread(rng, 8, 2048)
        return {"op": op, "dtype": dtype, "B": _spread(rng, 1, 4096), "H": h + 1 if h == 768 else h}
    if op == "scan":
        while True:
            b, t, h = _spread(rng, 1, 2048), _spread(rng, 1, 65536), _spread(rng, 8, 2048)
            if rng.random() < 0.5:
                h = 1 << max(3, h.bit_length() - 1)  # hidden sizes are often powers of two
            if b * t * h <= 30_000_000 and h != 768:
                break
        return {"op": op, "dtype": dtype, "B": b, "T": t, "H": h, "train": rng.random() < 0.6,
                "lens": rng.random() < 0.5}
    if op == "dropout":
        return {"op": op, "dtype": dtype, "n": _spread(rng, 1000, 1 << 25), "p": rng.choice([0.1, 0.2, 0.35, 0.5]),
                "residual": rng.random() < 0.5, "train": True}
    while True:
        m, n = _spread(rng, 1, 131072), _spread(rng, 8, 16384)
        if rng.random() < 0.5:
            n = 1 << max(3, n.bit_length() - 1)
        if m * n <= 1 << 25:
            break
    wdtype = rng.choice([dtype, "f32"])
    if op == "norm":
        pad = rng.choice([0, 0, n])
        return {"op": op, "dtype": dtype, "wdtype": wdtype, "M": m, "N": n, "pad": pad + 1 if n + pad == 3072 else pad,
                "train": rng.random() < 0.7}
    return {"op": op, "dtype": dtype, "rdtype": rng.choice([dtype, "f32"]), "wdtype": wdtype, "M": m, "N": n,
            "p": rng.choice([0.1, 0.2, 0.5]), "train": rng.random() < 0.7}


# ---- what a program has in hand -------------------------------------------------------------------------------------
def _size(name):
    return 4 if name == "f32" else 2


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _TYPES[case["dtype"]]
    s = dict(case)

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=gen, device="cuda", dtype=dtype)

    def grads(*names):
        if case.get("train"):
            for name in names:
                s[name].requires_grad_(True)

    if case["op"] in ("scan", "scan_step"):
        B, H = case["B"], case["H"]
        rows = (B, case["T"]) if case["op"] == "scan" else (B,)
        gates = normal(*rows, 4 * H)
        # Forget gates biased open, channel by channel, for memories from a few steps to a few hundred.
        gates[..., H:2 * H] += torch.linspace(1.0, 5.0, H, device="cuda").to(dt)
        s["gates"], s["c0"], s["lengths"] = gates, normal(B, H, dtype=torch.float32), None
        if case["op"] == "scan":
            if case["lens"]:
                T = case["T"]
                s["lengths"] = torch.randint(max(1, T // 5), T + 1, (B,), generator=gen, device="cuda",
                                             dtype=torch.int32)
            if case["train"]:
                s["dh"], s["dc_n"] = normal(*rows, H), normal(B, H, dtype=torch.float32)
            grads("gates", "c0")
        return s
    if case["op"] == "dropout":
        s["x"], s["seed"], s["offset"] = normal(case["n"]), 1234567 + 7919 * seed, seed % 1000
        s["res"] = normal(case["n"]) if case["residual"] else None
        s["dy"] = normal(case["n"])
        grads("x", *(["res"] if case["residual"] else []))
        return s
    M, N, wt = case["M"], case["N"], _TYPES[case["wdtype"]]
    s["weight"], s["bias"] = 1 + 0.1 * normal(N, dtype=wt), 0.1 * normal(N, dtype=wt)
    s["dy"] = normal(M, N)
    if case["op"] == "norm":
        s["x"] = (normal(M, N + case["pad"]) * 2 + 0.5)[:, case["pad"]:]
        s["x"] = s["x"].detach()
        grads("x", "weight", "bias")
        return s
    rt = _TYPES[case["rdtype"]]
    s["x"], s["res"], s["dz"] = normal(M, N), normal(M, N, dtype=rt) * 2, normal(M, N, dtype=rt)
    s["seed"], s["offset"] = 7654321 + 104729 * seed, seed % 1000
    grads("x", "res", "weight", "bias")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------
def _doubling(a, b):
    """All y_t = a_t y_{t-1} + b_t along axis 1 from y = 0, by recursive doubling: log2(T) whole-array steps."""
    d = 1
    while d < b.shape[1]:
        b = torch.cat([b[:, :d], b[:, d:] + a[:, d:] * b[:, :-d]], 1)
        a = torch.cat([a[:, :d], a[:, d:] * a[:, :-d]], 1)
        d *= 2
    return b


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _plain_step(s):
    i, f, g, o = s["gates"].float().chunk(4, -1)
    c = _sigmoid(f) * s["c0"] + _sigmoid(i) * torch.tanh(g)
    return (_sigmoid(o) * torch.tanh(c)).to(s["gates"].dtype), c


def _plain_scan(s):
    gates, c0, lens = s["gates"].detach(), s["c0"].detach(), s["lengths"]
    B, T, H = gates.shape[0], gates.shape[1], gates.shape[2] // 4
    i, f, g, o = gates.float().chunk(4, -1)
    i, f, g, o = _sigmoid(i), _sigmoid(f), torch.tanh(g), _sigmoid(o)
    u = i * g
    if lens is not None:
        live = (torch.arange(T, device=gates.device)[None, :] < lens[:, None])[:, :, None]
        f, u = torch.where(live, f, 1.0), torch.where(live, u, 0.0)
    u[:, 0] += f[:, 0] * c0
    c = _doubling(f, u)
    tc = torch.tanh(c)
    h = o * tc
    if lens is not None:
        h = torch.where(live, h, 0.0)
    h, c_n = h.to(gates.dtype), c[:, -1].clone()
    if not s["train"]:
        return h, c_n
    dh = s["dh"].float()
    e = dh * o * (1 - tc * tc)
    if lens is not None:
        e = torch.where(live, e, 0.0)
    e[:, -1] += s["dc_n"]
    # dc_t = e_t + f_{t+1} dc_{t+1}: the same recurrence in reversed time.
    ahead = torch.cat([f[:, 1:], torch.ones_like(f[:, :1])], 1)
    dc = _doubling(ahead.flip(1), e.flip(1)).flip(1)
    before = torch.cat([c0[:, None], c[:, :-1]], 1)
    d = torch.cat([dc * g * i * (1 - i), dc * before * f * (1 - f), dc * i * (1 - g * g), dh * tc * o * (1 - o)], -1)
    if lens is not None:
        d = torch.where(live, d, 0.0)
    return h, c_n, d.to(gates.dtype), f[:, 0] * dc[:, 0]


def _philox_keep(n, p, seed, offset, device):
    """Whether each of n elements is kept: Philox4x32-10 on whole arrays of counters, 32-bit words in int64."""
    low = 0xFFFFFFFF
    block = torch.arange((n + 3) // 4, device=device, dtype=torch.int64)
    w0, w1 = block & low, block >> 32
    w2, w3 = torch.full_like(block, offset & low), torch.full_like(block, offset >> 32 & low)
    k0, k1 = seed & low, seed >> 32 & low
    for _ in range(10):
        a, b = w0 * 0xD2511F53, w2 * 0xCD9E8D57  # the wrapped 64-bit product has the right 64 bits
        w0, w1, w2, w3 = (b >> 32 & low) ^ w1 ^ k0, b & low, (a >> 32 & low) ^ w3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack([w0, w1, w2, w3], 1).reshape(-1)[:n] >= int(p * 2.0 ** 32)


def _dropped(x, keep, p):
    return torch.where(keep, x.float() * (1 / (1 - p)), 0.0)


def _plain_dropout(s):
    x, p = s["x"].detach(), s["p"]
    keep = _philox_keep(x.numel(), p, s["seed"], s["offset"], x.device).view(x.shape)
    y = _dropped(x, keep, p)
    if s["res"] is not None:
        y = s["res"].detach().float() + y
    out = [y.to(x.dtype), _dropped(s["dy"], keep, p).to(x.dtype)]
    return out + ([s["dy"].clone()] if s["res"] is not None else [])


def _plain_norm_of(x, weight, bias, train, dy, dz=None):
    x32, w = x.float(), weight.float()
    mean = x32.mean(-1, keepdim=True)
    mid = x32 - mean
    rstd = 1 / torch.sqrt((mid * mid).mean(-1, keepdim=True) + _EPS)
    xh = mid * rstd
    y = (xh * w + bias.float()).to(dy.dtype)
    if not train:
        return y, None, None, None
    d = dy.float()
    dg = d * w
    dx = rstd * (dg - dg.mean(-1, keepdim=True) - xh * (dg * xh).mean(-1, keepdim=True))
    if dz is not None:
        dx = dx + dz.float()
    return y, dx, (d * xh).sum(0).to(weight.dtype), d.sum(0).to(weight.dtype)


def _plain_norm(s):
    x = s["x"].detach()
    y, dx, dw, db = _plain_norm_of(x, s["weight"].detach(), s["bias"].detach(), s["train"], s["dy"])
    return (y, dx.to(x.dtype), dw, db) if s["train"] else y


def _plain_fused(s):
    x, res, p = s["x"].detach(), s["res"].detach(), s["p"]
    keep = _philox_keep(x.numel(), p, s["seed"], s["offset"], x.device).view(x.shape)
    z = (res.float() + _dropped(x, keep, p)).to(res.dtype)
    y, dz, dw, db = _plain_norm_of(z, s["weight"].detach(), s["bias"].detach(), s["train"], s["dy"],
                                   s["dz"] if s["train"] else None)
    if not s["train"]:
        return y, z
    return y, z, _dropped(dz, keep, p).to(x.dtype), dz.to(res.dtype), dw, db


# ---- the framework's calls ----------------------------------------------------------------------------------------------
def _own(s):
    import persistent_lstm_hip_b200 as plstm

    grad = torch.autograd.grad
    if s["op"] == "scan_step":
        return plstm.gated_scan_step(s["gates"], s["c0"])
    if s["op"] == "scan":
        h, c_n = plstm.gated_scan(s["gates"], s["c0"], lengths=s["lengths"])
        return (h, c_n, *grad((h, c_n), (s["gates"], s["c0"]), (s["dh"], s["dc_n"]))) if s["train"] else (h, c_n)
    if s["op"] == "dropout":
        y = plstm.dropout(s["x"], s["p"], s["seed"], s["offset"], residual=s["res"])
        return [y, *grad(y, [s["x"]] + ([s["res"]] if s["res"] is not None else []), s["dy"])]
    w, b = s["weight"], s["bias"]
    if s["op"] == "norm":
        y = plstm.layer_norm(s["x"], w, b, _EPS)
        return (y, *grad(y, (s["x"], w, b), s["dy"])) if s["train"] else y
    y, z = plstm.dropout_add_layer_norm(s["x"], s["res"], w, b, s["p"], s["seed"], s["offset"], eps=_EPS)
    return (y, z, *grad((y, z), (s["x"], s["res"], w, b), (s["dy"], s["dz"]))) if s["train"] else (y, z)


_PLAIN = {"scan_step": _plain_step, "scan": _plain_scan, "dropout": _plain_dropout, "norm": _plain_norm,
          "fused": _plain_fused}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------
def work(case):
    e = _size(case["dtype"])
    if case["op"] in ("scan", "scan_step"):
        B, T, H = case["B"], case.get("T", 1), case["H"]
        train, n, state = case.get("train", False), B * T * H, 4 * B * H
        live = n * 0.6 if case.get("lens") else n  # lengths are uniform in [T / 5, T]; outputs are written whole
        if not train:
            return {"bytes": e * (4 * live + n) + 2 * state, "flops": 20 * live}
        return {"bytes": e * (5 * live + 5 * n) + 4 * state, "flops": 60 * live}
    if case["op"] == "dropout":
        n = case["n"]
        return {"bytes": e * n * (6 if case["residual"] else 4), "flops": 4 * n}
    n, w = case["M"] * case["N"], _size(case["wdtype"]) * case["N"]
    if case["op"] == "norm":
        return {"bytes": e * n * (4 if case["train"] else 2) + w * (4 if case["train"] else 2),
                "flops": (22 if case["train"] else 8) * n}
    r = _size(case["rdtype"])
    return {"bytes": (n * (4 * e + 4 * r) + 4 * w) if case["train"] else (n * (2 * e + 2 * r) + 2 * w),
            "flops": (26 if case["train"] else 10) * n}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------
def _exact_keep(n, p, seed, offset):
    import numpy as np

    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    at = np.arange((n + 3) // 4, dtype=np.uint64)
    ctr = [at & low, at >> half, np.uint64(offset) & low, np.uint64(offset) >> half]
    key = [np.uint64(seed & 0xFFFFFFFF), np.uint64(seed >> 32 & 0xFFFFFFFF)]
    for r in range(10):
        p0, p1 = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        bump = [np.uint64(r * 0x9E3779B9 & 0xFFFFFFFF), np.uint64(r * 0xBB67AE85 & 0xFFFFFFFF)]
        ctr = [(p1 >> half) ^ ctr[1] ^ (key[0] + bump[0] & low), p1 & low,
               (p0 >> half) ^ ctr[3] ^ (key[1] + bump[1] & low), p0 & low]
    words = np.empty((at.size, 4), np.uint32)
    for k in range(4):
        words[:, k] = ctr[k]
    return torch.from_numpy(words.reshape(-1)[:n] >= np.uint64(int(p * 2.0 ** 32))).cuda()


def _exact_norm(x, s):
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    r = (var + _EPS).rsqrt()
    xh = (x - mean) * r
    y = xh * w + b
    if not s["train"]:
        return y, None, None, None
    dy = s["dy"].double()
    gx = dy * w
    n = x.shape[-1]
    dx = r / n * (n * gx - gx.sum(-1, keepdim=True) - xh * torch.einsum("mn,mn->m", gx, xh)[:, None])
    return y, dx, torch.einsum("mn,mn->n", dy, xh), dy.sum(0)


def _exact_scan(s):
    """Step by step in time, whole rows at once."""
    gates, c = s["gates"].detach(), s["c0"].detach().double()
    if gates.dim() == 2:
        gates = gates[:, None]
    B, T, H = gates.shape[0], gates.shape[1], gates.shape[2] // 4
    gates = gates.double().transpose(0, 1).contiguous().view(T, B, 4, H)
    i, f, g, o = gates[:, :, 0].sigmoid(), gates[:, :, 1].sigmoid(), gates[:, :, 2].tanh(), gates[:, :, 3].sigmoid()
    del gates
    dead = None
    if s["lengths"] is not None:
        dead = torch.arange(T, device=c.device)[:, None, None] >= s["lengths"][None, :, None]
        f.masked_fill_(dead, 1)
        i.masked_fill_(dead, 0)
    cs = torch.empty(T + 1, B, H, device=c.device, dtype=torch.float64)
    cs[0] = c
    u = i * g
    for t in range(T):
        torch.addcmul(u[t], f[t], cs[t], out=cs[t + 1])
    del u
    tc = cs[1:].tanh()
    h = (o * tc) if dead is None else (o * tc).masked_fill_(dead, 0)
    h = h.transpose(0, 1)
    if s["op"] == "scan_step":
        return h[:, 0], cs[-1]
    if not s["train"]:
        return h, cs[-1]
    dh = s["dh"].double().transpose(0, 1)
    if dead is not None:
        dh = dh.masked_fill(dead, 0)
    dcs = dh * o * (1 - tc * tc)
    back = s["dc_n"].double()
    for t in reversed(range(T)):
        dcs[t] += back
        back = dcs[t] * f[t]
    d = torch.cat([dcs * g * i * (1 - i), dcs * cs[:-1] * f * (1 - f), dcs * i * (1 - g * g), dh * tc * o * (1 - o)], -1)
    return h, cs[-1], d.transpose(0, 1), back


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("scan", "scan_step"):
        return _exact_scan(s)
    if case["op"] == "norm":
        y, dx, dw, db = _exact_norm(s["x"].detach().double(), s)
        return (y, dx, dw, db) if case["train"] else y
    x, p = s["x"].detach().double(), s["p"]
    keep = _exact_keep(x.numel(), p, s["seed"], s["offset"]).view(x.shape)
    y = (x / (1 - p)).masked_fill_(~keep, 0)
    if case["op"] == "dropout":
        dx = (s["dy"].double() / (1 - p)).masked_fill_(~keep, 0)
        return [y, dx] if s["res"] is None else [y + s["res"].detach().double(), dx, s["dy"].double()]
    z = s["res"].detach().double() + y
    # The norm's input is z as stored.
    y, dx, dw, db = _exact_norm(z.to(s["res"].dtype).double(), s)
    if not case["train"]:
        return y, z
    dres = dx + s["dz"].double()
    return y, z, (dres / (1 - p)).masked_fill_(~keep, 0), dres, dw, db
