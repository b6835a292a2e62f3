"""64-bit plain forms of the training and streaming operators, with elementwise bounds on what
kernels that compute in f32 and round once may be off by.

The bounds follow from the arithmetic alone.  EPS (24 units of 2^-24) covers one evaluation of
sigmoid or tanh with the fast exponential and division plus the operations around it; ROUND is
half a unit in the last place of a stored type (and half its smallest subnormal step).  What f32
cannot hold as a normal number (below 2^-126, where 64 bits still do) may come out as zero.
"""
from __future__ import annotations

import numpy as np
import torch

EPS = 24 * 2.0 ** -24
TINY = 2.0 ** -126
ROUND = {torch.float32: (2.0 ** -24, TINY), torch.float16: (2.0 ** -11, 2.0 ** -25),
         torch.bfloat16: (2.0 ** -8, TINY)}


def f64(t):
    return None if t is None else t.detach().to("cpu", torch.float64)


def assert_within(got, ref, bound, what):
    """|got - ref| <= bound + the rounding of got's type, element by element."""
    rel, low = ROUND[got.dtype]
    got = f64(got)
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)}, expected {tuple(ref.shape)}"
    if ref.numel() == 0:
        return
    assert torch.isfinite(got).all(), f"{what}: not finite"
    excess = (got - ref).abs() - (bound + rel * (ref.abs() + bound) + low)
    worst = excess.argmax()
    assert excess.max() <= 0, (f"{what}: {got.flatten()[worst]} for {ref.flatten()[worst]} at {int(worst)}, "
                               f"over its bound by {float(excess.max()):.3g}")


# ---- gated scan -----------------------------------------------------------------------------
def scan_forward(gates, c0=None, lengths=None):
    """gates [B,T,4H] f64 -> dict of h, c_n, every intermediate, and the running error bounds.

    A step's errors (EPS of f, of u and of the sum) pass to later steps through f, whatever the
    order in which the steps are composed.
    """
    B, T, G = gates.shape
    H = G // 4
    i, f, g, o = (gates[..., k * H:(k + 1) * H] for k in range(4))
    live = torch.ones(B, T, 1, dtype=torch.bool) if lengths is None else \
        (torch.arange(T)[None, :] < lengths.clamp(0, T)[:, None])[..., None]
    i, f, g, o = (torch.where(live, x, torch.zeros(())) for x in (i, f, g, o))  # the dead may be NaN
    i, f, g, o = i.sigmoid(), f.sigmoid(), g.tanh(), o.sigmoid()
    c = torch.zeros(B, H, dtype=torch.float64) if c0 is None else c0
    err = torch.zeros_like(c)
    cs, errs = [c], [err]
    for t in range(T):
        new = f[:, t] * c + i[:, t] * g[:, t]
        bound = f[:, t] * err + EPS * (f[:, t] * c.abs() + (i * g).abs()[:, t] + new.abs())
        c, err = torch.where(live[:, t], new, c), torch.where(live[:, t], bound, err)
        cs.append(c)
        errs.append(err)
    cs, errs = torch.stack(cs, 1), torch.stack(errs, 1)
    tc = cs[:, 1:].tanh()
    h = torch.where(live, o * tc, torch.zeros((), dtype=torch.float64))
    h_err = torch.where(live, o * errs[:, 1:] + EPS * h.abs(), torch.zeros((), dtype=torch.float64))
    return dict(h=h, h_err=h_err, c_n=c, c_n_err=err, i=i, f=f, g=g, o=o, live=live, cs=cs, errs=errs, tc=tc)


def scan_backward(s, dh=None, dc_n=None):
    """Gradients (with bounds) of sum(h dh) + sum(c_n dc_n): dict of dgates, dc0."""
    i, f, g, o, live, cs, errs, tc = (s[k] for k in ("i", "f", "g", "o", "live", "cs", "errs", "tc"))
    B, T, H = f.shape
    zero = torch.zeros((), dtype=torch.float64)
    dh = torch.zeros(B, T, H, dtype=torch.float64) if dh is None else torch.where(live, dh, zero)
    G = torch.zeros(B, H, dtype=torch.float64) if dc_n is None else dc_n
    G_err = torch.zeros_like(G)
    e = dh * o * (1 - tc * tc)
    e_err = dh.abs() * o * 2 * (errs[:, 1:] + EPS)
    grads, bounds = [None] * T, [None] * T
    for t in reversed(range(T)):
        dc = e[:, t] + G
        dc_err = e_err[:, t] + G_err + EPS * (e[:, t].abs() + G.abs())
        it, ft, gt, ot, p, perr = i[:, t], f[:, t], g[:, t], o[:, t], cs[:, t], errs[:, t]
        w = [gt * it * (1 - it), p * ft * (1 - ft), it * (1 - gt * gt), tc[:, t] * ot * (1 - ot)]
        # 1 - s loses up to EPS absolutely where s is near 1.
        w_err = [EPS * (gt.abs() * it), EPS * (p.abs() * ft) + perr * ft * (1 - ft), 3 * EPS * it,
                 EPS * ot + errs[:, t + 1] * ot]
        by, by_err = [dc, dc, dc, dh[:, t]], [dc_err, dc_err, dc_err, torch.zeros_like(dc)]
        grads[t] = torch.cat([a * b for a, b in zip(by, w)], -1)
        bounds[t] = torch.cat([a.abs() * be + ae * b.abs() + ae * be + EPS * (a * b).abs()
                               for a, ae, b, be in zip(by, by_err, w, w_err)], -1)
        G_new, err_new = ft * dc, ft * dc_err + EPS * (ft * dc).abs()
        G, G_err = torch.where(live[:, t], G_new, G), torch.where(live[:, t], err_new, G_err)
    if T:
        d = torch.where(live, torch.stack(grads, 1), zero)
        d_err = torch.where(live, torch.stack(bounds, 1), zero)
    else:
        d = d_err = torch.zeros(B, 0, 4 * H, dtype=torch.float64)
    return dict(dgates=d, dgates_err=d_err, dc0=G, dc0_err=G_err)


# ---- layer norm -----------------------------------------------------------------------------
UNIT = 2.0 ** -24
DEPTH = 64  # additions on the longest path of a row sum


def norm_forward(x, weight, bias, eps):
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    big = x.abs().amax(-1, keepdim=True)
    # The mean is off by DEPTH roundings of the largest value, which shifts every difference;
    # rstd is off relatively by the roundings of the sum of squares and by that shift's part of it.
    shift = DEPTH * UNIT * big
    xh_err = shift * rstd * (1 + xh.abs()) + (DEPTH + 8) * UNIT * xh.abs()
    w = torch.ones_like(x[:1]) if weight is None else weight
    b = torch.zeros_like(x[:1]) if bias is None else bias
    y = xh * w + b
    return dict(y=y, y_err=xh_err * w.abs() + 4 * UNIT * ((xh * w).abs() + b.abs()), xh=xh, xh_err=xh_err, rstd=rstd,
                w=w, rstd_rel=(DEPTH + 8) * UNIT + shift * rstd)


def norm_backward(s, dy, dz=None):
    xh, xh_err, rstd, w = s["xh"], s["xh_err"], s["rstd"], s["w"]
    rows = xh.shape[0]
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
    dv = rstd * (g - m1 - xh * m2)
    a1, a2 = g.abs().mean(-1, keepdim=True), (g * xh).abs().mean(-1, keepdim=True)
    m2_err = (g.abs() * xh_err).mean(-1, keepdim=True) + (DEPTH + 4) * UNIT * a2
    err = rstd * (4 * UNIT * (g.abs() + a1 + (xh * m2).abs()) + (DEPTH + 4) * UNIT * a1 + xh_err * m2.abs() +
                  xh.abs() * m2_err) + s["rstd_rel"] * dv.abs()
    if dz is not None:
        dv = dv + dz
        err = err + 2 * UNIT * dv.abs()
    sums = (rows + DEPTH) * UNIT
    return dict(dv=dv, dv_err=err, dw=(dy * xh).sum(0), dw_err=sums * (dy * xh).abs().sum(0) +
                (dy.abs() * xh_err).sum(0), db=dy.sum(0), db_err=sums * dy.abs().sum(0))


# ---- dropout --------------------------------------------------------------------------------
def philox(counter, key):
    """Philox4x32-10 on four uint32 counter words and two key words (Python integers)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(elements, p, seed, offset):
    """Whether each of the given flattened element indices is kept (numpy uint64 arrays)."""
    m32, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    e = np.asarray(elements, dtype=np.uint64)
    block = e >> np.uint64(2)
    c = [block & m32, block >> s32, np.full_like(block, offset & 0xFFFFFFFF), np.full_like(block, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> s32) ^ c[1] ^ np.uint64(k0), b & m32, (a >> s32) ^ c[3] ^ np.uint64(k1), a & m32]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    word = np.choose((e & np.uint64(3)).astype(np.int64), c)
    return torch.from_numpy(word >= np.uint64(int(p * 2.0 ** 32)))


def dropped(x, p, seed, offset):
    """dropout(x) in f64 (flattened element order)."""
    if p == 1:
        return torch.zeros_like(x)
    keep = keep_mask(np.arange(x.numel()), p, seed, offset).view(x.shape)
    return torch.where(keep, x / (1 - p), torch.zeros((), dtype=x.dtype))
