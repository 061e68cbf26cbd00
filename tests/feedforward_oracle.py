"""The feed-forward operators from their definitions, in 64 bits, with a bound on what a kernel that
sums in fp32 and rounds once to its type may be off, for every element.

Units: U[t] = finfo(t).eps / 2, the largest relative error of one rounding; a sum of n products in
fp32, in any order, is off by at most G(n) = (n + 2) 2^-24 / (1 - (n + 2) 2^-24) of the sum of the
products' magnitudes. F32 functions (exp, erfc, reciprocal) are taken to be within 16 units of 2^-24
of their value; the sums they are made of are counted apart."""
import math

import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}
FN = 16 * 2.0 ** -24
# a rounding below the normal numbers is absolute
TINY = 2.0 ** -126


def G(n):
    e = (n + 2) * 2.0 ** -24
    return e / (1 - e)


def phi(x):
    return 0.5 * torch.special.erfc(-x / math.sqrt(2))


def act(name, g):
    if name == "relu":
        return g.clamp_min(0)
    if name == "gelu":
        return g * phi(g)
    return torch.sigmoid(g) * (g if name == "silu" else 1)


def slope(name, g):
    if name == "relu":
        return (g > 0).to(g.dtype)
    if name == "gelu":
        return phi(g) + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    s = torch.sigmoid(g)
    return s * (1 - s) if name == "sigmoid" else s + g * s * (1 - s)


# the largest |a'| and |a''| of each
LIP = {"silu": (1.1, 0.5), "gelu": (1.13, 0.8), "relu": (1.0, 0.0), "sigmoid": (0.25, 0.1)}


def gated(x, wg, wu, name, out_type, dh=None, ddh=None):
    """(h, bound) or, with dh (off by at most ddh), [(h, ..), (dx, ..), (dwg, ..), (dwu, ..)]. x, wg, wu,
    dh are the values the kernel reads, as fp64."""
    u = U[out_type]
    C, F, M = x.shape[1], wg.shape[0], x.shape[0]
    g, v = x @ wg.t(), x @ wu.t()
    eg, ev = G(C) * (x.abs() @ wg.abs().t()), G(C) * (x.abs() @ wu.abs().t())
    a = act(name, g)
    l1, l2 = LIP[name]
    # the value off by its argument's error and by the function's own; FN of |g| and 1 covers the
    # factors g s(g), g Phi(g), s(g)
    ea = l1 * eg + FN * (g.abs() + 1 if name != "relu" else 0)
    h = a * v
    eh = ea * (v.abs() + ev) + a.abs() * ev
    out = [(h, eh + u * (h.abs() + eh) + TINY)]
    if dh is None:
        return out[0]
    ddh = torch.zeros_like(dh) if ddh is None else ddh
    s = slope(name, g)
    es = l2 * eg + FN * (g.abs() + 2 if name != "relu" else 0)
    if name == "relu":  # the slope of a g that may lie on either side of zero
        es = torch.where(g.abs() <= eg, torch.ones_like(g), es)
    dg, du = dh * v * s, dh * a
    def times(p, ep, q, eq):
        return ep * (q.abs() + eq) + p.abs() * eq
    edv = times(dh, ddh, v, ev)
    edg = times(dh * v, edv, s, es) + 2 ** -23 * dg.abs()
    edu = times(dh, ddh, a, ea) + 2 ** -24 * du.abs()
    edg, edu = edg + u * (dg.abs() + edg) + TINY, edu + u * (du.abs() + edu) + TINY
    def product(parts, n):
        val = sum(p @ q for p, _, q in parts)
        mag = sum((p.abs() + ep) @ q.abs() for p, ep, q in parts)
        err = sum(ep @ q.abs() for p, ep, q in parts) + G(n) * mag
        return val, err + u * (val.abs() + err) + TINY
    out.append(product([(dg, edg, wg), (du, edu, wu)], 2 * F + 64))
    out.append(product([(dg.t(), edg.t(), x)], M + 64))
    out.append(product([(du.t(), edu.t(), x)], M + 64))
    return out


def threshold(p):
    return math.floor(p * 65536 + 0.5)


def scale(p):
    t = threshold(p)
    return 65536 / (65536 - t) if t < 65536 else 0.0


def philox(counter, key):
    """Philox4x32-10 of counters [n, 4] (uint64 holding 32-bit words) and two key words."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    low, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for i in range(10):
        k0 = np.uint64((key[0] + i * 0x9E3779B9) & 0xFFFFFFFF)
        k1 = np.uint64((key[1] + i * 0xBB67AE85) & 0xFFFFFFFF)
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ k0, b & low, (a >> sh) ^ c[3] ^ k1, a & low]
    return np.stack(c, 1)


def kept(rows, C, p, seed, offset, rows_per_mask=1, first=0):
    """bool [rows, C], from mask row `first` on"""
    masks, groups = -(-rows // rows_per_mask), -(-C // 8)
    gid = np.arange(first * groups, (first + masks) * groups, dtype=np.uint64)
    offset %= 1 << 64
    c = np.stack([gid & np.uint64(0xFFFFFFFF), gid >> np.uint64(32),
                  np.full_like(gid, offset & 0xFFFFFFFF), np.full_like(gid, offset >> 32)], 1)
    w = philox(c, (seed & 0xFFFFFFFF, seed >> 32)).astype(np.uint32)
    halves = np.stack([w & 0xFFFF, w >> 16], 2).reshape(masks, groups * 8)[:, :C]
    return torch.from_numpy(np.repeat(halves >= threshold(p), rows_per_mask, 0)[:rows])


def dropout_add(x, res, keep, p, out_type):
    """(y, bound)"""
    z = torch.where(keep, x * scale(p), torch.zeros_like(x))
    y = z if res is None else z + res
    e = 2 ** -23 * z.abs() + 2 ** -24 * y.abs()  # the factor's and the product's rounding, the sum's
    return y, e + U[out_type] * (y.abs() + e) + TINY


def linear(x, w, res, keep, p, out_type, dy=None, ddx=None):
    """(y, bound) or, with dy, [(y, ..), (dx, ..), (dw, ..)]; ddx: what x is off by"""
    u, sc = U[out_type], scale(p)
    K, N, M = x.shape[1], w.shape[0], x.shape[0]
    ddx = torch.zeros_like(x) if ddx is None else ddx
    z, mag = x @ w.t(), (x.abs() + ddx) @ w.abs().t()
    ez = ddx @ w.abs().t() + G(K + 64) * mag
    y = torch.where(keep, z * sc, torch.zeros_like(z))
    ey = torch.where(keep, (ez + 2 ** -23 * (z.abs() + ez)) * sc, torch.zeros_like(z))
    if res is not None:
        y = y + res
        ey = ey + 2 ** -24 * (y.abs() + ey)
    out = [(y, ey + u * (y.abs() + ey) + TINY)]
    if dy is None:
        return out[0]
    dz = torch.where(keep, dy, torch.zeros_like(dy))
    for a, b, eb, n in ((dz, w, torch.zeros_like(w), N), (dz.t(), x, ddx, M)):
        v = (a @ b) * sc
        e = (a.abs() @ eb + (G(n + 64) + 2 ** -23) * (a.abs() @ (b.abs() + eb))) * sc
        out.append((v, e + u * (v.abs() + e) + TINY))
    return out


def quantize(x):
    """(q int8, scale fp32) on the CPU: IEEE fp32 division"""
    x = x.float().cpu()
    s = x.abs().amax(-1) / 127
    s = torch.where(torch.isfinite(s), s, torch.full_like(s, float("nan")))
    q = torch.where(s[..., None] > 0, torch.round(x / s[..., None]), torch.zeros_like(x))
    return q.to(torch.int8), s


def product_i8(q, s, wq, ws):
    """(y, bound of the fp32 value) of the exact integer sums"""
    y = (q.double() @ wq.double().t()) * s.double()[:, None] * ws.double()
    return y, 3 * 2.0 ** -24 * y.abs() + TINY


def worst(got, want_and_bound, what=""):
    """asserts |got - want| <= bound everywhere"""
    want, bound = want_and_bound
    assert got.shape == want.shape, (what, got.shape, want.shape)
    if got.numel() == 0:
        return
    d = (got.double() - want.to(got.device)).abs()
    bad = ~(d <= bound.to(got.device))
    if bool(bad.any()):
        i = tuple(int(v) for v in torch.nonzero(bad)[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {got.numel()} outside the bound, first at {i}: "
                             f"{float(got[i])} for {float(want[i])}, bound {float(bound[i])}")
