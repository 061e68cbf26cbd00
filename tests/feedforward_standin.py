"""A stand-in for the launches of the feed-forward operators, so that what surrounds them in Python can be
tested without a GPU: fp32, relu, nothing dropped, the operators' formulas in numpy on the operands' memory."""
import ctypes

import numpy as np

from progressive_process_for_human_pose_estimation_amd import feedforward as F
from progressive_process_for_human_pose_estimation_amd import hgk as H


def at(p, *shape, of=ctypes.c_float):
    n = int(np.prod(shape))
    return None if p is None else np.ctypeslib.as_array((of * n).from_address(p)).reshape(shape)


def relu(v):
    return np.maximum(v, 0)


def rows_i8(x):
    s = np.abs(x).max(1) / np.float32(127)
    return np.rint(x / s[:, None]), s


def gated_fwd(dt, x, wg, wu, h, M, C, Fh, act, ws, n):
    x = at(x, M, C)
    at(h, M, Fh)[:] = relu(x @ at(wg, Fh, C).T) * (x @ at(wu, Fh, C).T)


def gated_bwd(dt, x, wg, wu, dh, dx, dwg, dwu, M, C, Fh, act, ws, n):
    x, wg, wu, dh = at(x, M, C), at(wg, Fh, C), at(wu, Fh, C), at(dh, M, Fh)
    g, u = x @ wg.T, x @ wu.T
    dg, du = dh * u * (g > 0), dh * relu(g)
    if dx:
        at(dx, M, C)[:] = dg @ wg + du @ wu
    if dwg:
        at(dwg, Fh, C)[:], at(dwu, Fh, C)[:] = dg.T @ x, du.T @ x


def linear_fwd(dt, x, w, res, y, M, K, N, p, seed, offset, step, ws, n):
    at(y, M, N)[:] = at(x, M, K) @ at(w, N, K).T + (at(res, M, N) if res else 0)


def linear_bwd(dt, x, w, dy, dx, dw, M, K, N, p, seed, offset, step, ws, n):
    x, w, dy = at(x, M, K), at(w, N, K), at(dy, M, N)
    if dx:
        at(dx, M, K)[:] = dy @ w
    if dw:
        at(dw, N, K)[:] = dy.T @ x


def dropout_add(dt, x, res, y, M, C, group, p, seed, offset, step):
    at(y, M, C)[:] = at(x, M, C) + (at(res, M, C) if res else 0)


def quantize_rows_i8(dt, x, q, s, M, K):
    at(q, M, K, of=ctypes.c_int8)[:], at(s, M)[:] = rows_i8(at(x, M, K))


def product_i8(x, w, s, M, K, N):
    q, sx = rows_i8(at(x, M, K))
    return (q @ at(w, N, K, of=ctypes.c_int8).T.astype(np.float32)) * sx[:, None] * at(s, N)


def linear_i8(dt, x, w, s, bias, res, y, M, K, N, ws, n):
    v = product_i8(x, w, s, M, K, N)
    at(y, M, N)[:] = v + (at(bias, N) if bias else 0) + (at(res, M, N) if res else 0)


def gated_i8(dt, x, wg, sg, wu, su, h, M, C, Fh, act, ws, n):
    at(h, M, Fh)[:] = relu(product_i8(x, wg, sg, M, C, Fh)) * product_i8(x, wu, su, M, C, Fh)


def install(monkeypatch):
    def launch(x, fn, *args):
        globals()[fn.__name__[4:]](*args)

    monkeypatch.setattr(F, "_gpu", lambda what, x: None)
    monkeypatch.setattr(F, "_launch", launch)
    H.load_library()
