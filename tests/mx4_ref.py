"""The MXFP4 row store in plain numpy float64, from the OCP microscaling format's definition (oracle of test_gpu_mx4.py)."""
import numpy as np

L2, IP, COSINE = 0, 1, 2


def micro(x, bits):
    """rows rounded in blocks of 32 to E2M1 (bits 4) or E2M3 (bits 6): float64 values, NaN for blocks that are not finite"""
    x = np.asarray(x, dtype=np.float64)
    m, dim = x.shape
    pad = np.zeros((m, -dim % 32 + dim))
    pad[:, :dim] = x
    b = pad.reshape(m, -1, 32)
    top = np.abs(b).max(axis=2, keepdims=True)
    finite = np.isfinite(top)
    e = np.where(finite & (top > 0), np.frexp(np.where(finite, top, 1))[1] - 1.0, -200.0)
    scale = np.ldexp(1.0, np.clip(e - 2, -127, 127).astype(int))
    digits, most = (1, 6.0) if bits == 4 else (3, 7.5)
    with np.errstate(invalid="ignore"):
        v = b / scale
        step = np.ldexp(1.0, np.maximum(np.frexp(np.where(np.isfinite(v), v, 0))[1] - 1, 0) - digits)
        r = np.clip(np.rint(v / step) * step, -most, most) * scale
    r = np.where(finite, r, np.nan)
    return r.reshape(m, -1)[:, :dim]


def scores(q, x, metric, bits):
    """float64 scores of queries q against stored values x (already rounded)"""
    with np.errstate(all="ignore"):
        q = micro(q, bits)
        dot = q @ x.T
        if metric == IP:
            return 1 - dot
        qq, xx = (q * q).sum(1)[:, None], (x * x).sum(1)[None]
        if metric == L2:
            return qq + xx - 2 * dot
        return 1 - dot / (np.sqrt(qq) * np.sqrt(xx))


def bound(q, x, metric, bits):
    """how far an fp32 score may be: each of the dim / 64 matrix instructions adds 64 products to its fp32 sum, 2^-22 of what it
    adds up each time (measured 2^-23.4); norms, products and the final operations half a step (2^-24) each"""
    ks = (x.shape[1] + 63) // 64
    q = micro(q, bits)
    nq, nx = np.sqrt((q * q).sum(1))[:, None], np.sqrt((x * x).sum(1))[None]
    dot = ks * 2.0 ** -22 * nq * nx
    if metric == IP:
        return dot + 2.0 ** -24 * (1 + nq * nx)
    if metric == L2:   # |q|^2, |x|^2: the norm's rounding twice and the square's; three sums of at most (|q| + |x|)^2
        return 2 * dot + 2.0 ** -24 * (3 * (nq * nq + nx * nx) + 3 * (nq + nx) ** 2)
    return np.full((len(q), len(x)), ks * 2.0 ** -22 + 2.0 ** -24 * 6)


def topk(q, x, k, metric, bits):
    """(ids, scores) of the k smallest by (score rounded to fp32, row), NaN scores left out, padded with -1"""
    s = scores(q, x, metric, bits)
    with np.errstate(over="ignore"):
        s = s.astype(np.float32)
    ids = np.full((len(q), k), -1, dtype=np.int64)
    out = np.full((len(q), k), -1.0, dtype=np.float32)
    for i in range(len(q)):
        order = np.argsort(s[i], kind="stable")
        order = order[~np.isnan(s[i][order])][:k]
        ids[i, :len(order)] = order
        out[i, :len(order)] = s[i][order]
    return ids, out
