"""The operators around a Mamba block in training, in FP64 numpy from their
definitions: layer norm and embedding with their gradients, dropout, and the
gradients of the causal convolution and the selective scan.

Beside most results the functions give a magnitude: the sum of the absolute
values of the terms that the result adds up, which is what rounding errors
of a lower-precision evaluation scale with."""
import numpy as np

from oracle.recurrent_block import sigmoid, softplus


def layer_norm(x, w, b, eps):
    """(out, mean, rstd), magnitude of out."""
    x = np.asarray(x, np.float64)
    w = np.ones(x.shape[1]) if w is None else np.asarray(w, np.float64)
    b = np.zeros(x.shape[1]) if b is None else np.asarray(b, np.float64)
    mean = x.mean(1)
    xc = x - mean[:, None]
    rstd = 1 / np.sqrt((xc ** 2).mean(1) + eps)
    mag = rstd[:, None] * np.abs(w) * (np.abs(x) + np.abs(x).mean(1, keepdims=True)) + np.abs(b)
    return (xc * rstd[:, None] * w + b, mean, rstd), mag


def layer_norm_backward(dout, x, mean, rstd, w):
    """Gradients and magnitudes, keys dx, dw, db, from the given statistics."""
    dout, x = np.asarray(dout, np.float64), np.asarray(x, np.float64)
    m, r = np.asarray(mean, np.float64)[:, None], np.asarray(rstd, np.float64)[:, None]
    w = np.ones(x.shape[1]) if w is None else np.asarray(w, np.float64)
    n, nm = (x - m) * r, (np.abs(x) + np.abs(m)) * r
    u = dout * w
    dx = r * (u - u.mean(1, keepdims=True) - n * (u * n).mean(1, keepdims=True))
    um = np.abs(u)
    mag = r * (um + um.mean(1, keepdims=True) + nm * (um * nm).mean(1, keepdims=True))
    g = {"dx": dx, "dw": (dout * n).sum(0), "db": dout.sum(0)}
    return g, {"dx": mag, "dw": (np.abs(dout) * nm).sum(0), "db": np.abs(dout).sum(0)}


def embedding(ids, table, scale):
    ids, table = np.asarray(ids), np.asarray(table, np.float64)
    out = np.zeros(ids.shape + table.shape[1:])
    inside = (ids >= 0) & (ids < table.shape[0])
    out[inside] = table[ids[inside]] * float(np.float32(scale))
    return out


def embedding_backward(dout, ids, vocab, scale):
    """(dtable, magnitude)."""
    ids = np.asarray(ids).reshape(-1)
    dout = np.asarray(dout, np.float64).reshape(ids.size, -1)
    g, m = np.zeros((vocab, dout.shape[1])), np.zeros((vocab, dout.shape[1]))
    for t, v in enumerate(ids):
        if 0 <= v < vocab:
            g[v] += dout[t]
            m[v] += np.abs(dout[t])
    s = float(np.float32(scale))
    return g * s, m * abs(s)


def philox(counter, key):
    """Philox4x32-10 (Salmon et al., SC 2011): four 32-bit words of a counter of four words and a key of two, by
    Python's whole numbers."""
    c, k, mask = list(counter), list(key), 0xFFFFFFFF
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & mask, (a >> 32) ^ c[3] ^ k[1], a & mask]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return c


def dropout_keep(first, n, p, seed, offset):
    """Which of elements first .. first + n - 1 a dropout call keeps."""
    border = round(float(np.float32(p)) * 2 ** 32)
    key = (seed & 0xFFFFFFFF, seed >> 32)
    out = []
    for g in range(first // 4, (first + n + 3) // 4):
        out += philox((g & 0xFFFFFFFF, g >> 32, offset & 0xFFFFFFFF, offset >> 32), key)
    at = first - first // 4 * 4
    return np.array(out[at:at + n], dtype=np.uint64) >= border


def dropout(x, p, seed, offset, residual=None):
    x = np.asarray(x, np.float64)
    p32 = float(np.float32(p))
    keep = dropout_keep(0, x.size, p, seed, offset).reshape(x.shape)
    out = np.where(keep, x / (1 - p32) if p32 < 1 else 0.0, 0.0)
    return out if residual is None else out + residual


def conv_backward(dy, x, w, bias, silu):
    """Gradients and magnitudes of the causal convolution, keys dx, dw, dbias."""
    dy, x, w = (np.asarray(v, np.float64) for v in (dy, x, w))
    B, L, D = x.shape
    K = w.shape[1]
    back = np.concatenate([np.zeros((B, K - 1, D)), x], 1)
    p, pm = dy, np.abs(dy)
    if silu:
        pre = np.zeros(x.shape) if bias is None else np.zeros(x.shape) + np.asarray(bias, np.float64)
        size = np.abs(pre)
        for k in range(K):
            pre = pre + back[:, k:k + L] * w[:, k]
            size = size + np.abs(back[:, k:k + L] * w[:, k])
        s = sigmoid(pre)
        p = dy * s * (1 + pre * sigmoid(-pre))
        # the slope of SiLU lies below 1.1, its own slope below 0.5
        pm = np.abs(dy) * (1.1 + 0.5 * size)
    g, m = {}, {}
    for out, v, taps in ((g, p, w), (m, pm, np.abs(w))):
        dback = np.zeros(back.shape)
        src = back if out is g else np.abs(back)
        for k in range(K):
            dback[:, k:k + L] += v * taps[:, k]
        out["dx"] = dback[:, K - 1:]
        out["dw"] = np.stack([(v * src[:, k:k + L]).sum((0, 1)) for k in range(K)], 1)
        out["dbias"] = v.sum((0, 1))
    return g, m


def _bend(v):
    """v e^v - (e^v - 1), by its series where that difference cancels."""
    near = np.abs(v) < 0.05
    u = np.where(near, v, 0.0)
    series = u * u * (1 / 2 + u * (1 / 3 + u * (1 / 8 + u * (1 / 30 + u * (1 / 144 + u * (1 / 840 + u / 5760))))))
    return np.where(near, series, v * np.exp(np.minimum(v, 700)) - np.expm1(np.minimum(v, 700)))


def scan_backward(dy, x, delta, A, B, C, D=None, z=None, dt_bias=None, h0=None, dfinal=None):
    """Gradients and magnitudes of the selective scan, keys dx, ddelta, dA, dB, dC, dD, dz, ddt_bias, dh0.

    dt = softplus(delta + dt_bias), a = e^(dt A), phi = (a - 1) / A (dt where |A| <= 1e-6),
    h_t = a h_{t-1} + phi B x, y = (sum_n C h + D x) SiLU(z)."""
    f = lambda v: np.asarray(v, np.float64)  # noqa: E731
    dy, x, A, B, C = f(dy), f(x), f(A), f(B), f(C)
    raw = f(delta) + (0 if dt_bias is None else f(dt_bias))
    bsz, L, dim = x.shape
    N = A.shape[1]
    Dk = np.zeros(dim) if D is None else f(D)
    dt = softplus(raw)
    big = np.abs(A) > 1e-6
    Ainv = np.where(big, 1 / np.where(big, A, 1.0), 0.0)

    def coef(t):
        d = dt[:, t, :, None]
        v = d * A
        a = np.exp(v)
        phi = np.where(big, np.expm1(v) * Ainv, d)
        psi = np.where(big, _bend(v) * Ainv * Ainv, d * d / 2)
        return d, a, phi, psi

    gate = np.ones(x.shape) if z is None else f(z) * sigmoid(f(z))
    slope = np.ones(x.shape) if z is None else sigmoid(f(z)) * (1 + f(z) * sigmoid(-f(z)))
    # SiLU' is a sum of two terms that cancels at z = -1.278: its rounding errors scale with the sum of their sizes
    slope_m = np.ones(x.shape) if z is None else sigmoid(f(z)) * (1 + np.abs(f(z)) * sigmoid(-f(z)))
    start = np.zeros((bsz, dim, N)) if h0 is None else f(h0)
    h, hm = [start], [np.abs(start)]
    y, ym = np.zeros(x.shape), np.zeros(x.shape)
    for t in range(L):
        _, a, phi, _ = coef(t)
        w = B[:, t, None] * x[:, t, :, None]
        h.append(a * h[-1] + phi * w)
        hm.append(a * hm[-1] + np.abs(phi * w))
        y[:, t] = (h[-1] * C[:, t, None]).sum(2) + Dk * x[:, t]
        ym[:, t] = (hm[-1] * np.abs(C[:, t, None])).sum(2) + np.abs(Dk * x[:, t])
    q = dy * gate
    keys = ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dh0")
    g = dict(zip(keys, (np.zeros(s) for s in (x.shape, x.shape, A.shape, B.shape, C.shape, dim, x.shape, dim,
                                                start.shape))))
    m = {k: v.copy() for k, v in g.items()}
    G = np.zeros(start.shape) if dfinal is None else f(dfinal)
    Gm = np.abs(G)
    sp = sigmoid(raw)
    for t in range(L - 1, -1, -1):
        d, a, phi, psi = coef(t)
        w = B[:, t, None] * x[:, t, :, None]
        qt = q[:, t, :, None]
        G, Gm = G + C[:, t, None] * qt, Gm + np.abs(C[:, t, None] * qt)
        for o, s, hh, hp in ((g, G, h[t + 1], h[t]), (m, Gm, hm[t + 1], hm[t])):
            ab = (lambda v: v) if o is g else np.abs
            o["dC"][:, t] = (ab(qt) * hh).sum(1)
            o["dB"][:, t] = (s * ab(phi * x[:, t, :, None])).sum(1)
            o["dx"][:, t] = ab(Dk * q[:, t]) + (s * ab(phi * B[:, t, None])).sum(2)
            u = (s * a * (ab(A) * hp + ab(w))).sum(2) * sp[:, t]
            o["ddelta"][:, t] = u
            o["ddt_bias"] += u.sum(0)
            # both parts of dA are within dt times this (the magnitude of its evaluation)
            o["dA"] += (s * (d * a * hp + ab(w) * psi)).sum(0)
            o["dD"] += ab(q[:, t] * x[:, t]).sum(0)
        G, Gm = a * G, a * Gm
    g["dh0"], m["dh0"] = G, Gm
    g["dz"], m["dz"] = dy * slope * y, np.abs(dy) * slope_m * ym
    return g, m
