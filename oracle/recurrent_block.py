"""The recurrent-block operators in FP64 numpy, from their definitions:
gated linear recurrence (forward, backward), block norm (forward, backward),
row quantisation and the 8-bit linear layer.

Beside each result the functions give a magnitude: the sum of the absolute
values of the terms that the result adds up, which is what rounding errors
of a lower-precision evaluation scale with."""
import numpy as np


def sigmoid(v):
    e = np.exp(-np.abs(v))
    return np.where(v >= 0, 1.0, e) / (1 + e)


def softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


def _gates(r, i, lam, c):
    y = c * softplus(lam) * sigmoid(r)
    return y, np.exp(-y), np.sqrt(-np.expm1(-2 * y)), sigmoid(i)


def gated_recurrence(x, r, i, lam, c, h0=None, lengths=None, resets=None):
    """Returns (h, final state, magnitude of h); positions behind a row's end are zero."""
    x, r, i, lam = (np.asarray(v, np.float64) for v in (x, r, i, lam))
    B, L, D = x.shape
    n = np.full(B, L) if lengths is None else np.clip(lengths, 0, L)
    h = np.zeros((B, D)) if h0 is None else np.asarray(h0, np.float64).copy()
    m = np.abs(h)
    out, mag = np.zeros((B, L, D)), np.zeros((B, L, D))
    for t in range(L):
        live = (t < n)[:, None]
        rt, it, xt = (np.where(live, v[:, t], 0.0) for v in (r, i, x))
        _, a, beta, si = _gates(rt, it, lam, c)
        if resets is not None:
            a = np.where(resets[:, t, None] != 0, 0.0, a)
        b = beta * si * xt
        h, m = np.where(live, a * h + b, h), np.where(live, a * m + np.abs(b), m)
        out[:, t], mag[:, t] = np.where(live, h, 0), np.where(live, m, 0)
    return out, h, mag


def gated_recurrence_backward(dh, x, r, i, lam, h, c, h0=None, lengths=None, resets=None, dfinal=None):
    """Returns dicts (gradients, magnitudes) with keys dx, dr, di, dlam, dh0; h_{t-1} is taken from h."""
    dh, x, r, i, lam, h = (np.asarray(v, np.float64) for v in (dh, x, r, i, lam, h))
    B, L, D = x.shape
    n = np.full(B, L) if lengths is None else np.clip(lengths, 0, L)
    C = np.zeros((B, D)) if dfinal is None else np.asarray(dfinal, np.float64).copy()
    Cm = np.abs(C)
    g = {k: np.zeros((B, L, D)) for k in ("dx", "dr", "di")}
    mag = {k: np.zeros((B, L, D)) for k in ("dx", "dr", "di")}
    dsp, dspm = np.zeros(D), np.zeros(D)
    first = np.zeros((B, D)) if h0 is None else np.asarray(h0, np.float64)
    for t in range(L - 1, -1, -1):
        live = (t < n)[:, None]
        rt, it, xt, dht = (np.where(live, v[:, t], 0.0) for v in (r, i, x, dh))
        y, a, beta, si = _gates(rt, it, lam, c)
        keep = np.ones((B, 1)) if resets is None else (resets[:, t, None] == 0).astype(float)
        prev = np.where(live & (keep > 0), h[:, t - 1] if t else first, 0.0)
        G, Gm = dht + C, np.abs(dht) + Cm
        dbeta_dy = np.where(beta > 0, a * a / np.where(beta > 0, beta, 1.0), 0.0)
        t1, t2 = si * xt * dbeta_dy, a * prev
        s = sigmoid(rt)
        dy_dr = c * softplus(lam) * s * sigmoid(-rt)
        for k, v, vm in (("dx", G * beta * si, Gm * beta * si),
                         ("di", G * beta * xt * si * sigmoid(-it), Gm * np.abs(beta * xt * si * sigmoid(-it))),
                         ("dr", G * (t1 - t2) * dy_dr, Gm * (np.abs(t1) + np.abs(t2)) * dy_dr)):
            g[k][:, t], mag[k][:, t] = np.where(live, v, 0), np.where(live, vm, 0)
        dsp += np.where(live, G * (t1 - t2) * s, 0).sum(0)
        dspm += np.where(live, Gm * (np.abs(t1) + np.abs(t2)) * s, 0).sum(0)
        C, Cm = np.where(live, keep * a * G, C), np.where(live, keep * a * Gm, Cm)
    g["dlam"], mag["dlam"] = c * sigmoid(lam) * dsp, c * sigmoid(lam) * dspm
    g["dh0"], mag["dh0"] = C, Cm
    return g, mag


def _silu(z):
    s = sigmoid(z)
    return z * s, s * (1 + z * sigmoid(-z))


def block_norm(y, residual, w_post, z, w_pre, rho, eps):
    """Returns (residual_out, out, rstd_post, rstd_pre) and the magnitudes of the first two."""
    y, residual = np.asarray(y, np.float64), np.asarray(residual, np.float64)
    wq = np.ones(y.shape[1]) if w_post is None else np.asarray(w_post, np.float64)
    wp = np.ones(y.shape[1]) if w_pre is None else np.asarray(w_pre, np.float64)
    g = 1.0 if z is None else _silu(np.asarray(z, np.float64))[0]
    rs = 1 / np.sqrt((y * y).mean(1) + eps)
    n = y * rs[:, None] * wq * g
    r1 = rho * residual + n
    rp = 1 / np.sqrt((r1 * r1).mean(1) + eps)
    mag = np.abs(rho * residual) + np.abs(n)
    return (r1, r1 * rp[:, None] * wp, rs, rp), (mag, mag * rp[:, None] * np.abs(wp))


def block_norm_backward(dres_out, dout, y, res_out, rstd_post, rstd_pre, w_post, z, w_pre, rho):
    """Returns dicts (gradients, magnitudes) with keys dy, dresidual, dw_post, dw_pre, dz (with a gate)."""
    y, r1 = np.asarray(y, np.float64), np.asarray(res_out, np.float64)
    wq = np.ones(y.shape[1]) if w_post is None else np.asarray(w_post, np.float64)
    wp = np.ones(y.shape[1]) if w_pre is None else np.asarray(w_pre, np.float64)
    rs = np.asarray(rstd_post, np.float64)[:, None]
    R = np.zeros(y.shape) if dres_out is None else np.asarray(dres_out, np.float64)
    Rm, g, mag = np.abs(R), {}, {}
    g["dw_pre"], mag["dw_pre"] = np.zeros(y.shape[1]), np.zeros(y.shape[1])
    if dout is not None:
        d, rp = np.asarray(dout, np.float64), np.asarray(rstd_pre, np.float64)[:, None]
        m, u = r1 * rp, d * wp
        R = R + rp * (u - m * (u * m).mean(1, keepdims=True))
        Rm = Rm + rp * (np.abs(u) + np.abs(m) * np.abs(u * m).mean(1, keepdims=True))
        g["dw_pre"], mag["dw_pre"] = (d * m).sum(0), np.abs(d * m).sum(0)
    gate, dgate = (1.0, 0.0) if z is None else _silu(np.asarray(z, np.float64))
    n = y * rs
    v, vm = R * wq * gate, Rm * np.abs(wq * gate)
    g["dresidual"], mag["dresidual"] = rho * R, abs(rho) * Rm
    g["dw_post"], mag["dw_post"] = (R * n * gate).sum(0), (Rm * np.abs(n * gate)).sum(0)
    g["dy"] = rs * (v - n * (v * n).mean(1, keepdims=True))
    mag["dy"] = rs * (vm + np.abs(n) * (vm * np.abs(n)).mean(1, keepdims=True))
    if z is not None:
        # SiLU'(z) = s + s z (1 - s) cancels near z = -1.278, so its two terms
        # count: an error e of either sigmoid is e s (1 + |z| (1 - s)) there,
        # however small the sum is.
        zz = np.asarray(z, np.float64)
        terms = sigmoid(zz) * (1 + np.abs(zz) * sigmoid(-zz))
        g["dz"], mag["dz"] = R * wq * n * dgate, Rm * np.abs(wq * n) * terms
    return g, mag


def quantize_rows(x):
    """(q int8, scale FP32).  Both quotients are exact enough in 64 bits to
    round like the exact ones: max / 127 to 32 bits (53 >= 2 * 24 + 2), and
    x / scale to a whole number (24-bit operands)."""
    x = np.asarray(x)
    with np.errstate(invalid="ignore"):
        amax = np.abs(x.astype(np.float64)).max(1, initial=0)
        scale = (amax / 127).astype(np.float32)
        scale[~np.isfinite(amax)] = np.nan
        div = np.where((scale == 0) | np.isnan(scale), np.inf, scale.astype(np.float64))
        q = np.nan_to_num(np.rint(x.astype(np.float64) / div[:, None]), nan=0.0)
    return np.clip(q, -127, 127).astype(np.int8), scale


def linear_i8(x, xs, w, ws, bias=None):
    """Returns the FP64 result and its magnitude."""
    v = (x.astype(np.float64) @ w.astype(np.float64).T) * xs.astype(np.float64)[:, None] * ws.astype(np.float64)
    b = 0.0 if bias is None else bias.astype(np.float64)
    return v + b, np.abs(v) + np.abs(b)
