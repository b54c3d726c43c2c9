"""Workloads of the training operators around a Mamba block: the embedding
lookup and its gradient, the layer norm (forward, backward), dropout, and the
backward passes of the causal convolution and of the selective scan.

Each case can be run in two ways: with `own` false through plain torch
operations in 32 bits, with `own` true through this library's entry points.
listed() gives the cases, draw() more of the same ranges, prepare() the
inputs a program holds before the call, run() one call, exact() the same
outputs in 64 bits and work() the bytes and operations of one call.
"""
import math

import numpy as np
import torch

own = False

EPS = 1e-5


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # The rows of a training batch of 8 x 4096 tokens at the stack workload's width, into the FP32 residual stream.
        {"name": "embedding 32768x2048 of 50000 f16 to f32", "op": "embed", "tokens": 32768, "vocab": 50000,
         "dim": 2048, "dtype": "f16", "out": "f32", "padded": False},
        # The table's gradient for the same batch, ids as skewed as words are.
        {"name": "embedding gradient 32768x2048 of 50000 f16", "op": "embed_bwd", "tokens": 32768, "vocab": 50000,
         "dim": 2048, "dtype": "f16", "out": "f16", "padded": False},
        # A small padded batch of odd sizes: latency of the sort and the sums counts.
        {"name": "embedding gradient padded 1777x1001 of 5003 f32", "op": "embed_bwd", "tokens": 1777, "vocab": 5003,
         "dim": 1001, "dtype": "f32", "out": "f32", "padded": True},
        # Between two layers of a decode step: 256 rows of the decode workload's d_model.
        {"name": "layer norm 256x2560 f16", "op": "ln", "rows": 256, "cols": 2560, "dtype": "f16", "out": "f16"},
        # The backward pass of a training step: FP32 residual stream, FP16 gradients from the block.
        {"name": "layer norm backward 32768x2048 f32 to f16", "op": "ln_bwd", "rows": 32768, "cols": 2048,
         "dtype": "f32", "out": "f16"},
        # The backward pass of a small model of odd width, all in 32 bits.
        {"name": "layer norm backward 3001x771 f32", "op": "ln_bwd", "rows": 3001, "cols": 771, "dtype": "f32",
         "out": "f32"},
        # Behind a block of a training step: dropout of its output, added to the FP32 residual stream.
        {"name": "dropout and residual 32768x2048 f16", "op": "dropout", "rows": 32768, "cols": 2048, "dtype": "f16",
         "out": "f32", "residual": True, "p": 0.1},
        # Dropout alone on a small activation of odd sizes.
        {"name": "dropout 999x1777 f32", "op": "dropout", "rows": 999, "cols": 1777, "dtype": "f32", "out": "f32",
         "residual": False, "p": 0.5},
        # The convolution's gradients in a training step at the stack workload's d_inner.
        {"name": "conv backward 8x4096x4096 f16", "op": "conv_bwd", "batch": 8, "seqlen": 4096, "dim": 4096, "K": 4,
         "dtype": "f16", "silu": True, "bias": True},
        # A small model of odd sizes with another tap count, no activation.
        {"name": "conv backward 3x1501x777 f32", "op": "conv_bwd", "batch": 3, "seqlen": 1501, "dim": 777, "K": 3,
         "dtype": "f32", "silu": False, "bias": False},
        # The scan's gradients in a training step: the stack workload's d_inner and states, the gate and the bias.
        {"name": "scan backward 8x2048x4096 f16", "op": "scan_bwd", "batch": 8, "seqlen": 2048, "dim": 4096,
         "states": 16, "dtype": "f16", "delta": "f16", "gate": True, "skip": True, "carried": False},
        # A short batch of odd sizes that continues from a state and hands one on (a slice of longer sequences).
        {"name": "scan backward carried 3x333x203 f32", "op": "scan_bwd", "batch": 3, "seqlen": 333, "dim": 203,
         "states": 7, "dtype": "f32", "delta": "f32", "gate": False, "skip": True, "carried": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["embed", "embed_bwd", "embed_bwd", "ln", "ln_bwd", "dropout", "conv_bwd", "scan_bwd", "scan_bwd"])
    dtype = rng.choice(["f16", "f16", "f32"])
    out = rng.choice(["f16", "f32"])
    if op in ("embed", "embed_bwd"):
        dim = _log_int(rng, 33, 8192)
        return {"op": op, "tokens": _log_int(rng, 1, min(65536, (1 << 26) // dim)),
                "vocab": _log_int(rng, 100, min(100000, 100000000 // dim)), "dim": dim, "dtype": dtype,
                "out": out if op == "embed" else dtype, "padded": rng.random() < 0.3}
    if op in ("ln", "ln_bwd", "dropout"):
        cols = _log_int(rng, 33, 8192)
        rows = _log_int(rng, 1, min(65536, (1 << 26) // cols))
        case = {"op": op, "rows": rows, "cols": cols, "dtype": dtype, "out": out}
        if op == "dropout":
            case["residual"] = rng.random() < 0.5
            case["p"] = round(rng.uniform(0.01, 0.6), 3)
        return case
    if op == "conv_bwd":
        dim = _log_int(rng, 33, 8192)
        seqlen = _log_int(rng, 1, min(16384, (1 << 26) // dim))
        batch = _log_int(rng, 1, max(1, min(64, (1 << 26) // (dim * seqlen))))
        return {"op": op, "batch": batch, "seqlen": seqlen, "dim": dim, "K": rng.choice([2, 3, 4, 4, 4]),
                "dtype": dtype, "silu": rng.random() < 0.8, "bias": rng.random() < 0.7}
    dim = _log_int(rng, 33, 8192)
    seqlen = _log_int(rng, 1, min(8192, (1 << 25) // dim))
    batch = _log_int(rng, 1, max(1, min(32, (1 << 25) // (dim * seqlen))))
    return {"op": op, "batch": batch, "seqlen": seqlen, "dim": dim, "states": rng.choice([4, 8, 11, 16, 16, 16]),
            "dtype": dtype, "delta": "f32" if dtype == "f32" else rng.choice(["f16", "f16", "f32"]),
            "gate": rng.random() < 0.7, "skip": rng.random() < 0.8, "carried": rng.random() < 0.4}


def _size(name):
    return 2 if name == "f16" else 4


def _distinct(tokens, vocab):
    """Table rows that a batch of ids as in _ids() touches, on average."""
    r = np.arange(vocab + 1, dtype=np.float64)
    share = np.diff(np.log1p(r)) / math.log(vocab + 1)
    return int(np.sum(-np.expm1(tokens * np.log1p(-share))))


def work(case):
    op, es = case["op"], _size(case["dtype"])
    if op in ("embed", "embed_bwd"):
        t, v, d = case["tokens"], case["vocab"], case["dim"]
        if op == "embed":
            return {"bytes": 8 * t + _distinct(t, v) * d * es + t * d * _size(case["out"]), "flops": t * d}
        return {"bytes": 8 * t + t * d * es + v * d * 4, "flops": 2 * t * d}
    if op in ("ln", "ln_bwd", "dropout"):
        n, eo = case["rows"] * case["cols"], _size(case["out"])
        if op == "ln":
            return {"bytes": n * (es + eo) + 8 * (case["cols"] + case["rows"]), "flops": 8 * n}
        if op == "ln_bwd":
            return {"bytes": n * (2 * es + eo) + 8 * case["rows"] + 12 * case["cols"], "flops": 14 * n}
        # ten rounds of two products and four exclusive ors for four numbers, then the scaling
        return {"bytes": n * (es + eo + (4 if case["residual"] else 0)), "flops": 17 * n}
    n = case["batch"] * case["seqlen"] * case["dim"]
    if op == "conv_bwd":
        return {"bytes": n * 3 * es + case["dim"] * (case["K"] + 1) * 8, "flops": n * (6 * case["K"] + 10)}
    gate = 1 if case["gate"] else 0
    N, ed = case["states"], _size(case["delta"])
    state = case["batch"] * case["dim"] * N * 4 * 3 if case["carried"] else 0
    side = case["batch"] * case["seqlen"] * N * 4 * es + case["dim"] * (N + 2) * 8 + state
    # per state: the forward step and its exponential, the reverse step and the sums of the gradients
    return {"bytes": n * (3 * es + 2 * gate * es + 2 * ed) + side, "flops": n * (N * 28 + 30)}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _dtype(name):
    return torch.float16 if name == "f16" else torch.float32


def _randn(gen, shape, dtype=torch.float32, scale=1.0):
    out = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, scale, generator=gen)
    return out.to(dtype)


def _ids(gen, case):
    """Token ids with the logarithm of their rank uniform (as words are about), spread over the table; a padded
    batch ends in ids of -1, which stand for no row."""
    t, v = case["tokens"], case["vocab"]
    u = torch.rand(t, device="cuda", dtype=torch.float64, generator=gen)
    rank = torch.clamp(torch.floor(torch.expm1(u * math.log(v + 1))), 0, v - 1).to(torch.int64)
    ids = (rank * 7919 + 13) % v if v % 7919 else rank
    if case["padded"]:
        ids[t - t // 5:] = -1
    return ids


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case}
    op, dt = case["op"], _dtype(case["dtype"])
    if op in ("embed", "embed_bwd"):
        s["ids"] = _ids(gen, case)
        s["scale"] = math.sqrt(case["dim"])
        if op == "embed":
            s["table"] = _randn(gen, (case["vocab"], case["dim"]), dt, 1.0 / math.sqrt(case["dim"]))
        else:
            s["dout"] = _randn(gen, (case["tokens"], case["dim"]), dt)
    elif op in ("ln", "ln_bwd"):
        t, d = case["rows"], case["cols"]
        s["x"] = (_randn(gen, (t, d), scale=2.0) + _randn(gen, (t, 1))).to(dt)
        s["w"] = 1.0 + _randn(gen, (d,), scale=0.2)
        s["b"] = _randn(gen, (d,), scale=0.2)
        if op == "ln_bwd":
            _, s["mean"], s["rstd"] = _plain_ln(s)
            s["dout"] = _randn(gen, (t, d), _dtype(case["out"]))
    elif op == "dropout":
        t, d = case["rows"], case["cols"]
        s["x"] = _randn(gen, (t, d), dt)
        s["residual"] = _randn(gen, (t, d), scale=2.0) if case["residual"] else None
        # the seed of a run, the number of this call in it
        s["seed"], s["offset"] = 0x9E3779B97F4A7C15 ^ seed, 1000003 * seed + 17
    elif op == "conv_bwd":
        shape = (case["batch"], case["seqlen"], case["dim"])
        s["x"], s["dy"] = _randn(gen, shape, dt), _randn(gen, shape, dt)
        s["w"] = torch.empty((case["dim"], case["K"]), device="cuda").uniform_(-0.5, 0.5, generator=gen)
        s["bias"] = None
        if case["bias"]:
            s["bias"] = torch.empty(case["dim"], device="cuda").uniform_(-0.5, 0.5, generator=gen)
    else:
        b, L, d, N = case["batch"], case["seqlen"], case["dim"], case["states"]
        s["x"], s["dy"] = _randn(gen, (b, L, d), dt), _randn(gen, (b, L, d), dt)
        s["B"], s["C"] = _randn(gen, (b, L, N), dt), _randn(gen, (b, L, N), dt)
        s["z"] = _randn(gen, (b, L, d), dt) if case["gate"] else None
        # raw step sizes from dt_proj around a bias whose softplus lies between 1e-3 and 1e-1
        s["delta"] = _randn(gen, (b, L, d), _dtype(case["delta"]), 0.5)
        step = torch.empty(d, device="cuda").uniform_(math.log(1e-3), math.log(1e-1), generator=gen).exp()
        s["dt_bias"] = torch.log(torch.expm1(step))
        s["A"] = -torch.arange(1, N + 1, device="cuda", dtype=torch.float32).repeat(d, 1) \
            * torch.exp(_randn(gen, (d, N), scale=0.1))
        s["D"] = 1.0 + _randn(gen, (d,), scale=0.2) if case["skip"] else None
        s["h0"] = _randn(gen, (b, d, N)) if case["carried"] else None
        s["dfinal"] = _randn(gen, (b, d, N)) if case["carried"] else None
    return s


# ---------------------------------------------------------------------------
# Plain forms
# ---------------------------------------------------------------------------
def _sigmoid(v):
    e = torch.exp(-v.abs())
    return torch.where(v >= 0, torch.ones_like(e), e) / (1 + e)


def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _plain_embed(s):
    ids, table = s["ids"], s["table"]
    inside = (ids >= 0) & (ids < table.shape[0])
    rows = table[torch.where(inside, ids, 0)].float() * np.float32(s["scale"])
    return torch.where(inside[:, None], rows, 0.0).to(_dtype(s["case"]["out"]))


def _plain_embed_bwd(s):
    """Sums of equal ids' rows: the sorted rows' running sums in 64 bits, differences at the ends of each id."""
    ids, dout, vocab = s["ids"], s["dout"], s["case"]["vocab"]
    out = torch.zeros((vocab, dout.shape[1]), dtype=torch.float32, device="cuda")
    order = torch.argsort(ids, stable=True)
    key = ids[order]
    order, key = order[key >= 0], key[key >= 0]
    if key.numel() == 0:
        return out
    rows, counts = torch.unique_consecutive(key, return_counts=True)
    end = torch.cumsum(counts, 0)
    for c in range(0, dout.shape[1], 512):  # a few columns at a time bounds the 64-bit copies
        sums = torch.cumsum(dout[:, c:c + 512][order].double(), 0)[end - 1]
        sums[1:] -= sums[:-1].clone()
        out[rows, c:c + 512] = (sums * float(np.float32(s["scale"]))).float()
    return out


def _plain_ln(s):
    x = s["x"].float()
    mean = x.mean(1)
    xc = x - mean[:, None]
    rstd = 1 / torch.sqrt((xc * xc).mean(1) + EPS)
    y = xc * rstd[:, None] * s["w"] + s["b"]
    return y.to(_dtype(s["case"]["out"])), mean, rstd


def _plain_ln_bwd(s):
    g, r = s["dout"].float(), s["rstd"][:, None]
    n = (s["x"].float() - s["mean"][:, None]) * r
    u = g * s["w"]
    dx = r * (u - u.mean(1, keepdim=True) - n * (u * n).mean(1, keepdim=True))
    return dx.to(s["x"].dtype), (g * n).double().sum(0).float(), g.double().sum(0).float()


def _words(n, seed, offset):
    """The first n numbers of 32 bits of the Philox4x32-10 stream (Salmon et al., 2011) of this seed and offset."""
    mask = 0xFFFFFFFF
    c0 = torch.arange((n + 3) // 4, dtype=torch.int64, device="cuda")
    c1 = c0 >> 32
    c0 = c0 & mask
    c2, c3 = torch.full_like(c0, offset & mask), torch.full_like(c0, (offset >> 32) & mask)
    k0, k1 = seed & mask, (seed >> 32) & mask

    def product(c, m):  # high and low word of c * m, by 16-bit halves (64-bit numbers have a sign)
        low, high = c * (m & 0xFFFF), c * (m >> 16)
        mid = high + (low >> 16)
        return mid >> 16, ((mid << 16) | (low & 0xFFFF)) & mask

    for _ in range(10):
        h0, l0 = product(c0, 0xD2511F53)
        h1, l1 = product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & mask, (k1 + 0xBB67AE85) & mask
    return torch.stack([c0, c1, c2, c3], 1).view(-1)[:n]


def _plain_dropout(s):
    x = s["x"]
    p = float(np.float32(s["case"]["p"]))
    keep = (_words(x.numel(), s["seed"], s["offset"]) >= round(p * 2 ** 32)).view(x.shape)
    out = torch.where(keep, x.float() * np.float32(1 / (1 - p)), 0.0)
    if s["residual"] is not None:
        out = out + s["residual"]
    return out.to(_dtype(s["case"]["out"]))


def _shift(v, k):
    """v[:, t - k] along time, zero outside (k may be negative)."""
    out = torch.zeros_like(v)
    if abs(k) >= v.shape[1]:
        return out
    if k > 0:
        out[:, k:] = v[:, :-k]
    elif k < 0:
        out[:, :k] = v[:, -k:]
    else:
        out = v
    return out


def _plain_conv_bwd(s):
    x, p, w, K = s["x"].float(), s["dy"].float(), s["w"], s["case"]["K"]
    if s["case"]["silu"]:
        pre = sum(_shift(x, K - 1 - k) * w[:, k] for k in range(K))
        if s["bias"] is not None:
            pre = pre + s["bias"]
        sg = _sigmoid(pre)
        p = p * (sg * (1 + pre * (1 - sg)))
    dx = sum(_shift(p, k + 1 - K) * w[:, k] for k in range(K))
    dw = torch.stack([(p * _shift(x, K - 1 - k)).double().sum((0, 1)) for k in range(K)], 1).float()
    out = [dx.to(s["x"].dtype), dw]
    if s["bias"] is not None:
        out.append(p.double().sum((0, 1)).float())
    return out


def _scan(a, b):
    """b[t] <- b[t] + a[t] * b[t - 1] along the first axis, by doubling; a and b are overwritten."""
    L, k = a.shape[0], 1
    while k < L:
        b[k:] += a[k:] * b[:-k]
        if 2 * k < L:
            a[k:] = a[k:] * a[:-k]
        k *= 2
    return b


def _plain_scan_bwd(s):
    case = s["case"]
    b, L, d, N = case["batch"], case["seqlen"], case["dim"], case["states"]
    dt_, dev = s["x"].dtype, "cuda"
    dx = torch.empty((b, L, d), dtype=dt_, device=dev)
    ddelta = torch.empty((b, L, d), dtype=s["delta"].dtype, device=dev)
    dz = torch.empty((b, L, d), dtype=dt_, device=dev) if case["gate"] else None
    dB, dC = (torch.zeros((b, L, N), dtype=torch.float64, device=dev) for _ in range(2))
    dA = torch.zeros((d, N), dtype=torch.float64, device=dev)
    dD, dbias = (torch.zeros(d, dtype=torch.float64, device=dev) for _ in range(2))
    dh0 = torch.empty((b, d, N), dtype=torch.float32, device=dev)
    wide = max(1, (1 << 26) // (L * N))  # channels at a time
    for i in range(b):
        Bm, Cm = s["B"][i].float()[:, None], s["C"][i].float()[:, None]  # [L, 1, N]
        for c0 in range(0, d, wide):
            c = slice(c0, min(d, c0 + wide))
            A = s["A"][c]
            x, dy = s["x"][i, :, c].float(), s["dy"][i, :, c].float()
            raw = s["delta"][i, :, c].float() + s["dt_bias"][c]
            dt = _softplus(raw)
            v = dt[:, :, None] * A
            em = torch.expm1(v)
            phi = torch.where(A.abs() > 1e-6, em / A, dt[:, :, None])
            w = x[:, :, None] * Bm
            h0 = s["h0"][i, c] if case["carried"] else torch.zeros_like(A)
            a = em + 1
            step = phi * w
            step[0] += a[0] * h0
            h = _scan(a.clone(), step)
            y = (h * Cm).sum(2)
            if case["skip"]:
                y = y + s["D"][c] * x
            q = dy
            if case["gate"]:
                z = s["z"][i, :, c].float()
                sg = _sigmoid(z)
                q = dy * (z * sg)
                dz[i, :, c] = (dy * y * (sg * (1 + z * (1 - sg)))).to(dt_)
            # g_t = C_t q_t + a_{t+1} g_{t+1}, as a scan over reversed time
            r = (Cm * q[:, :, None]).flip(0)
            if case["carried"]:
                r[0] += s["dfinal"][i, c]
            g = _scan(torch.cat([torch.ones_like(a[:1]), a[1:].flip(0)]), r).flip(0)
            dh0[i, c] = a[0] * g[0]
            dC[i] += (q[:, :, None] * h).double().sum(1)
            hp = torch.cat([h0[None], h[:-1]])
            del h, r
            gphi = g * phi
            dB[i] += (gphi * x[:, :, None]).double().sum(1)
            gx = (gphi * Bm).sum(2)
            if case["skip"]:
                gx = gx + s["D"][c] * q
                dD[c] += (q * x).double().sum(0)
            dx[i, :, c] = gx.to(dt_)
            u = (g * (a * (A * hp + w))).sum(2) * _sigmoid(raw)
            ddelta[i, :, c] = u.to(ddelta.dtype)
            dbias[c] += u.double().sum(0)
            # dphi/dA = (dt a - phi) / A, by its series where that difference cancels
            near = dt[:, :, None] ** 2 * (1 / 2 + v * (1 / 3 + v * (1 / 8 + v * (1 / 30 + v * (1 / 144 + v / 840)))))
            psi = torch.where(v.abs() < 0.1, near, (dt[:, :, None] * a - phi) / A)
            dA[c] += (g * (dt[:, :, None] * a * hp + w * psi)).double().sum(0)
    out = [dx, ddelta, dA.float(), dB.to(s["B"].dtype), dC.to(s["C"].dtype), dbias.float()]
    if case["skip"]:
        out.append(dD.float())
    if case["gate"]:
        out.append(dz)
    if case["carried"]:
        out.append(dh0)
    return out


# ---------------------------------------------------------------------------
# One call
# ---------------------------------------------------------------------------
def run(s):
    case = s["case"]
    op = case["op"]
    if not own:
        return {"embed": _plain_embed, "embed_bwd": _plain_embed_bwd, "ln": _plain_ln, "ln_bwd": _plain_ln_bwd,
                "dropout": _plain_dropout, "conv_bwd": _plain_conv_bwd, "scan_bwd": _plain_scan_bwd}[op](s)
    mb = _library()
    if op == "embed":
        return mb.embedding(s["ids"], s["table"], scale=s["scale"], out_dtype=_dtype(case["out"]))
    if op == "embed_bwd":
        return mb.embedding_backward(s["dout"], s["ids"], case["vocab"], scale=s["scale"])
    if op == "ln":
        return mb.layer_norm(s["x"], s["w"], s["b"], eps=EPS, out_dtype=_dtype(case["out"]), return_stats=True)
    if op == "ln_bwd":
        return mb.layer_norm_backward(s["dout"], s["x"], s["mean"], s["rstd"], w=s["w"])
    if op == "dropout":
        return mb.dropout(s["x"], case["p"], s["seed"], s["offset"], residual=s["residual"],
                          out_dtype=_dtype(case["out"]))
    if op == "conv_bwd":
        dx, dw, dbias = mb.causal_conv1d_backward(s["dy"], s["x"], s["w"], s["bias"], silu=case["silu"])
        return [dx, dw] + ([dbias] if s["bias"] is not None else [])
    dx, ddelta, dA, dB, dC, dD, dz, dbias, dh0 = mb.selective_scan_backward(
        s["dy"], s["x"], s["delta"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
        initial_state=s["h0"], dfinal_state=s["dfinal"])
    out = [dx, ddelta, dA, dB, dC, dbias]
    if case["skip"]:
        out.append(dD)
    if case["gate"]:
        out.append(dz)
    if case["carried"]:
        out.append(dh0)
    return out


_mb = None


def _library():
    global _mb
    if _mb is None:
        import os
        import sys
        path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mamba-metal_b200")
        if path not in sys.path:
            sys.path.insert(0, path)
        import mamba_b200
        _mb = mamba_b200
    return _mb


# ---------------------------------------------------------------------------
# The same outputs in 64 bits, step by step from the definitions
# ---------------------------------------------------------------------------
def _philox(index, seed, offset):
    """Words 4 * index .. 4 * index + 3 of the stream, by numpy's unsigned 64-bit integers: [len(index), 4]."""
    u = np.uint64
    lo = u(0xFFFFFFFF)
    ctr = [index & lo, index >> u(32), np.full_like(index, offset & 0xFFFFFFFF),
           np.full_like(index, (offset >> 32) & 0xFFFFFFFF)]
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for _ in range(10):
        a, b = ctr[0] * u(0xD2511F53), ctr[2] * u(0xCD9E8D57)
        ctr = [(b >> u(32)) ^ ctr[1] ^ u(key[0]), b & lo, (a >> u(32)) ^ ctr[3] ^ u(key[1]), a & lo]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(ctr, 1)


def _exact_scan_bwd(case, s):
    f = lambda name: s[name].double()  # noqa: E731
    L = case["seqlen"]
    A, x, dy, Bm, Cm = f("A"), f("x"), f("dy"), f("B"), f("C")
    raw = f("delta") + f("dt_bias")
    dt = torch.logaddexp(raw, torch.zeros_like(raw))
    D = f("D") if case["skip"] else torch.zeros_like(A[:, 0])
    gate = slope = torch.ones_like(x)
    if case["gate"]:
        z = f("z")
        gate = z * torch.special.expit(z)
        slope = torch.special.expit(z) * (1 + z * torch.special.expit(-z))
    start = f("h0") if case["carried"] else torch.zeros((case["batch"],) + tuple(A.shape), dtype=torch.float64,
                                                        device="cuda")
    h = [start]
    y = torch.empty_like(x)
    for t in range(L):
        v = dt[:, t, :, None] * A
        h.append(torch.exp(v) * h[-1] + torch.expm1(v) / A * Bm[:, t, None] * x[:, t, :, None])
        y[:, t] = (h[-1] * Cm[:, t, None]).sum(2) + D * x[:, t]
    q = dy * gate
    dx, ddt = torch.empty_like(x), torch.empty_like(x)
    dB, dC = torch.empty_like(Bm), torch.empty_like(Cm)
    dA = torch.zeros_like(A)
    carry = f("dfinal") if case["carried"] else torch.zeros_like(start)
    for t in range(L - 1, -1, -1):
        step = dt[:, t, :, None]
        v = step * A
        a, e = torch.exp(v), torch.expm1(v)
        G = carry + Cm[:, t, None] * q[:, t, :, None]
        dC[:, t] = (q[:, t, :, None] * h[t + 1]).sum(1)
        dB[:, t] = (G * (e / A) * x[:, t, :, None]).sum(1)
        dx[:, t] = (G * (e / A) * Bm[:, t, None]).sum(2) + D * q[:, t]
        da = G * h[t]
        dphi = G * Bm[:, t, None] * x[:, t, :, None]
        ddt[:, t] = (da * a * A + dphi * a).sum(2)
        # v e^v - (e^v - 1) cancels twice for short steps: there by its series
        bend = torch.where(v.abs() < 1e-2, v * v * (1 / 2 + v / 3 + v ** 2 / 8 + v ** 3 / 30 + v ** 4 / 144),
                           v * a - e)
        dA += (da * a * step + dphi * bend / (A * A)).sum(0)
        carry = a * G
        h.pop()
    dd = ddt * torch.special.expit(raw)
    out = [dx, dd, dA, dB, dC, dd.sum((0, 1))]
    if case["skip"]:
        out.append((q * x).sum((0, 1)))
    if case["gate"]:
        out.append(dy * y * slope)
    if case["carried"]:
        out.append(carry)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    f = lambda name: s[name].double()  # noqa: E731
    if op in ("embed", "embed_bwd"):
        scale, ids = float(np.float32(s["scale"])), s["ids"]
        if op == "embed":
            out = torch.zeros((case["tokens"], case["dim"]), dtype=torch.float64, device="cuda")
            out[ids >= 0] = f("table")[ids[ids >= 0]] * scale
            return out
        out = torch.zeros((case["vocab"], case["dim"]), dtype=torch.float64, device="cuda")
        return out.index_add_(0, ids[ids >= 0], f("dout")[ids >= 0]) * scale
    if op == "ln":
        x = f("x")
        mean = x.sum(1) / case["cols"]
        var = ((x - mean[:, None]) ** 2).sum(1) / case["cols"]
        return ((x - mean[:, None]) / (var + EPS).sqrt()[:, None] * f("w") + f("b")), mean, (var + EPS) ** -0.5
    if op == "ln_bwd":
        # the gradients of this call's own inputs: the saved means and reciprocal deviations are two of them
        g, r, cols = f("dout"), f("rstd")[:, None], case["cols"]
        xc = f("x") - f("mean")[:, None]
        v = g * f("w")
        dx = v * r - r * v.sum(1, keepdim=True) / cols - xc * r ** 3 * (v * xc).sum(1, keepdim=True) / cols
        return dx, (g * xc * r).sum(0), g.sum(0)
    if op == "dropout":
        p = float(np.float32(case["p"]))
        n = case["rows"] * case["cols"]
        keep = np.empty(((n + 3) // 4, 4), dtype=bool)
        for i in range(0, len(keep), 1 << 20):
            j = min(len(keep), i + (1 << 20))
            keep[i:j] = _philox(np.arange(i, j, dtype=np.uint64), s["seed"], s["offset"]) >= round(p * 2 ** 32)
        mask = torch.from_numpy(keep.reshape(-1)[:n]).cuda().view(case["rows"], case["cols"])
        out = mask * f("x") / (1 - p)
        return out + f("residual") if case["residual"] else out
    if op == "conv_bwd":
        K, L = case["K"], case["seqlen"]
        x, p, w = f("x"), f("dy"), f("w")
        back = torch.nn.functional.pad(x, (0, 0, K - 1, 0))  # back[:, t + k] = x[:, t - K + 1 + k]
        if case["silu"]:
            pre = f("bias").expand_as(x).clone() if case["bias"] else torch.zeros_like(x)
            for k in range(K):
                pre.addcmul_(back[:, k:k + L], w[:, k])
            p = p * torch.special.expit(pre) * (1 + pre * torch.special.expit(-pre))
        dback = torch.zeros_like(back)
        for k in range(K):
            dback[:, k:k + L].addcmul_(p, w[:, k])
        dw = torch.stack([(p * back[:, k:k + L]).sum((0, 1)) for k in range(K)], 1)
        return [dback[:, K - 1:], dw] + ([p.sum((0, 1))] if case["bias"] else [])
    return _exact_scan_bwd(case, s)
