"""The gated recurrence on the GPU where little of a batch is left, or little of
a value: padded batches of mostly empty rows, states that live for tens of
thousands of tokens, gates that are nearly closed or nearly open.  The
comparison is with the FP64 oracle on the same (rounded) inputs, element by
element."""
import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import recurrent_block as rb

pytestmark = pytest.mark.gpu

C = 8.0


def _dev(*arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(64, 2048, 64), (300, 700, 64), (5, 4096, 256)])
def test_mostly_empty_rows(cuda, B, L, D, dtype):
    """A padded batch whose rows end early: most tiles lie behind their row's
    end, several in a row for each CTA.  No wait runs out (bit 6), and
    every call gives the same bits."""
    rng = np.random.default_rng(B)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    x, r, i = (rng.standard_normal((B, L, D)).astype(np_t) for _ in range(3))
    lam = rng.uniform(-6, -3, D).astype(np.float32)
    h0 = rng.standard_normal((B, D)).astype(np.float32)
    lengths = np.where(rng.random(B) < 0.7, rng.integers(0, 3, B), rng.integers(0, 200, B)).astype(np.int32)
    lengths[B // 2] = L
    tx, tr, ti, tl, th, tn = _dev(x, r, i, lam, h0, lengths)
    mb.device_status(True)
    first = None
    for _ in range(40):
        out = mb.gated_recurrence(tx, tr, ti, tl, c=C, initial_state=th, lengths=tn, return_final_state=True)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))
    assert mb.device_status() == 0
    keep = [b for b in range(B) if lengths[b] < 200][:20] + [B // 2]
    ref, fin, mag = rb.gated_recurrence(x[keep], r[keep], i[keep], lam, C, h0[keep], lengths[keep])
    # gates: ~16 roundings of 2^-24, and 1e-5 for FP16 tensors' short series; a state of these
    # decays (0.98 and less at r = 0) is below 2^-24 of itself after 1000 tokens
    d = 2.0 ** -24 * 1016 + (1e-5 if dtype == torch.float16 else 0.0)
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    err = np.abs(first[0].double().cpu().numpy()[keep] - ref) - (u * np.abs(ref) + d * mag + 2.0 ** -25)
    assert err.max() <= 0
    last = np.maximum(lengths[keep] - 1, 0)
    fmag = np.where(lengths[keep, None] > 0, mag[np.arange(len(keep)), last], np.abs(h0[keep]))
    err = np.abs(first[1].double().cpu().numpy()[keep] - fin) - (d * fmag + 2.0 ** -25)
    assert err.max() <= 0


def _last(mag, lengths=None):
    return mag[:, -1] if lengths is None else mag[np.arange(len(lengths)), lengths - 1]


def _check(got, ref, mag, u, d, tiny, name):
    """|got - ref| <= u |ref| + d mag + tiny, every quantity of the element itself."""
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), name
    err = np.abs(got - ref)
    bad = err - (u * np.abs(ref) + d * mag + tiny)
    assert bad.max() <= 0, (name, float(bad.max()), float((err / np.maximum(mag, 1e-300)).max()))


def _slow(seed, B, L, D, dtype):
    """Gates whose decays at r = 0 lie between 1 - 1e-2 and 1 - 1e-5."""
    rng = np.random.default_rng(seed)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    v = {k: rng.standard_normal((B, L, D)).astype(np_t) for k in ("x", "r", "i", "dh")}
    y = 10.0 ** rng.uniform(-5, -2, D)
    v["lam"] = np.log(np.expm1(2 * y / C)).astype(np.float32)
    v["h0"], v["dfinal"] = (rng.standard_normal((B, D)).astype(np.float32) for _ in range(2))
    return v


def _slow_bound(dtype, L):
    """Errors of an FP32 state that lives for up to L tokens, relative to its
    terms.  Each token's gates: 16 roundings of 2^-24 (FP16 tensors: 1e-5 for
    the short series and the approximate exponentials), of which those in the
    decay's logarithm count once over the life of the state.  Along the
    sequence: three roundings a token (the decay, the product of decays, the
    sum), each at most 2^-24 of the state and as often up as down, since the
    gates differ from token to token.  By Hoeffding's inequality their sum
    exceeds 2^-24 sqrt(3 L) sqrt(2 ln(2 / p)) with probability p: 6.3 for the last factor is
    p = 5e-9 an element."""
    walk = 6.3 * 2.0 ** -24 * (3 * L) ** 0.5
    return walk + (1e-5 if dtype == torch.float16 else 2.0 ** -24 * 16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(1, 32768, 64), (1, 20000, 33), (64, 4096, 640)])
def test_states_that_live_long(cuda, B, L, D, dtype):
    """Decays up to 1 - 1e-5: what the approximation of the decay is off by adds
    up over the state's life, in the FP32 states and in every gradient."""
    rows = 1 if B > 1 else B  # the oracle follows one row of a batch
    v = _slow(L, rows, L, D, dtype)
    t = {k: torch.from_numpy(a).cuda() for k, a in v.items()}
    t = {k: a if k == "lam" else a.repeat((B // rows,) + (1,) * (a.dim() - 1)) for k, a in t.items()}
    h, hN = mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], c=C, initial_state=t["h0"], return_final_state=True)
    grads = mb.gated_recurrence_backward(t["dh"], t["x"], t["r"], t["i"], t["lam"], h, c=C, initial_state=t["h0"],
                                         dfinal_state=t["dfinal"])
    ref, fin, mag = rb.gated_recurrence(v["x"], v["r"], v["i"], v["lam"], C, v["h0"])
    d, u = _slow_bound(dtype, L), 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    _check(hN[-rows:], fin, _last(mag), 0, d, 0, "final state")
    _check(h[-rows:], ref, mag, u, d, tiny, "h")
    g, gm = rb.gated_recurrence_backward(v["dh"], v["x"], v["r"], v["i"], v["lam"], h[-rows:].cpu().numpy(), C, v["h0"],
                                         dfinal=v["dfinal"])
    for got, k in zip(grads, ("dx", "dr", "di")):
        # an error of the state's gradient and of the token's own gates
        _check(got[-rows:], g[k], gm[k], u, d + (1e-5 if dtype == torch.float16 else 2.0 ** -24 * 16), tiny, k)
    _check(grads[4][-rows:], g["dh0"], gm["dh0"], 0, d, 0, "dh0")
    # sums over the tokens: at most L / 32 (a warp's share) + 64 additions after one another
    _check(grads[3], B * g["dlam"], B * gm["dlam"], 0, 2 * d + 2.0 ** -24 * (L / 32 + 64 + B), 0, "dlam")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_many_single_tokens(cuda, dtype):
    """Decoding: the FP32 state carried through 6000 calls."""
    B, L, D = 2, 6000, 64
    v = _slow(7, B, L, D, dtype)
    t = {k: torch.from_numpy(a).cuda() for k, a in v.items()}
    s = t["h0"].clone()
    for k in range(L):
        h, _ = mb.gated_recurrence_step(t["x"][:, k], t["r"][:, k], t["i"][:, k], t["lam"], s, c=C, state_out=s)
    ref, fin, mag = rb.gated_recurrence(v["x"], v["r"], v["i"], v["lam"], C, v["h0"])
    d, u = _slow_bound(dtype, L), 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    _check(s, fin, _last(mag), 0, d, 0, "state")
    _check(h, ref[:, -1], mag[:, -1], u, d, 2.0 ** -25 if dtype == torch.float16 else 0.0, "h")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_the_decay_of_one_token(cuda, dtype):
    """A state of 1 and no input leave the decay itself, for y = -ln a from 1e-6
    to 10.  It is 1 - d with d by a series, rounded once (2^-25 below 1), while y is small:
    y and d are off by eight roundings of 2^-24 and by 2^-21 for the gate's exponential and
    reciprocal.  From y = 1/5 on the decay is the approximate exponential
    itself or close to it: 2^-20."""
    D = 1 << 18
    y = 10.0 ** np.random.default_rng(1).uniform(-6, 1, D)
    lam = np.log(np.expm1(2 * y / C)).astype(np.float32)
    y = C * rb.softplus(lam.astype(np.float64)) / 2
    z = torch.zeros((1, D), dtype=dtype, device="cuda")
    one = torch.ones((1, D), device="cuda")
    _, s = mb.gated_recurrence_step(z, z, z, torch.from_numpy(lam).cuda(), one, c=C)
    bound = 2.0 ** -25 + y * (2.0 ** -21 + 8 * 2.0 ** -24) + np.where(y < 0.2, 0.0, 2.0 ** -20)
    over = np.abs(s[0].double().cpu().numpy() - np.exp(-y)) - bound
    assert over.max() <= 0, (float(over.max()), float(y[over.argmax()]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(2, 130, 64), (40, 70, 640), (1, 300, 33)])
def test_nearly_closed_input_gates(cuda, B, L, D, dtype):
    """sigmoid(i) = exp(i) between 3e-20 and 1e-34: small, and not 0.  FP32
    results element by element; of FP16 tensors the FP32 state."""
    rng = np.random.default_rng(L)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    x, r, dh = (rng.standard_normal((B, L, D)).astype(np_t) for _ in range(3))
    i = rng.uniform(-78, -45, (B, L, D)).astype(np_t)
    lam = rng.uniform(-5, -2, D).astype(np.float32)
    tx, tr, ti, tl, tg = _dev(x, r, i, lam, dh)
    h, hN = mb.gated_recurrence(tx, tr, ti, tl, c=C, return_final_state=True)
    ref, fin, mag = rb.gated_recurrence(x, r, i, lam, C)
    # the exponent's product with log2(e), up to 113, is rounded once (FP16 tensors): 113 * 2^-24 * 1.5 < 1.1e-5
    d = 2.1e-5 if dtype == torch.float16 else 2.0 ** -24 * (16 + min(L, 2000))
    _check(hN, fin, _last(mag), 0, d, 0, "final state")
    s, _ = mb.gated_recurrence_step(tx[:, 0], tr[:, 0], ti[:, 0], tl, torch.zeros((B, D), device="cuda"), c=C)[::-1]
    _check(s, ref[:, 0], mag[:, 0], 0, d, 0, "step")
    if dtype == torch.float32:
        _check(h, ref, mag, 2.0 ** -24, d, 0, "h")
        grads = mb.gated_recurrence_backward(tg, tx, tr, ti, tl, h, c=C)
        g, gm = rb.gated_recurrence_backward(dh, x, r, i, lam, h.cpu().numpy(), C)
        for got, k in zip(grads, ("dx", "dr", "di")):
            _check(got, g[k], gm[k], 2.0 ** -24, d, 0, k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,D", [(2371, 8), (2370, 7), (4099, 520), (65537, 4), (131071, 3), (327680, 1)])
def test_steps_of_many_rows(cuda, B, D, dtype):
    """Several rows a thread, loaded ahead of the stores: odd counts of rows, more
    rows than a grid holds, and the state updated in place."""
    rng = np.random.default_rng(B)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    x, r, i = (rng.standard_normal((B, D)).astype(np_t) for _ in range(3))
    lam = rng.uniform(-6, -2, D).astype(np.float32)
    h0 = rng.standard_normal((B, D)).astype(np.float32)
    tx, tr, ti, tl, s = _dev(x, r, i, lam, h0)
    h, out = mb.gated_recurrence_step(tx, tr, ti, tl, s, c=C)
    h2, _ = mb.gated_recurrence_step(tx, tr, ti, tl, s, c=C, state_out=s)
    assert torch.equal(h, h2) and torch.equal(out, s)
    ref, fin, mag = rb.gated_recurrence(x[:, None], r[:, None], i[:, None], lam, C, h0)
    d = 2.0 ** -24 * 17 + (1e-5 if dtype == torch.float16 else 0.0)
    _check(s, fin, mag[:, 0], 0, d, 0, "state")
    u, tiny = (2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -24, 0.0)
    _check(h, ref[:, 0], mag[:, 0], u, d, tiny, "h")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(2, 130, 64), (40, 70, 640), (1, 300, 33)])
def test_gradients_of_nearly_open_gates(cuda, B, L, D, dtype):
    """1 - sigmoid(r) = exp(-r) for r of 8 to 17, under a loss scale of 20000:
    dr are ordinary numbers that a difference of 1 and the sigmoid would lose."""
    rng = np.random.default_rng(L + 1)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    x, i = (rng.standard_normal((B, L, D)).astype(np_t) for _ in range(2))
    r = rng.uniform(8, 17, (B, L, D)).astype(np_t)
    dh = (20000 * rng.uniform(-1, 1, (B, L, D))).astype(np_t)
    lam = rng.uniform(-3, 0, D).astype(np.float32)  # y of 0.4 to 5.5
    tx, tr, ti, tl, tg = _dev(x, r, i, lam, dh)
    h = mb.gated_recurrence(tx, tr, ti, tl, c=C)
    dr = mb.gated_recurrence_backward(tg, tx, tr, ti, tl, h, c=C)[1]
    g, gm = rb.gated_recurrence_backward(dh, x, r, i, lam, h.cpu().numpy(), C)
    # ~16 roundings in the gates, a state's gradient that lives for a few tokens; FP16 tensors 1e-5
    # each for the decay and for the gates' approximate exponentials
    d, u, tiny = (2.1e-5, 2.0 ** -11, 2.0 ** -25) if dtype == torch.float16 else (2.0 ** -24 * 64, 2.0 ** -24, 0.0)
    _check(dr, g["dr"], gm["dr"], u, d, tiny, "dr")


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_calls_that_share_the_gpu(cuda, dtype):
    """Forward and backward on two streams at once, each with tiles that wait for
    one another, beside a replayed graph of a third call: every call as alone."""
    cases = []
    for seed, (B, L, D) in enumerate(((2, 6000, 256), (3, 5000, 320), (1, 9000, 128))):
        v = _slow(50 + seed, B, L, D, dtype)
        cases.append({k: torch.from_numpy(a).cuda() for k, a in v.items()})

    def call(t):
        h, hN = mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], c=C, initial_state=t["h0"],
                                    return_final_state=True)
        return [h, hN, *mb.gated_recurrence_backward(t["dh"], t["x"], t["r"], t["i"], t["lam"], h, c=C,
                                                     initial_state=t["h0"], dfinal_state=t["dfinal"])]

    alone = [call(t) for t in cases]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = call(cases[2])
    torch.cuda.synchronize()
    mb.device_status(True)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for _ in range(5):
        outs = []
        for t, s in zip(cases[:2], streams):
            with torch.cuda.stream(s):
                outs.append(call(t))
        with torch.cuda.stream(streams[2]):
            graph.replay()
        for t, s in zip(cases[:2], streams):
            with torch.cuda.stream(s):
                call(t)
        torch.cuda.synchronize()
        for got, want in zip(outs + [captured], alone):
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert mb.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("ragged,resets", [(False, False), (True, True)])
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (2, 65, 130), (1, 257, 1001), (3, 300, 256), (24, 140, 1000), (2, 900, 72)])
def test_every_element_for_itself(cuda, B, L, D, ragged, resets, dtype):
    """The parity cases with each element's own magnitude in the bound: small
    states, closed gates and small gradients count as much as large ones."""
    rng = np.random.default_rng(B + L + D)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    x, r, i, dh = (rng.standard_normal((B, L, D)).astype(np_t) for _ in range(4))
    scale = 10.0 ** rng.uniform(-3, 1, D)  # channels of different sizes
    x, dh = (x * scale).astype(np_t), (dh / scale).astype(np_t)
    lam = np.log(np.expm1(10.0 ** rng.uniform(-4, 0, D))).astype(np.float32)
    h0, dfin = (rng.standard_normal((B, D)).astype(np.float32) for _ in range(2))
    lengths = cuts = None
    if ragged:
        lengths = rng.integers(1, L + 1, B).astype(np.int32)
        lengths[0] = L
    if resets:
        cuts = (rng.random((B, L)) < 0.05).astype(np.uint8)
    tx, tr, ti, tl, tg, th, tf, tn, tc = _dev(x, r, i, lam, dh, h0, dfin, lengths, cuts)
    kw = dict(c=C, initial_state=th, lengths=tn, resets=tc)
    h, hN = mb.gated_recurrence(tx, tr, ti, tl, return_final_state=True, **kw)
    grads = mb.gated_recurrence_backward(tg, tx, tr, ti, tl, h, dfinal_state=tf, **kw)
    # gates: 16 roundings (FP16 tensors: 1e-5 for the series and the approximate exponentials);
    # the state: three roundings a token at most, over its tokens
    gates = 1e-5 if dtype == torch.float16 else 2.0 ** -24 * 16
    d, u = gates + 2.0 ** -24 * 3 * L, 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126
    ref, fin, mag = rb.gated_recurrence(x, r, i, lam, C, h0, lengths, cuts)
    _check(h, ref, mag, u, d, tiny, "h")
    _check(hN, fin, _last(mag, lengths), 0, d, 2.0 ** -126, "final state")
    g, gm = rb.gated_recurrence_backward(dh, x, r, i, lam, h.cpu().numpy(), C, h0, lengths, cuts, dfin)
    for got, k in zip(grads, ("dx", "dr", "di")):
        _check(got, g[k], gm[k], u, d + gates, tiny, k)
    _check(grads[4], g["dh0"], gm["dh0"], 0, d, 2.0 ** -126, "dh0")
    _check(grads[3], g["dlam"], gm["dlam"], 0, d + gates + 2.0 ** -24 * (L + 64 + B), 2.0 ** -126, "dlam")
