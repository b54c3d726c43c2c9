"""Gradients of the selective scan where a step forgets nearly all of the state
before it, against the FP64 oracle.  There a = e^(dt A) is far below 1 and what it
scales (the state that is left, the gradient that goes on to it) is tiny, but
it is all of some outputs.

Tolerance, per element: u |ref| + d mag + tiny, mag the sum of the element's
absolute terms (with the exact a).  d: 2^-24 (64 + 8 L + n) for the FP32
evaluation and sums over n terms; 2^-16 for FP16 tensors' approximations (two
units of 2^-24 of an exponential of 1/16 or more, softplus and reciprocals); and
the exponent's own rounding: dt, A log2(e) and their product are off by 2^-24
each, which moves a by 3 2^-24 |dt A| of itself: below 2^-16 up to |dt A| = 80.
Terms beyond that are below e^-80 times values of at most 2^12: tiny = 2^-100
(for FP16 outputs half of their smallest step)."""
import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
KINDS = [(F32, F32, F32), (F16, F16, F16), (F16, F32, F16), (F16, F32, F32)]
KEYS = ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dh0")


def _np(dtype):
    return np.float16 if dtype == F16 else np.float32


def _inputs(seed, b, L, D, N, kind):
    rng = np.random.default_rng(seed)
    xt, dt, bt = (_np(k) for k in kind)
    v = {k: rng.standard_normal((b, L, D)).astype(xt) for k in ("dy", "x", "z")}
    v["delta"] = rng.uniform(4, 20, (b, L, D)).astype(dt)
    v["A"] = -np.arange(1, N + 1, dtype=np.float32) * np.ones((D, 1), np.float32)
    v["B"], v["C"] = (rng.standard_normal((b, L, N)).astype(bt) for _ in range(2))
    v["D"] = np.zeros(D, np.float32)
    v["initial_state"], v["dfinal_state"] = (100 * rng.standard_normal((b, D, N)).astype(np.float32)
                                             for _ in range(2))
    v["x"][:, ::5] = 0  # tokens that only forget
    return v


def _run(v):
    t = {k: torch.from_numpy(a).cuda() for k, a in v.items()}
    got = mb.selective_scan_backward(t["dy"], t["x"], t["delta"], t["A"], t["B"], t["C"], D=t["D"], z=t["z"],
                                     initial_state=t["initial_state"], dfinal_state=t["dfinal_state"])
    return dict(zip(KEYS, got))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("b,L,D,N", [(2, 1, 6, 1), (1, 7, 130, 4), (2, 40, 33, 16), (1, 300, 64, 5)])
def test_steps_that_forget(cuda, b, L, D, N, kind):
    v = _inputs(L + D, b, L, D, N, kind)
    ref, mag = tr.scan_backward(v["dy"], v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], None,
                                v["initial_state"], v["dfinal_state"])
    terms = {"dA": b * L, "dD": b * L, "dB": D, "dC": D}
    bad = []
    for k, g in _run(v).items():
        if g is None:
            continue
        u, tiny = (2.0 ** -11, 2.0 ** -25) if g.dtype == F16 else (2.0 ** -24, 2.0 ** -100)
        d = 2.0 ** -24 * (64 + 8 * L + terms.get(k, 0)) + 2.0 ** -16 + (2.0 ** -16 if kind[0] == F16 else 0)
        err = np.abs(g.double().cpu().numpy() - ref[k]) - (u * np.abs(ref[k]) + d * mag[k] + tiny)
        if not err.max() <= 0:  # a NaN too
            bad.append((k, err.max()))
    assert not bad, bad


@pytest.mark.parametrize("kind", KINDS)
def test_masked_steps(cuda, kind):
    """A delta of -inf, of the type's lowest value and of 16000: steps of length zero, which pass the state and
    its gradient on (dt = a - 1 = 0, nothing of delta's gradient), and steps that forget all of it."""
    b, L, D, N = 2, 37, 70, 6
    v = _inputs(1, b, L, D, N, kind)
    v["delta"] = (np.float32(0.3) * (v["delta"].astype(np.float32) - 16)).astype(_np(kind[1]))
    lowest = np.finfo(_np(kind[1])).min
    v["delta"][0, 3:7], v["delta"][1, 30:], v["delta"][0, 20], v["delta"][1, 9] = -np.inf, -np.inf, lowest, 16000
    ref, mag = tr.scan_backward(v["dy"], v["x"], np.maximum(v["delta"], -1e4), v["A"], v["B"], v["C"], v["D"], v["z"],
                                None, v["initial_state"], v["dfinal_state"])
    got = _run(v)
    terms = {"dA": b * L, "dD": b * L, "dB": D, "dC": D}
    for k, g in got.items():
        if g is None:
            continue
        u, tiny = (2.0 ** -11, 2.0 ** -25) if g.dtype == F16 else (2.0 ** -24, 2.0 ** -100)
        d = 2.0 ** -24 * (64 + 8 * L + terms.get(k, 0)) + 2.0 ** -16 + (2.0 ** -16 if kind[0] == F16 else 0)
        err = np.abs(g.double().cpu().numpy() - ref[k]) - (u * np.abs(ref[k]) + d * mag[k] + tiny)
        assert err.max() <= 0, (k, err.max())
    ddelta = got["ddelta"]
    assert (ddelta[0, 3:7] == 0).all() and (ddelta[1, 30:] == 0).all() and (ddelta[0, 20] == 0).all()


@pytest.mark.parametrize("dtype", [F16, F32])
def test_beside_tensor_core_products(cuda, dtype):
    """Two streams whose kernels both keep values in tensor memory, one of them with a round of CTAs that hold
    their columns for 256 tokens: results as alone."""
    g = torch.Generator(device="cpu").manual_seed(9)
    r = lambda *s: torch.randn(s, generator=g).cuda()  # noqa: E731
    xl, wl = r(4096, 1024).half(), r(1024, 1024).half()
    b, L, D = 4, 512, 128 * 74
    dy, x, z, delta = ((0.1 * r(b, L, 64)).to(dtype).repeat(1, 1, D // 64) for _ in range(4))
    B, C = r(b, L, 16).to(dtype), r(b, L, 16).to(dtype)
    A = -torch.arange(1, 17, device="cuda", dtype=torch.float32).repeat(D, 1)
    run = lambda: mb.selective_scan_backward(dy, x, delta, A, B, C, z=z)  # noqa: E731
    want, want_l = run(), mb.linear(xl, wl)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(one):
            got = run()
        with torch.cuda.stream(two):
            got_l = [mb.linear(xl, wl) for _ in range(20)][-1]
    torch.cuda.synchronize()
    assert torch.equal(got_l, want_l)
    assert all(p is q or torch.equal(p, q) for p, q in zip(got, want))
    assert mb.device_status() == 0
