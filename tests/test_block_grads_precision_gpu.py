"""FP32 tensors: the gradients of the selective scan in norm, against the FP64
oracle; tight enough to tell the evaluation in FP32 from the approximate one
that FP16 tensors take.

Independent roundings of at most u = 2^-24 each, N of them on the way to an
element, leave at most u sqrt(N) of a tensor's norm."""
import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

pytestmark = pytest.mark.gpu
KEYS = ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dh0")
U = 2.0 ** -24


def _run(v, dtype=torch.float32):
    t = {k: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for k, a in v.items()}
    for k in ("dy", "x", "z"):
        t[k] = None if t[k] is None else t[k].to(dtype)
    names = ("D", "z", "dt_bias", "initial_state", "dfinal_state")
    got = mb.selective_scan_backward(t["dy"], t["x"], t["delta"], t["A"], t["B"], t["C"], **{k: t[k] for k in names})
    return dict(zip(KEYS, got))


def _oracle(v):
    return tr.scan_backward(v["dy"], v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"],
                            v["initial_state"], v["dfinal_state"])[0]


def _error(got, ref):
    return np.linalg.norm(got.double().cpu().numpy() - ref) / np.linalg.norm(ref)


@pytest.mark.parametrize("carried", [False, True])
@pytest.mark.parametrize("b,L,D", [(8, 1, 300), (4, 64, 200), (1, 1000, 128)])
def test_gradients_in_norm(cuda, b, L, D, carried):
    """N: 64 for one token (delta + dt_bias is off by u |delta + dt_bias|, up to 7 u of dt; exponential and logarithm 4
    u each; the gate 3; A log2(e), its reciprocal, products and e some 12 more: 7^2 + ...).  A state rounds twice a
    step, and so does the carry, over its memory 1 / |dt A|, below 50 steps on average over these channels and states:
    4 min(L, 100).  Running sums of n terms: n / 4."""
    rng = np.random.default_rng(L + carried)
    f = np.float32
    v = {k: rng.standard_normal((b, L, D)).astype(f) for k in ("dy", "x", "z")}
    v["delta"] = (0.5 * rng.standard_normal((b, L, D))).astype(f)
    v["B"], v["C"] = (rng.standard_normal((b, L, 16)).astype(f) for _ in range(2))
    v["A"] = (-np.arange(1, 17) * np.exp(0.1 * rng.standard_normal((D, 16)))).astype(f)
    v["D"] = rng.standard_normal(D).astype(f)
    v["dt_bias"] = np.log(np.expm1(np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), D)))).astype(f)
    v["initial_state"], v["dfinal_state"] = ((rng.standard_normal((b, D, 16)).astype(f) if carried else None)
                                             for _ in range(2))
    ref = _oracle(v)
    terms = {"dA": b * L, "dD": b * L, "ddt_bias": b * L, "dB": D, "dC": D}
    errors = {k: _error(g, ref[k]) / (U * np.sqrt(64 + 4 * min(L, 100) + terms.get(k, 0) / 4))
              for k, g in _run(v).items() if g is not None}
    assert len(errors) == 8 + carried
    assert max(errors.values()) <= 1, errors


def test_no_approximate_exponentials(cuda):
    """One token, one state, |dt A| from 1/16 to 1/13: there 2^v - 1 loses most of an approximate 2^v.  N = 50: the
    exponential and the logarithm of dt 4 u each (16 + 16), and 18 products, sums and rounded constants.  The same
    values as FP16 x and dy, with their approximations, miss that bound: dA, dB and dC by 1.5, 2.1 and 1.8."""
    rng = np.random.default_rng(3)
    b, D, f = 8, 512, np.float32
    v = dict.fromkeys(("D", "z", "dt_bias", "initial_state", "dfinal_state"))
    v["dy"], v["x"] = (rng.standard_normal((b, 1, D)).astype(np.float16).astype(f) for _ in range(2))
    v["B"], v["C"] = (rng.standard_normal((b, 1, 1)).astype(f) for _ in range(2))
    v["A"] = -(1 + 0.01 * rng.random((D, 1))).astype(f)
    v["delta"] = np.log(np.expm1(rng.uniform(1 / 16, 1 / 13, (b, 1, D)))).astype(f)
    ref, got = _oracle(v), _run(v)
    errors = {k: _error(got[k], ref[k]) / (U * np.sqrt(50)) for k in ("dx", "dA", "dB", "dC")}
    assert max(errors.values()) <= 1, errors
