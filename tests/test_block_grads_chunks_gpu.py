"""Gradients of the convolution and the scan in the runs and chunks of time that
training batches take: convolution runs of 32, 64 and 128 tokens against the FP64
oracle, scan chunks of thousands of tokens against the same channels in chunks of
a few (which other tests compare with the oracle)."""
import ctypes

import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_memory():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _runs(b, L, D, K):
    """Runs of tokens a call is cut into, from its workspace: K + 1 FP32 rows of D for each run and sequence."""
    a = mb.MambaConvGradArgs()
    a.batch, a.seqlen, a.dim, a.K = b, L, D, K
    return mb.lib().mamba_causal_conv1d_backward_workspace(ctypes.byref(a)) // (4 * (K + 1) * D * b)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("b,L,D,K,runs", [(25, 90, 2048, 4, 3), (37, 100, 2047, 3, 2), (37, 129, 2048, 4, 2),
                                          (37, 131, 2046, 8, 2), (19, 400, 2048, 2, 4)])
def test_conv_backward_runs(cuda, b, L, D, K, runs, dtype):
    """Runs of 32, 64 and 128 tokens with a short last one, in groups of 4, 2 and 1 channels.

    Tolerance: the output's half step, 2^-24 (64 + n) of the sum of the absolute terms, and 2^-16 with FP16 tensors.
    n: additions that a token's term of dw or dbias passes through, at most 128 in its run, the partial rows of a warp
    (every 8th or fewer) and 32 warps' sums; one lost token would be 2^-13."""
    assert _runs(b, L, D, K) == runs
    n = 128 + -(-runs * b // 8) + 32
    rng = np.random.default_rng(L)
    t = np.float16 if dtype == F16 else np.float32
    dy, x = (rng.standard_normal((b, L, D), dtype=np.float32).astype(t) for _ in range(2))
    w, bias = (rng.uniform(-0.5, 0.5, s).astype(np.float32) for s in ((D, K), (D,)))
    ref, mag = tr.conv_backward(dy, x, w, bias, True)
    got = mb.causal_conv1d_backward(*(torch.from_numpy(v).cuda() for v in (dy, x, w, bias)))
    for g, k in zip(got, ("dx", "dw", "dbias")):
        u = 2.0 ** -11 if g.dtype == F16 else 2.0 ** -24
        d = 2.0 ** -24 * (64 + (n if k != "dx" else 0)) + (2.0 ** -16 if dtype == F16 else 0)
        err = np.abs(g.double().cpu().numpy() - ref[k]) - (u * np.abs(ref[k]) + d * mag[k] + 2.0 ** -25)
        assert err.max() <= 0, (k, err.max())


@pytest.mark.parametrize("dtype,L,N", [(F16, 17000, 2), (F32, 5000, 3)])
def test_scan_backward_long_chunks(cuda, dtype, L, N):
    """296 blocks of channels, two chunks of the sequence.  The channels repeat 64 different ones, which a second call
    has alone (in many short chunks): dB and dC are the repeats times that call's.

    Both are FP32 evaluations of one formula on the same values, which round apart.  A state and its carry round twice
    a step over a memory 1 / |dt A| below 10^4 steps: 2^-24 sqrt(2 10^4) in root mean square, seven times that for the
    largest of 10^8 elements: 2^-24 1024 of a tensor's largest value.  Sums over time round once a token: 2^-24 L of
    it.  FP16 outputs: a half step each, 2^-25 where numbers are subnormal."""
    rep, same = 592, 64
    g = torch.Generator(device="cuda").manual_seed(L)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)  # noqa: E731
    few = {k: r(1, L, same).to(dtype) for k in ("dy", "x", "z")}
    few["delta"] = (0.5 * r(1, L, same)).to(dtype)
    B, C = r(1, L, N).to(dtype), r(1, L, N).to(dtype)
    rows = {"A": -0.5 - torch.exp(r(same, N)), "D": r(same),
            "dt_bias": torch.empty(same, device="cuda").uniform_(-6.9, -2.3, generator=g)}
    h0, dh = r(1, same, N), r(1, same, N)

    def run(k):
        t = {n: v.repeat(1, 1, k) for n, v in few.items()}
        return mb.selective_scan_backward(t["dy"], t["x"], t["delta"], rows["A"].repeat(k, 1), B, C,
                                          D=rows["D"].repeat(k), z=t["z"], dt_bias=rows["dt_bias"].repeat(k),
                                          initial_state=h0.repeat(1, k, 1), dfinal_state=dh.repeat(1, k, 1))

    want, got = run(1), run(rep)
    assert mb.device_status() == 0
    for name, a, b in zip(("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dh0"), got, want):
        if name in ("dB", "dC"):
            a = a.double() / rep
        elif name in ("dx", "ddelta", "dz"):
            a = a.view(1, L, rep, same)
            b = b.view(1, L, 1, same)
        elif name == "dh0":
            a, b = a.view(1, rep, same, N), b.view(1, 1, same, N)
        else:
            a, b = a.view(rep, *b.shape), b.view(1, *b.shape)
        err = (a.double() - b.double()).abs()
        b = b.double().abs()
        tol = 2.0 ** -24 * (L if name in ("dA", "dD", "ddt_bias") else 1024) * b.max()
        if dtype == F16 and name in ("dx", "ddelta", "dB", "dC", "dz"):
            tol = tol + 2.0 ** -10 * b + 2.0 ** -24
        assert torch.isfinite(a).all() and bool((err <= tol).all()), (name, err.max().item(), b.max().item())
