"""Gated recurrence, without a GPU: the oracle's gradients against
differences of its forward, and the entry points' refusals (argument checks
run before any device work)."""
import ctypes

import numpy as np
import pytest

import mamba_b200 as mb
from oracle import recurrent_block as rb


def _problem(rng, B, L, D):
    x, r, i, dh = (rng.standard_normal((B, L, D)) for _ in range(4))
    lam, h0, dfin = rng.standard_normal(D) - 2, rng.standard_normal((B, D)), rng.standard_normal((B, D))
    return x, r, i, dh, lam, h0, dfin


@pytest.mark.parametrize("ragged", [False, True])
def test_oracle_gradients_match_differences(ragged):
    rng = np.random.default_rng(3)
    B, L, D, c = 3, 6, 2, 8.0
    x, r, i, dh, lam, h0, dfin = _problem(rng, B, L, D)
    lengths = np.array([6, 0, 4]) if ragged else None
    resets = (rng.random((B, L)) < 0.3) if ragged else None

    def loss(x, r, i, lam, h0):
        h, hN, _ = rb.gated_recurrence(x, r, i, lam, c, h0, lengths, resets)
        return (h * dh).sum() + (hN * dfin).sum()

    h, _, _ = rb.gated_recurrence(x, r, i, lam, c, h0, lengths, resets)
    g, _ = rb.gated_recurrence_backward(dh, x, r, i, lam, h, c, h0, lengths, resets, dfin)
    args = {"dx": x, "dr": r, "di": i, "dlam": lam, "dh0": h0}
    eps = 1e-5
    for name, v in args.items():
        num = np.zeros_like(v)
        for k in np.ndindex(v.shape):
            keep = v[k]
            v[k] = keep + eps
            up = loss(x, r, i, lam, h0)
            v[k] = keep - eps
            num[k] = (up - loss(x, r, i, lam, h0)) / (2 * eps)
            v[k] = keep
        # central differences: truncation ~eps^2, cancellation ~2^-52 |loss| / eps ~ 1e-9
        assert np.abs(num - g[name]).max() < 1e-7, name


def _args(B=2, L=4, D=8, dtype=mb.F32, ptr=4096):
    a = mb.MambaRecurrenceArgs()
    a.x = a.r = a.i = a.lambda_ = ptr  # never dereferenced: every call below is refused
    a.h = 2 * ptr
    a.batch, a.seqlen, a.dim, a.dtype, a.c = B, L, D, dtype, 8.0
    for s in (a.x_stride, a.r_stride, a.i_stride, a.h_stride):
        s[0], s[1] = L * D, D
    return a


def _forward(a, ws=None, n=0):
    return mb.lib().mamba_gated_recurrence(ctypes.byref(a), ws, n, None)


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(dtype=-1), "dtype"), (dict(batch=-1), "negative"), (dict(seqlen=-1), "negative"),
    (dict(dim=-1), "negative"), (dict(c=0.0), "c must be"), (dict(c=-1.0), "c must be"),
    (dict(c=float("nan")), "c must be"), (dict(c=float("inf")), "c must be"), (dict(x=None), "null"),
    (dict(r=None), "null"), (dict(i=None), "null"), (dict(h=None), "null"), (dict(lambda_=None), "null"),
    (dict(x=4098), "aligned"), (dict(lambda_=4098), "aligned"), (dict(initial_state=4098), "aligned"),
    (dict(final_state=4098), "aligned"), (dict(lengths=4098), "aligned"), (dict(h=4096), "one of the inputs"),
    (dict(initial_state=12288, final_state=12288), "may not be initial_state")])
def test_forward_refusals(change, text):
    a = _args()
    for k, v in change.items():
        setattr(a, k, v)
    assert _forward(a) == -1
    assert text in mb.last_error()


def test_forward_workspace_refusals():
    L = mb.lib()
    a = _args(L=5000)
    need = L.mamba_gated_recurrence_workspace(ctypes.byref(a), 0)
    assert need > 0
    for ws, n in ((None, need), (4096, need - 1), (4104, need)):
        assert _forward(a, ws, n) == -1 and "workspace" in mb.last_error()
    a = _args(B=2 ** 31 - 1, L=2 ** 31 - 1, D=2 ** 31 - 1)  # the count of tiles exceeds 64 bits
    assert _forward(a, 4096, 2 ** 62) == -1
    a = _args(B=60000, L=2 ** 31 - 1, D=2 ** 20)
    for s in (a.x_stride, a.r_stride, a.i_stride, a.h_stride):
        s[0], s[1] = 2 ** 52, 2 ** 20
    assert _forward(a, 4096, 2 ** 62) == -1 and "too many tiles" in mb.last_error()


def test_overlapping_output_rows_refused():
    a = _args()
    a.h_stride[1] = 7
    assert _forward(a) == -1 and "overlap" in mb.last_error()
    a = _args()
    a.h_stride[0] = 8  # batch rows start inside each other's time range
    assert _forward(a) == -1 and "overlap" in mb.last_error()


def test_null_structs_and_empty_sizes():
    L = mb.lib()
    assert L.mamba_gated_recurrence(None, None, 0, None) == -1 and "null" in mb.last_error()
    assert L.mamba_gated_recurrence_workspace(None, 0) == 0
    a = _args()
    assert L.mamba_gated_recurrence_backward(ctypes.byref(a), None, None, 0, None) == -1 and "null" in mb.last_error()
    assert _forward(_args(B=0)) == 0 and _forward(_args(D=0)) == 0  # nothing to do


def test_backward_refusals():
    L = mb.lib()

    def call(a, g, ws=4096, n=1 << 40):
        return L.mamba_gated_recurrence_backward(ctypes.byref(a), ctypes.byref(g), ws, n, None)

    def grads():
        g = mb.MambaRecurrenceGrads()
        g.dh, g.dx, g.dr, g.di, g.dlambda = 4096, 16384, 20480, 24576, 28672
        for s in (g.dh_stride, g.dx_stride, g.dr_stride, g.di_stride):
            s[0], s[1] = 32, 8
        return g

    for name in ("dh", "dx", "dr", "di", "dlambda"):
        g = grads()
        setattr(g, name, None)
        assert call(_args(), g) == -1, name
        g = grads()
        setattr(g, name, 4098)
        assert call(_args(), g) == -1, name
    for name, other in (("dx", 4096), ("dr", 8192), ("di", 16384)):  # an input, h, another gradient
        g = grads()
        setattr(g, name, other)
        assert call(_args(), g) == -1 and ("inputs" in mb.last_error() or "own" in mb.last_error())
    g = grads()
    g.dfinal_state = g.dinitial_state = 32768
    assert call(_args(), g) == -1 and "dinitial_state" in mb.last_error()
    g = grads()
    g.dr_stride[1] = 4
    assert call(_args(), g) == -1 and "overlap" in mb.last_error()
    need = L.mamba_gated_recurrence_workspace(ctypes.byref(_args()), 1)
    assert need > 0
    assert call(_args(), grads(), None, need) == -1 and "workspace" in mb.last_error()
    assert call(_args(), grads(), 4096, need - 1) == -1 and "workspace" in mb.last_error()
    assert call(_args(), grads(), 4104, need) == -1 and "workspace" in mb.last_error()


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(batch=-1), "negative"), (dict(dim=-1), "negative"), (dict(c=0.0), "c must be"),
    (dict(h=4096), "one of the inputs"), (dict(x=None), "null"), (dict(state_out=None), "null"), (dict(h=None), "null"),
    (dict(state_in=4098), "aligned"), (dict(hrs=7), "overlap")])
def test_step_refusals(change, text):
    v = dict(x=4096, xrs=8, r=4096, rrs=8, i=4096, irs=8, lam=4096, state_in=4096, state_out=4096, h=8192, hrs=8,
             batch=2, dim=8, c=8.0, dtype=mb.F32, stream=None)
    v.update(change)
    assert mb.lib().mamba_gated_recurrence_step(*v.values()) == -1
    assert text in mb.last_error()


def test_binding_refuses_wrong_tensors():
    import torch
    x = torch.zeros((2, 3, 8))
    lam = torch.zeros(8)
    for bad in (x.double(), x[0], x.half()):
        with pytest.raises(mb.MambaError):
            mb.gated_recurrence(x, bad, x, lam)
    with pytest.raises(mb.MambaError):
        mb.gated_recurrence(x, x, x, lam[:4])
    with pytest.raises(mb.MambaError):
        mb.gated_recurrence(x, x, x, lam, lengths=torch.zeros(2))
    with pytest.raises(mb.MambaError):
        mb.gated_recurrence(x, x, x, lam, resets=torch.zeros((2, 4), dtype=torch.uint8))
    with pytest.raises(mb.MambaError, match="CUDA"):
        mb.gated_recurrence(x, x, x, lam)
    with pytest.raises(mb.MambaError):
        mb.gated_recurrence(x.transpose(1, 2), x.transpose(1, 2), x.transpose(1, 2), torch.zeros(3))
    with pytest.raises(mb.MambaError):
        mb.gated_recurrence_step(x[0], x[0], x[0], lam, torch.zeros((3, 4)))
