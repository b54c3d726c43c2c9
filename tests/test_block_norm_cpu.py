"""Block norm, without a GPU: the oracle's gradients against differences and
the entry points' refusals (argument checks run before any device work)."""
import ctypes

import numpy as np
import pytest

import mamba_b200 as mb
from oracle import recurrent_block as rb


@pytest.mark.parametrize("gate", [False, True])
def test_oracle_gradients_match_differences(gate):
    rng = np.random.default_rng(4)
    T, D, rho, eps = 3, 5, 0.8, 1e-5
    v = {k: rng.standard_normal((T, D)) for k in ("y", "res", "z")}
    v["wq"], v["wp"] = rng.standard_normal(D), rng.standard_normal(D)
    dro, do = rng.standard_normal((T, D)), rng.standard_normal((T, D))

    def run():
        return rb.block_norm(v["y"], v["res"], v["wq"], v["z"] if gate else None, v["wp"], rho, eps)[0]

    r1, _, rs, rp = run()
    g, _ = rb.block_norm_backward(dro, do, v["y"], r1, rs, rp, v["wq"], v["z"] if gate else None, v["wp"], rho)
    for k, name in (("y", "dy"), ("res", "dresidual"), ("wq", "dw_post"), ("wp", "dw_pre")) + \
            ((("z", "dz"),) if gate else ()):
        num = np.zeros_like(v[k])
        for j in np.ndindex(num.shape):
            keep, f = v[k][j], []
            for e in (1e-5, -1e-5):
                v[k][j] = keep + e
                out = run()
                f.append((out[0] * dro).sum() + (out[1] * do).sum())
            v[k][j] = keep
            num[j] = (f[0] - f[1]) / 2e-5
        # central differences: truncation ~1e-10 times the third derivative, cancellation ~1e-10
        assert np.abs(num - g[name]).max() < 1e-7, name


def _args(**kw):
    a = mb.MambaBlockNormArgs()
    a.residual = a.residual_out = a.rstd_post = a.rstd_pre = 4096  # never dereferenced
    a.y, a.out = 8192, 12288
    a.rows, a.cols, a.dtype, a.residual_scale, a.eps = 4, 8, mb.F32, 1.0, 1e-5
    a.y_stride = a.z_stride = 8
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "negative"), (dict(cols=-1), "negative"), (dict(cols=16385), "16384"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(eps=float("inf")), "eps"),
    (dict(residual_scale=float("nan")), "residual_scale"), (dict(residual_scale=float("inf")), "residual_scale"),
    (dict(y=None), "null"), (dict(residual=None), "null"), (dict(residual_out=None), "null"),
    (dict(y=4098), "aligned"), (dict(z=4098), "aligned"), (dict(residual=4098), "aligned"), (dict(out=4098), "aligned"),
    (dict(w_post=4098), "aligned"), (dict(w_pre=4098), "aligned"), (dict(rstd_post=4098), "aligned"),
    (dict(out=8192), "own"), (dict(out=4096), "own"), (dict(residual_out=8192), "residual_out")])
def test_forward_refusals(change, text):
    assert mb.lib().mamba_block_norm(ctypes.byref(_args(**change)), None) == -1
    assert text in mb.last_error()


def test_empty_and_null():
    L = mb.lib()
    assert L.mamba_block_norm(None, None) == -1 and L.mamba_block_norm_workspace(None) == 0
    assert L.mamba_block_norm(ctypes.byref(_args(rows=0)), None) == 0
    assert L.mamba_block_norm(ctypes.byref(_args(cols=0)), None) == 0
    assert L.mamba_block_norm_backward(ctypes.byref(_args()), None, None, 0, None) == -1


@pytest.mark.parametrize("args,change,text", [
    ({}, dict(dresidual=None), "null"), ({}, dict(dy=None), "null"), ({}, dict(dout=None, dresidual_out=None), "null"),
    (dict(rstd_post=None), {}, "null"), (dict(rstd_pre=None), {}, "rstd_pre"), (dict(z=4096), dict(dz=None), "dz"),
    ({}, dict(dy=4098), "aligned"), ({}, dict(dout=4098), "aligned"), ({}, dict(dw_pre=4098), "aligned"),
    ({}, dict(dy_stride=7), "overlap"), (dict(z=28672), dict(dz=32768, dz_stride=7), "overlap"),
    ({}, dict(dy=8192), "inputs"), ({}, dict(dresidual=4096), "inputs"), ({}, dict(dresidual=24576), "own"),
    (dict(z=28672), dict(dz=24576), "own"), (dict(z=28672), dict(dz=28672), "inputs"),
    ({}, dict(ws=None), "workspace"), ({}, dict(short=1), "workspace"), ({}, dict(ws=4104), "workspace")])
def test_backward_refusals(args, change, text):
    a = _args(**args)
    g = mb.MambaBlockNormGrads()
    g.dresidual_out = g.dresidual = g.dw_post = g.dw_pre = 16384
    g.dout, g.dy = 20480, 24576
    g.dy_stride = g.dz_stride = 8
    ws, short = change.pop("ws", 4096), change.pop("short", 0)
    for k, v in change.items():
        setattr(g, k, v)
    need = mb.lib().mamba_block_norm_workspace(ctypes.byref(a))
    assert need > 0
    assert mb.lib().mamba_block_norm_backward(ctypes.byref(a), ctypes.byref(g), ws, need - short, None) == -1
    assert text in mb.last_error()


def test_binding_refuses_wrong_tensors():
    import torch
    y = torch.zeros((3, 8))
    for kw in (dict(z=y[:2]), dict(z=y.half()), dict(w_post=torch.zeros(7)), dict(w_pre=torch.zeros(8).half()),
               dict(out=y.half()), dict(residual_out=y.half())):
        with pytest.raises(mb.MambaError):
            mb.block_norm(y, y, **kw)
    with pytest.raises(mb.MambaError):
        mb.block_norm(y.double(), y)
    with pytest.raises(mb.MambaError):
        mb.block_norm(y, y.t().contiguous().t())
    with pytest.raises(mb.MambaError, match="rstd_pre"):
        mb.block_norm_backward(y, y, y, y, torch.zeros(3), None)
    with pytest.raises(mb.MambaError, match="CUDA"):
        mb.block_norm(y, y)
