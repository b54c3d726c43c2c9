"""8-bit rows and the 8-bit linear layer, without a GPU: the entry points'
refusals (argument checks run before any device work)."""
import numpy as np
import pytest

import mamba_b200 as mb
from oracle import recurrent_block as rb


@pytest.mark.parametrize("change,text", [
    (dict(dtype=2), "dtype"), (dict(rows=-1), "negative"), (dict(cols=-1), "negative"), (dict(x=None), "null"),
    (dict(q=None), "null"), (dict(scale=None), "null"), (dict(scale=4098), "null"), (dict(x=4098), "aligned"),
    (dict(ldq=7), "overlap")])
def test_quantize_refusals(change, text):
    v = dict(x=4096, ldx=8, q=4096, ldq=8, scale=4096, rows=4, cols=8, dtype=mb.F32, stream=None)
    v.update(change)
    assert mb.lib().mamba_quantize_rows(*v.values()) == -1
    assert text in mb.last_error()


@pytest.mark.parametrize("change,text", [
    (dict(mode=3), "mode"), (dict(mode=-1), "mode"), (dict(rows=-1), "negative"), (dict(n=-1), "negative"),
    (dict(k=-1), "negative"), (dict(k=131072, ldx=1 << 18, ldw=1 << 18), "131071"), (dict(x=None), "null"),
    (dict(w=None), "null"), (dict(y=None), "null"), (dict(xs=None), "null"), (dict(ws=None), "null"),
    (dict(xs=4098), "aligned"), (dict(ws=4098), "aligned"), (dict(bias=4098), "aligned"),
    (dict(mode=2, y=4098), "aligned"), (dict(y=4097), "aligned"), (dict(ldx=15), "stride"), (dict(ldw=15), "stride"),
    (dict(ldy=7), "stride")])
def test_linear_refusals(change, text):
    v = dict(x=4096, ldx=16, xs=4096, w=4096, ldw=16, ws=4096, bias=None, y=4096, ldy=8, rows=4, n=8, k=16, mode=0,
             stream=None)
    v.update(change)
    assert mb.lib().mamba_linear_i8(*v.values()) == -1
    assert text in mb.last_error()


def test_outputs_that_are_inputs_are_refused():
    L = mb.lib()
    for q, scale in ((4096, 8192), (8192, 8192)):  # x itself, scale itself
        assert L.mamba_quantize_rows(4096, 8, q, 8, scale, 4, 8, mb.F32, None) == -1
        assert "memory of its own" in mb.last_error()
    for y in (4096, 8192, 12288, 16384, 20480):
        assert L.mamba_linear_i8(4096, 16, 8192, 12288, 16, 16384, 20480, y, 8, 4, 8, 16, 2, None) == -1
        assert "one of the inputs" in mb.last_error()


def test_empty_calls():
    assert mb.lib().mamba_quantize_rows(None, 0, None, 0, None, 0, 8, mb.F32, None) == 0
    assert mb.lib().mamba_linear_i8(None, 0, None, None, 0, None, None, None, 0, 0, 8, 8, 0, None) == 0
    assert mb.lib().mamba_linear_i8(None, 0, None, None, 0, None, None, None, 0, 8, 0, 8, 0, None) == 0


def test_binding_refuses_wrong_tensors():
    import torch
    q, s, w, t = (torch.zeros((3, 16), dtype=torch.int8), torch.zeros(3), torch.zeros((5, 16), dtype=torch.int8),
                  torch.zeros(5))
    for args, kw in (((q.float(), s, w, t), {}), ((q, s, w[:, :8].contiguous(), t), {}), ((q, t, w, t), {}),
                     ((q, s, w, s), {}), ((q, s, w, t), dict(bias=s)), ((q, s, w, t), dict(mode=1)),
                     ((q, s, w, t), dict(mode=4)), ((q, s, w, t), dict(y=torch.zeros((3, 5)))),
                     ((q, s, w.t().contiguous().t(), t), {})):
        with pytest.raises(mb.MambaError):
            mb.linear_i8(*args, **kw)
    with pytest.raises(mb.MambaError):
        mb.quantize_rows(torch.zeros((2, 4), dtype=torch.float64))
    with pytest.raises(mb.MambaError, match="CUDA"):
        mb.linear_i8(q, s, w, t)


def test_oracle_quantiser():
    x = np.array([[127.0, 0.5, 1.5, -2.5, 126.5], [0, 0, 0, 0, 0], [1, np.inf, 0, 0, 0], [1, np.nan, 0, 0, 0]])
    q, s = rb.quantize_rows(x.astype(np.float32))
    assert q[0].tolist() == [127, 0, 2, -2, 126] and s[0] == 1
    assert not q[1:].any() and s[1] == 0 and np.isnan(s[2:]).all()
