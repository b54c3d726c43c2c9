"""The block norm on the GPU with narrow rows: one warp a row, many rows per
CTA, so that the shared-memory ring is refilled many times behind each warp's
reads.  Oracle and tolerance are those of the parity tests."""
import pytest
import torch

import mamba_b200 as mb
from test_block_norm_gpu import _backward, _case, _check_backward, _check_forward, _dev, _forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("T,D", [(28000, 72), (28001, 71), (14500, 256), (14500, 249)])
def test_one_warp_rows(cuda, T, D, gate, dtype):
    """Every refill of a place waits for all lanes' reads of it: with the second
    norm's gradient and without it, where the first sum of the backward
    pass depends on none of them."""
    v = _case(T + D, T, D, dtype, gate)
    t = _dev(v)
    mb.device_status(True)
    f = _forward(t)
    _check_forward(v, f, dtype)
    for part in (None, "dout", "dro"):
        w, u = dict(v), dict(t)
        if part:
            w[part] = u[part] = None
        grads = _backward(u, f)
        _check_backward(w, f, grads, dtype)
        again = _backward(u, f)
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(grads, again))
    assert mb.device_status() == 0
