"""Device-pointer calls on the model's own stream see what the default stream
was given before them, without a synchronisation by the caller."""
import numpy as np
import pytest
import torch

import mamba_b200 as mb

pytestmark = pytest.mark.gpu


def _late_copy(dst, src):
    """Fills dst on the default stream, about 0.1 s from now."""
    torch.cuda._sleep(200_000_000)
    dst.copy_(src)


def test_forward_waits_for_the_default_stream(cuda):
    m = mb.Model(128, 16, 4, 2, 2, mb.F16)
    m.init_random(5)
    h = np.random.default_rng(1).standard_normal((2, 300, 128)).astype(np.float32)
    want = m.forward(h)
    src = torch.from_numpy(h).cuda()
    x = torch.full_like(src, 7.0)
    out = torch.empty_like(src)
    torch.cuda.synchronize()
    _late_copy(x, src)
    m.forward_device(x.data_ptr(), out.data_ptr(), 2, 300)
    torch.cuda.synchronize()
    assert np.array_equal(out.cpu().numpy(), want)


def test_step_waits_for_the_default_stream(cuda):
    m = mb.Model(128, 16, 4, 2, 2, mb.F16)
    m.init_random(5)
    tok = np.random.default_rng(2).standard_normal((3, 4, 128)).astype(np.float32)
    a, b = m.create_state(4), m.create_state(4)
    src = torch.from_numpy(tok).cuda()
    x = torch.full_like(src[0], 7.0)
    out = torch.empty_like(x)
    torch.cuda.synchronize()
    for t in range(3):  # the first step captures the graph, the others replay it
        _late_copy(x, src[t])
        a.step_device(x.data_ptr(), out.data_ptr())
        torch.cuda.synchronize()
        same = np.array_equal(out.cpu().numpy(), b.step(tok[t]))
        assert same, t


def test_a_given_stream_is_left_alone(cuda):
    """Work on a stream of the caller does not wait for the default stream."""
    m = mb.Model(128, 16, 4, 2, 2, mb.F16)
    m.init_random(5)
    h = np.random.default_rng(3).standard_normal((1, 40, 128)).astype(np.float32)
    want = m.forward(h)
    x = torch.from_numpy(h).cuda()
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    m.forward_device(x.data_ptr(), out.data_ptr(), 1, 40, side.cuda_stream)
    torch.cuda.synchronize()
    for use in ("argument", "set_stream"):
        out.zero_()
        torch.cuda.synchronize()
        torch.cuda._sleep(1_000_000_000)
        busy = torch.cuda.Event()
        busy.record()
        if use == "argument":
            m.forward_device(x.data_ptr(), out.data_ptr(), 1, 40, side.cuda_stream)
        else:
            m.set_stream(side.cuda_stream)
            m.forward_device(x.data_ptr(), out.data_ptr(), 1, 40)
        side.synchronize()
        assert not busy.query()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
    m.set_stream(0)
