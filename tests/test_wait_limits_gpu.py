"""Waits of the recurrent-block operators that run out: with a short limit, on
conditions that nothing fulfils, each gives up, sets its bit of the device
status and leaves the context and the operators usable."""
import time

import pytest
import torch

import mamba_b200 as mb

pytestmark = pytest.mark.gpu


def test_every_wait_gives_up_and_reports(cuda):
    lib = mb.lib()
    lib.mamba_device_status(1)
    torch.manual_seed(0)
    x = torch.randn(3, 700, 64, device="cuda", dtype=torch.float16)
    lam = torch.full((64,), -4.0, device="cuda")
    lengths = torch.tensor([700, 0, 65], dtype=torch.int32, device="cuda")
    y, res = x.reshape(-1, 64), torch.randn(2100, 64, device="cuda")
    q, s = mb.quantize_rows(y)

    def run():
        h = mb.gated_recurrence(x, x, x, lam, lengths=lengths)
        g = mb.gated_recurrence_backward(x, x, x, x, lam, h, lengths=lengths)
        return [h, *g, *mb.block_norm(y, res), mb.linear_i8(q, s, q, s)]

    before = run()
    assert lib.mamba_device_status(0) == 0
    for _ in range(2):  # a second time: nothing of the first is left
        t0 = time.perf_counter()
        assert lib.mamba_selftest_bounded_wait(5000, None) == 0, mb.last_error()
        # one wait of 5 ms each; box and row waits give the copies in flight as long again
        assert 0.005 * 7 <= time.perf_counter() - t0 < 5.0
        assert lib.mamba_device_status(1) == 8 | 64 | 128 | 256
        assert lib.mamba_device_status(0) == 0
        assert all(torch.equal(a, b) for a, b in zip(before, run()))
        assert lib.mamba_device_status(0) == 0
