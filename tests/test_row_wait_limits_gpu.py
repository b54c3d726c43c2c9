"""Row waits of the layer norm and of the embedding's gradient that run out: with
a short limit, on rows that nothing fetches, each gives up, sets its bit of the
device status and leaves the context and the operators usable."""
import time

import pytest
import torch

import mamba_b200 as mb

pytestmark = pytest.mark.gpu


def test_row_waits_give_up_and_report(cuda):
    lib = mb.lib()
    lib.mamba_device_status(1)
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(15000, 131, device="cuda", generator=g).half()  # rows through the ring, both passes
    ids = torch.randint(-1, 40, (15000,), device="cuda", generator=g)

    def run():
        y, mean, rstd = mb.layer_norm(x, return_stats=True)
        return [y, *mb.layer_norm_backward(y, x, mean, rstd), mb.embedding_backward(x, ids, 40)]

    before = run()
    assert lib.mamba_device_status(0) == 0
    for _ in range(2):  # a second time: nothing of the first is left
        t0 = time.perf_counter()
        assert lib.mamba_selftest_row_waits(5000, None) == 0, mb.last_error()
        # two waits of 5 ms, each with as long again for the copies in flight
        assert 0.02 <= time.perf_counter() - t0 < 5.0
        assert lib.mamba_device_status(0) == 256 | 512
        assert lib.mamba_device_status(1) == 256 | 512
        assert lib.mamba_device_status(0) == 0
        assert all(torch.equal(a, b) for a, b in zip(before, run()))
        assert lib.mamba_device_status(0) == 0


def test_row_wait_limits_are_checked(cuda):
    lib = mb.lib()
    for limit in (0, 2000000):
        assert lib.mamba_selftest_row_waits(limit, None) == -1
        assert "limit" in mb.last_error()
