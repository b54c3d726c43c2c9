"""The largest sizes of the gated recurrence, without a GPU: what its 32-bit
positions cannot hold is refused before any device work."""
import ctypes

import pytest

import mamba_b200 as mb


def _args(B, L, D, dtype):
    a = mb.MambaRecurrenceArgs()
    a.x = a.r = a.i = a.lambda_ = 4096  # never dereferenced: the calls below are refused
    a.h = 8192
    a.batch, a.seqlen, a.dim, a.dtype, a.c = B, L, D, dtype, 8.0
    for s in (a.x_stride, a.r_stride, a.i_stride, a.h_stride):
        s[0], s[1] = L * D, D
    return a


@pytest.mark.parametrize("dtype", [mb.F16, mb.F32])
@pytest.mark.parametrize("backward", [0, 1])
def test_sequences_near_two_to_the_31(backward, dtype):
    """A tile's end has to be a 32-bit number: (k + 1) * tile wrapped for the last
    tile of longer sequences, whose final state was then never written."""
    lib = mb.lib()
    size = lambda L: lib.mamba_gated_recurrence_workspace(ctypes.byref(_args(1, L, 2, dtype)), backward)  # noqa: E731
    assert size(2 ** 31 - 257) > 0
    g = mb.MambaRecurrenceGrads()
    g.dh, g.dx, g.dr, g.di, g.dlambda = 4096, 16384, 20480, 24576, 28672
    for L in (2 ** 31 - 256, 2 ** 31 - 63, 2 ** 31 - 1):
        assert size(L) == 0
        for s in (g.dh_stride, g.dx_stride, g.dr_stride, g.di_stride):
            s[0], s[1] = 2 * L, 2
        a = _args(1, L, 2, dtype)
        if backward:
            rc = lib.mamba_gated_recurrence_backward(ctypes.byref(a), ctypes.byref(g), 4096, 1 << 60, None)
        else:
            rc = lib.mamba_gated_recurrence(ctypes.byref(a), 4096, 1 << 60, None)
        assert rc == -1 and "tokens" in mb.last_error()
