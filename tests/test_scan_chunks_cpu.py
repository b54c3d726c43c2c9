"""The chunks of time that the scan's backward pass cuts a sequence into, from the
size of its workspace (no GPU needed)."""
import ctypes

import pytest

import mamba_b200 as mb


def _workspace(b, L, dim):
    a = mb.MambaScanArgs()
    a.batch, a.seqlen, a.dim, a.dstate = b, L, dim, 16
    return mb.lib().mamba_selective_scan_backward_workspace(ctypes.byref(a))


def _expected(b, L, dim, chunks):
    """Bytes with so many chunks: states before every 8th token and partial rows of dB and dC for each 128 channels;
    with several chunks the sums of dt beside the states, and two sets of states and one of sums per chunk; a row of
    dA, dD and ddt_bias per chunk.  Each array takes whole 256 bytes."""
    per, subs = -(-dim // 4) * 64, -(-L // 8)
    several = chunks > 1
    floats = [b * subs * per, several * b * subs * -(-dim // 4) * 4, several * b * chunks * per,
              several * b * chunks * per, several * b * chunks * dim, -(-dim // 128) * b * L * 32,
              b * chunks * (per + -(-2 * dim // 4) * 4)]
    return sum(-(-4 * n // 256) * 256 for n in floats)


def _chunks(b, L, dim):
    found = [n for n in range(1, -(-L // 8) + 1) if _expected(b, L, dim, n) == _workspace(b, L, dim)]
    assert len(found) == 1, (b, L, dim, found)
    return found[0]


@pytest.mark.parametrize("b,L,dim", [(1, 16384, 37888), (2, 16384, 18944), (8, 1000, 4736)])
def test_one_round_of_channel_blocks_is_cut_in_at_most_two(b, L, dim):
    """296 blocks of channels, a round of CTAs: as long chunks as may be."""
    assert _chunks(b, L, dim) <= 2


@pytest.mark.parametrize("b,L,dim", [(1, 16385, 37888), (8, 40000, 4736), (296, 50001, 128), (8, 200000, 4736),
                                     (592, 33000, 100)])
def test_no_chunk_is_longer_than_16384_tokens(b, L, dim):
    """With the channels and the batch filling the GPU the bound is what cuts long sequences."""
    assert _chunks(b, L, dim) >= -(-L // 16384)


def test_few_channels_take_short_chunks():
    """One block of channels: CTAs for the GPU only by many chunks."""
    assert _chunks(1, 4096, 128) >= 100
    assert _chunks(1, 1, 1) == 1 and _chunks(3, 8, 40) == 1
