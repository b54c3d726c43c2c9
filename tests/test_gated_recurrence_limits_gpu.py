"""The gated recurrence on the GPU where little of a batch is left, or little of
a value: padded batches of mostly empty rows, states that live for tens of
thousands of tokens, gates that are nearly closed or nearly open.  The
comparison is with the FP64 oracle on the same (rounded) inputs, element by
element."""
import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import recurrent_block as rb

pytestmark = pytest.mark.gpu

C = 8.0


def _dev(*arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arrays]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(64, 2048, 64), (300, 700, 64), (5, 4096, 256)])
def test_mostly_empty_rows(cuda, B, L, D, dtype):
    """A padded batch whose rows end early: most tiles lie behind their row's
    end, several in a row for each CTA.  No wait runs out (bit 6), and
    every call gives the same bits."""
    rng = np.random.default_rng(B)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    x, r, i = (rng.standard_normal((B, L, D)).astype(np_t) for _ in range(3))
    lam = rng.uniform(-6, -3, D).astype(np.float32)
    h0 = rng.standard_normal((B, D)).astype(np.float32)
    lengths = np.where(rng.random(B) < 0.7, rng.integers(0, 3, B), rng.integers(0, 200, B)).astype(np.int32)
    lengths[B // 2] = L
    tx, tr, ti, tl, th, tn = _dev(x, r, i, lam, h0, lengths)
    mb.device_status(True)
    first = None
    for _ in range(40):
        out = mb.gated_recurrence(tx, tr, ti, tl, c=C, initial_state=th, lengths=tn, return_final_state=True)
        first = first or out
        assert all(torch.equal(a, b) for a, b in zip(first, out))
    assert mb.device_status() == 0
    keep = [b for b in range(B) if lengths[b] < 200][:20] + [B // 2]
    ref, fin, mag = rb.gated_recurrence(x[keep], r[keep], i[keep], lam, C, h0[keep], lengths[keep])
    # gates: ~16 roundings of 2^-24, and 1e-5 for FP16 tensors' short series; a state of these
    # decays (0.98 and less at r = 0) is below 2^-24 of itself after 1000 tokens
    d = 2.0 ** -24 * 1016 + (1e-5 if dtype == torch.float16 else 0.0)
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -24
    err = np.abs(first[0].double().cpu().numpy()[keep] - ref) - (u * np.abs(ref) + d * mag + 2.0 ** -25)
    assert err.max() <= 0
    last = np.maximum(lengths[keep] - 1, 0)
    fmag = np.where(lengths[keep, None] > 0, mag[np.arange(len(keep)), last], np.abs(h0[keep]))
    err = np.abs(first[1].double().cpu().numpy()[keep] - fin) - (d * fmag + 2.0 ** -25)
    assert err.max() <= 0
