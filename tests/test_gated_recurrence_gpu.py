"""GPU parity of the gated linear recurrence (forward, backward, step) against
the FP64 oracle on the same (rounded) inputs.

Tolerance, per element: |gpu - ref| <= u |ref| + d * mag + tiny, where u is the
output type's half step (2^-11 FP16, 2^-24 FP32), tiny half of FP16's smallest
step, and mag the largest magnitude (sum of absolute terms) in the tensor.
d bounds the FP32 evaluation: per token ~16 roundings of 2^-24 in the gates
and one in the running sum, which stays for at most 1/(1 - a) <= 2000 tokens
of these inputs: d = 2^-24 (16 + min(L, 2000)); FP16 tensors add 1e-5 for the
short series and the approximate exponentials."""
import ctypes

import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import recurrent_block as rb

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_memory():
    """Later tests find the allocator as a fresh process has it: with large
    cached blocks, tensors would no longer come from calls that synchronise."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()

C = 8.0


def _case(seed, B, L, D, dtype, ragged=False, resets=False, h0=True):
    rng = np.random.default_rng(seed)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    v = {k: rng.standard_normal((B, L, D)).astype(np_t) for k in ("x", "r", "i", "dh")}
    decay = rng.uniform(0.9, 0.999, D)
    v["lam"] = np.log(np.expm1(-np.log(decay) / C)).astype(np.float32)
    v["h0"] = rng.standard_normal((B, D)).astype(np.float32) if h0 else None
    v["dfinal"] = rng.standard_normal((B, D)).astype(np.float32) if h0 else None
    v["lengths"] = v["resets"] = None
    if ragged:
        v["lengths"] = rng.integers(0, L + 1, B).astype(np.int32)
        v["lengths"][-1] = 0
        v["lengths"][0] = L
    if resets:
        v["resets"] = (rng.random((B, L)) < 0.1).astype(np.uint8)
    return v


def _dev(v):
    return {k: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for k, a in v.items()}


def _tol(dtype, L):
    d = 2.0 ** -24 * (16 + min(L, 2000))
    return (2.0 ** -11, d + 1e-5) if dtype == torch.float16 else (2.0 ** -24, d)


def _close(got, ref, mag, u, d, name=""):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all(), name
    if not got.size:
        return
    err = np.abs(got - ref) - (u * np.abs(ref) + d * mag.max() + 2.0 ** -25)
    assert err.max() <= 0, (name, err.max(), np.unravel_index(err.argmax(), err.shape))


def _forward(t, **kw):
    return mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], c=C, initial_state=t["h0"], lengths=t["lengths"],
                               resets=t["resets"], return_final_state=True, **kw)


def _backward(t, h, **kw):
    return mb.gated_recurrence_backward(t["dh"], t["x"], t["r"], t["i"], t["lam"], h, c=C, initial_state=t["h0"],
                                        lengths=t["lengths"], resets=t["resets"], dfinal_state=t["dfinal"], **kw)


def _check_forward(v, h, hN, dtype):
    u, d = _tol(dtype, v["x"].shape[1])
    ref, fin, mag = rb.gated_recurrence(v["x"], v["r"], v["i"], v["lam"], C, v["h0"], v["lengths"], v["resets"])
    scale = np.concatenate([mag.ravel(), np.abs(fin).ravel()])
    _close(h, ref, scale, u, d, "h")
    _close(hN, fin, scale, 2.0 ** -24, d, "final state")


def _check_backward(v, h, grads, dtype):
    L = v["x"].shape[1]
    u, d = _tol(dtype, L)
    ref, mag = rb.gated_recurrence_backward(v["dh"], v["x"], v["r"], v["i"], v["lam"], h, C, v["h0"], v["lengths"],
                                            v["resets"], v["dfinal"])
    for got, k in zip(grads, ("dx", "dr", "di", "dlam", "dh0")):
        scale = mag[k] if mag[k].size else np.zeros(1)
        _close(got, ref[k], scale, u if k in ("dx", "dr", "di") else 2.0 ** -24, d, k)


SHAPES = [(1, 1, 1), (2, 1, 64), (1, 7, 3), (3, 64, 64), (2, 65, 130), (2, 129, 66), (1, 257, 1001), (2, 300, 256),
          (1, 2000, 96), (5, 17, 33), (2, 513, 72),
          (24, 140, 1000)]  # the last: enough rows and channels for CTAs to walk whole rows


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("ragged,resets,h0", [(False, False, False), (False, False, True), (True, False, True),
                                              (False, True, True), (True, True, False)])
@pytest.mark.parametrize("B,L,D", SHAPES)
def test_forward_and_backward(cuda, B, L, D, ragged, resets, h0, dtype):
    v = _case(B * 1000 + L + D, B, L, D, dtype, ragged, resets, h0)
    t = _dev(v)
    h, hN = _forward(t)
    grads = _backward(t, h)
    torch.cuda.synchronize()
    assert mb.device_status() == 0
    _check_forward(v, h, hN, dtype)
    _check_backward(v, h.cpu().numpy(), grads, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_strided_views(cuda, dtype, offset):
    """x, r, i as column blocks of one wide projection whose rows are not
    aligned to more than an element, time-major outputs, and a batch read
    through a transposed view."""
    B, L, D = 3, 150, 70
    v = _case(5, B, L, D, dtype)
    t = _dev(v)
    wide = torch.full((L, B, 3 * D + 9), float("nan"), dtype=dtype, device="cuda")
    views = {}
    for k, name in enumerate(("x", "r", "i")):
        views[name] = wide[:, :, offset + k * (D + 1):offset + k * (D + 1) + D].transpose(0, 1)
        views[name].copy_(t[name])
        t[name] = views[name]
    out = torch.full((L, B, D + 5), float("nan"), dtype=dtype, device="cuda")
    ho = out[:, :, offset:offset + D].transpose(0, 1)
    h, hN = _forward(t, h=ho)
    outs = [torch.full_like(out, float("nan")) for _ in range(3)]
    grads = _backward(t, h, **{n: o[:, :, offset:offset + D].transpose(0, 1) for n, o in zip(("dx", "dr", "di"), outs)})
    torch.cuda.synchronize()
    assert h.data_ptr() == ho.data_ptr()
    _check_forward(v, h, hN, dtype)
    _check_backward(v, h.cpu().numpy(), grads, dtype)
    for o in [out] + outs:  # nothing outside the views
        assert o[:, :, :offset].isnan().all() and o[:, :, offset + D:].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_padding_is_neither_read_nor_written(cuda, dtype):
    B, L, D = 4, 200, 64
    v = _case(9, B, L, D, dtype, ragged=True)
    t = _dev(v)
    for b, n in enumerate(v["lengths"]):
        for k in ("x", "r", "i", "dh"):
            t[k][b, n:] = float("nan") if b % 2 else float("inf")
    mark = 7.0
    h = torch.full((B, L, D), mark, dtype=dtype, device="cuda")
    h, hN = _forward(t, h=h)
    outs = [torch.full_like(h, mark) for _ in range(3)]
    h_in = h.clone()
    for b, n in enumerate(v["lengths"]):
        h_in[b, n:] = float("nan")
    grads = _backward(t, h_in, dx=outs[0], dr=outs[1], di=outs[2])
    torch.cuda.synchronize()
    for o in [h] + outs:
        for b, n in enumerate(v["lengths"]):
            assert (o[b, n:] == mark).all()
            o[b, n:] = 0
    _check_forward(v, h, hN, dtype)
    _check_backward(v, h.cpu().numpy(), grads, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_lengths_outside_the_range_are_clamped(cuda, dtype):
    v = _case(4, 3, 40, 32, dtype)
    v["lengths"] = np.array([1000, -5, 40], np.int32)
    t = _dev(v)
    h, hN = _forward(t)
    grads = _backward(t, h)
    _check_forward(v, h, hN, dtype)
    _check_backward(v, h.cpu().numpy(), grads, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_extreme_gates(cuda, dtype):
    """Gates that close or open completely, decays of 0 and 1: finite, and
    equal to the formulas' limits."""
    B, L, D = 2, 70, 40
    v = _case(2, B, L, D, dtype)
    big = np.float32(60000.0) if dtype == torch.float16 else np.float32(3e38)
    v["r"][:, ::3] = -big
    v["r"][:, 1::7] = big
    v["i"][:, ::5] = big
    v["i"][:, 2::5] = -big
    v["r"][:, 5::11] = -12.0
    v["lam"][:8] = [-90, -40, -25, -15, 10, 40, 100, 0]
    v["x"][:, ::13] = 0
    t = _dev(v)
    h, hN = _forward(t)
    grads = _backward(t, h)
    torch.cuda.synchronize()
    _check_forward(v, h, hN, dtype)
    _check_backward(v, h.cpu().numpy(), grads, dtype)


def test_gradients_against_differences(cuda):
    """FP32 gradients against central differences of the FP64 forward."""
    v = _case(8, 2, 12, 6, torch.float32, ragged=True, resets=True)
    v["lengths"] = np.array([12, 7], np.int32)
    t = _dev(v)
    h, _ = _forward(t)
    grads = dict(zip(("x", "r", "i", "lam", "h0"), _backward(t, h)))
    w = {k: v[k].astype(np.float64) for k in grads}

    def loss():
        hh, fin, _ = rb.gated_recurrence(w["x"], w["r"], w["i"], w["lam"], C, w["h0"], v["lengths"], v["resets"])
        return (hh * v["dh"]).sum() + (fin * v["dfinal"]).sum()

    for k, g in grads.items():
        num = np.zeros_like(w[k])
        for j in np.ndindex(num.shape):
            keep = w[k][j]
            w[k][j] = keep + 1e-5
            up = loss()
            w[k][j] = keep - 1e-5
            num[j] = (up - loss()) / 2e-5
            w[k][j] = keep
        # FP32 rounding of the gradients (~2^-24 * 40 of the largest) + differences (1e-8)
        assert np.abs(g.double().cpu().numpy() - num).max() < 1e-5 * max(1.0, np.abs(num).max()), k


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_empty_sizes(cuda, dtype):
    t = _dev(_case(1, 3, 5, 8, dtype))
    for k in ("x", "r", "i", "dh"):
        t[k] = t[k][:, :0]
    h, hN = _forward(t)
    assert h.shape == (3, 0, 8) and torch.equal(hN, t["h0"])
    dx, dr, di, dlam, dh0 = _backward(t, h)
    assert dx.shape == (3, 0, 8) and torch.equal(dh0, t["dfinal"]) and not dlam.any()
    t = _dev(_case(1, 3, 5, 8, dtype))
    t = {k: a[:0] if a is not None and k not in ("lam",) else a for k, a in t.items()}
    h, hN = _forward(t)
    dlam = _backward(t, h)[3]
    assert h.shape[0] == 0 and not dlam.any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(2, 1500, 200), (8, 700, 1024), (40, 200, 640)])
def test_repeated_calls_give_the_same_bits(cuda, dtype, B, L, D):
    t = _dev(_case(6, B, L, D, dtype))
    first = None
    for _ in range(5):
        h, hN = _forward(t)
        out = [h, hN] + list(_backward(t, h))
        if first is None:
            first = out
        assert all(torch.equal(a, b) for a, b in zip(first, out))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_pieces_of_a_sequence_join(cuda, dtype):
    """Prefill in two calls through the state, then single tokens: the same
    function as one call over the whole sequence."""
    B, L, D = 3, 90, 136
    v = _case(12, B, L, D, dtype)
    t = _dev(v)
    whole, hN = _forward(t)
    part = {k: a[:, :60] if k in ("x", "r", "i") else a for k, a in t.items()}
    h1, s = _forward(part)
    hs = [h1]
    for k in range(60, L):
        hk, s = mb.gated_recurrence_step(t["x"][:, k], t["r"][:, k], t["i"][:, k], t["lam"], s, c=C)
        hs.append(hk[:, None])
    h = torch.cat(hs, 1)
    _check_forward(v, h, s, dtype)
    _check_forward(v, whole, hN, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,D", [(1, 1), (1, 64), (7, 33), (256, 640), (3, 1001), (64, 1028)])
def test_step(cuda, dtype, B, D):
    v = _case(B + D, B, 1, D, dtype)
    t = _dev(v)
    keep = t["h0"].clone()
    x, r, i = (t[k][:, 0] for k in ("x", "r", "i"))
    h, s = mb.gated_recurrence_step(x, r, i, t["lam"], t["h0"], c=C)
    assert torch.equal(t["h0"], keep)
    _check_forward(v, h[:, None], s, dtype)
    # in place, from the column blocks of one wide projection
    wide = torch.zeros((B, 3 * D + 3), dtype=dtype, device="cuda")
    views = [wide[:, 1 + k * (D + 1):1 + k * (D + 1) + D] for k in range(3)]
    for w, a in zip(views, (x, r, i)):
        w.copy_(a)
    h2, s2 = mb.gated_recurrence_step(*views, t["lam"], keep, c=C, state_out=keep)
    assert s2.data_ptr() == keep.data_ptr()
    assert torch.equal(h2, h) and torch.equal(keep, s)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_streams_graphs_and_a_shared_workspace(cuda, dtype):
    """On a side stream, two differently sized calls in turn on one workspace,
    and a captured forward + backward replayed on new inputs."""
    cases = [_case(20, 2, 700, 96, dtype), _case(21, 1, 1111, 40, dtype, resets=True)]
    ts = [_dev(v) for v in cases]
    need = 0
    for t in ts:
        a = mb._recurrence_args("t", t["x"], t["r"], t["i"], t["lam"], C, None, None, None)
        need = max([need] + [mb.lib().mamba_gated_recurrence_workspace(ctypes.byref(a), k) for k in (0, 1)])
    ws = torch.full((max(need, 16),), 0xAB, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    results = []
    with torch.cuda.stream(side):
        for _ in range(2):
            for t in ts:
                h, hN = _forward(t, workspace=ws)
                results.append((h, hN, _backward(t, h, workspace=ws)))
    side.synchronize()
    for k, (h, hN, grads) in enumerate(results):
        _check_forward(cases[k % 2], h, hN, dtype)
        _check_backward(cases[k % 2], h.cpu().numpy(), grads, dtype)

    t = ts[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        h, hN = _forward(t)
        grads = _backward(t, h)
    for seed in (30, 31):
        v = _case(seed, 2, 700, 96, dtype)
        for k, a in _dev(v).items():
            if a is not None:
                t[k].copy_(a)
        graph.replay()
        torch.cuda.synchronize()
        _check_forward(v, h, hN, dtype)
        _check_backward(v, h.cpu().numpy(), grads, dtype)
    assert mb.device_status() == 0


def test_offsets_beyond_32_bits(cuda):
    """Rows that start more than 2^31 elements apart."""
    L, D, gap = 40, 64, (1 << 31) + 64
    free = torch.cuda.mem_get_info()[0]
    if free < 3 * 2 * (gap + L * D):
        pytest.skip("needs 13 GB of free device memory")
    v = _case(3, 2, L, D, torch.float16)
    t = _dev(v)
    big = torch.zeros(gap + L * D, dtype=torch.float16, device="cuda")
    out = torch.zeros(gap + L * D, dtype=torch.float16, device="cuda")
    view = lambda buf: buf.as_strided((2, L, D), (gap, D, 1))  # noqa: E731
    view(big).copy_(t["x"])
    t["x"] = view(big)
    h, hN = _forward(t, h=view(out))
    _check_forward(v, h, hN, torch.float16)
    t["h_big"] = h
    out2 = torch.zeros(gap + L * D, dtype=torch.float16, device="cuda")
    grads = _backward(t, h, dx=view(out2))
    _check_backward(v, h.cpu().numpy(), grads, torch.float16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_stream_argument(cuda, dtype):
    """On a given stream (object or handle), what the helper allocates and
    zeroes belongs to that stream: back-to-back calls from a busy current
    stream do not disturb each other's scratch."""
    v = _case(40, 4, 900, 128, dtype, ragged=True)
    t = _dev(v)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    outs = []
    for k in range(6):
        s = side if k % 2 else side.cuda_stream
        h, hN = _forward(t, stream=s)
        outs.append((h, hN, _backward(t, h, stream=s)))
        torch.full((1 << 22,), float("nan"), device="cuda")  # reuses whatever the current stream was given back
    torch.cuda.synchronize()
    for h, hN, grads in outs:
        _check_forward(v, h, hN, dtype)
        _check_backward(v, h.cpu().numpy(), grads, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("order", ["batch", "time"])
@pytest.mark.parametrize("B,L,D", [(3, 150, 72), (1, 300, 64), (24, 130, 1024), (5, 1, 64)])
def test_aligned_views(cuda, B, L, D, order, dtype):
    """Column blocks of a projection whose rows keep 16-byte alignment, with
    batch or time outermost: the kernels that fetch tiles by tensor maps."""
    v = _case(B + L + D, B, L, D, dtype, ragged=B > 1, resets=True)
    t = _dev(v)
    pitch = 3 * D + 16

    def buf():
        shape = (L, B, pitch) if order == "time" else (B, L, pitch)
        w = torch.full(shape, float("nan"), dtype=dtype, device="cuda")
        return w, (w.transpose(0, 1) if order == "time" else w)

    wide, view = buf()
    for k, name in enumerate(("x", "r", "i")):
        part = view[:, :, 8 + k * D:8 + (k + 1) * D]
        part.copy_(t[name])
        t[name] = part
    out, oview = buf()
    for b, n in enumerate(v["lengths"] if v["lengths"] is not None else []):
        oview[b, n:] = 0
    h, hN = _forward(t, h=oview[:, :, 16:16 + D])
    dwide, dview = buf()
    dview[:, :, 8:8 + 3 * D] = 0
    grads = _backward(t, h, **{n: dview[:, :, 8 + k * D:8 + (k + 1) * D] for k, n in enumerate(("dx", "dr", "di"))})
    torch.cuda.synchronize()
    assert mb.device_status() == 0
    _check_forward(v, h, hN, dtype)
    _check_backward(v, h.cpu().numpy(), grads, dtype)
    assert dwide[..., :8].isnan().all() and dwide[..., 8 + 3 * D:].isnan().all()


def test_many_rows(cuda):
    """More batch rows than a grid dimension holds."""
    B, L, D = 70000, 2, 8
    v = _case(1, B, L, D, torch.float16, ragged=True)
    t = _dev(v)
    h, hN = _forward(t)
    _check_forward(v, h, hN, torch.float16)
    _check_backward(v, h.cpu().numpy(), _backward(t, h), torch.float16)
    hs, s = mb.gated_recurrence_step(t["x"][:, 0], t["r"][:, 0], t["i"][:, 0], t["lam"], t["h0"], c=C)
    v1 = dict(v, x=v["x"][:, :1], r=v["r"][:, :1], i=v["i"][:, :1], lengths=None)
    _check_forward(v1, hs[:, None], s, torch.float16)


def test_keywords_and_refusals(cuda):
    t = _dev(_case(2, 2, 20, 16, torch.float32))
    a = mb.gated_recurrence(x=t["x"], r=t["r"], i=t["i"], lam=t["lam"], stream=torch.cuda.current_stream())
    assert torch.equal(a, mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"]))
    with pytest.raises(mb.MambaError, match="inputs"):
        mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], h=t["x"])
    with pytest.raises(mb.MambaError, match="workspace"):
        mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], workspace=torch.empty(8, dtype=torch.uint8, device="cuda"))
    with pytest.raises(mb.MambaError):
        mb.gated_recurrence(t["x"], t["r"], t["i"], t["lam"], lengths=torch.ones(2, dtype=torch.int32))  # on the CPU


def test_a_nan_stays_in_its_row_and_channel(cuda):
    """Without a reset a NaN gate or input reaches every later state of its own
    channel and no other; its gradient every earlier one."""
    for dtype in (torch.float16, torch.float32):
        for name in ("x", "r", "i"):
            for B, L, D in ((2, 200, 64), (2, 200, 33), (40, 70, 640)):
                t = _dev(_case(3, B, L, D, dtype))
                ref = _forward(t)[0]
                t[name][1, 50, 7] = float("nan")
                h, hN = _forward(t)
                assert h[1, 50:, 7].isnan().all() and hN[1, 7].isnan()
                h[1, 50:, 7] = ref[1, 50:, 7]
                assert torch.equal(h, ref)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("B,L,D", [(2, 300, 64), (2, 300, 33), (40, 130, 640), (40, 70, 641)])
def test_a_reset_stops_infinities_and_nan(cuda, B, L, D, dtype):
    """Documents that share a row do not see each other, whatever the one
    before holds: NaN and infinities stay before the reset going forward, and
    behind it going backward."""
    v = _case(5, B, L, D, dtype)
    v["resets"] = np.zeros((B, L), np.uint8)
    cuts = [0, 37, 64, 65, L - 3]
    v["resets"][:, cuts] = 1
    clean = _dev(v)
    href, fref = _forward(clean)
    gref = _backward(clean, href)
    for bad in (float("nan"), float("inf")):
        t = {k: None if a is None else a.clone() for k, a in clean.items()}
        t["x"][0, 40:44] = bad       # the document from 37 to 63
        t["h0"][1] = bad             # before a reset at the first token: unseen
        h, hN = _forward(t)
        assert not h[0, 44:64].isfinite().any()
        h[0, 40:64] = href[0, 40:64]
        assert torch.equal(h, href) and torch.equal(hN, fref)
        t = {k: None if a is None else a.clone() for k, a in clean.items()}
        t["dh"][0, 60:64] = bad
        dx, dr, di, dlam, dh0 = _backward(t, href)
        for got, ref in zip((dx, dr, di), gref):
            assert not got[0, 40:60].isfinite().all()
            got[0, 37:64] = ref[0, 37:64]
            assert torch.equal(got, ref)
        assert torch.equal(dh0, gref[4]) and not dh0.any()  # the first token resets
