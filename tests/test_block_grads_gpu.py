"""GPU parity of the gradients of the causal convolution and the selective scan
against the FP64 oracle on the same (rounded) inputs.

Tolerance, per element: |gpu - ref| <= u |ref| + d * mag + tiny, with u the
output type's half step, tiny half of FP16's smallest step and mag the sum of
the absolute terms of that element.  d bounds the FP32 evaluation: each of the
L steps of a state, forward and backward, rounds about 8 times relative to the
state's magnitude, and ~64 roundings outside these: d = 2^-24 (64 + 8 L).  FP16
tensors add 2^-16: e^v - 1 has a relative error up to 2e-6 (a relative error r
of it moves the state by r times its magnitude, however long its memory),
softplus and the reciprocals up to 4e-7, several of which multiply.  Sums over
n terms add 2^-24 n."""
import ctypes

import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
KINDS = [(F32, F32, F32), (F16, F16, F16), (F16, F32, F16), (F16, F32, F32)]


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_memory():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _np(dtype):
    return np.float16 if dtype == F16 else np.float32


def _dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _close(got, ref, mag, name, L, f16, terms=0, approx=2.0 ** -16):
    u = 2.0 ** -11 if got.dtype == F16 else 2.0 ** -24
    d = 2.0 ** -24 * (64 + 8 * L + terms) + (approx if f16 else 0.0)
    got = got.double().cpu().numpy()
    assert got.shape == ref.shape and np.isfinite(got).all(), name
    err = np.abs(got - ref) - (u * np.abs(ref) + d * mag + 2.0 ** -25)
    assert not err.size or err.max() <= 0, (name, err.max())


# ---- convolution ------------------------------------------------------------------
def _conv_case(seed, b, L, D, K, dtype, bias=True):
    rng = np.random.default_rng(seed)
    x, dy = (rng.standard_normal((b, L, D)).astype(_np(dtype)) for _ in range(2))
    w = rng.uniform(-0.5, 0.5, (D, K)).astype(np.float32)
    return dy, x, w, rng.uniform(-0.5, 0.5, D).astype(np.float32) if bias else None


def _conv_check(case, silu, got, dtype):
    ref, mag = tr.conv_backward(*case, silu)
    n = case[0].shape[0] * case[0].shape[1]
    _close(got[0], ref["dx"], mag["dx"], "dx", 0, dtype == F16)
    _close(got[1], ref["dw"], mag["dw"], "dw", 0, dtype == F16, n)
    if case[3] is None:
        assert got[2] is None
    else:
        _close(got[2], ref["dbias"], mag["dbias"], "dbias", 0, dtype == F16, n)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("b,L,D,K", [(1, 1, 1, 1), (1, 1, 4, 8), (2, 3, 5, 4), (3, 7, 12, 8), (2, 16, 130, 2),
                                     (1, 17, 516, 4), (2, 129, 64, 3), (1, 300, 260, 5), (2, 257, 33, 6),
                                     (5, 2, 1000, 7), (1, 4000, 8, 4), (8, 512, 768, 4)])
def test_conv_backward(cuda, b, L, D, K, dtype):
    for silu, bias in ((True, True), (False, True), (True, False), (False, False)):
        case = _conv_case(L + D, b, L, D, K, dtype, bias)
        dy, x, w, bv = (_dev(v) for v in case)
        _conv_check(case, silu, mb.causal_conv1d_backward(dy, x, w, bv, silu=silu), dtype)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_conv_backward_views(cuda, dtype):
    b, L, D, K = 2, 70, 36, 4
    case = _conv_case(9, b, L, D, K, dtype)
    w, bias = _dev(case[2]), _dev(case[3])
    for form in ("columns", "odd columns", "channels first", "one"):
        off = 4 if form == "columns" else 3
        views = []
        for v in (case[0], case[1], np.zeros((b, L, D), _np(dtype))):
            t = _dev(v)
            if form == "channels first":
                t = t.transpose(1, 2).contiguous().transpose(1, 2)
                whole = t
            else:
                whole = torch.full((b, L, D + 12), 7.0, dtype=dtype, device="cuda")
                whole[:, :, off:off + D] = t
                t = whole[:, :, off:off + D]
            views.append((whole, t))
        got = mb.causal_conv1d_backward(views[0][1], views[1][1], w, bias, dx=views[2][1])
        _conv_check(case, True, got, dtype)
        if form != "channels first":
            assert (views[2][0][:, :, :off] == 7).all() and (views[2][0][:, :, off + D:] == 7).all()


def test_conv_backward_extremes_bits_graph_and_empty(cuda):
    case = list(_conv_case(10, 3, 400, 96, 4, F16))
    case[1][0, 5:9] = 60000  # the activation saturates
    case[1][1, 5:9] = -60000
    t = [_dev(v) for v in case]
    _conv_check(case, True, mb.causal_conv1d_backward(*t), F16)
    want = mb.causal_conv1d_backward(*t)
    a = mb.MambaConvGradArgs()
    a.batch, a.seqlen, a.dim, a.K = 3, 400, 96, 4
    ws = torch.full((mb.lib().mamba_causal_conv1d_backward_workspace(ctypes.byref(a)),), 0xAB, dtype=torch.uint8,
                    device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = mb.causal_conv1d_backward(*t, workspace=ws, stream=side)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mb.causal_conv1d_backward(*t)
    new = _conv_case(11, 3, 400, 96, 4, F16)
    for p, q in zip(t, new):
        p.copy_(_dev(q))
    graph.replay()
    torch.cuda.synchronize()
    _conv_check(new, True, got, F16)
    e = torch.zeros((0, 5, 8), device="cuda")
    dx, dw, db = mb.causal_conv1d_backward(e, e, torch.ones((8, 4), device="cuda"), torch.ones(8, device="cuda"))
    assert dx.shape == (0, 5, 8) and (dw == 0).all() and (db == 0).all()


# ---- scan -------------------------------------------------------------------------
def _scan_case(seed, b, L, D, N, kind, gate=True, skip=True, carried=True, bias=True):
    rng = np.random.default_rng(seed)
    xt, dt, bt = (_np(k) for k in kind)
    v = {k: rng.standard_normal((b, L, D)).astype(xt) for k in ("x", "dy", "z")}
    v["delta"] = (0.5 * rng.standard_normal((b, L, D)) - (0 if bias else 3)).astype(dt)
    v["B"], v["C"] = (rng.standard_normal((b, L, N)).astype(bt) for _ in range(2))
    v["A"] = (-np.arange(1, N + 1) * np.exp(0.1 * rng.standard_normal((D, N)))).astype(np.float32)
    v["D"] = rng.standard_normal(D).astype(np.float32) if skip else None
    step = np.exp(rng.uniform(np.log(1e-3), np.log(1e-1), D))
    v["dt_bias"] = np.log(np.expm1(step)).astype(np.float32) if bias else None
    v["initial_state"] = rng.standard_normal((b, D, N)).astype(np.float32) if carried else None
    v["dfinal_state"] = rng.standard_normal((b, D, N)).astype(np.float32) if carried else None
    if not gate:
        v["z"] = None
    return v


def _scan_run(t, **kw):
    names = ("D", "z", "dt_bias", "initial_state", "dfinal_state")
    return mb.selective_scan_backward(t["dy"], t["x"], t["delta"], t["A"], t["B"], t["C"],
                                      **{k: t[k] for k in names}, **kw)


def _scan_check(v, got, kind):
    b, L, D = v["x"].shape
    ref, mag = tr.scan_backward(v["dy"], v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"],
                                v["initial_state"], v["dfinal_state"])
    terms = {"dA": b * L, "dD": b * L, "ddt_bias": b * L, "dB": D, "dC": D}
    absent = {"dD": "D", "dz": "z", "ddt_bias": "dt_bias", "dh0": "initial_state"}
    for g, k in zip(got, ("dx", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddt_bias", "dh0")):
        if k in absent and v[absent[k]] is None:
            assert g is None, k
            continue
        _close(g, ref[k], mag[k], k, L, kind[0] == F16, terms.get(k, 0))


SIZES = [(1, 1, 1, 1), (1, 1, 4, 16), (2, 2, 3, 3), (1, 7, 130, 16), (2, 8, 128, 16), (1, 9, 127, 5), (3, 33, 36, 16),
         (1, 64, 256, 16), (2, 65, 129, 12), (1, 333, 203, 7), (4, 100, 64, 8), (1, 1000, 16, 16), (2, 257, 384, 16)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("b,L,D,N", SIZES)
def test_scan_backward(cuda, b, L, D, N, kind):
    for k, opts in enumerate((dict(), dict(gate=False, carried=False), dict(skip=False, bias=False))):
        v = _scan_case(L + D + k, b, L, D, N, kind, **opts)
        _scan_check(v, _scan_run({n: _dev(a) for n, a in v.items()}), kind)
    assert mb.device_status() == 0


@pytest.mark.parametrize("kind", KINDS)
def test_scan_backward_many_channel_blocks(cuda, kind):
    """Enough blocks of channels for one chunk per sequence (no carries between chunks)."""
    v = _scan_case(1, 12, 40, 128 * 100, 4, kind)
    _scan_check(v, _scan_run({n: _dev(x) for n, x in v.items()}), kind)


@pytest.mark.parametrize("kind", KINDS)
def test_scan_backward_special_A_and_steps(cuda, kind):
    """A of zero, tiny, near the limit's border and positive; steps from e^-20 to 30."""
    v = _scan_case(2, 2, 50, 40, 16, kind, bias=False)
    v["A"][:8, 0] = 0.0
    v["A"][:8, 1] = [-1e-30, 1e-30, -1e-8, 1e-8, -9.9e-7, -1.01e-6, -1e-3, 1e-3]
    v["A"][:8, 2] = 0.01
    v["A"][:, 3] = -300
    v["delta"][:, 10:20] = -20
    v["delta"][0, 20:23] = 30
    v["delta"][1, 30] = -60
    v["A"][20:, 2] = np.linspace(-0.2, -20, 20)
    got = _scan_run({n: _dev(a) for n, a in v.items()})
    _scan_check(v, got, kind)


@pytest.mark.parametrize("kind", KINDS[1:])
@pytest.mark.parametrize("L", [1, 2])
def test_scan_backward_dA_of_short_rows(cuda, kind, L):
    """With no state before them dA is all (dt a - phi) / A, a difference that cancels twice.  Its relative errors:
    1.9e-6 of e (two units of 2^-24 over 1/16), 8e-7 of the series or the difference, twice 4e-7 of dt: 2^-18."""
    v = _scan_case(11 + L, 3, L, 300, 16, kind, carried=False)
    got = _scan_run({n: _dev(a) for n, a in v.items()})
    ref, mag = tr.scan_backward(v["dy"], v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"], v["dt_bias"])
    _close(got[2], ref["dA"], mag["dA"], "dA", L, True, 3 * L, 2.0 ** -18)


def test_scan_backward_long_sequence(cuda):
    """Longer than one chunk may be; sampled against the same call in two halves, joined by the state and its
    gradient (each half's own errors as above)."""
    kind, L, half = (F32, F32, F32), 40000, 17000
    v = _scan_case(12, 1, L, 5, 16, kind)
    t = {n: _dev(a) for n, a in v.items()}
    got = _scan_run(t)
    a, b = ({k: (x[:, s].contiguous() if k in ("x", "dy", "z", "delta", "B", "C") else x) for k, x in t.items()}
            for s in (slice(0, half), slice(half, L)))
    _, mid = mb.selective_scan(a["x"], a["delta"], a["A"], a["B"], a["C"], D=a["D"], z=a["z"], dt_bias=a["dt_bias"],
                               initial_state=a["initial_state"], return_final_state=True)
    b["initial_state"] = mid
    gb = _scan_run(b)
    a["dfinal_state"] = gb[8]
    ga = _scan_run(a)
    for k, name in ((0, "dx"), (1, "ddelta"), (3, "dB"), (4, "dC"), (6, "dz")):
        want = torch.cat([ga[k], gb[k]], 1)
        assert (got[k] - want).abs().max() <= 1e-4 * want.abs().max(), name
    for k, name in ((2, "dA"), (5, "dD"), (7, "ddt_bias")):
        assert (got[k] - ga[k] - gb[k]).abs().max() <= 1e-4 * got[k].abs().max(), name
    assert (got[8] - ga[8]).abs().max() <= 1e-4 * ga[8].abs().max()


@pytest.mark.parametrize("kind", KINDS)
def test_scan_backward_extreme_gates(cuda, kind):
    v = _scan_case(3, 2, 30, 36, 16, kind)
    big = 60000 if kind[0] == F16 else 3e38
    v["z"][0, 3] = -big
    v["z"][0, 4] = -90
    v["z"][1, 5] = 60
    v["dy"][1, 7] = 0
    _scan_check(v, _scan_run({n: _dev(a) for n, a in v.items()}), kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", ["columns", "channels first"])
def test_scan_backward_views(cuda, form, kind):
    """Rows inside wider rows (as projections make them), and channel-major tensors; outputs too."""
    b, L, D, N = 2, 45, 140, 9
    v = _scan_case(4, b, L, D, N, kind)
    t = {n: _dev(a) for n, a in v.items()}

    def view(x):
        if form == "channels first":
            return x, x.transpose(1, 2).contiguous().transpose(1, 2)
        wide = torch.full((b, L, x.shape[2] + 8), 7.0, dtype=x.dtype, device="cuda")
        wide[:, :, 3:3 + x.shape[2]] = x
        return wide, wide[:, :, 3:3 + x.shape[2]]

    for k in ("x", "dy", "z", "delta", "B", "C"):
        t[k] = view(t[k])[1]
    out = {k: view(torch.zeros((b, L, D), dtype=t[s].dtype, device="cuda"))
           for k, s in (("dx", "x"), ("dz", "x"), ("ddelta", "delta"))}
    got = _scan_run(t, **{k: o[1] for k, o in out.items()})
    _scan_check(v, got, kind)
    if form == "columns":
        for wide, _ in out.values():
            assert (wide[:, :, :3] == 7).all() and (wide[:, :, 3 + D:] == 7).all()


def test_scan_backward_broadcast_inputs(cuda):
    """delta shared by all channels and tokens shared by the batch, as expanded views."""
    kind = (F16, F16, F16)
    v = _scan_case(5, 3, 40, 64, 16, kind)
    v["delta"][:] = v["delta"][:, :, :1]
    v["x"][:] = v["x"][:1]
    t = {n: _dev(a) for n, a in v.items()}
    t["delta"] = t["delta"][:, :, :1].expand(3, 40, 64)
    t["x"] = t["x"][:1].expand(3, 40, 64)
    got = _scan_run(t)
    _scan_check(v, got, kind)


def test_scan_backward_bits_streams_graphs(cuda):
    kind = (F16, F16, F16)
    v = _scan_case(7, 2, 300, 200, 16, kind)
    t = {n: _dev(a) for n, a in v.items()}
    want = _scan_run(t)
    a = mb.MambaScanArgs()
    a.batch, a.seqlen, a.dim, a.dstate = 2, 300, 200, 16
    ws = torch.full((mb.lib().mamba_selective_scan_backward_workspace(ctypes.byref(a)),), 0xFF, dtype=torch.uint8,
                    device="cuda")  # NaN in every place of the workspace
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(2):
        got = _scan_run(t, workspace=ws, stream=side)
        side.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _scan_run(t)
    new = _scan_case(8, 2, 300, 200, 16, kind)
    for k, a in new.items():
        t[k].copy_(_dev(a))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    _scan_check(new, got, kind)


def test_scan_backward_empty(cuda):
    z = lambda *s: torch.zeros(s, device="cuda")  # noqa: E731
    h = torch.randn((2, 8, 4), device="cuda")
    got = mb.selective_scan_backward(z(2, 0, 8), z(2, 0, 8), z(2, 0, 8), z(8, 4), z(2, 0, 4), z(2, 0, 4), D=z(8),
                                     dt_bias=z(8), initial_state=h, dfinal_state=h)
    assert torch.equal(got[8], h) and (got[2] == 0).all() and (got[5] == 0).all() and (got[7] == 0).all()
    got = mb.selective_scan_backward(z(0, 5, 8), z(0, 5, 8), z(0, 5, 8), z(8, 4), z(0, 5, 4), z(0, 5, 4))
    assert (got[2] == 0).all() and got[0].shape == (0, 5, 8)
    got = mb.selective_scan_backward(z(2, 5, 0), z(2, 5, 0), z(2, 5, 0), z(0, 4), z(2, 5, 4), z(2, 5, 4))
    assert (got[3] == 0).all() and (got[4] == 0).all()
