"""GPU parity of the block norm (forward, backward) against the FP64 oracle on
the same (rounded) inputs.

Tolerance, per element: |gpu - ref| <= u |ref| + d * mag + tiny, with u the
output type's half step, tiny half of FP16's smallest step and mag the sum of
the absolute terms of that element.  d bounds the FP32 evaluation: a row sum
of squares (at most 16 terms in a thread, then 10 levels), rsqrtf (2 ulp), the
exponential and quotient of the gate and ~10 products: d = 2^-24 * 48; FP16
tensors add 2^-20 for the approximate exponential and reciprocal.  Column sums
add one rounding per row at most: d + 2^-24 * rows."""
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

EPS, RHO = 1e-5, 0.9


def _case(seed, T, D, dtype, gate=True, weights=True):
    rng = np.random.default_rng(seed)
    np_t = np.float16 if dtype == torch.float16 else np.float32
    v = {k: rng.standard_normal((T, D)).astype(np_t) for k in ("y", "z", "dout")}
    v.update({k: rng.standard_normal((T, D)).astype(np.float32) for k in ("res", "dro")})
    v["wq"] = v["wp"] = None
    if weights:
        v["wq"], v["wp"] = (rng.standard_normal(D).astype(np.float32) for _ in range(2))
    if not gate:
        v["z"] = None
    return v


def _dev(v):
    return {k: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda() for k, a in v.items()}


def _close(got, ref, mag, dtype, name, rows=0):
    f16 = got.dtype == torch.float16
    got = got.double().cpu().numpy()
    u = 2.0 ** -11 if f16 else 2.0 ** -24
    d = 2.0 ** -24 * (48 + rows) + (2.0 ** -20 if dtype == torch.float16 else 0.0)
    assert got.shape == ref.shape and not np.isnan(got).any(), name
    err = np.abs(got - ref) - (u * np.abs(ref) + d * mag + 2.0 ** -25)
    if f16:
        # A row of zeros has rstd = eps^-1/2 = 316 on both norms, so gradients
        # reach 1e5.  FP16 ends at 65504 and rounds what is 65520 or more to
        # infinity; within d * mag of that border either side may come out.
        over = np.abs(ref) + d * mag >= 65520
        assert (np.isinf(got) <= over).all(), name
        assert (np.isinf(got) >= (np.abs(ref) - d * mag >= 65520)).all(), name
        assert (np.sign(got) == np.sign(ref))[np.isinf(got)].all(), name
        err = np.where(np.isinf(got), 0.0, err)
    else:
        assert np.isfinite(got).all(), name
    assert not err.size or err.max() <= 0, (name, err.max())


def _forward(t, **kw):
    return mb.block_norm(t["y"], t["res"], w_post=t["wq"], z=t["z"], w_pre=t["wp"], residual_scale=RHO, eps=EPS,
                         return_rstd=True, **kw)


def _backward(t, f, **kw):
    return mb.block_norm_backward(t["dro"], t["dout"], t["y"], f[0], f[2], f[3], w_post=t["wq"], z=t["z"],
                                  w_pre=t["wp"], residual_scale=RHO, **kw)


def _check_forward(v, f, dtype):
    ref, mag = rb.block_norm(v["y"], v["res"], v["wq"], v["z"], v["wp"], RHO, EPS)
    _close(f[0], ref[0], mag[0], dtype, "residual_out")
    if f[1] is not None:
        _close(f[1], ref[1], mag[1], dtype, "out")
        np.testing.assert_allclose(f[3].cpu().numpy(), ref[3], rtol=2.0 ** -19)
    np.testing.assert_allclose(f[2].cpu().numpy(), ref[2], rtol=2.0 ** -24 * 48)


def _check_backward(v, f, grads, dtype):
    rp = None if f[3] is None else f[3].cpu().numpy()
    ref, mag = rb.block_norm_backward(v["dro"], v["dout"], v["y"], f[0].cpu().numpy(), f[2].cpu().numpy(), rp, v["wq"],
                                      v["z"], v["wp"], RHO)
    rows = v["y"].shape[0]
    for got, k in zip(grads, ("dy", "dresidual", "dw_post", "dw_pre", "dz")):
        if k == "dz" and v["z"] is None:
            assert got is None
            continue
        _close(got, ref[k], mag[k], dtype, k, rows if k.startswith("dw") else 0)


SHAPES = [(1, 1), (1, 8), (3, 7), (2, 64), (5, 256), (4, 264), (130, 1000), (9, 1001), (700, 72), (300, 2048),
          (64, 2560), (3, 4096), (3, 4099), (2, 8192), (2, 8200), (2, 16384), (2, 12001),
          # enough rows for persistent CTAs with rows fetched ahead: 1, 2, 8 and 16 warps, one and two rows of room
          (14500, 72), (7300, 264), (2000, 2048), (1000, 4096), (950, 8192),
          # and of rows that start and end anywhere
          (14500, 71), (3700, 513), (2000, 2045), (950, 7001)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("gate,weights", [(True, True), (False, True), (True, False)])
@pytest.mark.parametrize("T,D", SHAPES)
def test_forward_and_backward(cuda, T, D, gate, weights, dtype):
    v = _case(T + D, T, D, dtype, gate, weights)
    t = _dev(v)
    f = _forward(t)
    grads = _backward(t, f)
    torch.cuda.synchronize()
    _check_forward(v, f, dtype)
    _check_backward(v, f, grads, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 8])
@pytest.mark.parametrize("T,D", [(21, 40), (21, 136), (21, 1000), (4000, 500)])
def test_strided_views(cuda, dtype, offset, T, D):
    """y and the gate as column blocks of one projection, their gradients into
    column blocks of another."""
    v = _case(6, T, D, dtype)
    t = _dev(v)
    pitch = 2 * D + 32
    wide = torch.full((T, pitch), float("nan"), dtype=dtype, device="cuda")
    for k, name in enumerate(("y", "z")):
        view = wide[:, offset + k * (D + 8):offset + k * (D + 8) + D]
        view.copy_(t[name])
        t[name] = view
    f = _forward(t)
    dwide = torch.full((T, pitch), float("nan"), dtype=dtype, device="cuda")
    grads = _backward(t, f, dy=dwide[:, offset:offset + D], dz=dwide[:, offset + D + 8:offset + 2 * D + 8])
    torch.cuda.synchronize()
    _check_forward(v, f, dtype)
    _check_backward(v, f, grads, dtype)
    rest = torch.ones(pitch, dtype=torch.bool)
    rest[offset:offset + D] = False
    rest[offset + D + 8:offset + 2 * D + 8] = False
    assert dwide[:, rest.cuda()].isnan().all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("T,D", [(33, 520), (4000, 520), (4000, 523)])
def test_in_place_and_missing_parts(cuda, T, D, dtype):
    v = _case(7, T, D, dtype)
    t = _dev(v)
    f = _forward(t)
    res = t["res"].clone()
    f2 = mb.block_norm(t["y"], res, w_post=t["wq"], z=t["z"], w_pre=t["wp"], residual_scale=RHO, eps=EPS,
                       return_rstd=True, residual_out=res)
    assert f2[0].data_ptr() == res.data_ptr()
    assert all(torch.equal(a, b) for a, b in zip(f, f2))
    g = _backward(t, f)
    dro = t["dro"].clone()
    t2 = dict(t, dro=dro)
    g2 = _backward(t2, f, dresidual=dro)
    assert g2[1].data_ptr() == dro.data_ptr() and all(torch.equal(a, b) for a, b in zip(g, g2))
    # one output only: the last layer has no norm behind it, or only the norm's output is used
    f3 = _forward(t, second_norm=False)
    assert f3[1] is None and f3[3] is None and torch.equal(f3[0], f[0])
    for part in ("dout", "dro"):
        w, u = dict(v), dict(t)
        w[part] = u[part] = None
        _check_backward(w, f, _backward(u, f), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_rows_of_zeros_and_extreme_gates(cuda, dtype):
    v = _case(8, 6, 256, dtype)
    v["y"][0] = 0
    v["y"][1] = 0
    v["res"][1] = 0
    big = 60000 if dtype == torch.float16 else 3e38
    v["z"][2, ::2] = -big
    v["z"][3, 1::2] = -90
    v["z"][4, ::3] = 60
    t = _dev(v)
    f = _forward(t)
    _check_forward(v, f, dtype)
    _check_backward(v, f, _backward(t, f), dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_bits_streams_and_graphs(cuda, dtype):
    v = _case(9, 1500, 320, dtype)
    t = _dev(v)
    f, g = _forward(t), None
    g = _backward(t, f)
    a = mb._block_norm_args("t", t["y"], t["wq"], t["z"], t["wp"], RHO, EPS)
    ws = torch.full((mb.lib().mamba_block_norm_workspace(ctypes.byref(a)),), 0xAB, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            f2 = _forward(t)
            g2 = _backward(t, f2, workspace=ws)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(f + g, f2 + g2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f3 = _forward(t)
        g3 = _backward(t, f3)
    v2 = _case(10, 1500, 320, dtype)
    for k, x in _dev(v2).items():
        t[k].copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    _check_forward(v2, f3, dtype)
    _check_backward(v2, f3, g3, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_empty(cuda, dtype):
    t = {k: None if a is None else (a[:0] if a.dim() == 2 else a) for k, a in _dev(_case(1, 2, 40, dtype)).items()}
    f = _forward(t)
    g = _backward(t, f)
    assert f[0].shape == (0, 40) and not g[2].any() and not g[3].any()


def test_offsets_beyond_32_bits(cuda):
    rows, cols, pitch = 3, 64, (1 << 30) + 64
    if torch.cuda.mem_get_info()[0] < 3 * 4 * pitch * 2:
        pytest.skip("needs 26 GB of free device memory")
    v = _case(3, rows, cols, torch.float16)
    t = _dev(v)
    big = torch.zeros(rows * pitch, dtype=torch.float16, device="cuda").view(rows, pitch)
    big[:, :cols] = t["y"]
    t["y"] = big[:, :cols]
    f = _forward(t)
    dbig = torch.zeros(rows * pitch, dtype=torch.float16, device="cuda").view(rows, pitch)
    g = _backward(t, f, dy=dbig[:, :cols])
    _check_forward(v, f, torch.float16)
    _check_backward(v, f, g, torch.float16)
