"""GPU parity of the row quantiser (equal whole numbers and scales) and of the
8-bit linear layer against the FP64 oracle.

Tolerance of the product, per element: the integer sums are exact, so only
its conversion to FP32, two scalings and the bias round, one half step of
2^-24 each, on |sum * scales| + |bias|: 4 * 2^-24 of it, then the output
type's own half step and, for FP16, half of its smallest step."""
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



def _dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _check(y, ref, mag, before=None):
    u = 2.0 ** -11 if y.dtype == torch.float16 else 2.0 ** -24
    if before is not None:
        ref, mag = ref + before, mag + np.abs(before)
    got = y.double().cpu().numpy()
    err = np.abs(got - ref) - (u * np.abs(ref) + 5 * 2.0 ** -24 * mag + (2.0 ** -25 if u > 1e-4 else 1e-37))
    assert np.isfinite(got).all() and err.max() <= 0, (err.max(), np.unravel_index(err.argmax(), err.shape))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (5, 64), (2, 1000), (700, 72), (900, 1023), (33, 2560), (2, 8192),
                                       (3, 8200), (2, 20000), (1200, 1032)])
def test_quantize_rows(cuda, rows, cols, dtype):
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)).astype(dtype)
    if cols > 8:  # rows whose quotients are ties, zeros, subnormals
        x[0] = rng.integers(-254, 255, cols) * dtype(0.5)
        x[0, 0] = 127
        if rows > 2:
            x[1] = 0
            x[2] *= dtype(6e-8) if dtype == np.float16 else dtype(1e-42)
    q, s = mb.quantize_rows(_dev(x))
    rq, rs = rb.quantize_rows(x)
    assert torch.equal(s.cpu(), torch.from_numpy(rs))
    assert torch.equal(q.cpu(), torch.from_numpy(rq))


# Numbers of rows and channels on both sides of each choice of threads a row
# (32 to 256), with rows left over in the last block, vector and single loads.
@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("rows,cols", [(1205, 512), (1184, 512), (1203, 1024), (1203, 1032), (601, 2048), (599, 2056),
                                       (301, 4096), (299, 4104), (150, 8192), (3, 9000), (1205, 250), (601, 501),
                                       (301, 1001), (299, 1031), (150, 2051)])
def test_quantize_exact_halves(cuda, rows, cols, dtype):
    """Every half is met, exactly and one place above and below, for a
    scale that is a power of two, 3, or any number: equal whole numbers."""
    rng = np.random.default_rng(7 * rows + cols)
    # all but the scale's channel at halves; 3 (k + 1/2) and 127 * 3 are FP16 numbers too
    k = (rng.integers(-126, 127, (rows, cols)) + 0.5) * np.where(np.arange(rows) % 2, 3.0, 2.0 ** -6)[:, None]
    x = k.astype(dtype)
    near = rng.integers(0, 3, (rows, cols))
    x = np.where(near == 0, x, np.where(near == 1, np.nextafter(x, dtype(np.inf)), np.nextafter(x, dtype(-np.inf))))
    top = rng.integers(0, cols, rows)
    x[np.arange(rows), top] = (127 * np.where(np.arange(rows) % 2, 3.0, 2.0 ** -6)).astype(dtype)
    x[::5] = (rng.standard_normal((len(x[::5]), cols))).astype(dtype)  # any scale
    x = x.astype(dtype)
    q, s = mb.quantize_rows(_dev(x))
    rq, rs = rb.quantize_rows(x)
    assert torch.equal(s.cpu(), torch.from_numpy(rs))
    assert torch.equal(q.cpu(), torch.from_numpy(rq))


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_quantize_strides_and_padding(cuda, dtype):
    rng = np.random.default_rng(0)
    rows, cols = 50, 136
    x = rng.standard_normal((rows, cols)).astype(dtype)
    rq, rs = rb.quantize_rows(x)
    for off in (0, 1, 8):
        wide = torch.full((rows, cols + 24), float("nan"), dtype=_dev(x).dtype, device="cuda")
        wide[:, off:off + cols] = _dev(x)
        out = torch.full((rows, cols + 40), 99, dtype=torch.int8, device="cuda")
        q, s = mb.quantize_rows(wide[:, off:off + cols], q=out[:, off:off + cols])
        assert torch.equal(q.cpu(), torch.from_numpy(rq)) and torch.equal(s.cpu(), torch.from_numpy(rs))
        assert (out[:, :off] == 99).all() and (out[:, off + cols:] == 99).all()


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
def test_quantize_infinities_and_nan(cuda, dtype):
    x = np.random.default_rng(1).standard_normal((4, 300)).astype(dtype)
    x[0, 5], x[1, 299], x[2, 0] = np.inf, -np.inf, np.nan
    q, s = mb.quantize_rows(_dev(x))
    assert s[:3].isnan().all() and not q[:3].any() and s[3].isfinite()
    w, ws = mb.quantize_rows(_dev(np.ones((8, 300), dtype)))
    y = mb.linear_i8(q, s, w, ws)
    assert y[:3].isnan().all() and y[3].isfinite().all()


def _problem(seed, rows, n, k, bias, pad=True, full=True):
    rng = np.random.default_rng(seed)
    lo = -128 if full else -127
    x, w = (rng.integers(lo, 128, (m, k)).astype(np.int8) for m in (rows, n))
    xs, ws = (rng.uniform(0.001, 0.02, m).astype(np.float32) for m in (rows, n))
    b = rng.standard_normal(n).astype(np.float32) if bias else None

    def mat(a):
        if not pad:
            return _dev(a)
        buf = torch.full((a.shape[0], (k + 15) // 16 * 16), 77, dtype=torch.int8, device="cuda")  # padding is not read
        buf[:, :k] = _dev(a)
        return buf[:, :k]

    return (x, xs, w, ws, b), (mat(x), _dev(xs), mat(w), _dev(ws), _dev(b))


SHAPES = [(1, 1, 1), (1, 8, 16), (1, 200, 1000), (5, 96, 64), (17, 33, 130), (64, 300, 2560), (128, 1000, 260),
          (129, 256, 128), (256, 10240, 2560), (256, 192, 5120), (300, 203, 137), (513, 256, 256), (777, 203, 1000),
          (1000, 160, 4096), (2100, 2304, 520), (700, 5120, 96), (33, 40, 20000)]


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("rows,n,k", SHAPES)
def test_linear(cuda, rows, n, k, mode, bias):
    cpu, (x, xs, w, ws, b) = _problem(rows + n + k, rows, n, k, bias)
    if mode == 0:  # within FP16's range
        xs = xs / 100
        cpu = (cpu[0], xs.cpu().numpy()) + cpu[2:]
    before = np.random.default_rng(1).standard_normal((rows, n)).astype(np.float32)
    y = mb.linear_i8(x, xs, w, ws, bias=b, mode=mode, y=_dev(before) if mode == 1 else None)
    torch.cuda.synchronize()
    assert mb.device_status() == 0
    ref, mag = rb.linear_i8(*cpu)
    _check(y, ref, mag, before if mode == 1 else None)


@pytest.mark.parametrize("rows,n,k", [(3, 20, 37), (100, 70, 1001), (600, 130, 257)])
def test_unaligned_rows(cuda, rows, n, k):
    """Contiguous odd rows and starts: the kernel without alignment needs."""
    cpu, (x, xs, w, ws, b) = _problem(5, rows, n, k, True, pad=False)
    ref, mag = rb.linear_i8(*cpu)
    _check(mb.linear_i8(x, xs, w, ws, bias=b, mode=2), ref, mag)
    shifted = torch.zeros(w.numel() + 1, dtype=torch.int8, device="cuda")[1:].view(n, k)
    shifted.copy_(w)
    _check(mb.linear_i8(x, xs, shifted, ws, bias=b, mode=2), ref, mag)


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("rows,n,k,pad", [(40, 100, 64, 1), (40, 96, 64, 8), (700, 250, 128, 3), (700, 256, 128, 8),
                                          (256, 515, 64, 0)])
def test_strided_output_leaves_the_rest(cuda, rows, n, k, pad, mode):
    cpu, (x, xs, w, ws, b) = _problem(6, rows, n, k, True)
    dt = torch.float16 if mode == 0 else torch.float32
    wide = torch.full((rows + 1, n + 2 * pad), 3.0, dtype=dt, device="cuda")
    y = mb.linear_i8(x, xs, w, ws, bias=b, mode=mode, y=wide[:rows, pad:pad + n])
    ref, mag = rb.linear_i8(*cpu)
    _check(y, ref, mag, np.full(ref.shape, 3.0) if mode == 1 else None)
    assert (wide[:rows, :pad] == 3).all() and (wide[:rows, pad + n:] == 3).all() and (wide[rows:] == 3).all()


def test_largest_sums_are_exact(cuda):
    """-128 * -128 over the longest K: just below 2^31."""
    k = 131071
    for rows in (2, 600):
        x = torch.full((rows, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
        w = torch.full((3, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
        one = torch.ones(max(rows, 3), device="cuda")
        y = mb.linear_i8(x, one[:rows], w, one[:3], mode=2)
        assert (y == float(128 * 128 * k)).all()


def test_empty_and_zero_k(cuda):
    one = torch.ones(4, device="cuda")
    z = torch.zeros((4, 0), dtype=torch.int8, device="cuda")
    bias = torch.arange(4.0, device="cuda")
    y = mb.linear_i8(z, one, z, one, bias=bias, mode=2)
    assert torch.equal(y, bias.expand(4, 4))
    e = torch.zeros((0, 16), dtype=torch.int8, device="cuda")
    assert mb.linear_i8(e, one[:0], torch.zeros((4, 16), dtype=torch.int8, device="cuda"), one).shape == (0, 4)
    q, s = mb.quantize_rows(torch.zeros((3, 0), device="cuda"))
    assert q.shape == (3, 0) and not s.any()


@pytest.mark.parametrize("rows", [64, 1100])
def test_bits_streams_and_graphs(cuda, rows):
    cpu, (x, xs, w, ws, b) = _problem(7, rows, 512, 1024, True)
    y0 = mb.linear_i8(x, xs, w, ws, bias=b, mode=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ys = [mb.linear_i8(x, xs, w, ws, bias=b, mode=2) for _ in range(4)]
    side.synchronize()
    assert all(torch.equal(y0, y) for y in ys)
    src = torch.randn((rows, 1024), device="cuda", dtype=torch.float16)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, s = mb.quantize_rows(src)
        y = mb.linear_i8(q, s, w, ws, bias=b, mode=2)
    for seed in (1, 2):
        a = np.random.default_rng(seed).standard_normal((rows, 1024)).astype(np.float16)
        src.copy_(_dev(a))
        graph.replay()
        torch.cuda.synchronize()
        rq, rs = rb.quantize_rows(a)
        assert torch.equal(q.cpu(), torch.from_numpy(rq))
        _check(y, *rb.linear_i8(rq, rs, cpu[2], cpu[3], cpu[4]))


def test_quantised_product_approximates_the_product(cuda):
    """The two together: the error of a product of quantised operands is at
    most half a step of each operand per term."""
    rng = np.random.default_rng(2)
    x = rng.standard_normal((70, 512)).astype(np.float16)
    w = rng.standard_normal((90, 512)).astype(np.float32)
    (q, s), (wq, ws) = mb.quantize_rows(_dev(x)), mb.quantize_rows(_dev(w))
    y = mb.linear_i8(q, s, wq, ws, mode=2).double().cpu().numpy()
    x, w = x.astype(np.float64), w.astype(np.float64)
    ex, ew = s.double().cpu().numpy()[:, None] / 2, ws.double().cpu().numpy()[None] / 2
    bound = ex * np.abs(w).sum(1)[None] + ew * np.abs(x).sum(1)[:, None] + 512 * ex * ew
    assert (np.abs(y - x @ w.T) <= 1.0001 * bound).all()
