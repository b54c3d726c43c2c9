"""GPU parity of layer norm, embedding and dropout (and their gradients)
against the FP64 oracle on the same (rounded) inputs.

Tolerance, per element: |gpu - ref| <= u |ref| + d * mag + tiny, with u the
output type's half step, tiny half of FP16's smallest step and mag the sum of
the absolute terms of that element.  d bounds the FP32 evaluation: two row
sums (at most 16 terms in a thread, then 10 levels), rsqrtf (2 ulp) and ~10
products: d = 2^-24 * 64.  Sums over rows add one rounding per term at most:
d + 2^-24 * terms."""
import ctypes

import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32
TYPES = [(F16, F16), (F16, F32), (F32, F16), (F32, F32)]


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_memory():
    """Later tests find the allocator as a fresh process has it."""
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _np(dtype):
    return np.float16 if dtype == F16 else np.float32


def _dev(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _host(t):
    return t.double().cpu().numpy()


def _close(got, ref, mag, name, terms=0):
    u = 2.0 ** -11 if got.dtype == F16 else 2.0 ** -24
    got, d = _host(got), 2.0 ** -24 * (64 + terms)
    assert got.shape == ref.shape and np.isfinite(got).all(), name
    err = np.abs(got - ref) - (u * np.abs(ref) + d * mag + 2.0 ** -25)
    assert not err.size or err.max() <= 0, (name, err.max())


def _wide(t, offset, pitch, fill=float("nan")):
    """t as columns offset .. of rows of `pitch` elements."""
    w = torch.full((t.shape[0], pitch), fill, dtype=t.dtype, device="cuda")
    v = w[:, offset:offset + t.shape[1]]
    v.copy_(t)
    return w, v


# ---- layer norm -------------------------------------------------------------------
def _ln_case(seed, T, D, xt, ot, shift=0.0, weights=True):
    rng = np.random.default_rng(seed)
    x = (rng.standard_normal((T, D)) + shift).astype(_np(xt))
    w, b = (rng.standard_normal(D).astype(np.float32) if weights else None for _ in range(2))
    return x, w, b, rng.standard_normal((T, D)).astype(_np(ot))


def _ln_check(x, w, b, g, f, grads, eps=1e-5):
    ref, mag = tr.layer_norm(x, w, b, eps)
    _close(f[0], ref[0], mag, "out")
    _close(f[1], ref[1], np.abs(x.astype(np.float64)).mean(1), "mean")
    # centred values keep an error of d times the row's magnitude; rstd has its share of that
    rel = 2.0 ** -24 * 64 * (1 + np.abs(x.astype(np.float64)).mean(1) * ref[2])
    assert (np.abs(_host(f[2]) / ref[2] - 1) <= rel).all()
    ref, mag = tr.layer_norm_backward(g, x, _host(f[1]), _host(f[2]), w)
    for got, k in zip(grads, ("dx", "dw", "db")):
        _close(got, ref[k], mag[k], k, 0 if k == "dx" else x.shape[0])


SHAPES = [(1, 1), (1, 8), (3, 7), (2, 64), (4, 264), (130, 1000), (9, 1001), (64, 2560), (3, 4096), (3, 4099),
          (2, 8192), (2, 8200), (2, 16384), (2, 12001),
          # enough rows for persistent CTAs with rows fetched ahead, aligned and not
          (14500, 72), (7300, 264), (2000, 2048), (1000, 4096), (950, 8192), (14500, 71), (3700, 513), (950, 7001),
          (300, 16384), (320, 12001), (297, 40), (295, 40)]


@pytest.mark.parametrize("xt,ot", TYPES)
@pytest.mark.parametrize("T,D", SHAPES)
def test_layer_norm(cuda, T, D, xt, ot):
    for weights in (True, False):
        x, w, b, g = _ln_case(T + D, T, D, xt, ot, 0.5, weights)
        f = mb.layer_norm(_dev(x), _dev(w), _dev(b), out_dtype=ot, return_stats=True)
        grads = mb.layer_norm_backward(_dev(g), _dev(x), f[1], f[2], _dev(w))
        _ln_check(x, w, b, g, f, grads)


@pytest.mark.parametrize("xt,ot", TYPES)
@pytest.mark.parametrize("T,D,offset", [(21, 136, 8), (21, 40, 1), (4000, 520, 8), (4000, 520, 3), (4000, 523, 0)])
def test_layer_norm_strided(cuda, T, D, offset, xt, ot):
    x, w, b, g = _ln_case(5, T, D, xt, ot)
    pitch = D + 32
    _, xv = _wide(_dev(x), offset, pitch)
    _, gv = _wide(_dev(g), offset, pitch)
    ow, ov = _wide(torch.zeros((T, D), dtype=ot, device="cuda"), offset, pitch, 7.0)
    dw_, dv = _wide(torch.zeros((T, D), dtype=xt, device="cuda"), offset, pitch, 7.0)
    f = mb.layer_norm(xv, _dev(w), _dev(b), out=ov, return_stats=True)
    grads = mb.layer_norm_backward(gv, xv, f[1], f[2], _dev(w), dx=dv)
    _ln_check(x, w, b, g, f, grads)
    for wide in (ow, dw_):  # what lies around the rows is left alone
        assert (wide[:, :offset] == 7).all() and (wide[:, offset + D:] == 7).all()


def test_layer_norm_large_mean_constant_rows_and_bad_values(cuda):
    x, w, b, g = _ln_case(6, 40, 300, F32, F32, 1000.0)
    x[3] = 5.0
    x[4] = 0.0
    f = mb.layer_norm(_dev(x), _dev(w), _dev(b), return_stats=True)
    _ln_check(x, w, b, g, f, mb.layer_norm_backward(_dev(g), _dev(x), f[1], f[2], _dev(w)))
    clean = mb.layer_norm(_dev(x), _dev(w), _dev(b))
    x[7, 11], x[9, 0] = np.nan, np.inf
    out = mb.layer_norm(_dev(x), _dev(w), _dev(b))
    assert out[[7, 9]].isnan().all()
    rest = [i for i in range(40) if i not in (7, 9)]
    assert torch.equal(out[rest], clean[rest])


def test_layer_norm_bits_streams_graphs_and_empty(cuda):
    x, w, b, g = _ln_case(8, 3000, 320, F32, F16)
    t = [_dev(v) for v in (x, w, b, g)]

    def both(ws=None):
        f = mb.layer_norm(t[0], t[1], t[2], out_dtype=F16, return_stats=True)
        return f + mb.layer_norm_backward(t[3], t[0], f[1], f[2], t[1], workspace=ws)

    want = both()
    a = mb._layer_norm_args("t", t[0], t[1], None, None, None, F16, 1.0)
    ws = torch.full((mb.lib().mamba_layer_norm_workspace(ctypes.byref(a)),), 0xAB, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = both(ws)
    side.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = both()
    x2 = _ln_case(9, 3000, 320, F32, F16)
    for p, q in zip(t, x2):
        p.copy_(_dev(q))
    graph.replay()
    torch.cuda.synchronize()
    _ln_check(*x2, got[:3], got[3:])
    e = torch.zeros((0, 8), device="cuda")
    assert mb.layer_norm(e).shape == (0, 8)
    dx, dw, db = mb.layer_norm_backward(e, e, e[:, 0], e[:, 0])
    assert dx.shape == (0, 8) and (dw == 0).all() and (db == 0).all()
    assert mb.device_status() == 0


# ---- embedding --------------------------------------------------------------------
def _ids(rng, T, vocab, kind):
    if kind == "one":
        return np.full(T, vocab - 1)
    if kind == "skew":
        ids = np.minimum((rng.random(T) ** 4 * vocab).astype(np.int64), vocab - 1)
    elif kind == "distinct":
        ids = rng.permutation(max(T, vocab))[:T] % vocab
    else:  # ids outside the table too, among them ones whose low 32 bits lie inside
        ids = rng.integers(-3, vocab + 3, T)
        if T > 4:
            ids[:2] = -1, vocab
    return ids


CASES = [(1, 1, 1), (1, 7, 8), (5, 3, 33), (16, 5, 64), (17, 4, 40), (255, 300, 72), (4096, 50, 24), (4097, 256, 8),
         (2048, 255, 100), (9000, 70000, 16), (6000, 11, 1001), (700, 1000, 2056), (333, 257, 4100)]


@pytest.mark.parametrize("kind", ["skew", "one", "distinct", "outside"])
@pytest.mark.parametrize("T,vocab,dim", CASES)
def test_embedding(cuda, T, vocab, dim, kind):
    rng = np.random.default_rng(T + vocab)
    ids = _ids(rng, T, vocab, kind)
    for (tt, ot), wide in zip(TYPES, (torch.int32, torch.int64, torch.int32, torch.int64)):
        table = rng.standard_normal((vocab, dim)).astype(_np(tt))
        tok = _dev(ids).to(wide)
        out = mb.embedding(tok, _dev(table), scale=1.7, out_dtype=ot)
        ref = tr.embedding(ids, table, 1.7)
        _close(out, ref, np.abs(ref), "out")
        g = rng.standard_normal((T, dim)).astype(_np(ot))
        ref, mag = tr.embedding_backward(g, ids, vocab, 1.7)
        most = np.bincount(ids[(ids >= 0) & (ids < vocab)].astype(np.int64), minlength=1).max()
        dtable = mb.embedding_backward(_dev(g), tok, vocab, scale=1.7)
        _close(dtable, ref, mag, "dtable", most)
        start = rng.standard_normal((vocab, dim)).astype(np.float32)
        acc = mb.embedding_backward(_dev(g), tok, vocab, scale=1.7, dtable=_dev(start), accumulate=True)
        _close(acc, ref + start, mag + np.abs(start), "accumulated", most)
        absent = np.setdiff1d(np.arange(vocab), ids)
        assert (_host(acc)[absent] == start[absent]).all() and (_host(dtable)[absent] == 0).all()


@pytest.mark.parametrize("T,vocab,dim", [(32768, 70000, 8), (32769, 300, 16), (40000, 70000, 12), (65537, 1000, 8),
                                         (150000, 66000, 4)])
def test_embedding_many_tokens(cuda, T, vocab, dim):
    """Each of the sort's ways (one cluster, few and many tiles, one to three passes), and lookups with several tokens
    in flight."""
    rng = np.random.default_rng(T)
    ids = _ids(rng, T, vocab, "skew")
    ids[rng.random(T) < 0.05] = -1
    g = rng.standard_normal((T, dim)).astype(np.float32)
    inside = ids >= 0
    ref, mag = np.zeros((vocab, dim)), np.zeros((vocab, dim))
    np.add.at(ref, ids[inside], g[inside].astype(np.float64))
    np.add.at(mag, ids[inside], np.abs(g[inside].astype(np.float64)))
    got = mb.embedding_backward(_dev(g), _dev(ids), vocab)
    _close(got, ref, mag, "dtable", np.bincount(ids[inside]).max())
    assert torch.equal(got, mb.embedding_backward(_dev(g), _dev(ids).int(), vocab))
    wide = torch.randn((50, 2056 if T < 40000 else 1000), device="cuda")
    tok = _dev(ids[:6000] % 51 - 1)
    for dtype in (F16, F32):
        out = mb.embedding(tok, wide.to(dtype), scale=0.5, out_dtype=F32)
        want = torch.where((tok >= 0)[:, None], wide.to(dtype).float()[tok.clamp(min=0)] * 0.5, 0.0)
        assert torch.equal(out, want)  # halving is exact


def test_embedding_ids_beyond_32_bits(cuda):
    table = torch.randn((6, 16), device="cuda")
    tok = torch.tensor([2 ** 32 + 1, 3, -2 ** 32 + 2, 2 ** 62, -2 ** 63, 2 ** 63 - 1], device="cuda")
    out = mb.embedding(tok, table)
    assert torch.equal(out[1], table[3]) and (out[[0, 2, 3, 4, 5]] == 0).all()
    g = mb.embedding_backward(torch.ones_like(out), tok, 6)
    assert (g[3] == 1).all() and g.sum() == 16


@pytest.mark.parametrize("offset,dim", [(8, 64), (3, 64), (0, 61)])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_embedding_strided_and_shaped(cuda, dtype, offset, dim):
    rng = np.random.default_rng(3)
    ids, table = rng.integers(0, 50, 200), rng.standard_normal((50, dim)).astype(_np(dtype))
    g = rng.standard_normal((200, dim)).astype(_np(dtype))
    tok = _dev(ids)
    _, tv = _wide(_dev(table), offset, dim + 16)
    ow, ov = _wide(torch.zeros((200, dim), dtype=dtype, device="cuda"), offset, dim + 16, 7.0)
    assert mb.embedding(tok, tv, out=ov) is ov
    ref = tr.embedding(ids, table, 1.0)
    _close(ov, ref, np.abs(ref), "out")
    assert (ow[:, :offset] == 7).all() and (ow[:, offset + dim:] == 7).all()
    _, gv = _wide(_dev(g), offset, dim + 16)
    dw, dv = _wide(torch.full((50, dim), 3.0, device="cuda"), offset, dim + 16, 7.0)
    mb.embedding_backward(gv, tok, 50, dtable=dv)
    ref, mag = tr.embedding_backward(g, ids, 50, 1.0)
    _close(dv, ref, mag, "dtable", 200)
    assert (dw[:, :offset] == 7).all() and (dw[:, offset + dim:] == 7).all()
    shaped = mb.embedding(tok.view(8, 25), _dev(table))
    assert shaped.shape == (8, 25, dim) and torch.equal(shaped.view(200, dim), ov)
    assert torch.equal(mb.embedding_backward(_dev(g).view(8, 25, dim), tok.view(8, 25), 50), dv)


def test_embedding_bits_streams_graphs_and_empty(cuda):
    rng = np.random.default_rng(4)
    ids, g = _dev(_ids(rng, 30000, 900, "skew")), _dev(rng.standard_normal((30000, 96)).astype(np.float32))
    want = mb.embedding_backward(g, ids, 900)
    a = mb._embedding_args("t", ids, 900, 96, mb.F32, mb.F32, 1.0)
    ws = torch.full((mb.lib().mamba_embedding_workspace(ctypes.byref(a)),), 0xAB, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = mb.embedding_backward(g, ids, 900, workspace=ws, stream=side)
        side.synchronize()
        assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mb.embedding_backward(g, ids, 900)
    new = _dev(_ids(rng, 30000, 900, "outside"))
    ids.copy_(new)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, mb.embedding_backward(g, new, 900))
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    assert mb.embedding(none, g).shape == (0, 96)
    assert (mb.embedding_backward(g[:0], none, 5, dtable=torch.ones((5, 96), device="cuda")) == 0).all()
    assert mb.embedding_backward(g[:, :0], ids, 5).shape == (5, 0)
    assert (mb.embedding(ids[:4], g[:0]) == 0).all()
    assert mb.embedding_backward(g, ids, 0).shape == (0, 96)


# ---- dropout ----------------------------------------------------------------------
SEED, OFFSET = 0xF123456789ABCDEF, 0xFEDCBA9876543210


@pytest.mark.parametrize("xt,ot", TYPES)
@pytest.mark.parametrize("T,D", [(1, 1), (1, 3), (2, 4), (5, 8), (3, 41), (33, 128), (7, 1001)])
def test_dropout(cuda, T, D, xt, ot):
    rng = np.random.default_rng(T * D)
    x, res = rng.standard_normal((T, D)).astype(_np(xt)), rng.standard_normal((T, D)).astype(np.float32)
    for p in (0.0, 0.1, 0.5, 0.97, 1.0):
        for r in (None, res):
            out = mb.dropout(_dev(x), p, SEED, OFFSET, residual=_dev(r), out_dtype=ot)
            ref = tr.dropout(x, p, SEED, OFFSET, r)
            _close(out, ref, np.abs(tr.dropout(np.abs(x), p, SEED, OFFSET)) + (0 if r is None else np.abs(r)), "out")
            if r is None:
                keep = tr.dropout_keep(0, x.size, p, SEED, OFFSET).reshape(x.shape)
                assert ((_host(out) != 0) == (keep & (ref.astype(_np(ot)) != 0))).all()
        dx = mb.dropout_backward(_dev(x), p, SEED, OFFSET, out_dtype=ot)
        assert torch.equal(dx, mb.dropout(_dev(x), p, SEED, OFFSET, out_dtype=ot))


@pytest.mark.parametrize("offset,D,pitch", [(8, 64, 96), (4, 64, 100), (3, 64, 96), (0, 61, 80), (0, 8, 8)])
def test_dropout_mask_does_not_depend_on_strides(cuda, offset, D, pitch):
    x = torch.randn((50, D), device="cuda")
    res = torch.randn((50, D), device="cuda")
    for dtype in (F16, F32):
        want = mb.dropout(x.to(dtype), 0.3, 5, 6, residual=res)
        _, xv = _wide(x.to(dtype), offset, pitch + offset)
        _, rv = _wide(res, offset, pitch + offset)
        ow, ov = _wide(torch.zeros_like(x), offset, pitch + offset, 7.0)
        mb.dropout(xv, 0.3, 5, 6, residual=rv, out=ov)
        assert torch.equal(ov, want)
        assert (ow[:, :offset] == 7).all() and (ow[:, offset + D:] == 7).all()
        assert torch.equal(mb.dropout(xv, 0.3, 5, 6, residual=res), want)
        flat = mb.dropout(x.to(dtype).view(-1), 0.3, 5, 6, residual=res.view(-1))
        assert torch.equal(flat.view_as(want), want)


def test_dropout_in_place_and_bad_values(cuda):
    x = torch.randn((64, 200), device="cuda")
    want = mb.dropout(x, 0.4, 1, 2)
    y = x.clone()
    assert mb.dropout(y, 0.4, 1, 2, out=y) is y and torch.equal(y, want)
    res = torch.randn_like(x)
    want_r = mb.dropout(x, 0.4, 1, 2, residual=res)
    assert torch.equal(mb.dropout(x, 0.4, 1, 2, residual=res, out=res), want_r)
    keep = want != 0
    x[~keep] = float("nan")
    assert torch.equal(mb.dropout(x, 0.4, 1, 2), want)
    x[:] = float("inf")
    out = mb.dropout(x, 0.4, 1, 2)
    assert (out[keep] == float("inf")).all() and (out[~keep] == 0).all()
    assert (mb.dropout(x, 1.0, 1, 2) == 0).all()
    assert not torch.equal(mb.dropout(res, 0.4, 1, 3), mb.dropout(res, 0.4, 1, 2))


def test_dropout_counters_beyond_32_bits_of_elements(cuda):
    """Elements behind the first 2^32 + some: the mask there, and across the border of the low counter word's use."""
    n = (1 << 32) + 4096
    x = torch.ones(n, dtype=F16, device="cuda")
    out = mb.dropout(x, 0.5, SEED, OFFSET, out=x)
    for first in ((1 << 31) - 64, (1 << 32) - 64, n - 128):
        keep = tr.dropout_keep(first, 128, 0.5, SEED, OFFSET)
        assert ((_host(out[first:first + 128]) == 2) == keep).all()
    share = (out[:1 << 24] == 0).double().mean().item()
    assert abs(share - 0.5) < 5 * 0.5 / 2 ** 12  # five standard deviations


def test_dropout_state_streams_and_graphs(cuda):
    x = torch.randn((300, 128), device="cuda")
    state = torch.tensor([77, 1000], dtype=torch.int64, device="cuda")
    assert torch.equal(mb.dropout(x, 0.2, state=state, offset=5), mb.dropout(x, 0.2, 77, 1005))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mb.dropout(x, 0.2, state=state, offset=5)
        dx = mb.dropout_backward(x, 0.2, state=state, offset=5)
        state[1] += 1
    state[1] = 1000
    for k in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mb.dropout(x, 0.2, 77, 1005 + k)) and torch.equal(out, dx)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = mb.dropout(x, 0.2, 1, 2, stream=side)
    side.synchronize()
    assert torch.equal(got, mb.dropout(x, 0.2, 1, 2))
    assert mb.dropout(x[:0], 0.2).shape == (0, 128) and mb.dropout(x[:, :0], 0.2).shape == (300, 0)
