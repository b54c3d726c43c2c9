"""The training operators without a GPU: the oracle's gradients against
differences, its generator against published numbers, the C structs' layouts,
and the entry points' refusals (argument checks run before any device work)."""
import ctypes

import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

from test_recurrent_block_cpu import STRUCTS, layouts  # noqa: F401 (a fixture)
from test_recurrent_block_cpu import test_ctypes_layout_is_the_header_s as check_layout
from test_recurrent_block_cpu import test_packed_values_land_in_their_fields as check_packed

NEW_STRUCTS = {
    "MambaLayerNormArgs": (mb.MambaLayerNormArgs, mb._LAYER_NORM_ARGS),
    "MambaLayerNormGrads": (mb.MambaLayerNormGrads, mb._LAYER_NORM_GRADS),
    "MambaEmbeddingArgs": (mb.MambaEmbeddingArgs, mb._EMBEDDING_ARGS),
    "MambaDropoutArgs": (mb.MambaDropoutArgs, mb._DROPOUT_ARGS),
    "MambaScanArgs": (mb.MambaScanArgs, mb._SCAN_ARGS),
    "MambaScanGrads": (mb.MambaScanGrads, mb._SCAN_GRADS),
    "MambaConvGradArgs": (mb.MambaConvGradArgs, mb._CONV_GRAD_ARGS),
}


@pytest.fixture(scope="module", autouse=True)
def _structs():
    keep = dict(STRUCTS)
    STRUCTS.clear()
    STRUCTS.update(NEW_STRUCTS)
    yield
    STRUCTS.clear()
    STRUCTS.update(keep)


@pytest.mark.parametrize("name", sorted(NEW_STRUCTS))
def test_struct_layouts(layouts, name):  # noqa: F811
    check_layout(layouts, name)
    check_packed(name)


# Central differences with step 1e-5: truncation about 1e-10 times the third derivative, cancellation about 1e-10.
def _check_differences(values, run, grads, names, tol=1e-7):
    for name, key in names:
        v = values[name]
        num = np.zeros_like(v)
        for j in np.ndindex(v.shape):
            keep, f = v[j], []
            for e in (1e-5, -1e-5):
                v[j] = keep + e
                f.append(run())
            v[j] = keep
            num[j] = (f[0] - f[1]) / 2e-5
        assert np.abs(num - grads[key]).max() < tol, key


def test_layer_norm_gradients_match_differences():
    rng = np.random.default_rng(1)
    v = {"x": rng.standard_normal((3, 5)), "w": rng.standard_normal(5), "b": rng.standard_normal(5)}
    g = rng.standard_normal((3, 5))
    _, mean, rstd = tr.layer_norm(v["x"], v["w"], v["b"], 1e-2)[0]
    grads, _ = tr.layer_norm_backward(g, v["x"], mean, rstd, v["w"])
    _check_differences(v, lambda: (tr.layer_norm(v["x"], v["w"], v["b"], 1e-2)[0][0] * g).sum(), grads,
                       (("x", "dx"), ("w", "dw"), ("b", "db")))


def test_embedding_gradient_matches_differences():
    rng = np.random.default_rng(2)
    v = {"table": rng.standard_normal((4, 3))}
    ids, g = np.array([1, 3, -1, 1, 4, 0]), rng.standard_normal((6, 3))
    grad, _ = tr.embedding_backward(g, ids, 4, 1.5)
    _check_differences(v, lambda: (tr.embedding(ids, v["table"], 1.5) * g).sum(), {"d": grad}, (("table", "d"),))


@pytest.mark.parametrize("silu", [False, True])
def test_conv_gradients_match_differences(silu):
    rng = np.random.default_rng(3)
    v = {"x": rng.standard_normal((2, 5, 3)), "w": rng.standard_normal((3, 4)), "b": rng.standard_normal(3)}
    g = rng.standard_normal((2, 5, 3))

    def run():
        back = np.concatenate([np.zeros((2, 3, 3)), v["x"]], 1)
        pre = v["b"] + sum(back[:, k:k + 5] * v["w"][:, k] for k in range(4))
        return ((pre / (1 + np.exp(-pre)) if silu else pre) * g).sum()

    grads, _ = tr.conv_backward(g, v["x"], v["w"], v["b"], silu)
    _check_differences(v, run, grads, (("x", "dx"), ("w", "dw"), ("b", "dbias")))


@pytest.mark.parametrize("gate", [False, True])
def test_scan_gradients_match_differences(gate):
    rng = np.random.default_rng(4)
    b, L, D, N = 2, 4, 3, 2
    v = {k: rng.standard_normal((b, L, D)) for k in ("x", "delta", "z")}
    v.update({k: rng.standard_normal((b, L, N)) for k in ("B", "C")})
    v.update(A=-np.exp(rng.standard_normal((D, N))), D=rng.standard_normal(D), bias=rng.standard_normal(D),
             h0=rng.standard_normal((b, D, N)))
    v["A"][0, 0] = -1e-4  # where psi comes from its series
    g, gf = rng.standard_normal((b, L, D)), rng.standard_normal((b, D, N))

    def run():
        dt = np.logaddexp(0, v["delta"] + v["bias"])
        h, total = v["h0"], 0.0
        for t in range(L):
            d = dt[:, t, :, None]
            h = np.exp(d * v["A"]) * h + np.expm1(d * v["A"]) / v["A"] * v["B"][:, t, None] * v["x"][:, t, :, None]
            y = (h * v["C"][:, t, None]).sum(2) + v["D"] * v["x"][:, t]
            if gate:
                y = y * v["z"][:, t] / (1 + np.exp(-v["z"][:, t]))
            total += (y * g[:, t]).sum()
        return total + (h * gf).sum()

    grads, _ = tr.scan_backward(g, v["x"], v["delta"], v["A"], v["B"], v["C"], v["D"], v["z"] if gate else None,
                                v["bias"], v["h0"], gf)
    names = [("x", "dx"), ("delta", "ddelta"), ("B", "dB"), ("C", "dC"), ("D", "dD"), ("bias", "ddt_bias"),
             ("h0", "dh0")] + ([("z", "dz")] if gate else [])
    _check_differences(v, run, grads, names)
    # A's element near zero is moved by less than itself
    _check_differences(v, run, grads, (("A", "dA"),), 1e-6)


def test_generator_matches_published_numbers():
    """The known answers that accompany the generator's publication."""
    kat = [((0, 0, 0, 0), (0, 0), (0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8)),
           ((0xffffffff,) * 4, (0xffffffff,) * 2, (0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd)),
           ((0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344), (0xa4093822, 0x299f31d0),
            (0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1))]
    for counter, key, want in kat:
        assert tuple(tr.philox(counter, key)) == want


P = ctypes.byref


def _refused(fn, text, *args):
    assert fn(*args) == -1
    assert text in mb.last_error(), mb.last_error()


def _set(s, change):
    for k, v in change.items():
        if isinstance(v, tuple):
            getattr(s, k)[:] = v
        else:
            setattr(s, k, v)
    return s


# Addresses below are never dereferenced: every call is refused or empty.
def _ln(**kw):
    a = mb.MambaLayerNormArgs()
    a.x, a.out, a.mean, a.rstd, a.w, a.b = 4096, 8192, 12288, 16384, 20480, 24576
    a.rows, a.cols, a.x_dtype, a.out_dtype, a.eps = 4, 8, mb.F32, mb.F16, 1e-5
    a.x_stride = a.out_stride = 8
    return _set(a, kw)


@pytest.mark.parametrize("change,text", [
    (dict(x_dtype=2), "dtype"), (dict(out_dtype=-1), "dtype"), (dict(rows=-1), "negative"), (dict(cols=-1), "negative"),
    (dict(cols=16385), "16384"), (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(x=4098), "aligned"),
    (dict(out=8193), "aligned"), (dict(w=4098), "aligned"), (dict(b=4098), "aligned"), (dict(mean=4098), "aligned"),
    (dict(rstd=4098), "aligned"), (dict(out=4096), "own"), (dict(out_stride=7), "overlap")])
def test_layer_norm_refusals(change, text):
    _refused(mb.lib().mamba_layer_norm, text, P(_ln(**change)), None)


@pytest.mark.parametrize("args,change,text", [
    (dict(mean=None), {}, "null"), (dict(rstd=None), {}, "null"), ({}, dict(dout=None), "null"),
    ({}, dict(dx=None), "null"), ({}, dict(dx=4098), "aligned"), ({}, dict(dout=8193), "aligned"),
    ({}, dict(dw=4098), "aligned"), ({}, dict(db=4098), "aligned"), ({}, dict(dx=4096), "own"),
    ({}, dict(dx=28672), "own"), ({}, dict(dw=36864), "own"), ({}, dict(dx_stride=7), "overlap"),
    ({}, dict(ws=None), "workspace"), ({}, dict(ws=4104), "workspace"), ({}, dict(short=1), "workspace")])
def test_layer_norm_backward_refusals(args, change, text):
    a, g = _ln(**args), mb.MambaLayerNormGrads()
    change = dict(change)
    ws, short = change.pop("ws", 4096), change.pop("short", 0)
    g.dout, g.dx, g.dw, g.db, g.dout_stride, g.dx_stride = 28672, 32768, 40960, 36864, 8, 8
    need = mb.lib().mamba_layer_norm_workspace(P(a))
    assert need > 0
    _refused(mb.lib().mamba_layer_norm_backward, text, P(a), P(_set(g, change)), ws, need - short, None)


def _emb(**kw):
    a = mb.MambaEmbeddingArgs()
    a.ids, a.table, a.out = 4096, 8192, 12288
    a.tokens, a.vocab, a.dim, a.id_bytes, a.table_dtype, a.out_dtype, a.scale = 6, 5, 8, 8, mb.F16, mb.F32, 1.0
    a.table_stride = a.out_stride = 8
    return _set(a, kw)


BOTH = [(dict(tokens=-1), "negative"), (dict(vocab=-1), "negative"), (dict(dim=-1), "negative"),
        (dict(tokens=(1 << 30) + 1), "2^30"), (dict(vocab=1 << 31), "2^31"), (dict(id_bytes=2), "4 or 8"),
        (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(table_dtype=2), "dtype"),
        (dict(out_dtype=2), "dtype"), (dict(ids=4100), "aligned"), (dict(ids=None), "null")]


@pytest.mark.parametrize("change,text", BOTH + [
    (dict(table=None), "null"), (dict(out=None), "null"), (dict(table=8193), "aligned"), (dict(out=12290), "aligned"),
    (dict(out=8192), "own"), (dict(out=4096), "own"), (dict(out_stride=7), "overlap")])
def test_embedding_refusals(change, text):
    _refused(mb.lib().mamba_embedding, text, P(_emb(**change)), None)


@pytest.mark.parametrize("change,text", BOTH + [
    (dict(dtable=None), "null"), (dict(dout=None), "null"), (dict(dtable=12290), "aligned"),
    (dict(dout=16386), "aligned"), (dict(stride=7), "overlap"), (dict(dtable=16384), "own"), (dict(dtable=4096), "own"),
    (dict(ws=None), "workspace"), (dict(ws=4104), "workspace"), (dict(short=1), "workspace")])
def test_embedding_backward_refusals(change, text):
    change = dict(change)
    dout, dtable = change.pop("dout", 16384), change.pop("dtable", 20480)
    ws, short, stride = change.pop("ws", 4096), change.pop("short", 0), change.pop("stride", 8)
    need = mb.lib().mamba_embedding_workspace(P(_emb()))
    assert need > 0
    _refused(mb.lib().mamba_embedding_backward, text, P(_emb(**change)), dout, 8, dtable, stride, 0, ws, need - short,
             None)


def _drop(**kw):
    a = mb.MambaDropoutArgs()
    a.x, a.residual, a.out, a.rows, a.cols = 4096, 8192, 12288, 4, 8
    a.x_dtype, a.out_dtype, a.p = mb.F32, mb.F32, 0.5
    a.x_stride = a.residual_stride = a.out_stride = 8
    return _set(a, kw)


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "negative"), (dict(cols=-1), "negative"), (dict(x_dtype=2), "dtype"), (dict(out_dtype=2), "dtype"),
    (dict(p=-0.1), "p must"), (dict(p=1.1), "p must"), (dict(p=float("nan")), "p must"),
    (dict(rows=1 << 39, cols=4), "many"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(x=4098), "aligned"),
    (dict(residual=4098), "aligned"), (dict(out=4098), "aligned"), (dict(state=4100), "aligned"),
    (dict(out_stride=7), "overlap"), (dict(out=4096, out_stride=9), "out may be x"),
    (dict(out=4096, out_dtype=mb.F16), "out may be x"), (dict(out=8192, out_stride=9), "residual"),
    (dict(out=8192, out_dtype=mb.F16), "residual")])
def test_dropout_refusals(change, text):
    _refused(mb.lib().mamba_dropout, text, P(_drop(**change)), None)


def _conv(**kw):
    a = mb.MambaConvGradArgs()
    a.dy, a.x, a.w, a.bias, a.dx, a.dw, a.dbias = 4096, 8192, 12288, 16384, 20480, 24576, 28672
    a.batch, a.seqlen, a.dim, a.K, a.silu, a.dtype = 2, 5, 8, 4, 1, mb.F32
    for s in (a.dy_stride, a.x_stride, a.dx_stride):
        s[:] = (40, 8, 1)
    return _set(a, kw)


@pytest.mark.parametrize("change,text", [
    (dict(batch=-1), "negative"), (dict(seqlen=-1), "negative"), (dict(dim=-1), "negative"), (dict(K=0), "1..8"),
    (dict(K=9), "1..8"), (dict(dtype=2), "dtype"), (dict(seqlen=0x7fffffff), "long"), (dict(dy=None), "null"),
    (dict(x=None), "null"), (dict(w=None), "null"), (dict(dx=None), "null"), (dict(x=8194), "aligned"),
    (dict(dw=4098), "aligned"), (dict(bias=4098), "aligned"), (dict(dx=8192), "own"), (dict(dx=4096), "own"),
    (dict(dw=28672), "own"), (dict(dx_stride=(0, 8, 1)), "overlap"), (dict(dx_stride=(40, 0, 1)), "overlap"),
    (dict(dx_stride=(40, 8, 0)), "overlap"), (dict(ws=None), "workspace"), (dict(ws=4104), "workspace"), (dict(short=1), "workspace")])
def test_conv_backward_refusals(change, text):
    change = dict(change)
    ws, short = change.pop("ws", 4096), change.pop("short", 0)
    need = mb.lib().mamba_causal_conv1d_backward_workspace(P(_conv()))
    assert need > 0
    _refused(mb.lib().mamba_causal_conv1d_backward, text, P(_conv(**change)), ws, need - short, None)


def _scan(**kw):
    a = mb.MambaScanArgs()
    a.x, a.delta, a.B, a.C, a.A, a.D, a.z, a.dt_bias, a.initial_state = (4096 * k for k in range(1, 10))
    a.batch, a.seqlen, a.dim, a.dstate = 2, 5, 8, 4
    return _set(a, kw)


@pytest.mark.parametrize("args,change,text", [
    (dict(batch=-1), {}, "negative"), (dict(seqlen=-1), {}, "negative"), (dict(dim=-1), {}, "negative"),
    (dict(dstate=0), {}, "1..16"), (dict(dstate=17), {}, "1..16"), (dict(x_dtype=2), {}, "dtypes"),
    (dict(x_dtype=1), {}, None), (dict(delta_dtype=1), {}, "dtypes"), (dict(bc_dtype=1), {}, "dtypes"),
    (dict(x_dtype=1, delta_dtype=1), {}, "dtypes"), (dict(seqlen=0x7fffffff), {}, "many"),
    (dict(batch=1 << 16, seqlen=1 << 16), {}, "many"),
    (dict(x=None), {}, "null"), (dict(delta=None), {}, "null"), (dict(A=None), {}, "null"), (dict(B=None), {}, "null"),
    (dict(C=None), {}, "null"), ({}, dict(dy=None), "null"), ({}, dict(dx=None), "null"),
    ({}, dict(ddelta=None), "null"), ({}, dict(dz=None), "dz"), (dict(x=4098), {}, "aligned"),
    (dict(dt_bias=4098), {}, "aligned"), ({}, dict(dA=4098), "aligned"), ({}, dict(dB=4098), "aligned"),
    (dict(initial_state=4098), {}, "aligned"), ({}, dict(dfinal_state=4098), "aligned"), ({}, dict(dx=4096), "inputs"),
    ({}, dict(dB=4096 * 3), "inputs"), ({}, dict(dinitial_state=4096 * 9), "inputs"), ({}, dict(dz=4096 * 13), "own"),
    ({}, dict(dD=4096 * 18), "own"), ({}, dict(dx_stride=(40, 0, 1)), "overlap"),
    ({}, dict(ddelta_stride=(0, 8, 1)), "overlap"), ({}, dict(dz_stride=(40, 8, 0)), "overlap"),
    ({}, dict(dB_stride=(20, 4, 0)), "overlap"), ({}, dict(dC_stride=(20, 0, 1)), "overlap"), ({}, dict(ws=None), "workspace"), ({}, dict(ws=4104), "workspace"),
    ({}, dict(short=1), "workspace")])
def test_scan_backward_refusals(args, change, text):
    g, change = mb.MambaScanGrads(), dict(change)
    for k, (name, *_) in enumerate(mb.MambaScanGrads._fields_[:11]):
        setattr(g, name, 4096 * (11 + k))
    for st in (g.dy_stride, g.dx_stride, g.ddelta_stride, g.dz_stride):
        st[:] = (40, 8, 1)
    g.dB_stride[:] = g.dC_stride[:] = (20, 4, 1)
    ws, short = change.pop("ws", 4096), change.pop("short", 0)
    need = mb.lib().mamba_selective_scan_backward_workspace(P(_scan()))
    assert need > 0
    if text is None:  # FP16 rows with FP32 delta, B and C are supported
        _set(g, dict(dx=None))
        text = "null"
    _refused(mb.lib().mamba_selective_scan_backward, text, P(_scan(**args)), P(_set(g, change)), ws, need - short, None)


def test_empty_and_null():
    assert mb.lib().mamba_selective_scan_backward(None, None, None, 0, None) == -1
    assert mb.lib().mamba_selective_scan_backward(P(_scan()), None, None, 0, None) == -1
    assert mb.lib().mamba_causal_conv1d_backward(None, None, 0, None) == -1
    assert mb.lib().mamba_selective_scan_backward_workspace(None) == 0
    assert mb.lib().mamba_causal_conv1d_backward_workspace(None) == 0
    assert mb.lib().mamba_causal_conv1d_backward(P(_conv(dim=0)), None, 0, None) == 0
    L = mb.lib()
    for fn in (L.mamba_layer_norm, L.mamba_embedding, L.mamba_dropout):
        assert fn(None, None) == -1
    assert L.mamba_layer_norm(P(_ln(rows=0)), None) == 0 and L.mamba_layer_norm(P(_ln(cols=0)), None) == 0
    assert L.mamba_layer_norm_backward(P(_ln()), None, None, 0, None) == -1
    assert L.mamba_embedding(P(_emb(tokens=0)), None) == 0 and L.mamba_embedding(P(_emb(dim=0)), None) == 0
    assert L.mamba_embedding_backward(P(_emb(vocab=0)), None, 0, None, 0, 0, None, 0, None) == 0
    assert L.mamba_embedding_backward(P(_emb(tokens=0)), None, 0, 4096, 8, 1, None, 0, None) == 0
    assert L.mamba_dropout(P(_drop(rows=0)), None) == 0 and L.mamba_dropout(P(_drop(cols=0)), None) == 0
    assert L.mamba_layer_norm_workspace(None) == 0 and L.mamba_embedding_workspace(None) == 0


def test_binding_refuses_wrong_tensors():
    x, w, ids = torch.zeros((3, 8)), torch.zeros(8), torch.zeros(3, dtype=torch.int64)
    one = torch.zeros(3)
    for call in (lambda: mb.layer_norm(x.double()), lambda: mb.layer_norm(x[0]), lambda: mb.layer_norm(x, w[:7]),
                 lambda: mb.layer_norm(x, w, w.half()), lambda: mb.layer_norm(x.t().contiguous().t()),
                 lambda: mb.layer_norm(x, out=x.half(), out_dtype=torch.float32), lambda: mb.layer_norm(x, eps=1e300),
                 lambda: mb.layer_norm(x, out_dtype=torch.float64),
                 lambda: mb.layer_norm_backward(x[:2], x, one, one), lambda: mb.layer_norm_backward(x, x, one[:2], one),
                 lambda: mb.layer_norm_backward(x, x, one, one.double()),
                 lambda: mb.layer_norm_backward(x, x, one, one, dx=x.half()),
                 lambda: mb.embedding(ids.float(), x), lambda: mb.embedding(ids, x.double()),
                 lambda: mb.embedding(ids, x[0]), lambda: mb.embedding(ids.to(torch.int16), x),
                 lambda: mb.embedding(torch.zeros(6, dtype=torch.int64)[::2], x),
                 lambda: mb.embedding(ids, x, out=x[:2]), lambda: mb.embedding(ids, x, scale=1e300),
                 lambda: mb.embedding_backward(x[:2], ids, 5), lambda: mb.embedding_backward(x.double(), ids, 5), lambda: mb.embedding_backward(x, ids, -1),
                 lambda: mb.embedding_backward(x, ids, 5, dtable=x), lambda: mb.embedding_backward(x, ids, 5,
                                                                                                  accumulate=True),
                 lambda: mb.embedding_backward(x, ids, 1 << 31, dtable=x),
                 lambda: mb.dropout(x.double(), 0.1), lambda: mb.dropout(x, 0.1, residual=x.half()),
                 lambda: mb.dropout(x, 0.1, residual=x[:2]), lambda: mb.dropout(x, 0.1, seed=-1),
                 lambda: mb.dropout(x, 0.1, offset=1 << 64), lambda: mb.dropout(x, 0.1, state=ids),
                 lambda: mb.dropout(x.view(3, 2, 4).transpose(1, 2), 0.1), lambda: mb.dropout(x, 0.1, out=x[:2]),
                 lambda: mb.dropout_backward(x, 0.1, dx=x.half(), out_dtype=torch.float32)):
        with pytest.raises(mb.MambaError):
            call()
    v, A, bc, k = torch.zeros((2, 5, 8)), torch.zeros((8, 4)), torch.zeros((2, 5, 4)), torch.zeros((8, 3))
    h = torch.zeros((2, 8, 4))
    for call in (lambda: mb.causal_conv1d_backward(v, v[0], k), lambda: mb.causal_conv1d_backward(v[:1], v, k),
                 lambda: mb.causal_conv1d_backward(v.half(), v, k), lambda: mb.causal_conv1d_backward(v, v, k[:7]),
                 lambda: mb.causal_conv1d_backward(v, v, k, w[:7]), lambda: mb.causal_conv1d_backward(v, v, k.half()),
                 lambda: mb.selective_scan_backward(v[:1], v, v, A, bc, bc),
                 lambda: mb.selective_scan_backward(v.half(), v, v, A, bc, bc),
                 lambda: mb.selective_scan_backward(v, v, v[:, :4], A, bc, bc),
                 lambda: mb.selective_scan_backward(v, v, v, A[:7], bc, bc),
                 lambda: mb.selective_scan_backward(v, v, v, A.half(), bc, bc),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc[:1], bc),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc, bc.half()),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc, bc, D=w[:7]),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc, bc, z=v[:1]),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc, bc, dz=v),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc, bc, initial_state=h[:1]),
                 lambda: mb.selective_scan_backward(v, v, v, A, bc, bc, dfinal_state=h.half())):
        with pytest.raises(mb.MambaError):
            call()
    for call in (lambda: mb.layer_norm(x), lambda: mb.layer_norm_backward(x, x, one, one), lambda: mb.dropout(x, 0.1),
                 lambda: mb.causal_conv1d_backward(v, v, k), lambda: mb.selective_scan_backward(v, v, v, A, bc, bc),
                 lambda: mb.embedding(ids, x), lambda: mb.embedding_backward(x, ids, 5)):
        with pytest.raises(mb.MambaError, match="CUDA"):
            call()
