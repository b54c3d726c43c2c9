"""The training operators in a run, as a program uses them: token ids through
the embedding, the norm, one Mamba block (projections by torch), dropout with
the residual add, and all gradients back to the table, against autograd in FP64
over plain torch operations; the same step captured and replayed; and prompts
of token ids through the model.

Everything is FP32.  Each operator's own error is at most 2^-24 (64 + 8 L) =
2.7e-5 of its terms' magnitudes (L = 48, the scan; the others 4e-6).  Six of
them follow one another each way, terms are a few times their sums: 2e-4 of
the largest element bounds the chain."""
import numpy as np
import pytest
import torch

import mamba_b200 as mb
from oracle import training as tr

pytestmark = pytest.mark.gpu
BATCH, L, VOCAB, DM, DI, N, R = 2, 48, 37, 40, 72, 16, 5
P, SCALE, EPS = 0.2, 1.5, 1e-5


@pytest.fixture(scope="module", autouse=True)
def _leave_no_cached_memory():
    yield
    torch.cuda.synchronize()
    torch.cuda.empty_cache()


def _weights(seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(s, generator=g) * scale).cuda()  # noqa: E731
    return {"table": r(VOCAB, DM), "nw": 1 + r(DM, scale=0.1), "nb": r(DM, scale=0.1), "w_in": r(DM, 2 * DI, scale=0.15),
            "conv_w": r(DI, 4, scale=0.4), "conv_b": r(DI, scale=0.2), "w_x": r(DI, R + 2 * N, scale=0.15),
            "w_dt": r(R, DI, scale=0.3), "dt_bias": r(DI, scale=0.5) - 3,
            "A": -torch.exp(r(DI, N, scale=0.5)) * torch.arange(1, N + 1, device="cuda"), "D": 1 + r(DI, scale=0.1),
            "w_out": r(DI, DM, scale=0.15)}


def _step(w, tokens, dout, seed, offset=0, state=None):
    """The forward pass and the gradients of sum(out * dout), by the library's operators and torch's products."""
    T = BATCH * L
    e = mb.embedding(tokens, w["table"], SCALE).view(T, DM)
    n, mean, rstd = mb.layer_norm(e, w["nw"], w["nb"], EPS, return_stats=True)
    xz = (n @ w["w_in"]).view(BATCH, L, 2 * DI)
    x, z = xz[:, :, :DI], xz[:, :, DI:]
    u = mb.causal_conv1d(x, w["conv_w"], w["conv_b"])
    xdbc = u.view(T, DI) @ w["w_x"]
    v = xdbc.view(BATCH, L, R + 2 * N)
    delta = (xdbc[:, :R] @ w["w_dt"]).view(BATCH, L, DI)
    B, C = v[:, :, R:R + N], v[:, :, R + N:]
    y = mb.selective_scan(u, delta, w["A"], B, C, D=w["D"], z=z, dt_bias=w["dt_bias"])
    o = y.view(T, DI) @ w["w_out"]
    out = mb.dropout(o, P, seed, offset, residual=e, state=state)
    # and back
    g = {}
    do = mb.dropout_backward(dout, P, seed, offset, state=state)
    g["w_out"] = y.view(T, DI).t() @ do
    dy = (do @ w["w_out"].t()).view(BATCH, L, DI)
    dxz, dxdbc = torch.empty_like(xz), torch.empty_like(xdbc)
    du, ddelta, g["A"], dB, dC, g["D"], _, g["dt_bias"], _ = mb.selective_scan_backward(
        dy, u, delta, w["A"], B, C, D=w["D"], z=z, dt_bias=w["dt_bias"], dz=dxz[:, :, DI:])
    g["w_dt"] = xdbc[:, :R].t() @ ddelta.view(T, DI)
    dxdbc[:, :R] = ddelta.view(T, DI) @ w["w_dt"].t()
    dxdbc.view(BATCH, L, -1)[:, :, R:R + N] = dB
    dxdbc.view(BATCH, L, -1)[:, :, R + N:] = dC
    g["w_x"] = u.view(T, DI).t() @ dxdbc
    du = du + (dxdbc @ w["w_x"].t()).view(BATCH, L, DI)
    _, g["conv_w"], g["conv_b"] = mb.causal_conv1d_backward(du, x, w["conv_w"], w["conv_b"], dx=dxz[:, :, :DI])
    g["w_in"] = n.t() @ dxz.view(T, 2 * DI)
    de, g["nw"], g["nb"] = mb.layer_norm_backward(dxz.view(T, 2 * DI) @ w["w_in"].t(), e, mean, rstd, w["nw"])
    g["table"] = mb.embedding_backward(de + dout, tokens.view(-1), VOCAB, SCALE)
    return out, g


def _reference(w, tokens, dout, seed, offset):
    """The same by autograd in FP64, the mask from the oracle's generator."""
    w = {k: v.detach().double().requires_grad_() for k, v in w.items()}
    T = BATCH * L
    inside = (tokens >= 0) & (tokens < VOCAB)
    e = torch.where(inside[..., None], w["table"][tokens.clamp(0, VOCAB - 1)], 0.0).view(T, DM) * SCALE
    mean = e.mean(1, keepdim=True)
    n = (e - mean) / ((e - mean) ** 2).mean(1, keepdim=True).add(EPS).sqrt() * w["nw"] + w["nb"]
    xz = (n @ w["w_in"]).view(BATCH, L, 2 * DI)
    x, z = xz[:, :, :DI], xz[:, :, DI:]
    back = torch.nn.functional.pad(x, (0, 0, 3, 0))
    u = torch.nn.functional.silu(sum(back[:, k:k + L] * w["conv_w"][:, k] for k in range(4)) + w["conv_b"])
    xdbc = u.reshape(T, DI) @ w["w_x"]
    dt = torch.nn.functional.softplus((xdbc[:, :R] @ w["w_dt"]).view(BATCH, L, DI) + w["dt_bias"])
    v = xdbc.view(BATCH, L, R + 2 * N)
    h, ys = torch.zeros((BATCH, DI, N), dtype=torch.float64, device="cuda"), []
    for t in range(L):
        a = torch.exp(dt[:, t, :, None] * w["A"])
        h = a * h + (a - 1) / w["A"] * v[:, t, None, R:R + N] * u[:, t, :, None]
        ys.append((h * v[:, t, None, R + N:]).sum(2) + w["D"] * u[:, t])
    y = torch.stack(ys, 1) * torch.nn.functional.silu(z)
    keep = torch.from_numpy(tr.dropout_keep(0, T * DM, P, seed, offset).reshape(T, DM)).cuda()
    out = e + keep * (y.reshape(T, DI) @ w["w_out"]) / (1 - float(np.float32(P)))
    out.backward(dout.double())
    return out.detach(), {k: t.grad for k, t in w.items()}


def _compare(got, want):
    assert set(got[1]) == set(want[1])
    for k, a, b in [("out", got[0], want[0])] + [(k, got[1][k], want[1][k]) for k in want[1]]:
        assert (a.double() - b).abs().max() <= 2e-4 * b.abs().max(), k


def _tokens(seed):
    g = torch.Generator(device="cpu").manual_seed(seed)
    t = torch.randint(0, VOCAB, (BATCH, L), generator=g)
    t[0, -5:] = -1  # padding
    return t.cuda()


def test_training_step_against_autograd(cuda):
    w, tokens, dout = _weights(1), _tokens(2), torch.randn((BATCH * L, DM), device="cuda")
    _compare(_step(w, tokens, dout, 5, 6), _reference(w, tokens, dout, 5, 6))
    assert mb.device_status() == 0


def test_captured_step_draws_new_masks(cuda):
    """The whole step in a CUDA graph: new tokens, gradients and random numbers at each replay; an eager step of the
    same tensors in between changes nothing."""
    w, tokens, dout = _weights(3), _tokens(4), torch.randn((BATCH * L, DM), device="cuda")
    state = torch.tensor([11, 100], dtype=torch.int64, device="cuda")
    _step(w, tokens, dout, 0, state=state)  # loads the kernels
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _step(w, tokens, dout, 0, state=state)
        state[1] += 1
    state[1] = 100
    for k in range(3):
        tokens.copy_(_tokens(20 + k))
        dout.normal_()
        graph.replay()
        eager = _step(w, tokens, dout, 11, 100 + k)
        torch.cuda.synchronize()
        assert torch.equal(got[0], eager[0])
        for name in got[1]:
            if name.startswith("w_"):  # torch's products may take another algorithm in a graph
                continue
            assert (got[1][name] - eager[1][name]).abs().max() <= 1e-5 * eager[1][name].abs().max(), name
    _compare(got, _reference(w, tokens, dout, 11, 102))


def test_two_streams_at_once(cuda):
    """Two steps at the same time on two streams, each with its own tensors, equal to the steps alone."""
    jobs = [(_weights(5 + k), _tokens(6 + k), torch.randn((BATCH * L, DM), device="cuda")) for k in range(2)]
    want = [_step(*job, 1, k) for k, job in enumerate(jobs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = _step(*jobs[k], 1, k)
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0])
        for name in a[1]:
            if not name.startswith("w_"):
                assert (a[1][name] - b[1][name]).abs().max() <= 1e-5 * b[1][name].abs().max(), name


def test_scan_gradients_beside_tensor_core_products(cuda):
    """Both keep accumulators in tensor memory: calls on two streams wait for each other's columns, and give what they
    give alone."""
    g = torch.Generator(device="cpu").manual_seed(9)
    r = lambda *s: torch.randn(s, generator=g).half().cuda()  # noqa: E731
    xl, wl = r(4096, 1024), r(1024, 1024)
    dy, x, z, delta, B, C = r(4, 256, 1024), r(4, 256, 1024), r(4, 256, 1024), r(4, 256, 1024), r(4, 256, 16), r(4, 256, 16)
    A = -torch.arange(1, 17, device="cuda", dtype=torch.float32).repeat(1024, 1)
    run = lambda: mb.selective_scan_backward(dy, x, delta, A, B, C, z=z)  # noqa: E731
    want, want_l = run(), mb.linear(xl, wl)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(a):
            got = [run() for _ in range(3)][-1]
        with torch.cuda.stream(b):
            got_l = [mb.linear(xl, wl) for _ in range(20)][-1]
    torch.cuda.synchronize()
    assert torch.equal(got_l, want_l)
    assert all(p is q or torch.equal(p, q) for p, q in zip(got, want))
    assert mb.device_status() == 0


@pytest.mark.parametrize("side", [False, True])
def test_model_forward_of_tokens(cuda, side):
    m = mb.Model(32, 16, 4, 2, 2, mb.F16)
    m.init_random(3)
    table = torch.randn((50, 32), device="cuda").half()
    tokens = torch.randint(-1, 50, (3, 33), device="cuda")
    stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = m.forward_tokens(tokens, table, 0.7)
    torch.cuda.synchronize()
    rows = mb.embedding(tokens, table, 0.7, out_dtype=torch.float32)
    want = m.forward(rows.cpu().numpy())
    assert np.array_equal(got.cpu().numpy(), want)
    assert m.forward_tokens(tokens[:, :0].contiguous(), table).shape == (3, 0, 32)
    for bad in (lambda: m.forward_tokens(tokens[0], table), lambda: m.forward_tokens(tokens, table[:, :16]),
                lambda: m.forward_tokens(tokens.cpu(), table)):
        with pytest.raises(mb.MambaError):
            bad()
