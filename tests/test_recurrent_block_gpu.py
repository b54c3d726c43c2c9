"""The recurrent-block operators in a run, as a program uses them.

Training: norm -> projection -> gated recurrence -> projection -> norm, gate
and residual, and all gradients of a loss on its outputs, against torch
autograd of the same formulas in FP64.  Serving: the same block with 8-bit
projections, a prefill followed by single tokens, each operator against the
FP64 oracle on the inputs it got."""
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

C, EPS, RHO = 8.0, 1e-5, 0.9


def _params(dim, inner, seed, dtype=torch.float32):
    g = torch.Generator(device="cpu").manual_seed(seed)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    p = {"w0": 1 + 0.1 * rnd(dim), "win": rnd(4 * inner, dim) / dim ** 0.5, "wout": rnd(dim, inner) / inner ** 0.5,
         "wq": 1 + 0.1 * rnd(dim), "wp": 1 + 0.1 * rnd(dim),
         "lam": torch.log(torch.expm1(-torch.log(0.9 + 0.099 * torch.rand(inner, generator=g)) / C))}
    return {k: v.cuda().to(dtype) for k, v in p.items()}


def _plain(p, x, h0, wz, resets):
    """The block in torch, any dtype: returns (residual_out, out, final state)."""
    B, L, D = x.shape
    rms = lambda v: v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)  # noqa: E731
    u = (rms(x) * p["w0"]) @ p["win"].T
    n = p["lam"].numel()
    xr, r, i, _ = (u[..., k * n:(k + 1) * n] for k in range(4))
    y = C * torch.nn.functional.softplus(p["lam"]) * torch.sigmoid(r)
    a, b = torch.exp(-y), torch.sqrt(-torch.expm1(-2 * y)) * torch.sigmoid(i) * xr
    h, hs = h0, []
    for t in range(L):
        keep = (resets[:, t] == 0).to(x.dtype)[:, None]
        h = keep * a[:, t] * h + b[:, t]
        hs.append(h)
    o = torch.stack(hs, 1) @ p["wout"].T
    z = x @ wz
    res = RHO * x + rms(o) * p["wq"] * z * torch.sigmoid(z)
    return res, rms(res) * p["wp"], h


def test_training_step_matches_autograd(cuda):
    B, L, D, n = 3, 70, 96, 160
    p = _params(D, n, 1)
    g = torch.Generator(device="cpu").manual_seed(2)
    x, wz = torch.randn((B, L, D), generator=g).cuda(), (torch.randn((D, D), generator=g) / D ** 0.5).cuda()
    h0, dfin = torch.randn((B, n), generator=g).cuda(), torch.randn((B, n), generator=g).cuda()
    dres, dout = torch.randn((B * L, D), generator=g).cuda(), torch.randn((B * L, D), generator=g).cuda()
    resets = (torch.rand((B, L), generator=g) < 0.1).to(torch.uint8).cuda()

    # forward
    zeros = torch.zeros((B * L, D), device="cuda")
    x2 = x.view(B * L, D)
    # a norm alone: of the block norm's second half, with nothing added to the residual
    _, pn, _, rstd0 = mb.block_norm(zeros, x2, w_pre=p["w0"], eps=EPS, return_rstd=True)
    u = pn @ p["win"].T
    u3 = u.view(B, L, 4 * n)
    xr, r, i = (u3[..., k * n:(k + 1) * n] for k in range(3))  # strided views
    h, hN = mb.gated_recurrence(xr, r, i, p["lam"], c=C, initial_state=h0, resets=resets, return_final_state=True)
    o = h.view(B * L, n) @ p["wout"].T
    z = x2 @ wz
    res, out, rq, rp = mb.block_norm(o, x2, w_post=p["wq"], z=z, w_pre=p["wp"], residual_scale=RHO, eps=EPS,
                                     return_rstd=True)
    # backward
    do, dx, dwq, dwp, dz = mb.block_norm_backward(dres, dout, o, res, rq, rp, w_post=p["wq"], z=z, w_pre=p["wp"],
                                                  residual_scale=RHO)
    dx = dx + dz @ wz.T
    dh = (do @ p["wout"]).view(B, L, n)
    du = torch.zeros_like(u3)
    parts = [du[..., k * n:(k + 1) * n] for k in range(3)]
    _, _, _, dlam, dh0 = mb.gated_recurrence_backward(dh, xr, r, i, p["lam"], h, c=C, initial_state=h0, resets=resets,
                                                      dfinal_state=dfin, dx=parts[0], dr=parts[1], di=parts[2])
    du2 = du.view(B * L, 4 * n)
    _, dx0, _, dw0, _ = mb.block_norm_backward(None, du2 @ p["win"], zeros, x2, torch.ones(B * L, device="cuda"), rstd0,
                                               w_pre=p["w0"])
    got = {"x": dx + dx0, "w0": dw0, "win": du2.T @ pn, "wout": do.T @ h.view(B * L, n), "wq": dwq, "wp": dwp,
           "lam": dlam, "h0": dh0, "wz": x2.T @ dz}

    leaves = {k: v.double().requires_grad_() for k, v in list(p.items()) + [("x", x), ("h0", h0), ("wz", wz)]}
    rres, rout, rfin = _plain(leaves, leaves["x"], leaves["h0"], leaves["wz"], resets)
    loss = (rres.reshape(-1, D) * dres.double()).sum() + (rout.reshape(-1, D) * dout.double()).sum() + \
        (rfin * dfin.double()).sum()
    loss.backward()
    # FP32 products of up to 640 terms on the way: errors of a few 2^-24 * sqrt(640) of each tensor's size
    tol = 2e-5
    for name, a, ref in (("residual", res, rres), ("out", out, rout), ("final", hN, rfin)):
        ref = ref.detach().reshape(a.shape)
        assert (a.double() - ref).abs().max() <= tol * ref.abs().max(), name
    for k, v in got.items():
        ref = leaves[k].grad.reshape(v.shape)
        assert (v.double() - ref).abs().max() <= tol * ref.abs().max(), (k, (v.double() - ref).abs().max(), ref.abs().max())


def test_serving_prefill_and_steps(cuda):
    """FP16 activations, 8-bit projections, FP32 state and residual; padded
    prompts, then one token at a time."""
    B, L, D, n, steps = 4, 50, 256, 384, 3
    p = _params(D, n, 3)
    qin, sin = mb.quantize_rows(p["win"][:3 * n].contiguous())
    qout, sout = mb.quantize_rows(p["wout"])
    g = torch.Generator(device="cpu").manual_seed(4)
    lengths = torch.tensor([50, 17, 0, 33], dtype=torch.int32).cuda()
    prompt = torch.randn((B, L, D), generator=g).cuda()
    tokens = torch.randn((steps, B, D), generator=g).cuda()

    def check_linear(q, s, w, ws, y):
        ref, mag = rb.linear_i8(q.cpu().numpy(), s.cpu().numpy(), w.cpu().numpy(), ws.cpu().numpy())
        assert (np.abs(y.double().cpu().numpy() - ref) <= 2.0 ** -11 * np.abs(ref) + 2e-6 * mag + 2.0 ** -25).all()

    def project(v, w, ws):
        q, s = mb.quantize_rows(v)
        rq, rs = rb.quantize_rows(v.cpu().numpy())
        assert np.array_equal(q.cpu().numpy(), rq) and np.array_equal(s.cpu().numpy(), rs)
        y = mb.linear_i8(q, s, w, ws)
        check_linear(q, s, w, ws, y)
        return y

    def norm(x2):
        half = torch.zeros(x2.shape, dtype=torch.float16, device="cuda")
        return mb.block_norm(half, x2, w_pre=p["w0"], eps=EPS)[1]

    def join(o, x2):
        res, out, rq, rp = mb.block_norm(o, x2, w_post=p["wq"], w_pre=p["wp"], residual_scale=RHO, eps=EPS,
                                         return_rstd=True)
        ref, mag = rb.block_norm(o.cpu().numpy(), x2.cpu().numpy(), p["wq"].cpu().numpy(), None, p["wp"].cpu().numpy(),
                                 RHO, EPS)
        assert (np.abs(res.double().cpu().numpy() - ref[0]) <= 1e-5 * mag[0] + 1e-9).all()
        assert (np.abs(out.double().cpu().numpy() - ref[1]) <= 2.0 ** -11 * np.abs(ref[1]) + 1e-5 * mag[1] + 2.0 ** -25).all()
        return out

    u = project(norm(prompt.view(B * L, D)), qin, sin).view(B, L, 3 * n)
    parts = [u[..., k * n:(k + 1) * n] for k in range(3)]
    h, state = mb.gated_recurrence(*parts, p["lam"], c=C, lengths=lengths, return_final_state=True)
    lam, ln = p["lam"].cpu().numpy(), lengths.cpu().numpy()
    ref, fin, _ = rb.gated_recurrence(*(v.cpu().numpy() for v in parts), lam, C, lengths=ln)
    assert np.abs(h.double().cpu().numpy() - ref).max() <= (2.0 ** -11 + 2e-5) * np.abs(ref).max()
    assert np.abs(state.double().cpu().numpy() - fin).max() <= 2e-5 * np.abs(fin).max()
    join(project(h.view(B * L, n), qout, sout), prompt.view(B * L, D))

    seqs = [[v[b, :ln[b]] for b in range(B)] for v in parts]
    for k in range(steps):
        ut = project(norm(tokens[k]), qin, sin)
        step = [ut[:, j * n:(j + 1) * n] for j in range(3)]
        ht, state = mb.gated_recurrence_step(*step, p["lam"], state, c=C, state_out=state)
        join(project(ht, qout, sout), tokens[k])
        for j in range(3):
            for b in range(B):
                seqs[j][b] = torch.cat([seqs[j][b], step[j][b:b + 1]])
    # the state after the steps is that of each row's whole sequence
    for b in range(B):
        _, fin, _ = rb.gated_recurrence(*(seqs[j][b][None].cpu().numpy() for j in range(3)), lam, C)
        assert np.abs(state[b].double().cpu().numpy() - fin[0]).max() <= 3e-5 * np.abs(fin).max()
    assert mb.device_status() == 0
