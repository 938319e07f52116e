"""The learner's operators (alphazero_amd.learn) against plain implementations in 64 bits.

Tolerances.  A result is compared with the 64-bit value of the same (already rounded) inputs:
  fp32 results        sums of n terms in 32 bits: |error| <= n 2^-24 sum |terms| at the very worst; partial sums stay near
                      sqrt(n) of that, 64 * 2^-24 of the sum of magnitudes is allowed
  16-bit results      one rounding of the result (eps / 2 of its value) on top of one rounding of dz for d_features (eps / 2 of
                      the sum of magnitudes |w| |dz|): eps / 2 (|value| + sum of magnitudes) and the fp32 part
  16-bit dz in d_weight   dz enters as hi + lo: 2 (eps / 2)^2 of the sum of magnitudes, at most 2^-16 (bfloat16)
Exponentials: exp(z - lse) with fp32 z: |z - lse| 2^-23 relative, plus the error of z itself, 2^-24 (C + 2) of sum |w h|.
"""
import math

import numpy as np
import pytest
import torch

from alphazero_amd import capi, learn

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
F24 = 2.0 ** -24


def _rows(B, N, C, O, dtype, layout="nchw", sparse=False, legal=0.0, seed=0, cap=None, empty=()):
    g = torch.Generator().manual_seed(seed)
    A = O * N * N
    x = torch.randn(B, C, N, N, generator=g).relu().to(DT[dtype])
    w = (torch.randn(O, C, generator=g) * 2 / math.sqrt(C)).to(DT[dtype])
    b = (torch.randn(O, generator=g) * 0.3).to(DT[dtype])
    ok = torch.rand(B, A, generator=g) < legal if legal else None
    if sparse:
        cap = cap or min(A, 17)
        counts = torch.randint(0, cap + 1, (B,), generator=g, dtype=torch.int32)
        acts = torch.randint(0, A, (B, cap), generator=g, dtype=torch.int32)
        probs = torch.rand(B, cap, generator=g)
        probs = probs / probs.sum(1, keepdim=True).clamp_min(1e-9)
        for r in empty:
            counts[r] = 0
        t = torch.zeros(B, A, dtype=torch.float64)
        for r in range(B):
            for e in range(int(counts[r])):
                t[r, acts[r, e]] += float(probs[r, e])
                if ok is not None:
                    ok[r, acts[r, e]] = True
        tgt = (counts, acts, probs)
    else:
        t = torch.rand(B, A, generator=g) ** 4
        if ok is not None:
            t = t * ok
        t = (t / t.sum(1, keepdim=True).clamp_min(1e-9) * 0.97).float()
        for r in empty:
            t[r] = 0
        tgt = t.view(B, O, N, N).clone()
        t = t.double()
    words = None
    if ok is not None:
        bits = (ok.view(B, O * N, N).long() << torch.arange(N)).sum(2)
        words = torch.where(bits >= 2 ** 31, bits - 2 ** 32, bits).to(torch.int32)
    return dict(x=x, w=w, b=b, t=t, ok=ok, tgt=tgt, words=words, B=B, N=N, C=C, O=O, dtype=dtype, layout=layout)


def _cuda(p):
    mv = lambda v: None if v is None else tuple(q.cuda() for q in v) if isinstance(v, tuple) else v.cuda()     # noqa: E731
    x = p["x"].cuda()
    if p["layout"] == "nhwc":
        x = x.contiguous(memory_format=torch.channels_last)
    return x, mv(p["w"]), mv(p["b"]), mv(p["tgt"]), mv(p["words"])


def _exact(p, r):
    """(loss, dx, dw, db, magnitudes) in 64 bits; r: row scales [B]"""
    B, N, C, O = p["B"], p["N"], p["C"], p["O"]
    S, A = N * N, O * N * N
    h = p["x"].double().reshape(B, C, S)
    w, b = p["w"].double(), p["b"].double()
    z = torch.einsum("oc,bcs->bos", w, h) + b[None, :, None]
    zmag = torch.einsum("oc,bcs->bos", w.abs(), h.abs()) + b.abs()[None, :, None]
    z = z.reshape(B, A)
    ok = p["ok"] if p["ok"] is not None else torch.ones(B, A, dtype=torch.bool)
    zm = z.masked_fill(~ok, -math.inf)
    t = p["t"]
    lse = torch.logsumexp(zm, 1, keepdim=True)
    loss = torch.where(t != 0, t * (lse - zm), 0.0).sum(1)
    bad = ((t != 0) & ~ok).any(1)
    loss[bad] = math.inf
    T = t.sum(1, keepdim=True)
    prob = torch.where(ok, torch.exp(zm - torch.where(torch.isinf(lse), 0.0, lse)), 0.0)
    dz = torch.where(ok, (prob * T - t), 0.0) * r[:, None]
    # error of a dz: its probability's relative error (logit error twice, once through lse) and the subtraction
    zerr = (C + 4) * F24 * zmag.reshape(B, A).amax(1, keepdim=True) + 4 * F24 * (zm.clamp_min(-1e30) - torch.where(torch.isinf(lse), 0.0, lse)).abs()
    dzerr = (prob * T.abs() * (2 * zerr + 8 * F24) + 2 * F24 * (prob * T + t).abs()) * r[:, None].abs()
    dzerr = torch.where(ok, dzerr, 0.0)
    q = dz.view(B, O, S)
    dx = torch.einsum("oc,bos->bcs", w, q).view(B, C, N, N)
    dw = torch.einsum("bos,bcs->oc", q, h)
    db = q.sum((0, 2))
    mag = dict(z=zerr.amax(1), dx=torch.einsum("oc,bos->bcs", w.abs(), q.abs()).view(B, C, N, N), dw=torch.einsum("bos,bcs->oc", q.abs(), h.abs()),
               db=q.abs().sum((0, 2)), dxe=torch.einsum("oc,bos->bcs", w.abs(), dzerr.view(B, O, S)).view(B, C, N, N),
               dwe=torch.einsum("bos,bcs->oc", dzerr.view(B, O, S), h.abs()), dbe=dzerr.view(B, O, S).sum((0, 2)), T=t.abs().sum(1))
    return loss, dx, dw, db, mag


def _check(p, got, r):
    loss, dx, dw, db = [v.cpu() for v in got]
    eloss, edx, edw, edb, m = _exact(p, r)
    half = torch.finfo(DT[p["dtype"]]).eps / 2
    fin = torch.isfinite(eloss)
    assert torch.equal(torch.isfinite(loss), fin)
    tol = m["T"] * (2 * m["z"] + 64 * F24) + 64 * F24 * eloss.abs()
    assert ((loss.double() - eloss)[fin].abs() <= tol[fin]).all(), (loss.double() - eloss)[fin].abs().max()
    sixteen = p["dtype"] != "f32"
    assert dx.dtype == DT[p["dtype"]] and dx.shape == p["x"].shape
    # (fp16's smallest step is 2^-24: a rounding is at least half of it)
    tiny = 2.0 ** -25 if p["dtype"] == "f16" else 0.0
    tol = m["dxe"] + 64 * F24 * m["dx"] + (half * (edx.abs() + m["dx"]) if sixteen else F24 * edx.abs()) + tiny
    assert ((dx.double() - edx).abs() <= tol).all(), ((dx.double() - edx).abs() - tol).max()
    tol = m["dwe"] + 64 * F24 * m["dw"] + (2 * half * half * m["dw"] if sixteen else 0.0) + F24 * edw.abs()
    assert ((dw.double() - edw).abs() <= tol).all(), ((dw.double() - edw).abs() / tol).max()
    if p["O"] == 1 and bool(fin.all()):
        assert (db == 0).all()
    else:
        tol = m["dbe"] + 64 * F24 * m["db"]
        assert ((db.double() - edb).abs() <= tol).all(), ((db.double() - edb).abs() / tol).max()


CASES = [
    # B, N, C, O, sparse, legal
    (1, 1, 1, 1, False, 0.0), (1, 3, 16, 1, False, 0.0), (5, 3, 17, 2, True, 0.0), (3, 15, 128, 1, False, 0.0),
    (2, 20, 128, 91, True, 0.02), (9, 9, 100, 3, False, 0.5), (4, 8, 129, 17, True, 0.3), (2, 5, 256, 128, False, 0.2),
    (3, 7, 250, 33, True, 0.0), (70, 2, 40, 65, False, 0.6), (200, 1, 31, 7, True, 0.0), (1, 32, 64, 5, True, 0.4), (2, 19, 200, 100, True, 0.05),
]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["nchw", "nhwc"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "b%d-n%d-c%d-o%d%s%s" % (c[0], c[1], c[2], c[3], "-sparse" if c[4] else "", "-legal" if c[5] else ""))
def test_loss_and_gradients_match_the_formula(case, layout, dtype):
    B, N, C, O, sparse, legal = case
    p = _rows(B, N, C, O, dtype, layout, sparse, legal, seed=B * 1000 + N * 31 + C, empty=(0,) if B > 1 else ())
    x, w, b, tgt, words = _cuda(p)
    r = torch.linspace(0.5, -1.5, B, dtype=torch.float64) if B > 1 else torch.ones(1, dtype=torch.float64)
    r = r.float().double()
    got = learn.policy_loss_grad(x, w, b, tgt, row_scale=r.float().cuda(), legal=words)
    assert got[1].stride() == x.stride()
    _check(p, got, r)
    alone = learn.policy_loss(x, w, b, tgt, legal=words)
    assert torch.equal(alone, got[0])


def _matrix_exact(u, steps=5, coef=learn.NEWTON_SCHULZ, eps=1e-7):
    a, b, c = [float(np.float32(v)) for v in coef]
    out = []
    for m in u.double():
        q = m.t() if m.shape[0] > m.shape[1] else m
        q = q / (torch.linalg.vector_norm(q) + float(np.float32(eps)))
        for _ in range(steps):
            s = q @ q.t()
            q = a * q + (b * s + c * (s @ s)) @ q
        out.append(q.t() if m.shape[0] > m.shape[1] else q)
    return torch.stack(out)


MATS = [(1, 1, 1), (1, 1, 7), (2, 9, 1), (3, 27, 128), (2, 128, 27), (1, 64, 225), (2, 65, 64), (1, 128, 1152), (2, 200, 136), (1, 129, 513), (5, 3, 900), (1, 256, 256)]


def _mats(n, R, K, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = max(1, min(R, K) // 6)
    u = torch.randn(n, R, r, generator=g) @ torch.randn(n, r, K, generator=g) + 0.5 * torch.randn(n, R, K, generator=g)
    return (u * 1e-3).to(DT[dtype])


# Error of the orthogonalised update, relative to its largest singular value (<= 1.3): A's arithmetic holds 2^-22 of A's
# largest eigenvalue (pairs of fp16; products of pairs drop lo * lo, 2^-22); a stage of m steps carries an absolute error
# of A on to a relative one of Q of at most 1.4 a^2 (a^2)^(m - 2) times it for the smallest singular values, and every
# step adds its own: under 2^-22 * 1.4 * 2 * 11.9^(m - 1) = 1e-4 (m = 3), 1.3e-2 (m = 5) in the direction of a vanishing
# singular value, and 2^-22 times some tens where the value is not small.  The inputs here have no vanishing ones (noise of
# half the strong part's scale): 3e-5 absolute of the matrix's norm, and half a step of the output type.
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", MATS, ids=lambda s: "%dx%dx%d" % s)
def test_orthogonalize_matches_the_iteration(shape, dtype):
    n, R, K = shape
    u = _mats(n, R, K, dtype, seed=R * 7 + K)
    want = _matrix_exact(u)
    got = learn.orthogonalize(u.cuda()).cpu()
    assert got.dtype == u.dtype and got.shape == u.shape
    half = 0.0 if dtype == "f32" else torch.finfo(DT[dtype]).eps / 2
    err = (got.double() - want).abs()
    for i in range(n):
        nrm = torch.linalg.matrix_norm(got[i].double() - want[i], 2)
        lim = 3e-5 * 1.3 + half * torch.linalg.vector_norm(want[i])
        assert nrm <= lim, (i, float(nrm), float(lim))
    assert torch.isfinite(err).all()


@pytest.mark.parametrize("gdtype", ["f32", "bf16"])
@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shape", [(1, 128, 27), (3, 64, 225), (2, 160, 100)], ids=lambda s: "%dx%dx%d" % s)
def test_optimiser_step_matches_the_formula(shape, nesterov, gdtype):
    n, R, K = shape
    grad, mom = _mats(n, R, K, gdtype, 1), _mats(n, R, K, "f32", 2)
    w = torch.randn(n, R, K, generator=torch.Generator().manual_seed(3))
    lr, beta, wd, scale = 0.03, 0.9, 0.1, 1.7
    f = lambda v: float(np.float32(v))                                                                        # noqa: E731
    m2 = f(beta) * mom.double() + grad.double()
    u = grad.double() + f(beta) * m2 if nesterov else m2
    want = w.double() * (1 - f(lr) * f(wd)) - f(lr) * f(scale) * _matrix_exact(u)
    wg, mg = w.cuda(), mom.cuda()
    rw, rm = learn.muon_step(wg, mg, grad.cuda(), lr=lr, beta=beta, nesterov=nesterov, weight_decay=wd, scale=scale)
    assert rw is wg and rm is mg
    assert ((mg.cpu().double() - m2).abs() <= 3 * F24 * (mom.abs() + grad.abs()).double()).all()
    # the orthogonalised part: 3e-5 of its norm as above, times lr * scale; the weight: two roundings
    tol = lr * scale * 4e-5 + 4 * F24 * w.abs().double()
    assert ((wg.cpu().double() - want).abs() <= tol).all(), ((wg.cpu().double() - want).abs() - tol).max()
    w2, m3 = torch.empty_like(wg), torch.empty_like(mg)
    learn.muon_step(w.cuda(), mom.cuda(), grad.cuda(), lr=lr, beta=beta, nesterov=nesterov, weight_decay=wd, scale=scale, weight_out=w2, momentum_out=m3)
    assert torch.equal(w2, wg) and torch.equal(m3, mg)                                                        # in place and apart: the same bits


# ---- the calls around the products: edges, streams, graphs, sizes -----------------------------------------------------------

def _grad(p, scale=1.0, **kw):
    x, w, b, tgt, words = _cuda(p)
    return learn.policy_loss_grad(x, w, b, kw.get("tgt", tgt), row_scale=scale, legal=kw.get("words", words))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("N", [3, 9])
def test_boards_without_targets_or_without_allowed_actions(N, dtype):
    """No target: loss 0, no gradient.  No allowed action and no target: the same.  A target on an action that is not
    allowed: loss inf, the gradient still finite and 0 at that entry."""
    B, C, O = 6, 32, 3
    p = _rows(B, N, C, O, dtype, legal=0.5, seed=5, empty=(1,))
    p["ok"][2] = False                                    # nothing allowed, targets there: inf
    p["ok"][3] = False
    p["t"][3] = 0                                         # nothing allowed, no target
    p["tgt"].view(B, -1)[3] = 0
    p["ok"][4, 7] = False
    p["t"][4, 7] = 0.25                                   # one target outside
    p["tgt"].view(B, -1)[4, 7] = 0.25
    bits = (p["ok"].view(B, O * N, N).long() << torch.arange(N)).sum(2)
    p["words"] = bits.to(torch.int32)
    loss, dx, dw, db = [v.cpu().double() for v in _grad(p)]
    assert loss[1] == 0 and loss[3] == 0 and math.isinf(loss[2]) and math.isinf(loss[4]) and torch.isfinite(loss[[0, 5]]).all()
    assert (dx[[1, 2, 3]] == 0).all()
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
    _check(p, _grad(p), torch.ones(B, dtype=torch.float64))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["nchw", "nhwc"])
def test_what_lies_behind_a_mask_does_not_matter_for_the_loss(layout, dtype):
    """NaN and inf in the features of cells none of whose actions is allowed: the loss and the other cells' feature gradients
    are those of a clean board."""
    B, N, C, O = 3, 8, 64, 2
    p = _rows(B, N, C, O, dtype, layout, legal=0.6, seed=9)
    ok = p["ok"].view(B, O, N, N)
    ok[:, :, 2, 3] = False
    ok[:, :, 7, 7] = False
    p["t"] = (p["t"].view(B, O, N, N) * ok).view(B, -1)
    p["tgt"] = p["t"].float().view(B, O, N, N).contiguous()
    p["words"] = (ok.reshape(B, O * N, N).long() << torch.arange(N)).sum(2).to(torch.int32)
    clean = [v.cpu() for v in _grad(p)]
    p["x"][:, :, 2, 3] = float("nan")
    p["x"][:, :, 7, 7] = float("inf")
    dirty = [v.cpu() for v in _grad(p)]
    assert torch.equal(clean[0], dirty[0])
    keep = torch.ones(N, N, dtype=torch.bool)
    keep[2, 3] = keep[7, 7] = False
    assert torch.equal(clean[1][:, :, keep], dirty[1][:, :, keep]) and (dirty[1][:, :, ~keep] == 0).all()


def test_the_same_action_twice_entries_outside_and_counts_beyond_the_list():
    B, N, C, O = 5, 9, 48, 4
    A = O * N * N
    p = _rows(B, N, C, O, "f32", "nhwc", sparse=True, seed=3, cap=12)
    counts, acts, probs = p["tgt"]
    counts[:] = torch.tensor([12, 12, 0, 99, -4], dtype=torch.int32)
    acts[0, :6] = 17                                      # six times the same
    acts[1, 3] = -1
    acts[1, 4] = A
    acts[1, 5] = 2 ** 31 - 1
    acts[1, 6] = -2 ** 31
    p["t"] = torch.zeros(B, A, dtype=torch.float64)
    for r in range(B):
        for e in range(max(0, min(int(counts[r]), 12))):
            if 0 <= int(acts[r, e]) < A:
                p["t"][r, acts[r, e]] += float(probs[r, e])
    got = _grad(p)
    _check(p, got, torch.ones(B, dtype=torch.float64))
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(got, _grad(p)))


@pytest.mark.parametrize("case", [(2, 32, 256, 128, 1024, "f16"), (2, 32, 128, 128, 1024, "f32"), (1, 20, 128, 91, 5000, "bf16"), (3, 32, 128, 96, 1024, "bf16"),
                                  (40, 2, 16, 5, 30, "f32"), (2, 4, 256, 128, 2048, "f16")], ids=lambda c: "b%d-n%d-c%d-o%d-cap%d-%s" % c)
def test_long_target_lists_and_the_largest_heads(case):
    B, N, C, O, cap, dtype = case
    p = _rows(B, N, C, O, dtype, "nhwc", sparse=True, legal=0.3, seed=cap, cap=min(cap, 5000))
    _check(p, _grad(p), torch.ones(B, dtype=torch.float64))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_tensors_at_odd_addresses(dtype):
    """Views that are aligned to their element type only."""
    B, N, C, O = 3, 7, 64, 5
    p = _rows(B, N, C, O, dtype, "nhwc", seed=1)
    x, w, b, tgt, _ = _cuda(p)

    def shift(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        buf[1:] = t.flatten()
        return buf[1:].view(t.shape)
    xs = shift(x.permute(0, 2, 3, 1).contiguous()).permute(0, 3, 1, 2)
    got = learn.policy_loss_grad(xs, shift(w), shift(b), shift(tgt))
    want = learn.policy_loss_grad(x, w, b, tgt)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    u = _mats(2, 33, 70, dtype).cuda()
    assert torch.equal(learn.orthogonalize(shift(u)), learn.orthogonalize(u))


def test_empty_batches():
    x, w, b = torch.empty(0, 8, 5, 5, device="cuda"), torch.randn(2, 8, device="cuda"), torch.zeros(2, device="cuda")
    t = torch.empty(0, 2, 5, 5, device="cuda")
    assert learn.policy_loss(x, w, b, t).shape == (0,)
    loss, dx, dw, db = learn.policy_loss_grad(x, w, b, t)
    assert loss.shape == (0,) and dx.shape == x.shape and (dw == 0).all() and (db == 0).all()
    assert learn.orthogonalize(torch.empty(0, 4, 6, device="cuda")).shape == (0, 4, 6)


def test_autograd_gives_the_same_gradients_and_checks_its_inputs():
    p = _rows(4, 9, 40, 3, "f32", legal=0.7, seed=8)
    x, w, b, tgt, words = _cuda(p)
    xr, wr, br = x.clone().requires_grad_(), w.view(3, 40, 1, 1).clone().requires_grad_(), b.clone().requires_grad_()
    g = torch.tensor([0.5, -1.0, 2.0, 0.0], device="cuda")
    (learn.policy_loss(xr, wr, br, tgt, legal=words) * g).sum().backward()
    _, dx, dw, db = learn.policy_loss_grad(x, w, b, tgt, row_scale=g, legal=words)
    assert torch.equal(xr.grad, dx) and torch.equal(wr.grad.view(3, 40), dw) and torch.equal(br.grad, db)
    learn.policy_loss(xr, wr, br, tgt, legal=words).mean().backward()        # an expanded gradient
    loss = learn.policy_loss(xr, wr, br, tgt, legal=words)
    with torch.no_grad():
        wr.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.sum().backward()


def test_gradients_against_differences():
    """d/dx and d/dw of the summed loss along random directions, central differences of the 64-bit loss."""
    p = _rows(2, 5, 20, 3, "f32", seed=4)
    _, dx, dw, db = [v.cpu().double() for v in _grad(p)]
    r = torch.ones(2, dtype=torch.float64)
    g = torch.Generator().manual_seed(0)
    for key, d in (("x", dx), ("w", dw), ("b", db)):
        v = torch.randn(p[key].shape, generator=g, dtype=torch.float64)
        base, h, side = p[key], 1e-5, []
        for s in (1, -1):
            q = dict(p)
            q[key] = base.double() + s * h * v
            side.append(float(_exact(q, r)[0].sum()))
        num = (side[0] - side[1]) / (2 * h)
        assert abs(num - float((d * v).sum())) <= 1e-5 * float((d * v).abs().sum()) + 1e-7


def test_another_stream_than_the_default_one():
    p = _rows(32, 15, 128, 1, "bf16", "nhwc", seed=2)
    want = _grad(p)
    x, w, b, tgt, words = _cuda(p)
    u = _mats(3, 100, 300, "f32").cuda()
    o = learn.orthogonalize(u)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        xs = x * 1.0                                      # made on this stream: the call has to be ordered behind it
        got = learn.policy_loss_grad(xs, w, b, tgt)
        o2 = learn.orthogonalize(u * 1.0)
    s.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(want, got)) and torch.equal(o, o2)


def test_two_captured_steps_replayed_between_eager_ones():
    """Forward, gradients and the optimiser step of two heads, each captured into a graph of its own, replayed several times
    with other inputs, eager calls and synchronisations between the replays: every replay against the eager result."""
    ps = [_rows(8, 9, 64, 3, "bf16", "nhwc", sparse=True, seed=s) for s in (1, 2)]
    static, graphs = [], []
    for p in ps:
        x, w, b, tgt, _ = _cuda(p)
        wm, mm = torch.randn(3, 64, device="cuda"), torch.zeros(3, 64, device="cuda")
        st = dict(x=x, w=w, b=b, tgt=tgt, wm=wm, mm=mm)

        def step(st=st):
            st["loss"], st["dx"], st["dw"], st["db"] = learn.policy_loss_grad(st["x"], st["w"], st["b"], st["tgt"], row_scale=1.0 / 8)
            st["wm2"], st["mm2"] = learn.muon_step(st["wm"], st["mm"], st["dw"], lr=0.1, weight_out=torch.empty_like(st["wm"]), momentum_out=torch.empty_like(st["mm"]))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        static.append(st)
        graphs.append(g)
    for rep in range(4):
        for st in static:
            st["x"].copy_((torch.randn(st["x"].shape, device="cuda") + rep).relu())
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for st in static:
            loss, dx, dw, db = learn.policy_loss_grad(st["x"], st["w"], st["b"], st["tgt"], row_scale=1.0 / 8)
            wm, mm = learn.muon_step(st["wm"].clone(), st["mm"].clone(), dw, lr=0.1)
            for a, c in ((loss, st["loss"]), (dx, st["dx"]), (dw, st["dw"]), (db, st["db"]), (wm, st["wm2"]), (mm, st["mm2"])):
                assert torch.equal(a, c)


def test_offsets_beyond_32_bits():
    """More than 2^31 features: the last boards of a large batch come out as alone."""
    B, N, C = 21100, 20, 256
    x = torch.zeros(B, N, N, C, dtype=torch.float16, device="cuda").permute(0, 3, 1, 2)
    assert x.numel() > 2 ** 31
    g = torch.Generator().manual_seed(0)
    tail = torch.randn(3, C, N, N, generator=g).relu().half().cuda().contiguous(memory_format=torch.channels_last)
    x[-3:] = tail
    w, b = (torch.randn(1, C, generator=g) / 8).half().cuda(), torch.zeros(1, dtype=torch.float16, device="cuda")
    t = torch.zeros(B, 1, N, N, device="cuda")
    t[:, 0, 3, 4] = 1.0
    loss, dx, _, _ = learn.policy_loss_grad(x, w, b, t)
    l3, d3, _, _ = learn.policy_loss_grad(tail, w, b, t[-3:].contiguous())
    assert torch.equal(loss[-3:], l3) and torch.equal(dx[-3:], d3)
    assert torch.allclose(loss[:5], torch.full((5,), math.log(400.0), device="cuda"), rtol=1e-6)


def test_weight_blob_in_place():
    """The convolutions of all blocks as strided batches of a flat blob: one call each for conv1 and conv2, everything else in the
    blob left as it was; the result is taken by az_load_weights_dev."""
    from alphazero_amd import synth
    N, Cs = 9, [64] * 4
    blob = torch.from_numpy(synth.make_blob(N, 3, Cs, 5)).cuda()
    before = blob.clone()
    layout, at, off = synth.blob_layout(N, 3, Cs), 0, {}
    for name, shape in layout:
        off[name] = at
        at += int(np.prod(shape))
    stride = off["RBlock_1.conv1.weight"] - off["RBlock_0.conv1.weight"]
    assert stride == off["RBlock_2.conv2.weight"] - off["RBlock_1.conv2.weight"]
    grad, mom = torch.randn(at, generator=torch.Generator().manual_seed(1)).cuda() * 1e-3, torch.zeros(at, device="cuda")
    touched = torch.zeros(at, dtype=torch.bool)
    for conv in ("conv1", "conv2"):
        o = off["RBlock_0.%s.weight" % conv]
        view = lambda t: t.as_strided((3, 64, 64, 3, 3), (stride, 64 * 9, 9, 3, 1), o)                          # noqa: E731
        want_w, want_m = learn.muon_step(view(blob).contiguous(), view(mom).contiguous(), view(grad).contiguous(), lr=0.02)
        learn.muon_step(view(blob), view(mom), view(grad), lr=0.02)
        assert torch.equal(view(blob), want_w) and torch.equal(view(mom), want_m)
        for i in range(3):
            touched[o + i * stride:o + i * stride + 64 * 64 * 9] = True
    same = (blob == before).cpu()
    assert same[~touched].all() and not same[touched].all() and (mom.cpu()[~touched] == 0).all()
    eng = capi.Engine(N, 5, 2, Cs=Cs)
    eng.load_weights_dev(blob.data_ptr(), blob.numel())
    eng.sync()
    eng.close()


def test_zero_and_nonfinite_updates():
    z = torch.zeros(2, 20, 50, device="cuda")
    assert (learn.orthogonalize(z) == 0).all()
    z[1, 3, 4] = float("nan")
    z[0, 0, 0] = 2.0
    out = learn.orthogonalize(z)
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1]).all()
    for s in (1e-30, 1e30):                               # far from 1: the norm is taken in 64 bits
        u = _mats(1, 40, 90, "f32", 5)
        a, b = learn.orthogonalize((u * s).cuda(), eps=0.0), learn.orthogonalize(u.cuda(), eps=0.0)
        assert torch.allclose(a, b, atol=1e-5)


@pytest.mark.parametrize("steps", [0, 1, 2, 4, 7, 12])
@pytest.mark.parametrize("shape", [(2, 50, 130), (1, 140, 90), (1, 300, 200)], ids=lambda s: "%dx%dx%d" % s)
def test_any_number_of_steps(shape, steps):
    n, R, K = shape
    u = _mats(n, R, K, "f32", 11)
    coef = (1.875, -1.25, 0.375)                          # converges: every number of steps stays bounded
    want = _matrix_exact(u, steps, coef)
    got = learn.orthogonalize(u.cuda(), steps=steps, coefficients=coef).cpu().double()
    for i in range(n):
        # as above: 3e-5 of the norm for up to three steps after the last formation of X, and what the earlier ones left
        assert torch.linalg.matrix_norm(got[i] - want[i], 2) <= 4e-5 * max(1.0, float(torch.linalg.matrix_norm(want[i], 2)))


@pytest.mark.parametrize("shape", [(260, 40, 500), (300, 600, 64), (90, 200, 200), (3, 65, 64), (2, 64, 481)], ids=lambda s: "%dx%dx%d" % s)
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_matrices(shape, dtype):
    """Batches that fill the chip with large tiles, shapes at the borders between the kernels; a few matrices against 64 bits."""
    n, R, K = shape
    u = _mats(n, R, K, dtype, 21)
    got = learn.orthogonalize(u.cuda())
    half = 0.0 if dtype == "f32" else torch.finfo(DT[dtype]).eps / 2
    for i in sorted({0, 1, n // 2, n - 1}):
        want = _matrix_exact(u[i:i + 1])[0]
        err = got[i].cpu().double() - want
        # as above, and the rounding of the result: each element by half a step
        assert torch.linalg.matrix_norm(err, 2) <= 4e-5 * max(1.0, float(torch.linalg.matrix_norm(want, 2))) + half * float(want.norm())


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["nchw", "nhwc"])
@pytest.mark.parametrize("case", [(90, 15, 128, 1, False, 0.0), (150, 9, 100, 3, False, 0.5), (300, 7, 48, 17, True, 0.3), (2000, 3, 40, 65, True, 0.0),
                                  (2200, 3, 33, 2, False, 0.6), (40, 20, 128, 91, True, 0.02), (38, 20, 64, 40, False, 0.0), (5000, 1, 31, 7, True, 0.0), (17, 32, 96, 33, True, 0.2)],
                         ids=lambda c: "b%d-n%d-c%d-o%d%s%s" % (c[0], c[1], c[2], c[3], "-sparse" if c[4] else "", "-legal" if c[5] else ""))
def test_gradients_of_more_than_a_step_a_workgroup(case, layout, dtype):
    B, N, C, O, sparse, legal = case
    p = _rows(B, N, C, O, dtype, layout, sparse, legal, seed=B + N, empty=(0, B - 1))
    r = torch.linspace(0.5, -1.5, B, dtype=torch.float64)
    r = r.float()
    _check(p, _grad(p, r.cuda()), r.double())


def test_gradients_through_autograd_are_refused_under_capture():
    p = _rows(2, 5, 16, 1, "f32", seed=1)
    x, w, b, tgt, _ = _cuda(p)
    xr = x.clone().requires_grad_()
    policy = learn.policy_loss(xr, w, b, tgt)             # an eager graph of the same leaf lives
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        with pytest.raises(capi.AzError, match="policy_loss_grad"):
            learn.policy_loss(xr, w, b, tgt)
        out = learn.policy_loss(x, w, b, tgt)             # without gradients it can be captured
    for _ in range(3):
        x.copy_(torch.randn_like(x).relu())
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, learn.policy_loss(x, w, b, tgt))
    policy.sum().backward()
    assert torch.isfinite(xr.grad).all()


def test_matrices_that_are_not_contiguous_are_refused():
    u = torch.randn(4, 12, 20, device="cuda")
    for bad in (u.transpose(1, 2), u[:, :, ::2], u[:, ::2], torch.randn(2, 8, 3, 3, 4, device="cuda").permute(0, 1, 4, 2, 3)):
        with pytest.raises(capi.AzError, match="contiguous"):
            learn.orthogonalize(bad)
    for good in (u[::2], u[1:2, :, :], u[:, :1], u.view(4, 12, 5, 4)[0], u[0], u.view(4, 12, 5, 2, 2)[::3], u[:, 3:7]):
        assert torch.equal(learn.orthogonalize(good), learn.orthogonalize(good.contiguous()))


@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
@pytest.mark.parametrize("N", [3, 9, 20])
def test_a_nan_target_counts_for_the_gradients_only(N, sparse):
    B, C, O = 6, 24, 5
    p = _rows(B, N, C, O, "f32", sparse=sparse, seed=N, cap=9)
    if sparse:
        p["tgt"][0][2] = 9
        p["tgt"][2][2] = 0.1
        p["tgt"][1][2] = torch.arange(9, dtype=torch.int32)
        p["tgt"][2][2, 4] = float("nan")
        p["t"][2] = 0
        p["t"][2, :9] = 0.1
        p["t"][2, 4] = 0
        p["t"] = p["t"].float().double()
    else:
        p["tgt"].view(B, -1)[2, 4] = float("nan")
        p["t"][2, 4] = 0
    loss, dx, dw, db = _grad(p)
    want = _exact(p, torch.ones(B, dtype=torch.float64))[0]
    assert torch.allclose(loss.cpu().double(), want, rtol=1e-5, atol=1e-5)      # (sums of at most 2000 fp32 terms: 2^-13 of them at worst)
    keep = torch.arange(B) != 2
    assert torch.isnan(dx[2]).all() and torch.isfinite(dx.cpu()[keep]).all()
    assert torch.isnan(dw).all() and torch.isnan(db).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("case", [(5, 3, 20, 1), (200, 9, 64, 2), (3, 20, 200, 91), (40, 20, 128, 91)], ids=lambda c: "b%d-n%d-c%d-o%d" % c)
def test_a_board_with_one_allowed_action_has_exactly_no_loss(case, dtype):
    B, N, C, O = case
    p = _rows(B, N, C, O, dtype, "nhwc", legal=0.5, seed=3)
    A = O * N * N
    at = torch.randint(0, A, (B,), generator=torch.Generator().manual_seed(1))
    ok = torch.zeros(B, A, dtype=torch.bool)
    ok[torch.arange(B), at] = True
    p["tgt"] = ok.view(B, O, N, N).float() * torch.linspace(0.3, 1.0, B).view(B, 1, 1, 1)
    p["words"] = (ok.view(B, O * N, N).long() << torch.arange(N)).sum(2).to(torch.int32)
    loss, dx, dw, db = _grad(p, 1.0 / 3)
    assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all() and (db == 0).all()
