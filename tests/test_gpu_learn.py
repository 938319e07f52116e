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
