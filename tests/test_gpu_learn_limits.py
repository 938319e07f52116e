"""The learner's operators at the limits of their number types, against 64 bits: what 16-bit features and updates may cost,
and values that overflow a narrower step on the way.

Tolerances, beside those that test_gpu_learn.py derives for 32-bit sums (F24 = 2^-24, half = half a step of the type):
  d_features, 16 bits  one rounding of the result, half of its value.  dz enters its product as hi + lo, so a term is off by
                       half^2 of itself at most; fp16's lo has steps of 2^-24 where the largest dz is put at 2^9 or more:
                       2^-34 of the largest |r T|.
"""
import math

import pytest
import torch

from alphazero_amd import learn
from test_gpu_learn import DT, F24, _check, _cuda, _exact, _matrix_exact, _rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("layout", ["nchw", "nhwc"])
@pytest.mark.parametrize("case", [(3, 9, 100, 1, False, 0.0), (4, 8, 129, 17, True, 0.3), (2, 9, 256, 128, False, 0.0), (1, 20, 128, 91, True, 0.0), (70, 2, 40, 65, False, 0.6),
                                  (90, 15, 128, 1, False, 0.0), (150, 9, 100, 3, False, 0.5), (2000, 3, 40, 30, True, 0.0), (70, 15, 60, 40, False, 0.0), (40, 20, 128, 91, True, 0.0)],
                         ids=lambda c: "b%d-n%d-c%d-o%d%s%s" % (c[0], c[1], c[2], c[3], "-sparse" if c[4] else "", "-legal" if c[5] else ""))
def test_gradient_of_16_bit_features_is_off_by_its_own_rounding(case, layout, dtype):
    B, N, C, O, sparse, legal = case
    p = _rows(B, N, C, O, dtype, layout, sparse, legal, seed=B + C)
    r = torch.linspace(0.5, -1.5, B).double() if B > 1 else torch.ones(1, dtype=torch.float64)
    x, w, b, tgt, words = _cuda(p)
    dx = learn.policy_loss_grad(x, w, b, tgt, row_scale=r.float().cuda(), legal=words)[1].cpu().double()
    _, want, _, _, m = _exact(p, r.float().double())
    half = torch.finfo(DT[dtype]).eps / 2
    before = m["dxe"] + (64 * F24 + half * half) * m["dx"]
    if dtype == "f16":
        before = before + 2.0 ** -34 * float((r.abs() * m["T"]).max()) * p["w"].double().abs().sum(0).view(1, C, 1, 1)
    tol = half * want.abs() + (1 + half) * before + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert ((dx - want).abs() <= tol).all(), ((dx - want).abs() / tol).max()


# d_weight where no error can average out: channel c is 1 in one cell of board c alone, so d_weight[o, c] is one dz, r T p.  The
# weights are 0, so logits are the biases and p is known exactly.  Roundings, in F24 of the value: the sum of exponentials, at most
# 62 additions one after another on the way (two tiles of 96 planes in a lane, 64 lanes, 8 waves); exp2 and its argument, 7 in
# the sum and 7 in dz; products and the division, 6; parts of dz: the third one leaves 1 (bfloat16), two of fp16 4.  100 in all.
# Two parts of bfloat16 would leave up to 128.  (fp16: steps of 2^-34 of the largest r T besides.)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
@pytest.mark.parametrize("N,O", [(5, 3), (5, 91), (5, 120), (15, 2), (15, 17), (15, 40), (15, 91), (15, 128)])
def test_gradient_of_the_weight_holds_32_bits(N, O, sparse, dtype):
    B = C = 128
    S = N * N
    g = torch.Generator().manual_seed(N + O)
    at = torch.randint(0, S - 1, (B,), generator=g)
    x = torch.zeros(B, C, S, dtype=DT[dtype])
    x[torch.arange(B), torch.arange(B), at] = 1
    w, b = torch.zeros(O, C, dtype=DT[dtype]), (torch.rand(O, generator=g) * 1.5).to(DT[dtype])
    T, r = torch.rand(B, generator=g) + 0.5, torch.rand(B, generator=g) + 0.5
    if sparse:
        tgt = (torch.ones(B, dtype=torch.int32), torch.full((B, 3), S - 1, dtype=torch.int32), T.view(B, 1).repeat(1, 3))     # (plane 0, the last cell)
    else:
        tgt = torch.zeros(B, O, S)
        tgt[:, 0, S - 1] = T
        tgt = tgt.view(B, O, N, N)
    tgt = tuple(t.cuda() for t in tgt) if sparse else tgt.cuda()
    dw = learn.policy_loss_grad(x.view(B, C, N, N).cuda(), w.cuda(), b.cuda(), tgt, row_scale=r.cuda())[2].cpu().double()
    p = torch.softmax(b.double(), 0) / S
    want = p.view(O, 1) * (r.double() * T.double()).view(1, C)
    tol = 100 * F24 * want + (2.0 ** -34 * float((r * T).max()) if dtype == "f16" else 0.0)
    assert ((dw - want).abs() <= tol).all(), (((dw - want).abs() / want).max() / F24, dw.shape)


def _values(n, R, K, s, seed):
    """n matrices R x K with the singular values s"""
    g = torch.Generator().manual_seed(seed)
    r = min(R, K)
    left, right = (torch.linalg.qr(torch.randn(n, m, r, generator=g, dtype=torch.float64))[0] for m in (R, K))
    return (left * s) @ right.transpose(1, 2)


# One direction that is most of the norm, the others far below: what A = X X^T holds of them it holds against the largest.
# Three steps on one A leave up to 1e-4 of a value's own size, and two up to 1e-5 (test_gpu_learn.py); a step behind them
# magnifies a relative error by |x f'(x) / f(x)|.  An element is off by that before it is rounded, and then by half a step of
# the type.
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rest", [1e-3, 1e-4])
@pytest.mark.parametrize("shape", [(2, 128, 1152), (1, 256, 600), (1, 600, 200), (2, 100, 300), (1, 64, 700)], ids=lambda s: "%dx%dx%d" % s)
def test_orthogonalize_16_bits_with_one_strong_direction(shape, rest, dtype):
    r = min(shape[1:])
    s = torch.full((r,), rest, dtype=torch.float64)
    s[0] = 1
    u = (_values(*shape, s, seed=r) * 1e-2).to(DT[dtype])
    want, got = _matrix_exact(u), learn.orthogonalize(u.cuda()).cpu().double()
    x = torch.linalg.svdvals(u.double())
    x, magnified = x / torch.linalg.vector_norm(x, dim=1, keepdim=True), 1.0
    a, b, c = learn.NEWTON_SCHULZ
    for step in range(5):
        f = a + b * x ** 2 + c * x ** 4
        if step >= 3:
            magnified = magnified * ((a + 3 * b * x ** 2 + 5 * c * x ** 4) / f).abs().clamp_min(1.0)
        x = (x * f).abs()
    tol = torch.linalg.vector_norm(x * (1e-4 * magnified + 1e-5), dim=1)
    over = ((got - want).abs() - torch.finfo(DT[dtype]).eps / 2 * want.abs() - (2.0 ** -25 if dtype == "f16" else 0.0)).clamp_min(0)
    assert (torch.linalg.matrix_norm(over) <= tol).all(), torch.linalg.matrix_norm(over) / tol


@pytest.mark.parametrize("gdtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(3, 64, 225), (2, 100, 300), (2, 128, 1152), (1, 600, 200), (1, 256, 600)], ids=lambda s: "%dx%dx%d" % s)
def test_optimiser_step_orthogonalises_as_exactly_as_orthogonalize(shape, gdtype):
    """Weights 0, no momentum, lr 1: minus what orthogonalize makes of the gradient in fp32, bit for bit."""
    s = torch.logspace(0, -3, min(shape[1:]), dtype=torch.float64)
    grad = (_values(*shape, s, seed=3) * 1e-2).to(DT[gdtype]).cuda()
    w, _ = learn.muon_step(torch.zeros(shape, device="cuda"), torch.zeros(shape, device="cuda"), grad, lr=1.0, beta=0.0)
    assert torch.equal(-w, learn.orthogonalize(grad.float()))


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
@pytest.mark.parametrize("B,N,O", [(3, 9, 1), (5, 5, 7), (90, 15, 1), (90, 15, 3), (150, 9, 17), (2000, 5, 2), (40, 20, 91)])
def test_logits_far_below_the_bias(B, N, O, sparse, dtype):
    """Features of one sign against weights of the other: every logit is 128 below the bias, which is what a row beyond the board's last
    would have.  All values are exact in the types: p = 1 / (S O)."""
    C, S = 64, N * N
    x = torch.ones(B, C, N, N, dtype=DT[dtype])
    w, b = torch.full((O, C), -2.0, dtype=DT[dtype]), torch.zeros(O, dtype=DT[dtype])
    if sparse:
        tgt = (torch.ones(B, dtype=torch.int32), torch.full((B, 2), N + 1, dtype=torch.int32), torch.ones(B, 2))
    else:
        tgt = torch.zeros(B, O, N, N)
        tgt[:, 0, 1, 1] = 1.0
    p = dict(x=x, w=w, b=b, t=torch.zeros(B, O * S, dtype=torch.float64), ok=None, tgt=tgt, words=None, B=B, N=N, C=C, O=O, dtype=dtype, layout="nhwc")
    p["t"][:, N + 1] = 1.0
    xg, wg, bg, tg, _ = _cuda(p)
    _check(p, learn.policy_loss_grad(xg, wg, bg, tg), torch.ones(B, dtype=torch.float64))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("B,O", [(2, 3), (90, 3), (90, 17), (90, 91)])
def test_infinite_feature_whose_logits_are_all_minus_infinity(B, O, dtype):
    """That cell's actions have probability 0 and the gradient of its features is 0, as anywhere (planes are padded inside)."""
    N, C = 15, 64
    x = torch.rand(B, C, N, N, generator=torch.Generator().manual_seed(1)).to(DT[dtype])
    x[1, 5, 3, 3] = math.inf
    w, b = torch.full((O, C), -0.125, dtype=DT[dtype]), torch.zeros(O, dtype=DT[dtype])
    tgt = torch.zeros(B, O, N, N)
    tgt[:, 0, 1, 1] = 1.0
    loss, dx, _, db = [v.cpu() for v in learn.policy_loss_grad(x.cuda(), w.cuda(), b.cuda(), tgt.cuda())]
    assert torch.isfinite(loss).all() and torch.isfinite(dx).all() and torch.isfinite(db).all()
    assert (dx[1, :, 3, 3] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
@pytest.mark.parametrize("B,N,O", [(2, 15, 1), (6, 4, 3), (90, 15, 1), (2000, 4, 3), (90, 15, 17)])
def test_targets_of_both_signs(B, N, O, sparse, dtype):
    """Targets that nearly cancel: no sum of theirs bounds a gradient's terms, their magnitudes do."""
    C = 48
    p = _rows(B, N, C, O, dtype, "nhwc", sparse, seed=B + O, cap=8)
    g = torch.Generator().manual_seed(1)
    if sparse:
        counts, acts, probs = p["tgt"]
        counts[:] = 8
        acts[:] = torch.stack([torch.randperm(O * N * N, generator=g)[:8] for _ in range(B)]).int()
        probs[:, ::2] = 1.0
        probs[:, 1::2] = -0.999
        p["t"] = torch.zeros(B, O * N * N, dtype=torch.float64).scatter_(1, acts.long(), probs.double())
    else:
        t = torch.randn(B, O * N * N, generator=g)
        t[:, 0] -= t.sum(1) - 1e-3
        p["t"], p["tgt"] = t.double(), t.view(B, O, N, N).clone()
    x, w, b, tgt, _ = _cuda(p)
    loss, dx, dw, db = [v.cpu().double() for v in learn.policy_loss_grad(x, w, b, tgt, row_scale=1.0 / 32)]
    r = torch.full((B,), 1.0 / 32, dtype=torch.float64)
    eloss, edx, edw, edb, m = _exact(p, r)
    # the sum of the targets in 32 bits: 64 F24 of their magnitudes, which reaches the loss with lse and a dz with its probability
    S, half = N * N, torch.finfo(DT[dtype]).eps / 2 if dtype != "f32" else F24
    h, wd = p["x"].double().reshape(B, C, S), p["w"].double()
    z = (torch.matmul(wd, h) + p["b"].double().view(1, O, 1)).reshape(B, O * S)
    tol = m["T"] * (2 * m["z"] + 64 * F24 * (torch.logsumexp(z, 1).abs() + z.abs().amax(1)))
    assert ((loss - eloss).abs() <= tol).all(), ((loss - eloss).abs() / tol).max()
    e = ((64 * F24 * m["T"].view(B, 1) * torch.softmax(z, 1) + 4 * F24 * p["t"].abs()) / 32).view(B, O, S)
    if dtype == "f16":
        e = e + 2.0 ** -34 / 32 * float(m["T"].max())
    before = m["dxe"] + torch.matmul(wd.abs().t(), e).view(B, C, N, N) + (64 * F24 + half * half) * m["dx"]
    tol = half * edx.abs() + (1 + half) * before + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert ((dx - edx).abs() <= tol).all(), ((dx - edx).abs() / tol).max()
    tol = m["dwe"] + torch.matmul(e, h.transpose(1, 2)).sum(0) + (64 * F24 + half * half) * m["dw"]
    assert ((dw - edw).abs() <= tol).all(), ((dw - edw).abs() / tol).max()
    tol = m["dbe"] + e.sum((0, 2)) + 64 * F24 * m["db"]
    assert (db == 0).all() if O == 1 else ((db - edb).abs() <= tol).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
@pytest.mark.parametrize("N", [3, 9])
def test_any_target_outside_the_allowed_actions_makes_the_loss_infinite(N, sparse, dtype):
    """Positive, negative, one of each; board 0 has none, board 4 negative ones on allowed actions only."""
    B, C, O = 5, 32, 2
    S = N * N
    p = _rows(B, N, C, O, dtype, legal=0.5, seed=N)
    ok = torch.ones(B, O * S, dtype=torch.bool)
    ok[:, 4] = ok[:, S + 5] = False
    acts = torch.tensor([0, 4, S + 5]).repeat(B, 1)
    vals = torch.tensor([[0.5, 0.0, 0.0], [0.5, 0.25, 0.0], [0.5, 0.0, -0.25], [0.5, 0.25, -0.25], [0.5, 0.0, 0.0]])
    acts[4], vals[4] = torch.tensor([0, 1, S]), torch.tensor([0.5, -0.25, -0.125])
    t = torch.zeros(B, O * S).scatter_(1, acts, vals)
    tgt = (torch.full((B,), 3, dtype=torch.int32), acts.int(), vals) if sparse else t.view(B, O, N, N)
    words = (ok.view(B, O * N, N).long() << torch.arange(N)).sum(2).to(torch.int32).cuda()
    p["t"], p["ok"] = t.double(), ok
    tgt = tuple(v.cuda() for v in tgt) if sparse else tgt.cuda()
    x, w, b, _, _ = _cuda(p)
    loss, dx, dw, db = [v.cpu() for v in learn.policy_loss_grad(x, w, b, tgt, legal=words)]
    assert loss[[1, 2, 3]].tolist() == [math.inf] * 3 and torch.isfinite(loss[[0, 4]]).all()
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all() and torch.isfinite(db).all()
    assert torch.equal(learn.policy_loss(x, w, b, tgt, legal=words).cpu(), loss)


@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_one_plane_bias_gradient_with_a_target_outside_the_allowed_actions(sign):
    """sum dz = r (T - the targets on allowed actions), not zero there."""
    N, C = 5, 16
    p = _rows(2, N, C, 1, "f32", seed=1)
    t = torch.zeros(2, 1, N, N)
    t[:, 0, 0, 0], t[1, 0, 1, 1] = 0.5, 0.25 * sign
    words = torch.full((2, N), 31, dtype=torch.int32)
    words[1, 1] = 31 - 2
    x, w, b, _, _ = _cuda(p)
    loss, _, _, db = learn.policy_loss_grad(x, w, b, t.cuda(), legal=words.cuda())
    assert loss[1] == math.inf and abs(float(db) - 0.25 * sign) <= 64 * F24


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("what", ["target", "feature"])
@pytest.mark.parametrize("B,N", [(3, 4), (2, 15), (90, 15)])
def test_one_plane_bias_gradient_of_a_nan(B, N, what, dtype):
    """A NaN target, or a NaN logit, makes the board's gradients NaN: d_bias too, which is zero for one plane otherwise."""
    p = _rows(B, N, 32, 1, dtype, "nhwc", seed=1)
    if what == "target":
        p["tgt"].view(B, -1)[1, 5] = float("nan")
    else:
        p["x"][1, 3, 2, 2] = float("nan")
    x, w, b, tgt, _ = _cuda(p)
    loss, dx, dw, db = [v.cpu() for v in learn.policy_loss_grad(x, w, b, tgt)]
    keep = torch.arange(B) != 1
    assert torch.isfinite(loss[keep]).all() and bool(torch.isnan(loss[1])) == (what == "feature")
    assert torch.isnan(dx[1]).all() and torch.isfinite(dx[keep]).all() and torch.isnan(dw).all() and torch.isnan(db).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shape", [(64, 1 << 22), (1 << 22, 64), (600, 1 << 19)], ids=lambda s: "%dx%d" % s)
def test_one_element_of_a_large_matrix_is_all_of_its_norm(shape, dtype):
    """2^28 and more elements: scaled by their root mean square the one would leave fp16.  Its result is the scalar iteration's."""
    u = torch.zeros(shape, dtype=DT[dtype], device="cuda")
    u[7, 33] = 1.0
    got = learn.orthogonalize(u)
    x = 1.0 / (1.0 + 1e-7)
    a, b, c = learn.NEWTON_SCHULZ
    for _ in range(5):
        x = a * x + b * x ** 3 + c * x ** 5
    assert abs(float(got[7, 33]) - x) <= 3e-5 + torch.finfo(DT[dtype]).eps * x     # (3e-5: test_gpu_learn.py)
    assert int(torch.count_nonzero(got)) == 1


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("coef,steps", [((2.0, 0.0, 0.0), 3), ((-2.0, 0.0, 0.0), 3), ((4.0, 0.0, 0.0), 2), ((32.0, 0.0, 0.0), 1), ((0.0, 6.9, 0.0), 1), ((0.0, 1.5, 0.0), 2), ((20.0, -10.0, -2.0), 1),
                                        ((6.9, 0.0, 0.0), 1), ((0.0, 0.0, 1.2), 3), ((0.0, 4.0, 0.0), 2)], ids=str)
@pytest.mark.parametrize("shape", [(1, 64, 225), (2, 100, 300), (1, 256, 256), (1, 300, 200)], ids=lambda s: "%dx%dx%d" % s)
def test_coefficients_that_enlarge(shape, coef, steps, dtype):
    """One singular value is the whole norm, in one element or spread over all, and grows to the borders of what is taken.  Its
    result is the scalar iteration's: each step's 3e-5 of the value (test_gpu_learn.py), which two later steps may magnify by
    |x f' / f| <= 5 each, and half a step of the type."""
    x, most = 1.0, 1.0
    f = [float(torch.tensor(v, dtype=torch.float32)) for v in coef]
    for _ in range(steps):
        x = f[0] * x + f[1] * x ** 3 + f[2] * x ** 5
        most = max(most, abs(x))
    g = torch.Generator().manual_seed(1)
    n, R, K = shape
    left, right = (torch.sign(torch.randn(n, m, generator=g)) for m in (R, K))
    one = torch.zeros(shape)
    one[:, R // 2, K // 3] = 1.0
    half = 0.0 if dtype == "f32" else torch.finfo(DT[dtype]).eps / 2
    for u, norm in ((left[:, :, None] * right[:, None, :], math.sqrt(R * K)), (one, 1.0)):    # exact in every type
        got = learn.orthogonalize(u.to(DT[dtype]).cuda(), steps=steps, coefficients=coef).cpu().double()
        err = torch.linalg.vector_norm((got - u.double() * (x / norm)).flatten(1), dim=1)
        assert (err <= 25 * 3e-5 * most + half * abs(x)).all(), err


@pytest.mark.parametrize("norm", [1e-6, 1e-9, 1e-11, 1e-14])
@pytest.mark.parametrize("shape", [(1, 64, 225), (1, 128, 600), (1, 256, 300)], ids=lambda s: "%dx%dx%d" % s)
def test_updates_far_smaller_than_eps(shape, norm):
    """The result shrinks with the update; its error is that of singular values near 1 (3e-5: test_gpu_learn.py)."""
    u = torch.randn(shape, generator=torch.Generator().manual_seed(2))
    u = u * (norm / float(u.norm()))
    want, got = _matrix_exact(u), learn.orthogonalize(u.cuda()).cpu().double()
    assert torch.linalg.matrix_norm(got - want, 2).max() <= 3e-5 * 1.3
    assert torch.isfinite(got).all() and float(got.norm()) <= 1.01 * float(want.norm()) + 3e-5 * math.sqrt(min(shape[1:]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", [(17, 32, 128, 96, 1024, 0.3), (17, 32, 100, 65, 1025, 0.0), (70, 12, 128, 96, 1024, 0.0), (2000, 2, 16, 91, 64, 0.0), (2000, 3, 32, 17, 147, 0.3)],
                         ids=lambda c: "b%d-n%d-c%d-o%d-cap%d%s" % (c[:5] + ("-legal" if c[5] else "",)))
def test_lists_that_just_fit_beside_more_than_a_step_a_workgroup(case, dtype):
    """The largest boards and heads of the paired kernel, with lists at the border of what LDS keeps of a workgroup's boards (1 024)."""
    B, N, C, O, cap, legal = case
    p = _rows(B, N, C, O, dtype, "nhwc", sparse=True, legal=legal, seed=cap + N, cap=cap, empty=(0,))
    x, w, b, tgt, words = _cuda(p)
    _check(p, learn.policy_loss_grad(x, w, b, tgt, legal=words), torch.ones(B, dtype=torch.float64))
