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
from test_gpu_learn import DT, F24, _cuda, _exact, _rows

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
