"""The learner's operators inside torch: what autograd, forward mode and tracing may rely on, and runs of the operators together
with the engines that they stand between."""
import pytest
import torch
from torch.autograd import forward_ad

from alphazero_amd import learn
from alphazero_amd.capi import AzError
from test_gpu_learn import _cuda, _rows

pytestmark = pytest.mark.gpu


def test_a_tensor_that_orthogonalize_overwrites_is_a_new_version():
    """A backward that saved it says so instead of using the new contents."""
    u = torch.randn(2, 20, 30, device="cuda")
    out, x = torch.randn(2, 20, 30, device="cuda"), torch.ones(2, 20, 30, device="cuda", requires_grad=True)
    y = (x * out).sum()
    before = out._version
    assert learn.orthogonalize(u, out=out) is out and out._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    w, m = torch.randn(2, 20, 30, device="cuda"), torch.zeros(2, 20, 30, device="cuda")
    before = w._version, m._version
    learn.muon_step(w, m, u, lr=0.1)
    assert w._version > before[0] and m._version > before[1]
    with torch.inference_mode():
        assert torch.equal(learn.orthogonalize(u, out=torch.empty_like(u)), learn.orthogonalize(u))


@pytest.mark.parametrize("needs_grad", [False, True])
def test_forward_mode_tangents_are_refused(needs_grad):
    """There is none of these operators' derivatives in it; without the check the result had no tangent, without a word."""
    p = _rows(2, 5, 16, 2, "f32", seed=1)
    x, w, b, tgt, _ = _cuda(p)
    m = torch.randn(1, 16, 20, device="cuda")
    with forward_ad.dual_level():
        assert learn.policy_loss(x, w, b, tgt).shape == (2,)                                   # (no tangent among them: fine)
        for at in range(4):
            args = [x, w, b, tgt]
            args[at] = forward_ad.make_dual(args[at].clone().requires_grad_(needs_grad and at < 3), torch.ones_like(args[at]))
            for call in (learn.policy_loss, learn.policy_loss_grad):
                with pytest.raises(AzError, match="tangent"):
                    call(*args)
        d = forward_ad.make_dual(m.clone(), torch.ones_like(m))
        with pytest.raises(AzError, match="tangent"):
            learn.orthogonalize(d)
        for at in range(3):
            args = [m.clone(), m.clone(), m.clone()]
            args[at] = d
            with pytest.raises(AzError, match="tangent"):
                learn.muon_step(*args, lr=0.1)


def test_tracing_is_refused():
    """A trace would hold the empty results alone."""
    p = _rows(2, 5, 16, 2, "f32", seed=1)
    x, w, b, tgt, _ = _cuda(p)
    m = torch.randn(1, 16, 20, device="cuda")
    for call, args in ((lambda x: learn.policy_loss(x, w, b, tgt), x), (lambda x: learn.policy_loss_grad(x, w, b, tgt), x), (learn.orthogonalize, m),
                       (lambda g: learn.muon_step(m.clone(), m.clone(), g, lr=0.1), m)):
        with pytest.raises(AzError, match="trace"):
            torch.jit.trace(call, (args,))


@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
def test_targets_that_require_a_gradient_are_refused(sparse):
    p = _rows(2, 5, 16, 2, "f32", sparse=sparse, seed=1)
    x, w, b, tgt, _ = _cuda(p)
    want = learn.policy_loss(x, w, b, tgt)
    asks = tgt[:2] + (tgt[2].clone().requires_grad_(),) if sparse else tgt.clone().requires_grad_()
    for xs in (x, x.clone().requires_grad_()):
        with pytest.raises(AzError, match="detach"):
            learn.policy_loss(xs, w, b, asks)
    with torch.no_grad():
        assert torch.equal(learn.policy_loss(x, w, b, asks), want)
    assert torch.equal(learn.policy_loss_grad(x, w, b, asks)[0], want)                         # (its gradients are named)


def test_words_and_targets_without_a_dimension_are_refused():
    x, w, b = torch.zeros(1, 4, 1, 1, device="cuda"), torch.zeros(1, 4, device="cuda"), torch.zeros(1, device="cuda")
    t = torch.ones(1, 1, device="cuda")
    assert learn.policy_loss(x, w, b, t, legal=torch.ones(1, 1, dtype=torch.int32, device="cuda")).tolist() == [0.0]
    for kw in (dict(legal=torch.tensor(1, dtype=torch.int32, device="cuda")), dict(legal=t.int()[:0])):
        with pytest.raises(AzError, match="words"):
            learn.policy_loss(x, w, b, t, **kw)
    for bad in (t[0, :0], None, 1.0, (t.int()[0],)):
        with pytest.raises(AzError, match="targets"):
            learn.policy_loss(x, w, b, bad)
