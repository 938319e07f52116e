"""The learner's operators inside torch: what autograd, forward mode and tracing may rely on, and runs of the operators together
with the engines that they stand between."""
import ctypes as C

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

from alphazero_amd import capi, learn, synth
from alphazero_amd.capi import AzError
from test_gpu_learn import DT, _check, _cuda, _rows

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
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda v: learn.policy_loss(v, w, b, tgt), (x,), (torch.ones_like(x),))
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


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
@pytest.mark.parametrize("B", [4, 90])
def test_autograd_gives_the_same_gradients_in_16_bits(B, sparse, dtype):
    """Those of policy_loss_grad, with the weight's and the bias's rounded to their type."""
    p = _rows(B, 15, 40, 3, dtype, "nhwc", sparse=sparse, legal=0.7, seed=8)
    x, w, b, tgt, words = _cuda(p)
    xr, wr, br = x.clone().requires_grad_(), w.view(3, 40, 1, 1).clone().requires_grad_(), b.clone().requires_grad_()
    g = torch.linspace(-1.0, 2.0, B, device="cuda")
    loss = learn.policy_loss(xr, wr, br, tgt, legal=words)
    (loss * g).sum().backward()
    want, dx, dw, db = learn.policy_loss_grad(x, w, b, tgt, row_scale=g, legal=words)
    assert torch.equal(loss, want) and torch.equal(xr.grad, dx) and xr.grad.stride() == x.stride()
    assert torch.equal(wr.grad, dw.view(3, 40, 1, 1).to(DT[dtype])) and torch.equal(br.grad, db.to(DT[dtype]))


def test_rows_of_selfplay_through_a_training_step_and_back():
    """m,n,k rows as az_replay_drain leaves them -> features of a torch convolution, the blob's policy head on them, loss and
    gradients, the optimiser step inside the blob -> az_load_weights_dev, whose games go on."""
    N, K, budget, G, Ch = 5, 4, 32, 8, 32
    eng = capi.Engine(N, K, G, eval_mode=capi.AZ_EVAL_HASH, max_budget=budget, seed=7)
    eng.selfplay_begin(budget)
    eng.selfplay_run((2 * budget + 1 + 24 * budget) + 8)
    cells, tm, pol, _ = eng.replay_drain()
    eng.close()
    B = len(tm)
    assert B >= 40 and (pol.sum(1) > 0).all()
    blob = torch.from_numpy(synth.make_blob(N, 3, [Ch, Ch], 5)).cuda()
    off, at = {}, 0
    for name, shape in synth.blob_layout(N, 3, [Ch, Ch]):
        off[name] = at, shape
        at += int(np.prod(shape))
    part = lambda t, name: t[off[name][0]:off[name][0] + int(np.prod(off[name][1]))].view(off[name][1])       # noqa: E731
    planes = torch.from_numpy(np.stack([cells == 1, cells == 2, np.repeat(tm[:, None], N * N, 1) == 0], 1).astype(np.float32)).view(B, 3, N, N).cuda()
    stem = part(blob, "CBlock.conv.weight").clone().requires_grad_()
    x = torch.relu(torch.nn.functional.conv2d(planes, stem, padding=1))
    w, b, tgt = part(blob, "PHead.conv.weight"), part(blob, "PHead.conv.bias"), torch.from_numpy(pol).cuda()
    learn.policy_loss(x, w, b, tgt).mean().backward()
    loss, dx, dw, db = learn.policy_loss_grad(x.detach(), w, b, tgt, row_scale=1.0 / B)
    p = dict(x=x.detach().cpu(), w=w.view(1, Ch).cpu(), b=b.cpu(), t=torch.from_numpy(pol).double(), ok=None, B=B, N=N, C=Ch, O=1, dtype="f32")
    _check(p, (loss, dx, dw, db), torch.full((B,), 1.0 / B, dtype=torch.float32).double())
    momentum, before = torch.zeros_like(blob), blob.clone()
    learn.muon_step(part(blob, "CBlock.conv.weight"), part(momentum, "CBlock.conv.weight"), stem.grad, lr=0.02)
    learn.muon_step(w, part(momentum, "PHead.conv.weight"), dw.view(1, Ch, 1, 1), lr=0.02)
    b -= 0.02 * db
    changed = (blob != before).cpu()
    for name, (o, shape) in off.items():
        assert changed[o:o + int(np.prod(shape))].any() == (name in ("CBlock.conv.weight", "PHead.conv.weight")), name
    after = learn.policy_loss(torch.relu(torch.nn.functional.conv2d(planes, part(blob, "CBlock.conv.weight"), padding=1)), w, b, tgt)
    assert torch.isfinite(after).all()
    play = capi.Engine(N, K, G, Cs=[Ch, Ch], max_budget=budget, seed=8)
    play.load_weights_dev(blob.data_ptr(), blob.numel())
    play.selfplay_begin(budget)
    play.selfplay_run(4 * budget)
    play.sync()
    assert play.stats()["moves"] > 0 and play.stats()["error_games"] == 0
    play.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("reuse", [False, True], ids=["fresh", "reuse"])
def test_blokus_rows_as_they_are_drained(reuse, dtype):
    """Sparse search policies of whole games; with the tree reused a row has room for 4 * budget entries, more than LDS keeps
    (1 040 here), and most of it is empty."""
    G, budget, O, N, C, B = 2, 260, 91, 20, 32, 48
    dev = capi.Blokus(G, seed=3)
    dev.search_config(max_budget=budget, reuse=reuse)
    dev.selfplay_config(ring_rows=G * 84, max_budget=budget)
    dev.selfplay_moves(budget, 86)
    got = dev.replay_drain(G * 84)
    dev.close()
    assert len(got["counts"]) >= B and (got["actions"].shape[1] > 1024) == reuse
    n, acts, probs = (np.ascontiguousarray(got[k][:B]) for k in ("counts", "actions", "probs"))
    g = torch.Generator().manual_seed(1)
    x = torch.randn(B, C, N, N, generator=g).relu().to(DT[dtype])
    w, b = (torch.randn(O, C, generator=g) / 4).to(DT[dtype]), (torch.randn(O, generator=g) * 0.1).to(DT[dtype])
    t = torch.from_numpy(capi.Blokus.dense_policy(acts, probs, n)).view(B, -1).double()
    p = dict(x=x, w=w, b=b, t=t, ok=None, tgt=tuple(torch.from_numpy(v) for v in (n, acts, probs)), words=None, B=B, N=N, C=C, O=O, dtype=dtype, layout="nhwc")
    xg, wg, bg, tg, _ = _cuda(p)
    _check(p, learn.policy_loss_grad(xg, wg, bg, tg, row_scale=1.0 / B), torch.full((B,), 1.0 / B, dtype=torch.float32).double())


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("B,N", [(3, 4), (90, 15)])
def test_lists_without_room_are_boards_without_targets(B, N, dtype):
    p = _rows(B, N, 32, 3, dtype, "nhwc", seed=1)
    x, w, b, _, _ = _cuda(p)
    none = (torch.full((B,), 5, dtype=torch.int32, device="cuda"), torch.empty(B, 0, dtype=torch.int32, device="cuda"), torch.empty(B, 0, device="cuda"))
    assert all((v == 0).all() for v in learn.policy_loss_grad(x, w, b, none))


def test_calls_at_the_same_time_on_two_streams():
    """Each has its workspace: results are those of the calls one after the other."""
    heads = [_cuda(_rows(90, 15, 128, O, "bf16", "nhwc", sparse=True, seed=O)) for O in (3, 91)]
    mats = [torch.randn(4, 256, 600, device="cuda") for _ in range(2)]
    call = lambda i: learn.policy_loss_grad(*heads[i][:4]) + (learn.orthogonalize(mats[i]),)                   # noqa: E731
    want = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    for s in streams:
        s.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(r, want[i]))


@pytest.mark.parametrize("steps", [2, 3, 4, 5, 6, 7, 9, 10])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_no_call_leaves_its_workspace(steps, dtype):
    """Guards around the workspace and the result of every number of stages, through the C entry."""
    n, R, K = 3, 130, 200
    u = torch.randn(n, R, K, device="cuda").to(DT[dtype])
    a = capi.AzOrthogonalizeArgs()
    a.device, a.n, a.rows, a.cols, a.dtype, a.steps = u.device.index, n, R, K, {"f32": capi.AZ_F32, "bf16": capi.AZ_BF16}[dtype], steps
    a.a, a.b, a.c = learn.NEWTON_SCHULZ
    a.eps, a.scale = 1e-7, 1.0
    L = capi.load()
    size, guard = L.az_orthogonalize_workspace(C.byref(a)), 4096
    ws = torch.full((size + 2 * guard,), 0xA5, dtype=torch.uint8, device="cuda")
    out = torch.full((n * R * K + 256,), 7.0, dtype=DT[dtype], device="cuda")
    a.update, a.update_stride, a.out, a.out_stride = u.data_ptr(), R * K, out.data_ptr() + 128 * out.element_size(), R * K
    capi._chk(L.az_orthogonalize_dev(C.byref(a), ws.data_ptr() + guard, size, torch.cuda.current_stream().cuda_stream))
    assert (ws[:guard] == 0xA5).all() and (ws[-guard:] == 0xA5).all() and (out[:128] == 7).all() and (out[-128:] == 7).all()
    assert torch.equal(out[128:-128].view(n, R, K), learn.orthogonalize(u, steps=steps))


@pytest.mark.parametrize("case", [(3, 9, 100, 3, "f32"), (2, 20, 250, 91, "f32"), (90, 15, 128, 17, "bf16"), (90, 15, 128, 1, "f16"), (40, 20, 128, 91, "bf16"), (5, 3, 200, 128, "f16")], ids=str)
@pytest.mark.parametrize("sparse", [False, True], ids=["dense", "sparse"])
def test_no_loss_leaves_its_workspace_or_outputs(case, sparse):
    """Guards around everything az_policy_loss_dev writes, and the statistics handed from a call for the losses to one for the
    gradients."""
    B, N, ch, O, dtype = case
    p = _rows(B, N, ch, O, dtype, "nchw", sparse=sparse, seed=B)
    x, w, b, tgt, _ = _cuda(p)
    want = learn.policy_loss_grad(x, w, b, tgt, row_scale=0.25)
    L, a = capi.load(), capi.AzPolicyLossArgs()
    a.device, a.B, a.N, a.C, a.c_out, a.scale, a.layout = x.device.index, B, N, ch, O, 0.25, capi.AZ_CHANNELS_FIRST
    a.dtype = {"f32": capi.AZ_F32, "f16": capi.AZ_F16, "bf16": capi.AZ_BF16}[dtype]
    a.features, a.weight, a.bias = x.data_ptr(), w.data_ptr(), b.data_ptr()
    if sparse:
        a.counts, a.actions, a.probs, a.cap = tgt[0].data_ptr(), tgt[1].data_ptr(), tgt[2].data_ptr(), tgt[1].shape[1]
    else:
        a.target = tgt.data_ptr()
    guarded = []

    def room(nbytes):
        t = torch.full((nbytes + 1024,), 0xA5, dtype=torch.uint8, device="cuda")
        guarded.append(t)
        return t[512:-512]

    def call():
        ws = room(L.az_policy_loss_workspace(C.byref(a)))
        capi._chk(L.az_policy_loss_dev(C.byref(a), ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    loss, stats, dx, dw, db = room(B * 4), room(B * 16), room(x.numel() * x.element_size()), room(O * ch * 4), room(O * 4)
    a.loss, a.stats = loss.data_ptr(), stats.data_ptr()
    call()
    a.loss, a.stats_given, a.d_features, a.d_weight, a.d_bias = None, 1, dx.data_ptr(), dw.data_ptr(), db.data_ptr()
    call()
    got = loss.view(torch.float32), dx.view(x.dtype).view(x.shape), dw.view(torch.float32).view(O, ch), db.view(torch.float32)
    assert all(torch.equal(g, v) for g, v in zip(got, want))
    for t in guarded:
        assert (t[:512] == 0xA5).all() and (t[-512:] == 0xA5).all()
