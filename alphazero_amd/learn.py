"""The learner's operators on torch tensors: the policy head's loss with its gradients over the rows that self-play
leaves (az_replay_drain, az_blokus_replay_drain), and the update of weight matrices by orthogonalised momentum.  The
result goes back into self-play as the blob of Engine.load_weights_dev.

Every call runs on the current stream of its tensors' device and returns without waiting; workspaces come from torch's
allocator, one per call.  Nothing here falls back to torch arithmetic: the compute is libazhip.so's (include/az_hip.h,
az_policy_loss_dev, az_orthogonalize_dev, az_muon_step_dev), and a call it does not take raises AzError.

The gradients that autograd asks for (policy_loss(...).backward()) are computed by the same kernels.  A training step that
is captured into a HIP graph uses policy_loss_grad, which involves no autograd graph.
"""
import ctypes as C

import torch
from torch.autograd import forward_ad

from . import capi
from .capi import AzError

NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)      # singular values x -> a x + b x^3 + c x^5, five times: about 0.7 .. 1.2
_DTYPES = {torch.float32: capi.AZ_F32, torch.float16: capi.AZ_F16, torch.bfloat16: capi.AZ_BF16}


def _need(ok, msg, *a):
    if not ok:
        raise AzError(msg % a)


def _untraced():
    _need(not torch.jit.is_tracing(), "torch.jit.trace records torch's own operators, not this call's kernels")


def _run(name, args, device):
    L = capi.load()
    ref = C.byref(args)
    size = getattr(L, "az_%s_workspace" % name)(ref)
    if size == 0:
        capi._chk(capi.AZ_E_ARG)
    ws = torch.empty(size, dtype=torch.uint8, device=device)
    capi._chk(getattr(L, "az_%s_dev" % name)(ref, ws.data_ptr(), size, torch.cuda.current_stream(device).cuda_stream))


def _dual(t):
    return getattr(forward_ad, "_current_level", 0) >= 0 and forward_ad.unpack_dual(t).tangent is not None


def _on(t, device, what):
    _need(isinstance(t, torch.Tensor) and t.device == device, "%s is not a tensor on %s", what, device)
    _need(not _dual(t), "%s carries a tangent: there is no forward-mode derivative", what)


def _loss_args(features, weight, bias, targets, legal):
    _untraced()
    _need(isinstance(features, torch.Tensor) and features.is_cuda and features.dim() == 4, "features: a [B, C, N, N] tensor on the GPU")
    dev = features.device
    _on(features, dev, "features")
    B, ch, N, N2 = features.shape
    _need(N == N2, "features: board %d x %d is not square", N, N2)
    _need(features.dtype in _DTYPES, "features: %s (float32, float16 or bfloat16)", features.dtype)
    _on(weight, dev, "weight")
    _on(bias, dev, "bias")
    if weight.dim() == 4:                                    # the 1x1 convolution's own shape
        _need(weight.shape[2] == 1 and weight.shape[3] == 1, "weight: a 1x1 convolution's")
        weight = weight.flatten(1)
    _need(weight.dim() == 2 and weight.shape[1] == ch, "weight: [c_out, %d]", ch)
    O = weight.shape[0]
    _need(bias.shape == (O,), "bias: [%d]", O)
    _need(weight.dtype == features.dtype and bias.dtype == features.dtype, "weight and bias are not of the features' type %s", features.dtype)
    _need(weight.is_contiguous() and bias.is_contiguous(), "weight and bias have to be contiguous")
    a = capi.AzPolicyLossArgs()
    a.device, a.B, a.N, a.C, a.c_out = dev.index, B, N, ch, O
    a.dtype = _DTYPES[features.dtype]
    if features.is_contiguous():
        a.layout = capi.AZ_CHANNELS_FIRST
    else:
        _need(features.is_contiguous(memory_format=torch.channels_last), "features: contiguous or channels_last, not strides %s", features.stride())
        a.layout = capi.AZ_CHANNELS_LAST
    a.features, a.weight, a.bias = features.data_ptr(), weight.data_ptr(), bias.data_ptr()
    if isinstance(targets, torch.Tensor):
        _on(targets, dev, "targets")
        _need(targets.dtype == torch.float32 and targets.is_contiguous() and targets.numel() == B * O * N * N and
              (targets.dim() == 0 or targets.shape[0] == B), "targets: contiguous float32 [%d, %d, %d, %d]", B, O, N, N)
        a.target = targets.data_ptr()
    else:
        _need(isinstance(targets, (tuple, list)) and len(targets) == 3, "targets: a dense tensor or (counts, actions, probs)")
        counts, actions, probs = targets
        for t, n, dt in ((counts, "counts", torch.int32), (actions, "actions", torch.int32), (probs, "probs", torch.float32)):
            _on(t, dev, n)
            _need(t.dtype == dt and t.is_contiguous(), "%s: contiguous %s", n, dt)
        _need(counts.shape == (B,) and actions.dim() == 2 and actions.shape[0] == B and actions.shape == probs.shape, "counts [B], actions and probs [B, cap]")
        a.counts, a.actions, a.probs, a.cap = counts.data_ptr(), actions.data_ptr(), probs.data_ptr(), actions.shape[1]
    if legal is not None:
        _on(legal, dev, "legal")
        _need(legal.dtype in (torch.int32, torch.uint32) and legal.is_contiguous() and legal.numel() == B * O * N and legal.dim() > 0 and legal.shape[0] == B,
              "legal: contiguous 32-bit words [%d, %d]", B, O * N)
        a.legal = legal.data_ptr()
    a.scale = 1.0
    return a


def _loss(features, weight, bias, targets, legal, keep=False):
    a = _loss_args(features, weight, bias, targets, legal)
    loss = torch.empty(a.B, dtype=torch.float32, device=features.device)
    stats = torch.empty(a.B, 4, dtype=torch.float32, device=features.device) if keep else None
    if a.B:
        a.loss = loss.data_ptr()
        if keep:
            a.stats = stats.data_ptr()
        _run("policy_loss", a, features.device)
    return loss, stats


def _grad(features, weight, bias, targets, legal, row_scale, stats=None):
    a = _loss_args(features, weight, bias, targets, legal)
    dev = features.device
    d = torch.empty_like(features), torch.empty(a.c_out, a.C, dtype=torch.float32, device=dev), torch.empty(a.c_out, dtype=torch.float32, device=dev)
    if isinstance(row_scale, torch.Tensor):
        _on(row_scale, dev, "row_scale")
        _need(row_scale.dtype == torch.float32 and row_scale.shape == (a.B,) and row_scale.is_contiguous(), "row_scale: contiguous float32 [%d]", a.B)
        a.row_scale = row_scale.data_ptr()
    elif row_scale is not None:
        a.scale = float(row_scale)
    loss = None
    if stats is not None:
        a.stats, a.stats_given = stats.data_ptr(), 1 if a.B else 0
    else:
        loss = torch.empty(a.B, dtype=torch.float32, device=dev)
        a.loss = loss.data_ptr()
    a.d_features, a.d_weight, a.d_bias = (t.data_ptr() for t in d)
    _run("policy_loss", a, dev)
    return (loss,) + d


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, features, weight, bias, legal, *targets):
        tgt = targets[0] if len(targets) == 1 else targets
        loss, stats = _loss(features, weight, bias, tgt, legal, keep=True)
        ctx.save_for_backward(features, weight, bias, legal, stats, *targets)
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        features, weight, bias, legal, stats, *targets = ctx.saved_tensors
        tgt = targets[0] if len(targets) == 1 else tuple(targets)
        _, dx, dw, db = _grad(features, weight, bias, tgt, legal, g.contiguous(), stats)
        return (dx, dw.view(weight.shape).to(weight.dtype), db.to(bias.dtype), None) + (None,) * len(targets)


def policy_loss(features, weight, bias, targets, legal=None):
    """Cross entropy of the policy head, one fp32 loss a board: sum t (lse - z) over the c_out * N * N actions, z the 1x1
    convolution (network.hpp:46-65; the policy term of train.cpp:90-112 before its mean).  Differentiable in features,
    weight and bias.

    features  [B, C, N, N], contiguous or channels_last, float32 / float16 / bfloat16; weight [c_out, C] or [c_out, C, 1, 1]
              and bias [c_out] of the same type
    targets   float32 [B, c_out, N, N] (or [B, c_out * N * N]), or (counts int32 [B], actions int32 [B, cap], probs float32
              [B, cap]) as the Blokus rows are drained; they need not sum to 1
    legal     None, or int32 words [B, c_out * N]: bit x of word co * N + y allows action (co, y, x); the softmax runs
              over the allowed actions.  A target outside them makes that board's loss inf; a board without targets has
              loss 0.  They get no gradient
    """
    _need(isinstance(targets, (torch.Tensor, tuple, list)), "targets: a dense tensor or (counts, actions, probs)")
    tgt = (targets,) if isinstance(targets, torch.Tensor) else tuple(targets)
    _need(not (torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tgt)), "targets get no gradient: detach() them")
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (features, weight, bias)):
        _need(not torch.cuda.is_current_stream_capturing(), "policy_loss with gradients cannot be captured into a graph: policy_loss_grad can")
        for t in (features, weight, bias) + tgt:
            _need(not (isinstance(t, torch.Tensor) and _dual(t)), "an argument carries a tangent: there is no forward-mode derivative")
        return _PolicyLoss.apply(features, weight, bias, legal, *tgt)
    return _loss(features, weight, bias, targets, legal)[0]


@torch.no_grad()
def policy_loss_grad(features, weight, bias, targets, row_scale=None, legal=None):
    """policy_loss and the gradients of sum_b row_scale_b * loss_b in one call: (loss [B], d_features like features,
    d_weight float32 [c_out, C], d_bias float32 [c_out]).  row_scale: None = 1, a number (1 / B for the mean), or float32
    [B].  For c_out = 1 the bias shifts every logit alike and its gradient is zero (NaN
    where a board's are)."""
    return _grad(features, weight, bias, targets, legal, row_scale)


def _batch(t, what):
    """(n, rows, cols, stride) of a matrix [R, K], a batch [n, R, K], a convolution's weight [O, I, kh, kw] (as O x I kh kw)
    or a batch of those."""
    _need(isinstance(t, torch.Tensor) and t.is_cuda and 2 <= t.dim() <= 5, "%s: a matrix or a batch of matrices on the GPU", what)
    shape, strides = t.shape, t.stride()
    lead = len(shape) & 1
    want = 1
    for d in range(len(shape) - 1, lead, -1):
        _need(strides[d] == want or shape[d] == 1 or 0 in shape, "%s: every matrix has to be contiguous (strides %s)", what, strides)
        want *= shape[d]
    rows = shape[lead]
    _need(strides[lead] == want or rows == 1 or 0 in shape, "%s: every matrix has to be contiguous (strides %s)", what, strides)
    return (shape[0], rows, want, strides[0]) if lead else (1, rows, want, rows * want)


def _coef(a, coefficients, eps, steps):
    a.a, a.b, a.c = coefficients
    a.eps, a.steps = eps, steps


@torch.no_grad()
def orthogonalize(update, scale=1.0, steps=5, coefficients=NEWTON_SCHULZ, eps=1e-7, out=None):
    """scale times the update with its singular values brought near 1 by `steps` Newton-Schulz products, matrix by matrix.

    update: [R, K], [n, R, K], a convolution's weight [O, I, kh, kw] or [n, O, I, kh, kw]; float32 / float16 / bfloat16; the
    batch may be strided (the convolutions of all blocks in the weight blob), each matrix contiguous.  out: like update,
    apart from it.  coefficients that take singular values of up to 1 beyond 7 ahead of a step, or enlarge one more than 200
    times in a step, are refused."""
    _untraced()
    n, R, K, stride = _batch(update, "update")
    _on(update, update.device, "update")
    _need(update.dtype in _DTYPES, "update: %s (float32, float16 or bfloat16)", update.dtype)
    if out is None:
        out = torch.empty(update.shape, dtype=update.dtype, device=update.device)
    _on(out, update.device, "out")
    _need(out.dtype == update.dtype and out.shape == update.shape, "out: %s %s", update.dtype, tuple(update.shape))
    a = capi.AzOrthogonalizeArgs()
    a.device, a.n, a.rows, a.cols, a.dtype = update.device.index, n, R, K, _DTYPES[update.dtype]
    _coef(a, coefficients, eps, steps)
    a.scale = scale
    a.update, a.update_stride, a.out, a.out_stride = update.data_ptr(), stride, out.data_ptr(), _batch(out, "out")[3]
    _run("orthogonalize", a, update.device)
    torch.autograd.graph.increment_version(out)              # the kernels wrote where autograd cannot see
    return out


@torch.no_grad()
def muon_step(weight, momentum, grad, lr, beta=0.95, nesterov=True, weight_decay=0.0, scale=1.0, steps=5, coefficients=NEWTON_SCHULZ,
              eps=1e-7, weight_out=None, momentum_out=None):
    """One optimiser step of weight matrices by orthogonalised momentum:
        momentum' = beta momentum + grad;  u = grad + beta momentum' (nesterov) or momentum'
        weight' = (1 - lr weight_decay) weight - lr orthogonalize(u, scale)
    weight and momentum: float32, shapes as in orthogonalize (views into the weight blob may be strided batches); grad of any
    of the three types.  Without weight_out / momentum_out the step is in place.  Returns (weight', momentum')."""
    _untraced()
    n, R, K, ws = _batch(weight, "weight")
    a = capi.AzMuonStepArgs()
    w_out = weight if weight_out is None else weight_out
    m_out = momentum if momentum_out is None else momentum_out
    for t, what in ((weight, "weight"), (momentum, "momentum"), (grad, "grad"), (w_out, "weight_out"), (m_out, "momentum_out")):
        _on(t, weight.device, what)
        _need(t.shape == weight.shape, "%s: shape %s is not the weight's %s", what, t.shape, weight.shape)
    for t, what in ((weight, "weight"), (momentum, "momentum"), (w_out, "weight_out"), (m_out, "momentum_out")):
        _need(t.dtype == torch.float32, "%s: %s (float32)", what, t.dtype)
    _need(grad.dtype in _DTYPES, "grad: %s (float32, float16 or bfloat16)", grad.dtype)
    a.device, a.n, a.rows, a.cols, a.grad_dtype = weight.device.index, n, R, K, _DTYPES[grad.dtype]
    _coef(a, coefficients, eps, steps)
    a.scale, a.lr, a.beta, a.weight_decay, a.nesterov = scale, lr, beta, weight_decay, int(bool(nesterov))
    a.grad, a.grad_stride = grad.data_ptr(), _batch(grad, "grad")[3]
    a.weight, a.weight_stride = weight.data_ptr(), ws
    a.momentum, a.momentum_stride = momentum.data_ptr(), _batch(momentum, "momentum")[3]
    a.weight_out, a.weight_out_stride = w_out.data_ptr(), _batch(w_out, "weight_out")[3]
    a.momentum_out, a.momentum_out_stride = m_out.data_ptr(), _batch(m_out, "momentum_out")[3]
    _run("muon_step", a, weight.device)
    torch.autograd.graph.increment_version(w_out)
    torch.autograd.graph.increment_version(m_out)
    return w_out, m_out
