"""Argument checks of the learner's operators (no GPU: every refusal comes before any HIP call), the ctypes mirrors of
their structures, and the store scan over their kernels."""
import concurrent.futures
import ctypes as C
import os
import subprocess
import sys

import pytest
import torch

from alphazero_amd import capi, learn

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                                   # an address no call may touch


def _policy(**kw):
    a = capi.AzPolicyLossArgs()
    v = dict(B=4, N=9, C=64, c_out=3, dtype=capi.AZ_F32, layout=capi.AZ_CHANNELS_LAST, features=P, weight=P, bias=P, target=P, scale=1.0, loss=P)
    v.update(kw)
    for k, x in v.items():
        setattr(a, k, x)
    return a


def _ortho(**kw):
    a = capi.AzOrthogonalizeArgs()
    v = dict(n=2, rows=64, cols=225, dtype=capi.AZ_F32, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, scale=1.0, update=P, update_stride=64 * 225,
             out=2 * P, out_stride=64 * 225)
    v.update(kw)
    for k, x in v.items():
        setattr(a, k, x)
    return a


def _muon(**kw):
    a = capi.AzMuonStepArgs()
    s = 64 * 225
    v = dict(n=2, rows=64, cols=225, grad_dtype=capi.AZ_F32, steps=5, a=3.4445, b=-4.775, c=2.0315, eps=1e-7, scale=1.0, lr=0.1, beta=0.9, grad=P, grad_stride=s,
             weight=2 * P, weight_stride=s, momentum=3 * P, momentum_stride=s, weight_out=2 * P, weight_out_stride=s, momentum_out=3 * P, momentum_out_stride=s)
    v.update(kw)
    for k, x in v.items():
        setattr(a, k, x)
    return a


def _call(name, a, ws=P, size=1 << 40):
    L = capi.load()
    rc = getattr(L, "az_%s_dev" % name)(C.byref(a) if a is not None else None, ws, size, None)
    return rc, L.az_last_error().decode()


@pytest.mark.parametrize("kw,word", [
    (dict(B=-1), "negative"), (dict(N=0), "board side"), (dict(N=33), "board side"), (dict(C=0), "channels"), (dict(C=257), "channels"),
    (dict(c_out=0), "policy channels"), (dict(c_out=129), "policy channels"), (dict(dtype=3), "element type"), (dict(layout=2), "layout"),
    (dict(B=1 << 30, N=32), "too many cells"), (dict(features=None), "features"), (dict(weight=None), "weight"), (dict(bias=None), "bias"),
    (dict(target=None), "target"), (dict(counts=P, actions=P, probs=P, cap=4), "not both"), (dict(target=None, counts=P, cap=4), "actions"),
    (dict(target=None, counts=P, actions=P, probs=P, cap=-1), "cap"), (dict(features=P + 2), "aligned"), (dict(dtype=capi.AZ_F16, bias=P + 1), "aligned"),
    (dict(target=P + 2), "aligned"), (dict(stats=P + 8), "16-byte"), (dict(loss=None), "nothing to compute"), (dict(d_weight=P), "come together"),
    (dict(d_weight=P, d_bias=P), "come together"), (dict(stats_given=1, stats=P), "stats_given"), (dict(stats_given=1, d_features=P, d_weight=P, d_bias=P), "stats_given"),
], ids=lambda v: "-".join(v) if isinstance(v, dict) else v.replace(" ", "_"))
def test_policy_loss_refuses(kw, word):
    rc, msg = _call("policy_loss", _policy(**kw))
    assert rc == capi.AZ_E_ARG and word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(n=-1), "-1 matrices"), (dict(n=65536), "too many"), (dict(rows=0), "matrix 0"), (dict(cols=0), "x 0"), (dict(rows=1 << 16, cols=1 << 16), "too many elements"),
    (dict(rows=8193, cols=8193, update_stride=1 << 40, out_stride=1 << 40), "8192"), (dict(rows=(1 << 24) + 1, cols=1, update_stride=1 << 40, out_stride=1 << 40), "2^24"), (dict(steps=-1), "steps"), (dict(steps=101), "steps"), (dict(a=40.0), "coefficients"),
    (dict(b=float("nan")), "coefficients"), (dict(eps=-1.0), "eps"), (dict(eps=float("inf")), "eps"), (dict(eps=float("nan")), "eps"), (dict(dtype=7), "element type"),
    (dict(update=None), "update"), (dict(out=None), "out"), (dict(update=P + 2), "aligned"), (dict(update_stride=10), "stride"), (dict(out_stride=0), "stride"),
    (dict(out=P), "overlaps"), (dict(out=P + 64 * 225 * 4), "overlaps"),
], ids=lambda v: "-".join(v) if isinstance(v, dict) else v.replace(" ", "_"))
def test_orthogonalize_refuses(kw, word):
    rc, msg = _call("orthogonalize", _ortho(**kw))
    assert rc == capi.AZ_E_ARG and word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(n=-1), "matrices"), (dict(grad_dtype=-1), "element type"), (dict(steps=200), "steps"), (dict(grad=None), "grad"), (dict(weight=None), "weight"),
    (dict(momentum=None), "momentum"), (dict(weight_out=None), "weight_out"), (dict(momentum_out=None), "momentum_out"), (dict(weight=P + 1), "aligned"),
    (dict(momentum_stride=5), "momentum"), (dict(weight_out=2 * P + 4), "overlaps"), (dict(weight_out_stride=64 * 225 + 4), "overlaps"), (dict(momentum_out=2 * P), "overlaps"),
    (dict(weight_out=P), "overlaps"), (dict(weight_out=3 * P), "overlaps"),
], ids=lambda v: "-".join(v) if isinstance(v, dict) else v)
def test_muon_step_refuses(kw, word):
    rc, msg = _call("muon_step", _muon(**kw))
    assert rc == capi.AZ_E_ARG and word in msg, msg


@pytest.mark.parametrize("name,make", [("policy_loss", _policy), ("orthogonalize", _ortho), ("muon_step", _muon)])
def test_workspace_is_checked(name, make):
    L = capi.load()
    size = getattr(L, "az_%s_workspace" % name)(C.byref(make()))
    assert size > 0
    assert _call(name, None)[0] == capi.AZ_E_ARG and getattr(L, "az_%s_workspace" % name)(None) == 0
    rc, msg = _call(name, make(), None, size)
    assert rc == capi.AZ_E_ARG and "workspace" in msg
    rc, msg = _call(name, make(), P + 16, size)
    assert rc == capi.AZ_E_ARG and "256-byte" in msg
    rc, msg = _call(name, make(), P, size - 1)
    assert rc == capi.AZ_E_CAPACITY and str(size - 1) in msg
    assert getattr(L, "az_%s_workspace" % name)(C.byref(make(**{"N": 99} if name == "policy_loss" else {"rows": -3}))) == 0
    if not torch.cuda.is_available():
        assert _call(name, make(), P, size)[0] == capi.AZ_E_HIP                      # every check passed: only the device is missing


def test_tensors_that_are_not_on_the_gpu_are_refused():
    x, w, b, t = torch.zeros(2, 8, 3, 3), torch.zeros(1, 8), torch.zeros(1), torch.zeros(2, 1, 3, 3)
    for call in (lambda: learn.policy_loss(x, w, b, t), lambda: learn.policy_loss_grad(x, w, b, t), lambda: learn.orthogonalize(w),
                 lambda: learn.muon_step(w, w.clone(), w.clone(), lr=0.1)):
        with pytest.raises(capi.AzError, match="GPU"):
            call()


def test_ctypes_structures_match_the_header_layout(tmp_path):
    structs = {"az_policy_loss_args": capi.AzPolicyLossArgs, "az_orthogonalize_args": capi.AzOrthogonalizeArgs, "az_muon_step_args": capi.AzMuonStepArgs}
    src = ['#include <stdio.h>', '#include <stddef.h>', '#include "az_hip.h"', 'int main(void) {']
    for st, cls in structs.items():
        src.append('printf("%s %%zu\\n", sizeof(%s));' % (st, st))
        src += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (st, f, st, f) for f, _ in cls._fields_]
    src.append('return 0; }')
    c, exe = tmp_path / "probe.c", tmp_path / "probe"
    c.write_text("\n".join(src))
    subprocess.check_call(["gcc", "-std=c99", "-I", os.path.join(ROOT, "include"), str(c), "-o", str(exe)])
    got = dict(line.split() for line in subprocess.check_output([str(exe)], text=True).splitlines())
    for st, cls in structs.items():
        assert int(got[st]) == C.sizeof(cls), st
        for f, _ in cls._fields_:
            assert int(got["%s.%s" % (st, f)]) == getattr(cls, f).offset, (st, f)


@pytest.mark.skipif(not os.path.exists("/opt/rocm/bin/hipcc"), reason="no hipcc")
def test_kernels_hold_no_packed_fp32_and_no_write_behind_a_wide_store(tmp_path):
    """Compiled with the Makefile's flags: packed fp32 instructions are off for these sources, and no data register of a
    wide store is written too soon behind it (tools/probe/wide_store_overwrite_scan.py)."""
    def asm(src):
        out = str(tmp_path / (src + ".s"))
        subprocess.run(["/opt/rocm/bin/hipcc", "--offload-arch=gfx950", "-O3", "-std=c++17", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
                        "--cuda-device-only", "-S", os.path.join(ROOT, "alphazero_amd", "csrc", src), "-o", out], check=True, capture_output=True, timeout=900)
        return out
    with concurrent.futures.ThreadPoolExecutor(5) as pool:
        files = list(pool.map(asm, ["policy_f32.hip", "policy_f16.hip", "policy_bf16.hip", "orthogonalize.hip", "policy_loss.hip"]))
    for f in files:
        text = open(f).read()
        assert not any("v_pk_%s_f32" % op in text for op in ("add", "mul", "fma"))
    r = subprocess.run([sys.executable, os.path.join(ROOT, "tools", "probe", "wide_store_overwrite_scan.py"), *files], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout[-3000:]


@pytest.mark.parametrize("coef,steps,fine", [
    ((2.0, 0.0, 0.0), 3, True), ((2.0, 0.0, 0.0), 4, False), ((2.0, 0.0, 0.0), 5, False), ((32.0, 0.0, 0.0), 1, True), ((32.0, 0.0, 0.0), 2, False),
    ((-2.0, 0.0, 0.0), 5, False), ((0.0, 8.0, 0.0), 2, False), ((0.0, 6.9, 0.0), 2, False), ((0.0, 4.0, 0.0), 2, True), ((0.0, 0.0, 2.0), 2, True), ((0.0, 0.0, 2.0), 3, False), ((0.0, 0.0, 3.2), 2, False), ((7.0, 0.0, 0.0), 1, True), ((4.0, 0.0, 0.0), 2, True),
    ((4.0, 0.0, 0.0), 3, False), ((0.0, 0.0, 1.0), 100, True), ((3.4445, -4.775, 2.0315), 100, True), ((1.875, -1.25, 0.375), 100, True), ((1.5, -0.5, 0.0), 100, True), ((0.0, 0.0, 0.0), 100, True),
], ids=str)
def test_coefficients_that_leave_the_arithmetics_range_are_refused(coef, steps, fine):
    """Singular values of up to 1 may reach 7 ahead of a step, which may enlarge them 200 times: beyond that A = X X^T or its
    products leave fp16.  Both sides of the rule, and the usual coefficients with any number of steps."""
    L = capi.load()
    for make, name in ((_ortho, "orthogonalize"), (_muon, "muon_step")):
        a = make(a=coef[0], b=coef[1], c=coef[2], steps=steps)
        size = getattr(L, "az_%s_workspace" % name)(C.byref(a))
        assert (size > 0) == fine, L.az_last_error()
        if not fine:
            rc, msg = _call(name, a)
            assert rc == capi.AZ_E_ARG and "singular values" in msg, msg


@pytest.mark.parametrize("targets", [None, 3.0, "abc", {}])
def test_targets_of_another_kind_are_refused(targets):
    x, w, b = torch.zeros(2, 8, 3, 3), torch.zeros(1, 8), torch.zeros(1)
    for call in (learn.policy_loss, learn.policy_loss_grad):
        with pytest.raises(capi.AzError):
            call(x, w, b, targets)


def test_target_lists_beyond_what_an_int_counts_are_refused():
    """Sixteen small boards' entries are counted together."""
    for cap, word in (((1 << 26) + 1, "too many"), (1 << 27, "too many"), ((1 << 31) - 1, "too many"), (1 << 26, "workspace")):
        rc, msg = _call("policy_loss", _policy(N=1, target=None, counts=P, actions=P, probs=P, cap=cap), None)
        assert rc == capi.AZ_E_ARG and word in msg, msg


@pytest.mark.parametrize("kw,word", [
    (dict(d_features=1 * P), "d_features overlaps features"), (dict(d_features=1 * P + 4 * 81 * 64 * 2 - 2), "d_features overlaps features"), (dict(d_features=2 * P), "d_features overlaps weight"),
    (dict(d_features=3 * P), "d_features overlaps bias"), (dict(d_features=4 * P + 4 * 3 * 81 * 4 - 2), "d_features overlaps target"), (dict(d_features=6 * P), "d_features overlaps row_scale"),
    (dict(d_features=7 * P), "d_features overlaps legal"), (dict(loss=1 * P), "loss overlaps features"), (dict(loss=4 * P), "loss overlaps target"), (dict(loss=6 * P), "loss overlaps row_scale"),
    (dict(loss=8 * P), "loss overlaps d_features"), (dict(stats=9 * P), "d_weight overlaps stats"), (dict(stats=4 * P), "stats overlaps target"), (dict(d_weight=8 * P), "d_weight overlaps d_features"),
    (dict(d_bias=9 * P + 4 * 3 * 64 - 4), "d_bias overlaps d_weight"), (dict(d_bias=5 * P), "d_bias overlaps loss"), (dict(stats_given=1, stats=8 * P, loss=None), "d_features overlaps stats"),
    (dict(target=None, counts=8 * P, actions=11 * P, probs=12 * P, cap=5), "d_features overlaps counts"), (dict(target=None, counts=11 * P, actions=8 * P, probs=12 * P, cap=5), "d_features overlaps actions"),
    (dict(target=None, counts=11 * P, actions=12 * P, probs=8 * P - 4 * 5 * 4 + 4, cap=5), "d_features overlaps probs"),
    (dict(d_weight=2 * P, d_bias=3 * P), "workspace"), (dict(d_features=1 * P + 4 * 81 * 64 * 2), "workspace"), (dict(), "workspace"),
], ids=lambda v: "-".join(v) if isinstance(v, dict) else v.replace(" ", "_"))
def test_policy_loss_gradients_refuse_outputs_that_overlap(kw, word):
    """The tensors lie P apart; "workspace": everything before was in order (the head in place of its own gradient is)."""
    v = dict(dtype=capi.AZ_F16, features=1 * P, weight=2 * P, bias=3 * P, target=4 * P, loss=5 * P, row_scale=6 * P, legal=7 * P, d_features=8 * P, d_weight=9 * P, d_bias=10 * P)
    v.update(kw)
    rc, msg = _call("policy_loss", _policy(**v), None)
    assert rc == capi.AZ_E_ARG and word in msg, msg


def test_more_tiles_than_a_launch_takes_are_refused():
    """Rows of 2^24 elements, 2^18 tiles each: 63 of them are taken, 64 would be 2^32 threads."""
    L = capi.load()
    for make, name in ((_ortho, "orthogonalize"), (_muon, "muon_step")):
        for n, fine in ((63, True), (64, False)):
            strides = {k: 1 << 24 for k, _ in type(make())._fields_ if k.endswith("_stride")}
            at = {k: (i + 1) << 40 for i, k in enumerate(("update", "out") if name == "orthogonalize" else ("grad", "weight", "momentum"))}
            if name == "muon_step":
                at.update(weight_out=at["weight"], momentum_out=at["momentum"])
            a = make(n=n, rows=1, cols=1 << 24, **strides, **at)
            assert (getattr(L, "az_%s_workspace" % name)(C.byref(a)) > 0) == fine
            rc, msg = _call(name, a, None)
            assert rc == capi.AZ_E_ARG and ("workspace" if fine else "too many tiles") in msg, msg
