"""The token operators' argument checks, which need no GPU: at the C entries and in Python."""

import ctypes as C
import math

import pytest
import torch

import token_reference as R
from appfl_amd import _native as N
from appfl_amd import token_ops


def _logits(**change):
    f = dict(data=256, outer=2, inner=3, stride_outer=30, stride_inner=10, vocab=10, dtype=0)
    f.update(change)
    return N.Logits(*f.values())


def _teacher(**change):
    f = dict(ids=256, logprobs=256, id_stride=4, lp_stride=4, row_weight=None, temperature=1.0, k=4)
    f.update(change)
    return N.Teacher(*f.values())


def _tops(**change):
    f = dict(ids=256, logprobs=256, id_client=12, id_row=4, lp_client=12, lp_row=4, token_weight=None, unit_client=0,
             unit_row=0, k=4)
    f.update(change)
    return N.Tops(*f.values())


INVALID, ALIGN, LARGE = -1, -2, -4


@pytest.mark.parametrize("change,code", [
    (dict(vocab=0), INVALID), (dict(vocab=-3), INVALID), (dict(outer=-1), INVALID), (dict(inner=-1), INVALID),
    (dict(dtype=3), INVALID), (dict(dtype=-1), INVALID), (dict(stride_outer=-1), INVALID),
    (dict(stride_inner=-1), INVALID), (dict(data=None), INVALID), (dict(data=258), ALIGN),
    (dict(data=257, dtype=1), ALIGN), (dict(outer=1 << 20, inner=1 << 11), LARGE)])
def test_logits_are_checked_by_every_entry(change, code):
    lib = N.load()
    x, t = _logits(**change), _teacher()
    assert lib.fa_token_scores(C.byref(x), None, 0, 0, None, 256, 256, None, None, None) == code
    assert lib.fa_distill_loss(C.byref(x), C.byref(t), 256, 256, None) == code
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), 256, None, 256, 30, 10, None) == code
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), 256, 256, 30, 10, None, None) == code


@pytest.mark.parametrize("change", [
    dict(ids=None), dict(logprobs=None), dict(k=0), dict(k=257), dict(id_stride=-1), dict(lp_stride=-1),
    dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf)])
def test_teachers_are_checked(change):
    lib = N.load()
    x, t = _logits(), _teacher(**change)
    assert lib.fa_distill_loss(C.byref(x), C.byref(t), 256, 256, None) == INVALID
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), 256, None, 256, 30, 10, None) == INVALID
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), 256, 256, 30, 10, None, None) == INVALID


def test_outputs_and_null_pointers_are_checked():
    lib = N.load()
    x, t = _logits(), _teacher()
    scores = lambda **c: lib.fa_token_scores(C.byref(x), *{**dict(
        targets=None, ignore=0, top=0, logprob=None, entropy=256, lse=256, ids=None, lps=None, st=None), **c}.values())
    for change in (dict(entropy=None), dict(lse=None), dict(targets=256), dict(top=2), dict(top=2, ids=256), dict(top=11),
                   dict(top=-1)):
        assert scores(**change) == INVALID, change
    x.vocab = 1000
    assert scores(top=129, ids=256, lps=256) == INVALID
    x.vocab = 10
    assert lib.fa_distill_loss(C.byref(x), None, 256, 256, None) == INVALID
    assert lib.fa_distill_loss(C.byref(x), C.byref(t), None, 256, None) == INVALID
    assert lib.fa_distill_loss(C.byref(x), C.byref(t), 256, None, None) == INVALID
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), None, None, 256, 30, 10, None) == INVALID
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), 256, None, None, 30, 10, None) == INVALID
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), 256, None, 256, -1, 10, None) == INVALID
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), 256, None, 258, 30, 10, None) == ALIGN
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), 256, None, 30, 10, None, None) == INVALID
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), None, 256, 30, 10, None, None) == INVALID
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), 256, 256, 30, -10, None, None) == INVALID
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), 256, 257, 30, 10, None, None) == ALIGN
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), 256, 256, 30, 10, 258, None) == ALIGN


def test_merge_arguments_are_checked():
    lib = N.load()
    w = N.double_array([0.25] * 4)
    merge = lambda tops=_tops(), w=w, K=4, rows=3, top=4, ids=256, lps=256: lib.fa_merge_tops(
        C.byref(tops) if tops else None, w, K, rows, top, ids, lps, None)
    assert merge(tops=None) == INVALID and merge(w=None) == INVALID
    assert merge(K=0) == INVALID and merge(K=129) == INVALID and merge(rows=-1) == INVALID
    assert merge(top=0) == INVALID and merge(top=17) == INVALID and merge(ids=None) == INVALID and merge(lps=None) == INVALID
    assert merge(w=N.double_array([1.0, -1.0, 1.0, 1.0])) == INVALID
    assert merge(w=N.double_array([1.0, math.nan, 1.0, 1.0])) == INVALID
    assert merge(w=N.double_array([1.0, math.inf, 1.0, 1.0])) == INVALID
    assert merge(rows=1 << 31) == LARGE
    assert merge(tops=_tops(k=256), w=N.double_array([1.0] * 33), K=33) == LARGE
    for change in (dict(k=0), dict(k=257), dict(ids=None), dict(logprobs=None), dict(id_client=-1), dict(id_row=-1),
                   dict(lp_client=-1), dict(lp_row=-1), dict(unit_client=-1), dict(unit_row=-1)):
        assert merge(tops=_tops(**change)) == INVALID, change


def test_empty_calls_do_nothing():
    lib = N.load()
    x, t = _logits(outer=0, data=None), _teacher()
    assert lib.fa_token_scores(C.byref(x), None, 0, 0, None, None, None, None, None, None) == 0
    assert lib.fa_distill_loss(C.byref(x), C.byref(t), None, None, None) == 0
    assert lib.fa_distill_grad(C.byref(x), C.byref(t), None, None, None, 0, 0, None) == 0
    assert lib.fa_distill_loss_grad(C.byref(x), C.byref(t), None, None, 0, 0, None, None) == 0
    tops = _tops()
    assert lib.fa_merge_tops(C.byref(tops), N.double_array([1.0]), 1, 0, 4, None, None, None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 5)
    ids, lp = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, 3)
    for call in (lambda: token_ops.token_scores(x), lambda: token_ops.distill_loss(x, ids, lp),
                 lambda: token_ops.distill_loss_grad(x, ids, lp), lambda: token_ops.merge_tops(ids[None], lp[None], [1.0], 1)):
        with pytest.raises(N.NativeLibraryError):
            call()
    with pytest.raises(TypeError):
        token_ops.token_scores([1.0, 2.0])


def test_reference_agrees_with_torch():
    """The plain forms the GPU tests compare with, against torch's own in 64 bits."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4, 33, generator=g, dtype=torch.float64) * 3
    t = torch.tensor([0, 5, -100, 32])
    want = torch.log_softmax(x, dim=1)
    out, _ = R.scores(x, t, 33)
    assert torch.allclose(out["logprob"][[0, 1, 3]], want[[0, 1, 3], t[[0, 1, 3]]]) and float(out["logprob"][2]) == 0
    assert torch.allclose(out["entropy"], -(want.exp() * want).sum(1)) and torch.allclose(out["lse"], torch.logsumexp(x, 1))
    assert torch.equal(out["top_ids"].long(), x.argsort(1, descending=True))
    ids = torch.stack([torch.randperm(33, generator=g)[:5] for _ in range(4)]).to(torch.int32)
    lp = torch.randn(4, 5, generator=g)
    leaf = x.clone().requires_grad_(True)
    target = torch.zeros(4, 33, dtype=torch.float64).scatter_(1, ids.long(), torch.softmax(lp.double() / 2, 1))
    kl = torch.nn.functional.kl_div(torch.log_softmax(leaf / 2, 1), target, reduction="none").sum(1) * 4
    kl.sum().backward()
    loss, grad, _, _ = R.distill(x, ids, lp, 2.0)
    assert torch.allclose(loss, kl.detach()) and torch.allclose(grad, leaf.grad)


def test_the_package_imports_without_a_gpu_build_of_torch():
    """Such a build lacks the calls that read the current stream and device; host tensors are refused as ever."""
    import os
    import subprocess
    import sys

    code = ("import torch\n"
            "for name in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, name): delattr(torch._C, name)\n"
            "import appfl_amd, appfl_amd.aggregator\n"
            "from appfl_amd import _native, token_ops\n"
            "try: token_ops.token_scores(torch.zeros(2, 5))\n"
            "except _native.NativeLibraryError: print('refused')\n")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    done = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=600)
    assert done.returncode == 0 and done.stdout.strip() == "refused", done.stderr
