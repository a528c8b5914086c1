"""Operators on answers: log probabilities and top alternatives of logits, the merge of the clients'
top lists, and distillation from such lists with its gradient.

A federation whose clients cannot share weights (other architectures, models too large to send)
shares what its models answer on a public set: for every position the most probable tokens (or
classes) with their log probabilities.  `token_scores` makes such answers from logits, `merge_tops`
is the client-weighted mean of them (what :func:`appfl_amd.ops.reduce_opt` is for weights), and
`distill_loss` / `distill_loss_grad` teach a model the merged answers.

Every function enqueues its kernels on the CURRENT torch stream of the tensors' device and returns
at once; results are new tensors of that device.  Logits are fp32, bfloat16 or float16 of shape
``[rows, vocab]`` or ``[batch, rows, vocab]`` with adjacent elements along the vocabulary and any
other strides (``logits[:, :-1]`` is taken as it is).  Lists hold int32 ids (negative: absent) and
fp32 log probabilities.  The arithmetic is in ``libappfl_amd.so``.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _native as N

DTYPES = {torch.float32: N.FA_LOGITS_F32, torch.bfloat16: N.FA_LOGITS_BF16, torch.float16: N.FA_LOGITS_F16}
TOP_MAX, SCORES_TOP_MAX = N.FA_TOP_MAX, N.FA_SCORES_TOP_MAX

# The smallest calls take less time on the GPU than in Python, so the checks below look at each
# property once, the stream's handle is read without making a Stream object, and results are
# allocated without the dispatcher (0.7 instead of 1.4-1.9 us each) where torch has those calls.  A
# torch that was built without a GPU lacks them, and imports this module all the same.
_f32, _i32, _i64 = torch.float32, torch.int32, torch.int64

try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream, _cuda_getDevice as _current_device
except ImportError:
    def _raw_stream(index):
        return torch.cuda.current_stream(index).cuda_stream

    _current_device = torch.cuda.current_device

try:
    from torch._C._dynamo.guards import _empty_strided_cuda as _empty_strided
except ImportError:
    def _empty_strided(shape, stride, dtype):
        return torch.empty_strided(shape, stride, dtype=dtype, device="cuda")


def _new(shape, dtype: torch.dtype) -> torch.Tensor:
    """A contiguous tensor on the current device."""
    if len(shape) == 1:
        return _empty_strided((shape[0],), (1,), dtype)
    if len(shape) == 2:
        return _empty_strided((shape[0], shape[1]), (shape[1], 1), dtype)
    return torch.empty(shape, dtype=dtype, device="cuda")


class TokenScores(NamedTuple):
    logprob: Optional[torch.Tensor]        # of the given targets; None without targets
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: Optional[torch.Tensor]        # None with top = 0
    top_logprobs: Optional[torch.Tensor]


def _check(name: str, t: torch.Tensor, dtype: torch.dtype, index: int, shape) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise N.NativeLibraryError(f"libappfl_amd kernels take device tensors; {name} is a CPU tensor")
    if t.get_device() != index:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{index}")
    if t.dtype is not dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _logits(x: torch.Tensor) -> N.Logits:
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"logits must be a tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise N.NativeLibraryError("libappfl_amd kernels take device tensors; logits is a CPU tensor")
    code = DTYPES.get(x.dtype)
    if code is None:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {x.dtype}")
    shape, stride = x.shape, x.stride()
    if len(shape) == 2:
        outer, inner, so, si = 1, shape[0], 0, stride[0]
    elif len(shape) == 3:
        outer, inner, so, si = shape[0], shape[1], stride[0], stride[1]
    else:
        raise ValueError(f"logits must be [rows, vocab] or [batch, rows, vocab], got shape {tuple(shape)}")
    vocab = shape[-1]
    if not 1 <= vocab <= N.FA_VOCAB_MAX:
        raise ValueError(f"a vocabulary of {vocab} tokens")
    if stride[-1] != 1 and vocab > 1:
        raise ValueError("logits must have adjacent elements along the vocabulary")
    if outer * inner > 0x7FFFFFFF:
        raise ValueError("too many rows")
    return N.Logits(x.data_ptr(), outer, inner, so, si, vocab, code)


def _lists(ids: torch.Tensor, logprobs: torch.Tensor, index: int, lead) -> int:
    """Checks a pair of lists for rows of shape `lead`; their length."""
    if not isinstance(ids, torch.Tensor):
        raise TypeError(f"ids must be a tensor, got {type(ids).__name__}")
    shape = ids.shape
    k = shape[-1] if len(shape) else 0
    _check("ids", ids, _i32, index, lead + (k,))
    _check("logprobs", logprobs, _f32, index, shape)
    if not 1 <= k <= TOP_MAX:
        raise ValueError(f"lists hold 1..{TOP_MAX} entries, got {k}")
    if k > 1 and (ids.stride(-1) != 1 or logprobs.stride(-1) != 1):
        raise ValueError("a list's entries must be adjacent")
    return k


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def token_scores(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0,
                 ignore_index: int = -100) -> TokenScores:
    """Scores of every row of `logits` (fa_token_scores): ``lse = log sum_v exp x_v``, the entropy
    of ``softmax(x)`` in nats, the log probability of ``targets`` (int64, the shape of the rows; 0
    where it is `ignore_index`, NaN where it is outside the vocabulary) and the `top` most probable
    tokens, best first (ties to the lower id), with their log probabilities.  The results carry no
    gradient, also of logits that require one."""
    x = _logits(logits)
    index = logits.get_device()
    if _current_device() != index:           # launches go to the current device
        with torch.cuda.device(index):
            return token_scores(logits, targets, top, ignore_index)
    if type(top) is not int:
        raise TypeError("top must be an int")
    if not 0 <= top <= min(N.FA_SCORES_TOP_MAX, x.vocab):
        raise ValueError(f"top must be in 0..{min(N.FA_SCORES_TOP_MAX, x.vocab)}, got {top}")
    lead = logits.shape[:-1]
    logprob = ids = tops = None
    if targets is not None:
        _check("targets", targets, _i64, index, lead)
        targets = targets.contiguous()
        logprob = _new(lead, _f32)
    entropy = _new(lead, _f32)
    lse = _new(lead, _f32)
    if top:
        ids = _new((*lead, top), _i32)
        tops = _new((*lead, top), _f32)
    rc = N.load().fa_token_scores(C.byref(x), _ptr(targets), ignore_index, top, _ptr(logprob), entropy.data_ptr(),
                                  lse.data_ptr(), _ptr(ids), _ptr(tops), _raw_stream(index))
    if rc:
        N.check(rc, "fa_token_scores")
    return TokenScores(logprob, entropy, lse, ids, tops)


def merge_tops(ids: torch.Tensor, logprobs: torch.Tensor, weights: Sequence[float], top: int,
               token_weight: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Weighted mean of K clients' answers (fa_merge_tops): `ids` / `logprobs` ``[K, rows, k]``, one
    weight per client (as in :func:`appfl_amd.ops.reduce_opt`), optionally a weight per client and
    row (``[K, rows]`` float32; nothing above zero leaves the client out of the row).  Returns ids
    and log probabilities ``[rows, top]``, best first; id -1 and -inf where a row has fewer tokens."""
    if not isinstance(ids, torch.Tensor):
        raise TypeError(f"ids must be a tensor, got {type(ids).__name__}")
    if ids.dim() != 3:
        raise ValueError(f"ids must be [clients, rows, k], got shape {tuple(ids.shape)}")
    index = ids.get_device()
    K, rows, _ = ids.shape
    k = _lists(ids, logprobs, index, ids.shape[:2])
    if _current_device() != index:
        with torch.cuda.device(index):
            return merge_tops(ids, logprobs, weights, top, token_weight)
    if len(weights) != K:
        raise ValueError("one weight per client")
    if not 1 <= K <= N.FA_MERGE_CLIENTS or K * k > N.FA_MERGE_ENTRIES:
        raise ValueError(f"one merge takes 1..{N.FA_MERGE_CLIENTS} clients and {N.FA_MERGE_ENTRIES} entries a row, "
                         f"got {K} clients of {k}")
    try:
        w = N.double_array(weights)
    except TypeError:                        # 0-d tensors, other libraries' numbers
        w = N.double_array([float(v) for v in weights])
    if not all(0.0 <= v < math.inf for v in w):
        raise ValueError("client weights must be finite and not negative")
    if type(top) is not int:
        raise TypeError("top must be an int")
    if not 1 <= top <= min(K * k, TOP_MAX):
        raise ValueError(f"top must be in 1..{min(K * k, TOP_MAX)}, got {top}")
    unit, unit_stride = None, (0, 0)
    if token_weight is not None:
        _check("token_weight", token_weight, _f32, index, ids.shape[:2])
        unit, unit_stride = token_weight.data_ptr(), token_weight.stride()
    out_ids = _new((rows, top), _i32)
    out_lp = _new((rows, top), _f32)
    tops = N.Tops(ids.data_ptr(), logprobs.data_ptr(), *ids.stride()[:2], *logprobs.stride()[:2], unit, *unit_stride, k)
    rc = N.load().fa_merge_tops(C.byref(tops), w, K, rows, top, out_ids.data_ptr(), out_lp.data_ptr(), _raw_stream(index))
    if rc:
        N.check(rc, "fa_merge_tops")
    return out_ids, out_lp


def _teacher(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float,
             row_weight: Optional[torch.Tensor]):
    """The C structure and the tensors it points into (keep them until the call has returned)."""
    lead = logits.shape[:-1]
    index = logits.get_device()
    k = _lists(ids, logprobs, index, lead)
    tau = float(temperature)
    if not 1e-3 <= tau <= 1e3:
        raise ValueError(f"temperature must be in 1e-3..1e3, got {temperature}")
    if row_weight is not None:
        _check("row_weight", row_weight, _f32, index, lead)
        row_weight = row_weight.contiguous()
    if len(lead) == 2:                       # rows of a batch have to be one axis with one stride
        ids, logprobs = ids.reshape(-1, k), logprobs.reshape(-1, k)
    t = N.Teacher(ids.data_ptr(), logprobs.data_ptr(), ids.stride(0), logprobs.stride(0), _ptr(row_weight), tau, k)
    return t, (ids, logprobs, row_weight)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, temperature, row_weight):
        x = _logits(logits)                  # the logits' device is the current one here and in backward
        t, keep = _teacher(logits, ids, logprobs, temperature, row_weight)
        lead = logits.shape[:-1]
        loss = _new(lead, _f32)
        stat = _new((x.outer * x.inner, N.FA_DISTILL_STAT), _f32)
        rc = N.load().fa_distill_loss(C.byref(x), C.byref(t), loss.data_ptr(), stat.data_ptr(),
                                      _raw_stream(logits.get_device()))
        if rc:
            N.check(rc, "fa_distill_loss")
        ctx.save_for_backward(logits, stat, *keep)
        ctx.call = x, t, logits.stride(), t.id_stride, t.lp_stride
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, row_grad):
        # Python costs three times as much in autograd's threads: the forward call's structures are used
        # again, unless hooks on saved tensors handed back other memory than was saved.  They are never
        # written to: another backward pass of the graph may be under way.
        logits, stat, ids, logprobs, row_weight = ctx.saved_tensors
        x, t, strides, id_stride, lp_stride = ctx.call
        if (logits.data_ptr() != (x.data or 0) or ids.data_ptr() != (t.ids or 0) or
                logprobs.data_ptr() != (t.logprobs or 0) or (_ptr(row_weight) or 0) != (t.row_weight or 0) or
                logits.stride() != strides or ids.stride(0) != id_stride or logprobs.stride(0) != lp_stride):
            x = _logits(logits)
            t = N.Teacher(ids.data_ptr(), logprobs.data_ptr(), ids.stride(0), logprobs.stride(0), _ptr(row_weight),
                          t.temperature, t.k)
        if not row_grad.is_contiguous():
            row_grad = row_grad.contiguous()
        grad = _new(logits.shape, logits.dtype)
        rc = N.load().fa_distill_grad(C.byref(x), C.byref(t), stat.data_ptr(), row_grad.data_ptr(), grad.data_ptr(),
                                      x.inner * x.vocab, x.vocab, _raw_stream(logits.get_device()))
        if rc:
            N.check(rc, "fa_distill_grad")
        return grad, None, None, None, None


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float = 1.0,
                 row_weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Distillation loss of every row, differentiable with respect to `logits` (fa_distill_loss,
    fa_distill_grad).  The teacher's list (`ids` int32, `logprobs` float32 log probabilities or
    logits, ``[rows..., k]``) is made a distribution of its own, ``t = softmax(logprobs / T)``, and
    ``loss = row_weight * T**2 * sum_j t_j (log t_j - log softmax(x / T)[ids_j])``.  Rows of weight 0
    or without an entry have loss and gradient 0; an id outside the vocabulary makes its row NaN.
    Only `logits` get a gradient: `logprobs` and `row_weight` are taken as constants, also where they
    require one.  The log probabilities are fp32, off by some ``2**-20``, the loss by ``T**2`` times
    that: 2e-5 at ``T = 4``, but 1e-2 at 100 and 1 at 1000."""
    if isinstance(logits, torch.Tensor) and logits.is_cuda and _current_device() != logits.get_device():
        with torch.cuda.device(logits.get_device()):
            return _Distill.apply(logits, ids, logprobs, temperature, row_weight)
    return _Distill.apply(logits, ids, logprobs, temperature, row_weight)


def distill_loss_grad(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float = 1.0,
                      row_weight: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`distill_loss` and the gradient of its sum in one call (fa_distill_loss_grad): the training
    step of a caller that runs the model's backward from the logits' gradient.  `out` receives the
    gradient (the logits' shape and type; `logits` itself: written over them)."""
    x = _logits(logits)
    index = logits.get_device()
    if _current_device() != index:
        with torch.cuda.device(index):
            return distill_loss_grad(logits, ids, logprobs, temperature, row_weight, out)
    t, keep = _teacher(logits, ids, logprobs, temperature, row_weight)
    lead = logits.shape[:-1]
    if out is None:
        out = _new(logits.shape, logits.dtype)
        so, si = x.inner * x.vocab, x.vocab
    else:
        _check_out(out, logits)
        torch.autograd.graph.increment_version(out)          # a graph that saved it must not use it
        so, si = (0, out.stride(0)) if len(lead) == 1 else out.stride()[:2]
    loss = _new(lead, _f32)
    ws = None
    if x.outer * x.inner <= N.FA_DISTILL_WS_ROWS and x.vocab * logits.element_size() >= N.FA_DISTILL_WS_BYTES:
        ws = _new((N.FA_DISTILL_WS_FLOATS,), _f32)
    rc = N.load().fa_distill_loss_grad(C.byref(x), C.byref(t), loss.data_ptr(), out.data_ptr(), so, si, _ptr(ws),
                                       _raw_stream(index))
    if rc:
        N.check(rc, "fa_distill_loss_grad")
    return loss, out


def _span(t: torch.Tensor) -> Tuple[int, int]:
    size = t.element_size()
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * size


def _check_out(out: torch.Tensor, logits: torch.Tensor) -> None:
    _check("out", out, logits.dtype, logits.get_device(), logits.shape)
    if out.numel() == 0:
        return
    strides = sorted((s, n) for s, n in zip(out.stride(), out.shape) if n > 1)
    reach = 1
    for s, n in strides:                     # every stride past all that the smaller ones reach: no overlap
        if s < reach:
            raise ValueError("out's rows overlap")
        reach = s * (n - 1) + reach
    if out.shape[-1] > 1 and out.stride(-1) != 1:
        raise ValueError("out must have adjacent elements along the vocabulary")
    same = out.data_ptr() == logits.data_ptr() and out.stride() == logits.stride()
    a, b = _span(out), _span(logits)
    if not same and a[0] < b[1] and b[0] < a[1]:
        raise ValueError("out overlaps logits; pass logits itself to write the gradient over them")
