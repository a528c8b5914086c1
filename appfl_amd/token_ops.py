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

import contextlib
import ctypes as C
import math
from typing import NamedTuple, Optional, Sequence, Tuple

import torch

from . import _native as N
from .ops import _stream

DTYPES = {torch.float32: N.FA_LOGITS_F32, torch.bfloat16: N.FA_LOGITS_BF16, torch.float16: N.FA_LOGITS_F16}
TOP_MAX = N.FA_TOP_MAX


class TokenScores(NamedTuple):
    logprob: Optional[torch.Tensor]        # of the given targets; None without targets
    entropy: torch.Tensor
    lse: torch.Tensor
    top_ids: Optional[torch.Tensor]        # None with top = 0
    top_logprobs: Optional[torch.Tensor]


_here = contextlib.nullcontext()


def _on(device: torch.device):
    """The tensors' device as the current one (launches go to the current device)."""
    return _here if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def _on_device(name: str, t: torch.Tensor, device: Optional[torch.device] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise N.NativeLibraryError(f"libappfl_amd kernels take device tensors; {name} is a CPU tensor")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")


def _shape(name: str, t: torch.Tensor, shape) -> None:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")


def _logits(x: torch.Tensor) -> N.Logits:
    _on_device("logits", x)
    if x.dtype not in DTYPES:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {x.dtype}")
    if x.dim() == 2:
        outer, inner, so, si = 1, x.shape[0], 0, x.stride(0)
    elif x.dim() == 3:
        outer, inner, so, si = x.shape[0], x.shape[1], x.stride(0), x.stride(1)
    else:
        raise ValueError(f"logits must be [rows, vocab] or [batch, rows, vocab], got shape {tuple(x.shape)}")
    vocab = x.shape[-1]
    if vocab < 1 or vocab > N.FA_VOCAB_MAX:
        raise ValueError(f"a vocabulary of {vocab} tokens")
    if x.stride(-1) != 1 and vocab > 1:
        raise ValueError("logits must have adjacent elements along the vocabulary")
    if outer * inner > 0x7FFFFFFF:
        raise ValueError("too many rows")
    return N.Logits(x.data_ptr(), outer, inner, so, si, vocab, DTYPES[x.dtype])


def _list_pair(ids: torch.Tensor, logprobs: torch.Tensor, device: torch.device) -> None:
    _on_device("ids", ids, device)
    _on_device("logprobs", logprobs, device)
    if ids.dtype != torch.int32:
        raise TypeError(f"ids must be int32, got {ids.dtype}")
    if logprobs.dtype != torch.float32:
        raise TypeError(f"logprobs must be float32, got {logprobs.dtype}")
    _shape("logprobs", logprobs, ids.shape)
    k = ids.shape[-1]
    if not 1 <= k <= TOP_MAX:
        raise ValueError(f"lists hold 1..{TOP_MAX} entries, got {k}")
    if k > 1 and (ids.stride(-1) != 1 or logprobs.stride(-1) != 1):
        raise ValueError("a list's entries must be adjacent")


def _workspace(x: N.Logits, top: int, device: torch.device) -> Optional[torch.Tensor]:
    need = C.c_size_t()
    N.check(N.load().fa_token_workspace(C.byref(x), top, C.byref(need)), "fa_token_workspace")
    return torch.empty(need.value, dtype=torch.uint8, device=device) if need.value else None


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def token_scores(logits: torch.Tensor, targets: Optional[torch.Tensor] = None, top: int = 0,
                 ignore_index: int = -100) -> TokenScores:
    """Scores of every row of `logits` (fa_token_scores): ``lse = log sum_v exp x_v``, the entropy
    of ``softmax(x)`` in nats, the log probability of ``targets`` (int64, the shape of the rows; 0
    where it is `ignore_index`, NaN where it is outside the vocabulary) and the `top` most probable
    tokens, best first (ties to the lower id), with their log probabilities."""
    x = _logits(logits)
    device = logits.device
    if not isinstance(top, int) or isinstance(top, bool):
        raise TypeError("top must be an int")
    if not 0 <= top <= min(TOP_MAX, x.vocab):
        raise ValueError(f"top must be in 0..{min(TOP_MAX, x.vocab)}, got {top}")
    lead = logits.shape[:-1]
    if targets is not None:
        _on_device("targets", targets, device)
        if targets.dtype != torch.int64:
            raise TypeError(f"targets must be int64, got {targets.dtype}")
        _shape("targets", targets, lead)
        targets = targets.contiguous()
    with _on(device):
        entropy = torch.empty(lead, dtype=torch.float32, device=device)
        lse = torch.empty(lead, dtype=torch.float32, device=device)
        logprob = torch.empty(lead, dtype=torch.float32, device=device) if targets is not None else None
        ids = torch.empty(lead + (top,), dtype=torch.int32, device=device) if top else None
        tops = torch.empty(lead + (top,), dtype=torch.float32, device=device) if top else None
        ws = _workspace(x, top, device)
        rc = N.load().fa_token_scores(C.byref(x), _ptr(targets), int(ignore_index), top, _ptr(logprob),
                                      entropy.data_ptr(), lse.data_ptr(), _ptr(ids), _ptr(tops), _ptr(ws),
                                      _stream(logits))
        N.check(rc, "fa_token_scores")
    return TokenScores(logprob, entropy, lse, ids, tops)


def merge_tops(ids: torch.Tensor, logprobs: torch.Tensor, weights: Sequence[float], top: int,
               token_weight: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Weighted mean of K clients' answers (fa_merge_tops): `ids` / `logprobs` ``[K, rows, k]``, one
    weight per client (as in :func:`appfl_amd.ops.reduce_opt`), optionally a weight per client and
    row (``[K, rows]`` float32; nothing above zero leaves the client out of the row).  Returns ids
    and log probabilities ``[rows, top]``, best first; id -1 and -inf where a row has fewer tokens."""
    _on_device("ids", ids)
    if ids.dim() != 3:
        raise ValueError(f"ids must be [clients, rows, k], got shape {tuple(ids.shape)}")
    device = ids.device
    _list_pair(ids, logprobs, device)
    K, rows, k = ids.shape
    if len(weights) != K:
        raise ValueError("one weight per client")
    w = [float(v) for v in weights]
    if not 1 <= K <= N.FA_MERGE_CLIENTS or K * k > N.FA_MERGE_ENTRIES:
        raise ValueError(f"one merge takes 1..{N.FA_MERGE_CLIENTS} clients and {N.FA_MERGE_ENTRIES} entries a row, "
                         f"got {K} clients of {k}")
    if not all(v >= 0.0 and math.isfinite(v) for v in w):
        raise ValueError("client weights must be finite and not negative")
    if not isinstance(top, int) or isinstance(top, bool):
        raise TypeError("top must be an int")
    if not 1 <= top <= min(K * k, TOP_MAX):
        raise ValueError(f"top must be in 1..{min(K * k, TOP_MAX)}, got {top}")
    unit_client = unit_row = 0
    if token_weight is not None:
        _on_device("token_weight", token_weight, device)
        if token_weight.dtype != torch.float32:
            raise TypeError(f"token_weight must be float32, got {token_weight.dtype}")
        _shape("token_weight", token_weight, (K, rows))
        unit_client, unit_row = token_weight.stride()
    with _on(device):
        out_ids = torch.empty((rows, top), dtype=torch.int32, device=device)
        out_lp = torch.empty((rows, top), dtype=torch.float32, device=device)
        tops = N.Tops(ids.data_ptr(), logprobs.data_ptr(), ids.stride(0), ids.stride(1), logprobs.stride(0),
                      logprobs.stride(1), _ptr(token_weight), unit_client, unit_row, k)
        rc = N.load().fa_merge_tops(C.byref(tops), N.double_array(w), K, rows, top, out_ids.data_ptr(),
                                    out_lp.data_ptr(), _stream(ids))
        N.check(rc, "fa_merge_tops")
    return out_ids, out_lp


def _teacher(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float,
             row_weight: Optional[torch.Tensor]):
    """The C structure and the tensors it points into (keep them until the call has returned)."""
    lead = logits.shape[:-1]
    device = logits.device
    _list_pair(ids, logprobs, device)
    _shape("ids", ids, lead + ids.shape[-1:])
    tau = float(temperature)
    if not 1e-30 <= tau <= 1e30:
        raise ValueError(f"temperature must be positive and finite, got {temperature}")
    if row_weight is not None:
        _on_device("row_weight", row_weight, device)
        if row_weight.dtype != torch.float32:
            raise TypeError(f"row_weight must be float32, got {row_weight.dtype}")
        _shape("row_weight", row_weight, lead)
        row_weight = row_weight.contiguous()
    k = ids.shape[-1]
    if ids.dim() == 3:                       # rows of a batch have to be one axis with one stride
        ids, logprobs = ids.reshape(-1, k), logprobs.reshape(-1, k)
    t = N.Teacher(ids.data_ptr(), logprobs.data_ptr(), ids.stride(0), logprobs.stride(0), _ptr(row_weight), tau, k)
    return t, (ids, logprobs, row_weight)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, logprobs, temperature, row_weight):
        x = _logits(logits)
        t, keep = _teacher(logits, ids, logprobs, temperature, row_weight)
        device = logits.device
        with _on(device):
            loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=device)
            stat = torch.empty(logits.shape[:-1] + (N.FA_DISTILL_STAT,), dtype=torch.float32, device=device)
            ws = _workspace(x, 0, device)
            N.check(N.load().fa_distill_loss(C.byref(x), C.byref(t), loss.data_ptr(), stat.data_ptr(), _ptr(ws),
                                             _stream(logits)), "fa_distill_loss")
        ctx.save_for_backward(logits, keep[0], keep[1], keep[2], stat)
        ctx.temperature = t.temperature
        return loss

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, row_grad):
        logits, ids, logprobs, row_weight, stat = ctx.saved_tensors
        x = _logits(logits)
        t = N.Teacher(ids.data_ptr(), logprobs.data_ptr(), ids.stride(0), logprobs.stride(0), _ptr(row_weight),
                      ctx.temperature, ids.shape[-1])
        row_grad = row_grad.contiguous()
        with _on(logits.device):
            grad = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            so, si = (0, grad.stride(0)) if grad.dim() == 2 else grad.stride()[:2]
            N.check(N.load().fa_distill_grad(C.byref(x), C.byref(t), stat.data_ptr(), row_grad.data_ptr(),
                                             grad.data_ptr(), so, si, _stream(logits)), "fa_distill_grad")
        return grad, None, None, None, None


def distill_loss(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float = 1.0,
                 row_weight: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Distillation loss of every row, differentiable with respect to `logits` (fa_distill_loss,
    fa_distill_grad).  The teacher's list (`ids` int32, `logprobs` float32 log probabilities or
    logits, ``[rows..., k]``) is made a distribution of its own, ``t = softmax(logprobs / T)``, and
    ``loss = row_weight * T**2 * sum_j t_j (log t_j - log softmax(x / T)[ids_j])``.  Rows of weight 0
    or without an entry have loss and gradient 0; an id outside the vocabulary makes its row NaN."""
    return _Distill.apply(logits, ids, logprobs, temperature, row_weight)


def distill_loss_grad(logits: torch.Tensor, ids: torch.Tensor, logprobs: torch.Tensor, temperature: float = 1.0,
                      row_weight: Optional[torch.Tensor] = None,
                      out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`distill_loss` and the gradient of its sum in one call (fa_distill_loss_grad): the training
    step of a caller that runs the model's backward from the logits' gradient.  `out` receives the
    gradient (the logits' shape and type; `logits` itself: written over them)."""
    x = _logits(logits)
    t, keep = _teacher(logits, ids, logprobs, temperature, row_weight)
    device = logits.device
    with _on(device):
        if out is None:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=device)
        else:
            _check_out(out, logits)
            torch.autograd.graph.increment_version(out)      # a graph that saved it must not use it
        loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=device)
        so, si = (0, out.stride(0)) if out.dim() == 2 else out.stride()[:2]
        ws = _workspace(x, 0, device)
        N.check(N.load().fa_distill_loss_grad(C.byref(x), C.byref(t), loss.data_ptr(), out.data_ptr(), so, si,
                                              _ptr(ws), _stream(logits)), "fa_distill_loss_grad")
    return loss, out


def _span(t: torch.Tensor) -> Tuple[int, int]:
    size = t.element_size()
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * size


def _check_out(out: torch.Tensor, logits: torch.Tensor) -> None:
    _on_device("out", out, logits.device)
    if out.dtype != logits.dtype:
        raise TypeError(f"out must be {logits.dtype}, got {out.dtype}")
    _shape("out", out, logits.shape)
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
