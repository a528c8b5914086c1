"""Aggregation by distillation: the clients send what their models ANSWER on a public set, not the
models, so that they may differ in architecture, in size or in what they are allowed to share.

A client's update is a dict of CPU tensors like any other update, with the entries

* ``top_ids``       ``[rows, k]``  the k most probable tokens (classes) of every position, negative: none
* ``top_logprobs``  ``[rows, k]``  their log probabilities
* ``token_weight``  ``[rows]``     optional, how much the client's answer to each position counts

(`answer` makes the first two from logits); k may differ between clients.  `aggregate` returns their
client-weighted mean, cut to `top` entries, in the same form -- the teacher every client then learns
from, and the server's own model through `loss`.  The weights are FedAvg's
(algorithm/aggregator/fedavg_aggregator.py:343-358: data share or equal); the class has no
counterpart among the reference's aggregators.
"""

from __future__ import annotations

import math
from typing import Any, Dict, List, Optional, Tuple

import torch

from .. import token_ops
from .base_aggregator import BaseAggregator, DeviceStateMixin, cfg_get, resolve_device


class FedDistillAggregator(BaseAggregator, DeviceStateMixin):
    """
    :param `model`: optional model; `get_parameters` hands out its state before the first round.
    :param `aggregator_configs`: `client_weights_mode` ("equal" or "sample_size"), `top` (entries of
        the teacher's lists, with absent ones behind where a round brings fewer; default: as many as
        the longest client list), `temperature` (of `loss`, default 1.0), `device`.
    :param `logger`: optional logger.
    """

    def __init__(self, model: Optional[torch.nn.Module] = None, aggregator_configs: Any = None,
                 logger: Optional[Any] = None):
        self.model = model
        self.logger = logger
        self.aggregator_configs = aggregator_configs if aggregator_configs is not None else {}
        self.client_weights_mode = cfg_get(self.aggregator_configs, "client_weights_mode", "equal")
        self.top = cfg_get(self.aggregator_configs, "top", None)
        self.temperature = float(cfg_get(self.aggregator_configs, "temperature", 1.0))
        self.device = resolve_device(self.aggregator_configs)
        self.teacher: Optional[Tuple[torch.Tensor, torch.Tensor]] = None      # ids, log probabilities on the device
        self._init_lock()

    def get_parameters(self, **kwargs) -> Dict:
        with self._lock:
            if self.teacher is not None:
                return self._download()
            if self.model is None:
                raise ValueError("Model is not provided to the aggregator.")
            with torch.no_grad():
                return {k: v.clone().detach() for k, v in self.model.state_dict().items()}

    def aggregate(self, local_models: Dict, **kwargs) -> Dict[str, torch.Tensor]:
        with self._lock:
            if not local_models:
                raise ValueError("no client answers to aggregate")
            ids, logprobs, unit = self._stack(local_models)
            top = int(self.top) if self.top is not None else ids.shape[2]
            most = ids.shape[0] * ids.shape[2]                   # entries a row can have; behind them absent ones
            merged = token_ops.merge_tops(ids, logprobs, self._weights(local_models),
                                          top if top > token_ops.TOP_MAX else min(top, most), token_weight=unit)
            if top > most:
                merged = tuple(torch.nn.functional.pad(t, (0, top - most), value=v) for t, v in zip(merged, (-1, -math.inf)))
            self.teacher = merged
            return self._download()

    def answer(self, logits: torch.Tensor, targets: Optional[torch.Tensor] = None) -> Dict[str, torch.Tensor]:
        """A client's update from its model's logits (``[rows, vocab]`` or ``[batch, rows, vocab]`` on
        the GPU), as tensors of that GPU with one row per position, with the `entropy` of every
        position and, if `targets` are given, their `logprob`.  The lists hold `top` entries, or
        as many as there are tokens (classes), and at most 128."""
        if self.top is None:
            raise ValueError("answer needs the configuration's `top`")
        top = min(int(self.top), token_ops.SCORES_TOP_MAX)
        if isinstance(logits, torch.Tensor) and logits.dim():
            top = min(top, logits.shape[-1])
        s = token_ops.token_scores(logits, targets, top=top)
        out = {"top_ids": s.top_ids.flatten(0, -2), "top_logprobs": s.top_logprobs.flatten(0, -2),
               "entropy": s.entropy.flatten()}
        if targets is not None:
            out["logprob"] = s.logprob.flatten()
        return out

    def loss(self, logits: torch.Tensor, first: int = 0, row_weight: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Distillation losses of positions ``first .. first + rows`` against the current teacher,
        differentiable with respect to `logits` (on the aggregator's GPU; ``[rows, vocab]`` or
        ``[batch, rows, vocab]``, batch-major positions)."""
        ids, logprobs = self._teacher_rows(logits, first)
        return token_ops.distill_loss(logits, ids, logprobs, temperature=self.temperature, row_weight=row_weight)

    def loss_grad(self, logits: torch.Tensor, first: int = 0, row_weight: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """`loss` and the gradient of its sum in one call, for a caller that continues the backward
        pass from the logits' gradient."""
        ids, logprobs = self._teacher_rows(logits, first)
        return token_ops.distill_loss_grad(logits, ids, logprobs, temperature=self.temperature,
                                           row_weight=row_weight, out=out)

    # ---- helpers ---------------------------------------------------------------------------------

    def _teacher_rows(self, logits: torch.Tensor, first: int):
        with self._lock:
            if self.teacher is None:
                raise ValueError("no answers have been aggregated yet")
            ids, logprobs = self.teacher
            # the caller's stream may still read them when a later round replaces them
            stream = torch.cuda.current_stream(self.device)
            ids.record_stream(stream)
            logprobs.record_stream(stream)
        lead = tuple(logits.shape[:-1])
        rows = 1
        for n in lead:
            rows *= n
        if not 0 <= first <= first + rows <= ids.shape[0]:
            raise ValueError(f"positions {first}..{first + rows} of a teacher of {ids.shape[0]}")
        part = slice(first, first + rows)
        shape = lead + (ids.shape[1],)
        return ids[part].view(shape), logprobs[part].view(shape)

    def _weights(self, local_models: Dict) -> List[float]:
        sizes = getattr(self, "client_sample_size", None) or {}
        total = sum(sizes.get(c, 0) for c in local_models)
        if self.client_weights_mode == "sample_size" and total > 0 and all(c in sizes for c in local_models):
            return [sizes[c] / total for c in local_models]
        return [1.0 / len(local_models)] * len(local_models)

    def _stack(self, local_models: Dict):
        """The clients' lists as [K, rows, k] device tensors; shorter lists end with absent entries."""
        updates = list(local_models.values())
        rows = k = None
        for c, u in local_models.items():
            for name in ("top_ids", "top_logprobs"):
                if name not in u:
                    raise KeyError(name)
            ids, lp = u["top_ids"], u["top_logprobs"]
            if ids.dim() != 2 or ids.shape != lp.shape:
                raise ValueError(f"client {c}: top_ids and top_logprobs must be [rows, k], got {tuple(ids.shape)} "
                                 f"and {tuple(lp.shape)}")
            if ids.dtype not in (torch.int32, torch.int64) or not lp.dtype.is_floating_point:
                raise TypeError(f"client {c}: top_ids must be integers and top_logprobs floats, got {ids.dtype} and {lp.dtype}")
            if rows is None:
                rows, k = ids.shape
            if ids.shape[0] != rows:
                raise ValueError(f"client {c} answers {ids.shape[0]} positions, the others {rows}")
            if ids.dtype == torch.int64 and ids.numel() and int(ids.max()) > 0x7FFFFFFF:
                raise ValueError(f"client {c}: a token id beyond 31 bits")
            w = u.get("token_weight")
            if w is not None and tuple(w.shape) != (rows,):
                raise ValueError(f"client {c}: token_weight has shape {tuple(w.shape)}, expected {(rows,)}")
            k = max(k, ids.shape[1])
        K = len(updates)
        host_ids = torch.full((K, rows, k), -1, dtype=torch.int32, pin_memory=True)
        host_lp = torch.full((K, rows, k), float("-inf"), dtype=torch.float32, pin_memory=True)
        unit = None
        if any(u.get("token_weight") is not None for u in updates):
            unit = torch.ones((K, rows), dtype=torch.float32, pin_memory=True)
        for i, u in enumerate(updates):
            n = u["top_ids"].shape[1]
            host_ids[i, :, :n].copy_(u["top_ids"].detach().clamp(min=-1))
            host_lp[i, :, :n].copy_(u["top_logprobs"].detach())
            if u.get("token_weight") is not None:
                unit[i].copy_(u["token_weight"].detach())
        up = lambda t: None if t is None else t.to(self.device, non_blocking=True)
        return up(host_ids), up(host_lp), up(unit)

    def _download(self) -> Dict[str, torch.Tensor]:
        ids, logprobs = self.teacher
        return {"top_ids": ids.cpu(), "top_logprobs": logprobs.cpu()}
