"""The token operators in 64 bits, plainly, on the CPU, with the bounds their fp32 kernels are held to."""

import math

import torch

EPS = 2.0 ** -22     # an fp32 operation is off by 2^-24 of its result; a term goes through exp2 (1 ulp = 2^-23) and
                     # the scaling of its argument on top, so 2^-22 covers each term and each addition


def _chain(vocab):
    """Longest chain of additions (and rescalings) a value goes through: a lane's share of a row when one
    wave of 64 lanes takes it all, plus the joins of lanes, waves and parts."""
    return vocab / 64 + 64


def softmax_terms(x, tau=1.0):
    """x [rows, vocab] double -> peak, distance in log2 units (0 where p = 0), sum, p; a row of -inf has p = 0."""
    peak = x.amax(dim=1, keepdim=True)
    ref = torch.where(peak == -math.inf, torch.zeros_like(peak), peak)
    d = (x - ref) / tau
    t = d.exp()
    s = t.sum(dim=1, keepdim=True)
    p = torch.where(s == 0, torch.zeros_like(t), t / s)
    y = torch.where(t == 0, torch.zeros_like(d), d.abs() / math.log(2))
    return peak, y, s, p


def delta(vocab, mean_y):
    """Relative error of a row's sum of exponentials: every term's own (its argument is rounded
    relative to its size) and the additions."""
    return EPS * (_chain(vocab) + 2 + mean_y)


def scores(x, targets, top, ignore_index=-100):
    """(values, bounds) of a [rows, vocab] tensor of any float type; targets [rows] int64 or None."""
    vocab = x.shape[1]
    x = x.double()
    peak, y, s, p = softmax_terms(x)
    lse = (peak + s.log()).squeeze(1)
    lse = torch.where(peak.squeeze(1) == -math.inf, peak.squeeze(1), lse)
    mean_y = (p * y).sum(dim=1)
    nat = torch.where(p == 0, torch.zeros_like(x), s.log() - (x - peak))
    entropy = torch.where(s.squeeze(1) == 0, torch.zeros_like(lse), (p * nat).sum(dim=1))
    entropy = torch.where(s.squeeze(1).isnan(), s.squeeze(1), entropy)
    d = delta(vocab, mean_y)
    finite = lambda v: torch.where(v.isfinite(), v.abs(), torch.zeros_like(v))
    out = {"lse": lse, "entropy": entropy}
    tol = {"lse": d + EPS * (finite(lse) + finite(peak.squeeze(1))),
           "entropy": d * (2 + 2 * mean_y) + EPS * (1 + finite(entropy) + mean_y)}

    def log_p(v):
        row = lambda c: c.reshape([-1] + [1] * (v.dim() - 1)).expand_as(v)
        r = (v - row(peak)) - row(s.log())             # not v - lse: a peak of -1e38 swallows the logarithm
        r = torch.where(v == -math.inf, torch.full_like(r, -math.inf), r)
        return torch.where(row(s.isnan()), torch.full_like(r, math.nan), r)

    if targets is not None:
        inside = (targets >= 0) & (targets < vocab)
        lp = log_p(x.gather(1, targets.clamp(0, vocab - 1)[:, None]).squeeze(1))
        lp = torch.where(inside, lp, torch.full_like(lp, math.nan))
        lp = torch.where(targets == ignore_index, torch.zeros_like(lp), lp)
        out["logprob"], tol["logprob"] = lp, d + EPS * (finite(lp) + 1)
    if top:
        key = torch.where(x.isnan(), torch.full_like(x, math.inf), x)
        nan_first = torch.where(x.isnan(), torch.ones_like(x), torch.zeros_like(x))
        # NaN before everything, then by value, then by index: a stable sort, the last key first
        order = torch.argsort(key + 0.0, dim=1, descending=True, stable=True)
        order = order.gather(1, torch.argsort(nan_first.gather(1, order), dim=1, descending=True, stable=True))
        ids = order[:, :top]
        lp = log_p(x.gather(1, ids))
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), lp
        tol["top_logprobs"] = d[:, None] + EPS * (finite(lp) + 1)
    return out, tol


def distill(x, ids, lp, tau, row_weight=None, row_grad=None):
    """Losses, gradients and their bounds for [rows, vocab] logits of any float type."""
    dtype = x.dtype
    rows, vocab = x.shape
    xd = x.double()
    w = torch.ones(rows, dtype=torch.float64) if row_weight is None else row_weight.double()
    g = torch.ones(rows, dtype=torch.float64) if row_grad is None else row_grad.double()
    loss, grad = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, vocab, dtype=torch.float64)
    loss_tol, grad_tol = torch.zeros_like(loss), torch.zeros_like(grad)
    half_ulp = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + 2.0 ** -125   # underflow of type and exp2
    for r in range(rows):
        keep = (ids[r] >= 0) & (lp[r] != -math.inf)
        if float(w[r]) == 0.0 or not bool(keep.any()):
            continue
        if bool((ids[r] >= vocab).any()) or bool(lp[r][ids[r] >= 0].isnan().any()):
            loss[r] = math.nan
            grad[r] = math.nan
            continue
        idx = ids[r][keep].long()
        log_t = torch.log_softmax(lp[r][keep].double() / tau, dim=0)
        t = log_t.exp()
        peak, y, s, q = softmax_terms(xd[r:r + 1], tau)
        peak, y, s, q = peak[0, 0], y[0], s[0, 0], q[0]
        log_q = (xd[r] - peak) / tau - s.log() if peak != -math.inf else torch.full_like(xd[r], -math.inf)
        lq = log_q[idx]
        loss[r] = w[r] * tau ** 2 * (t * (log_t - lq)).sum()
        d = delta(vocab, float((q * y).sum()))
        spread = float((t * (log_t.max() - log_t)).sum()) / math.log(2)
        d_t = EPS * (len(idx) + 4 + spread)
        err = (t * ((log_t - lq).abs() * (d_t + EPS * (2 + (log_t.max() - log_t)))
                    + EPS * (log_t.abs() + lq.abs() + 1) + d + d_t)).sum()
        loss_tol[r] = abs(float(w[r])) * tau ** 2 * float(err) + EPS * abs(float(loss[r]))
        target = torch.zeros(vocab, dtype=torch.float64).index_add_(0, idx, t)
        slack = torch.zeros(vocab, dtype=torch.float64).index_add_(
            0, idx, t * (d_t + EPS * (2 + (log_t.max() - log_t))))
        c = float(w[r] * g[r]) * tau
        grad[r] = c * (q - target)
        grad_tol[r] = abs(c) * (q * (d + EPS * (3 + y)) + slack) + (half_ulp + EPS) * grad[r].abs() + tiny
    return loss, grad, loss_tol, grad_tol


def merge(ids, lp, weights, top, token_weight=None):
    """ids / lp [K, rows, k] on the CPU -> ids, log probabilities (double), by dictionaries."""
    K, rows, k = ids.shape
    out_ids = torch.full((rows, top), -1, dtype=torch.int32)
    out_lp = torch.full((rows, top), -math.inf, dtype=torch.float64)
    ids_l, lp_l = ids.tolist(), lp.tolist()
    for r in range(rows):
        acc, total = {}, 0.0
        for c in range(K):
            share = float(weights[c]) * (1.0 if token_weight is None else float(token_weight[c, r]))
            if not share > 0.0 or all(i < 0 for i in ids_l[c][r]):
                continue
            total += share
            for i, v in zip(ids_l[c][r], lp_l[c][r]):
                if i >= 0:
                    p = share * math.exp(v) if v == v else math.nan
                    acc[i] = acc.get(i, 0.0) + p
        best = sorted(acc.items(), key=lambda kv: (0 if kv[1] != kv[1] else 1, -kv[1] if kv[1] == kv[1] else 0.0, kv[0]))
        for j, (i, p) in enumerate(best[:top]):
            out_ids[r, j] = i
            q = p / total
            out_lp[r, j] = math.log(q) if q > 0 else (-math.inf if q == 0 else math.nan)
    return out_ids, out_lp


def close(got, want, tol, what=""):
    """Equal infinities and NaNs, everything else within its bound (tol broadcasts)."""
    got, want = got.detach().cpu().double(), want.double()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | (want.isfinite() & ((got - want).abs() <= tol)))
    if bool(bad.any()):
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {at}: got {float(got[at])}, "
                             f"want {float(want[at])}, bound {float(tol[at])}")
