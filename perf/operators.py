"""Cases, inputs and plain forms of the token operators: scoring tokens (log probability, entropy, top
alternatives), merging the clients' top lists into one teacher, and distilling from it.

With ``own`` false `run` computes an operator from elementary torch operations; with ``own`` true it makes
the calls a user makes of :mod:`appfl_amd.token_ops`.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    return [
        # one generated token scored on the server: a single row, latency is what counts
        {"name": "scores_one_token", "op": "scores", "batch": 1, "rows": 1, "vocab": 32000, "dtype": "bf16", "top": 8},
        # a batch of an image classifier (1000 classes, as the ResNet / ViT workloads), fp32
        {"name": "scores_classes", "op": "scores", "batch": 1, "rows": 512, "vocab": 1000, "dtype": "f32", "top": 5},
        # prompts shifted by one (every row but the last of each sequence), odd vocabulary: unaligned rows
        {"name": "scores_prompts", "op": "scores", "batch": 4, "rows": 511, "vocab": 50261, "dtype": "bf16", "top": 32},
        # a public set of 8192 positions over a large vocabulary: the client's upload of a whole round
        {"name": "scores_public_set", "op": "scores", "batch": 8, "rows": 1024, "vocab": 128000, "dtype": "f16", "top": 64},
        # two clients' answers to a handful of positions
        {"name": "merge_two", "op": "merge", "clients": 2, "rows": 60, "vocab": 32000, "k": 8, "top": 8},
        # a round of 16 clients, some positions left out by some of them
        {"name": "merge_sixteen", "op": "merge", "clients": 16, "rows": 2047, "vocab": 50261, "k": 32, "top": 32},
        # a round of 100 clients over the whole public set
        {"name": "merge_hundred", "op": "merge", "clients": 100, "rows": 8192, "vocab": 128000, "k": 32, "top": 64},
        # a small classifier (10 classes) learning from a merged teacher, forward and backward
        {"name": "distill_digits", "op": "distill", "rows": 128, "vocab": 10, "dtype": "f32", "k": 4, "tau": 2.0},
        # a bfloat16 model with an odd vocabulary, forward and backward through autograd
        {"name": "distill_odd", "op": "distill", "rows": 2047, "vocab": 32003, "dtype": "bf16", "k": 32, "tau": 1.0},
        # loss and gradient in one call: a micro batch of fp32 logits
        {"name": "step_micro", "op": "step", "rows": 96, "vocab": 50261, "dtype": "f32", "k": 16, "tau": 1.5},
        # the largest training step: 8192 positions over a large vocabulary in bfloat16
        {"name": "step_large", "op": "step", "rows": 8192, "vocab": 128000, "dtype": "bf16", "k": 64, "tau": 2.0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scores", "merge", "distill", "step"])
    if op == "merge":
        clients = _log_int(rng, 1, 100)
        k = _log_int(rng, 1, 64)
        rows = _log_int(rng, 1, max(1, min(8192, 26214400 // (clients * k))))
        return {"op": op, "clients": clients, "rows": rows, "vocab": _log_int(rng, max(2 * k + 2, 10), 131072), "k": k,
                "top": rng.randint(1, min(64, clients * k))}
    vocab = _log_int(rng, 10, 131072)
    rows = _log_int(rng, 1, max(1, min(8192, 800000000 // vocab)))
    case = {"op": op, "rows": rows, "vocab": vocab, "dtype": rng.choice(["bf16", "f16", "f32"])}
    if case["dtype"] == "f32":
        case["rows"] = max(1, rows // 2)
    if op == "scores":
        case["batch"] = rng.randint(1, 4)
        case["rows"] = max(1, case["rows"] // case["batch"])
        case["top"] = rng.randint(0, min(64, vocab))
    else:
        case["k"] = _log_int(rng, 1, min(64, vocab // 2))
        case["tau"] = rng.choice([1.0, 1.5, 2.0, 4.0])
    return case


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _distinct(rows, count, vocab, gen):
    """`count` different ids a row, in random order."""
    ids = torch.randint(0, vocab - count + 1, (rows, count), device="cuda", generator=gen).sort(dim=1).values
    ids = ids + torch.arange(count, device="cuda")
    order = torch.rand(rows, count, device="cuda", generator=gen).argsort(dim=1)
    return ids.gather(1, order)


def _logits(shape, dtype, gen):
    """Logits of a model: a broad bulk, and one row in two sure of a few tokens."""
    x = torch.empty(shape, device="cuda", dtype=dtype).normal_(0.0, 2.0, generator=gen)
    flat = x.view(-1, shape[-1])
    rows, vocab = flat.shape
    picks = torch.randint(0, vocab, (rows, 4), device="cuda", generator=gen)
    lift = 10.0 * torch.rand(rows, 4, device="cuda", generator=gen)
    lift = lift * (torch.rand(rows, 1, device="cuda", generator=gen) < 0.5)
    for j in range(4):
        index = picks[:, j:j + 1]
        flat.scatter_(1, index, flat.gather(1, index) + lift[:, j:j + 1].to(dtype))
    return x


def _top_lists(shape, gen):
    """Log probabilities of a row's best tokens, descending; the rest of the vocabulary holds some mass too."""
    score = torch.empty(shape, device="cuda").normal_(0.0, 2.5, generator=gen).sort(dim=-1, descending=True).values
    rest = torch.empty(shape[:-1] + (1,), device="cuda").normal_(0.0, 1.0, generator=gen)
    every = torch.cat([score, rest], dim=-1)
    return torch.log_softmax(every, dim=-1)[..., :-1].contiguous()


def prepare(case, seed):
    gen = _generator(seed)
    state = {"case": case}
    if case["op"] == "merge":
        clients, rows, k = case["clients"], case["rows"], case["k"]
        pool = _distinct(rows, 2 * k, case["vocab"], gen)        # clients answer from the same neighbourhood
        ids = torch.empty(clients, rows, k, device="cuda", dtype=torch.int32)
        for c in range(clients):
            pick = torch.rand(rows, 2 * k, device="cuda", generator=gen).argsort(dim=1)[:, :k]
            ids[c] = pool.gather(1, pick).to(torch.int32)
        state["ids"] = ids
        state["logprobs"] = _top_lists((clients, rows, k), gen)
        state["token_weight"] = (torch.rand(clients, rows, device="cuda", generator=gen) < 0.9).float() * (
            0.5 + torch.rand(clients, rows, device="cuda", generator=gen))
        sizes = [50 + (37 * c + seed) % 101 for c in range(clients)]          # samples a client holds
        state["weights"] = [n / sum(sizes) for n in sizes]
        return state
    dtype = DTYPES[case["dtype"]]
    rows, vocab = case["rows"], case["vocab"]
    if case["op"] == "scores":
        full = _logits((case["batch"], rows + 1, vocab), dtype, gen)
        state["logits"] = full[:, :-1]                           # position s predicts token s + 1
        targets = torch.randint(0, vocab, (case["batch"], rows), device="cuda", generator=gen)
        targets[torch.rand(case["batch"], rows, device="cuda", generator=gen) < 0.05] = -100
        state["targets"] = targets
        return state
    k = case["k"]
    state["logits"] = _logits((rows, vocab), dtype, gen)
    state["ids"] = _distinct(rows, k, vocab, gen).to(torch.int32)
    state["logprobs"] = _top_lists((rows, k), gen)
    keep = (torch.rand(rows, device="cuda", generator=gen) < 0.95).float()    # the rest is padding
    state["row_weight"] = keep / max(rows, 1)
    if case["op"] == "distill":
        state["logits"].requires_grad_(True)
        state["row_grad"] = torch.rand(rows, device="cuda", generator=gen)
    return state


def run(state):
    op = state["case"]["op"]
    if own:
        from appfl_amd import token_ops
        case = state["case"]
        if op == "scores":
            s = token_ops.token_scores(state["logits"], state["targets"], top=case["top"])
            lists = [s.top_ids, s.top_logprobs]
            if case["top"] == 0:                                 # no lists; the plain form's are empty
                lists = [s.lse.new_empty((*s.lse.shape, 0), dtype=t) for t in (torch.int32, torch.float32)]
            return [s.logprob, s.entropy, s.lse, *lists]
        if op == "merge":
            return list(token_ops.merge_tops(state["ids"], state["logprobs"], state["weights"], case["top"],
                                             token_weight=state["token_weight"]))
        if op == "distill":
            losses = token_ops.distill_loss(state["logits"], state["ids"], state["logprobs"],
                                            temperature=case["tau"], row_weight=state["row_weight"])
            grad, = torch.autograd.grad(losses, state["logits"], state["row_grad"])
            return [losses.detach(), grad]
        return list(token_ops.distill_loss_grad(state["logits"], state["ids"], state["logprobs"],
                                                temperature=case["tau"], row_weight=state["row_weight"]))
    with torch.no_grad():
        return {"scores": _scores, "merge": _merge, "distill": _distill, "step": _distill}[op](state)


def _scores(state):
    x = state["logits"].float()
    top = state["case"]["top"]
    peak = x.amax(dim=-1, keepdim=True)
    lse = peak + (x - peak).exp().sum(dim=-1, keepdim=True).log()
    away = lse - x
    entropy = ((-away).exp() * away).sum(dim=-1)
    del away
    targets = state["targets"]
    given = targets != -100
    logprob = x.gather(-1, targets.clamp(min=0).unsqueeze(-1)).squeeze(-1) - lse.squeeze(-1)
    logprob = torch.where(given, logprob, torch.zeros_like(logprob))
    # value and index in one whole number: the top ones of it are unique, ties go to the lowest index
    bits = (x + 0.0).view(torch.int32)
    keys = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32
    keys |= x.shape[-1] - 1 - torch.arange(x.shape[-1], device=x.device)
    ids = x.shape[-1] - 1 - (keys.topk(top, dim=-1).values & 0xFFFFFFFF)
    return [logprob, entropy, lse.squeeze(-1), ids.to(torch.int32), x.gather(-1, ids) - lse]


def _merge(state):
    ids, logprobs, unit = state["ids"], state["logprobs"], state["token_weight"]
    clients, rows, k = ids.shape
    top = state["case"]["top"]
    w = torch.tensor(state["weights"], device="cuda", dtype=torch.float64)
    share = w[:, None] * unit.double()                            # [clients, rows]
    p = share[:, :, None] * logprobs.double().exp()
    total = share.sum(dim=0)
    here = (share > 0)[:, :, None].expand_as(ids)
    far = torch.iinfo(torch.int32).max
    flat_ids = torch.where(here, ids, torch.full_like(ids, far)).permute(1, 0, 2).reshape(rows, clients * k)
    flat_p = p.permute(1, 0, 2).reshape(rows, clients * k)
    flat_ids, order = flat_ids.sort(dim=1, stable=True)
    flat_p = flat_p.gather(1, order)
    first = torch.ones_like(flat_ids, dtype=torch.bool)
    first[:, 1:] = flat_ids[:, 1:] != flat_ids[:, :-1]
    group = first.long().cumsum(dim=1) - 1
    sums = torch.zeros_like(flat_p).scatter_add_(1, group, flat_p)
    names = torch.full_like(flat_ids, far).scatter_(1, group, flat_ids)
    sums = torch.where(names == far, torch.full_like(sums, -1.0), sums)
    sums, order = sums.sort(dim=1, descending=True, stable=True)
    sums, names = sums[:, :top], names.gather(1, order)[:, :top]
    empty = sums < 0
    out = torch.where(empty, torch.full_like(sums, -math.inf), (sums.clamp(min=0) / total[:, None]).log())
    return [torch.where(empty, torch.full_like(names, -1), names), out.float()]


def _distill(state):
    tau = state["case"]["tau"]
    x = state["logits"].detach().float() / tau
    ids = state["ids"].long()
    teacher = state["logprobs"] / tau
    teacher = teacher - teacher.amax(dim=1, keepdim=True)
    t = teacher.exp()
    total = t.sum(dim=1, keepdim=True)
    log_t = teacher - total.log()
    t = t / total
    peak = x.amax(dim=1, keepdim=True)
    q = (x - peak).exp()
    mass = q.sum(dim=1, keepdim=True)
    log_q = x.gather(1, ids) - peak - mass.log()
    weight = state["row_weight"]
    losses = weight * (tau * tau) * (t * (log_t - log_q)).sum(dim=1)
    q = (q / mass).scatter_add_(1, ids, -t)
    scale = weight * tau
    if "row_grad" in state:
        scale = scale * state["row_grad"]
    return [losses, (q * scale[:, None]).to(state["logits"].dtype)]


def work(case):
    if case["op"] == "merge":
        entries = case["clients"] * case["rows"] * case["k"]
        return {"bytes": 8 * entries + 4 * case["clients"] * case["rows"] + 8 * case["rows"] * case["top"],
                "flops": 4 * entries}
    size = 4 if case["dtype"] == "f32" else 2
    rows = case["rows"] * case.get("batch", 1)
    elements = rows * case["vocab"]
    if case["op"] == "scores":
        return {"bytes": elements * size + rows * (20 + 8 * case["top"]), "flops": 6 * elements}
    return {"bytes": 2 * elements * size + rows * (8 + 8 * case["k"]), "flops": 6 * elements}


def exact(case, seed):
    """The definitions in 64 bits, a block of rows at a time."""
    state = prepare(case, seed)
    if case["op"] == "merge":
        return _exact_merge(case, state)
    logits = state["logits"].detach()
    lead, vocab = logits.shape[:-1], logits.shape[-1]
    rows = logits.numel() // vocab
    flat = logits.reshape(rows, vocab)
    step = max(1, (1 << 26) // vocab)
    parts = [(_exact_scores if case["op"] == "scores" else _exact_distill)(case, state, flat[a:a + step], a)
             for a in range(0, rows, step)]
    out = [torch.cat(column) for column in zip(*parts)]
    return [o.reshape(lead + o.shape[1:]) for o in out]


def _exact_scores(case, state, block, first):
    x = block.double()
    log_p = torch.log_softmax(x, dim=1)
    p = log_p.exp()
    targets = state["targets"].reshape(-1)[first:first + len(block)]
    logprob = log_p[torch.arange(len(block), device="cuda"), targets.clamp(min=0)]
    logprob = logprob.masked_fill(targets == -100, 0.0)
    value, ids = (x + 0.0).sort(dim=1, descending=True, stable=True)
    ids = ids[:, :case["top"]]
    lse = torch.logsumexp(x, dim=1)
    return logprob, -(p * log_p).sum(dim=1), lse, ids.to(torch.int32), value[:, :case["top"]] - lse[:, None]


def _exact_distill(case, state, block, first):
    tau = case["tau"]
    x = block.double() / tau
    pick = slice(first, first + len(block))
    ids = state["ids"][pick].long()
    log_t = torch.log_softmax(state["logprobs"][pick].double() / tau, dim=1)
    log_q = torch.log_softmax(x, dim=1)
    weight = state["row_weight"][pick].double()
    losses = weight * tau ** 2 * (log_t.exp() * (log_t - log_q.gather(1, ids))).sum(dim=1)
    target = torch.zeros_like(x).scatter_(1, ids, log_t.exp())
    scale = weight * tau
    if case["op"] == "distill":
        scale = scale * state["row_grad"][pick].double()
    return losses, scale[:, None] * (log_q.exp() - target)


def _exact_merge(case, state):
    clients, rows, k, vocab, top = (case[n] for n in ("clients", "rows", "k", "vocab", "top"))
    names, values = [], []
    step = max(1, (1 << 26) // vocab)
    for a in range(0, rows, step):
        n = min(step, rows - a)
        dense = torch.zeros(n, vocab, device="cuda", dtype=torch.float64)
        seen = torch.zeros(n, vocab, device="cuda", dtype=torch.bool)
        total = torch.zeros(n, 1, device="cuda", dtype=torch.float64)
        line = torch.arange(n, device="cuda")[:, None].expand(n, k)
        for c in range(clients):                                  # ids of one client's row are different
            share = state["weights"][c] * state["token_weight"][c, a:a + n].double()[:, None]
            ids = state["ids"][c, a:a + n].long()
            dense[line, ids] += share * state["logprobs"][c, a:a + n].double().exp()
            seen[line, ids] |= share > 0
            total += share
        value, ids = dense.masked_fill(~seen, -1.0).topk(min(top, vocab), dim=1)
        ids = torch.where(value < 0, torch.full_like(ids, -1), ids).to(torch.int32)
        value = torch.where(value < 0, torch.full_like(value, -math.inf), (value.clamp(min=0) / total).log())
        pad = top - ids.shape[1]
        names.append(torch.nn.functional.pad(ids, (0, pad), value=-1))
        values.append(torch.nn.functional.pad(value, (0, pad), value=-math.inf))
    return [torch.cat(names), torch.cat(values)]
