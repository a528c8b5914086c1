"""The token operators (scores, merge of top lists, distillation) against their definitions in 64 bits."""

import math

import pytest
import torch

import token_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def ops():
    from appfl_amd import token_ops
    return token_ops


def logits(rows, vocab, dtype, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g) * scale
    if vocab > 8:
        x[:, int(torch.randint(0, vocab, (1,), generator=g))] += 6.0
    return x.to(DTYPES[dtype])


def check_scores(x, targets, top, view=None):
    """`x` [rows, vocab] on the CPU; `view` the same values on the device (any strides)."""
    dev = x.cuda() if view is None else view
    lead = dev.shape[:-1]
    s = ops().token_scores(dev, None if targets is None else targets.cuda().reshape(lead), top=top)
    want, tol = R.scores(x, targets, top)
    for name in want:
        got = getattr(s, name)
        assert got.shape[:len(lead)] == lead
        got = got.reshape(want[name].shape)
        if name == "top_ids":
            assert torch.equal(got.cpu(), want[name]), (got.cpu() != want[name]).nonzero()[:4]
        else:
            R.close(got, want[name], tol[name], name)
    assert (s.logprob is None) == (targets is None) and (s.top_ids is None) == (top == 0)


def some_targets(rows, vocab, seed=1):
    t = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(seed))
    t[::5] = -100
    return t


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (5, 7, 7), (4, 10, 3), (2, 63, 63), (2, 64, 8), (3, 65, 64), (9, 255, 5), (2, 256, 128),
    (2, 257, 128), (2, 128, 128), (2, 129, 127), (33, 1000, 5), (3, 1023, 17), (2, 2049, 33), (3, 4097, 1), (1, 8191, 64), (5, 16385, 9),
    (1, 32003, 128), (2, 50261, 32), (1, 131075, 40), (2, 300007, 12), (70, 5003, 0), (600, 1003, 4), (300, 9001, 16)])
def test_scores(rows, vocab, top, dtype):
    check_scores(logits(rows, vocab, dtype, seed=rows + vocab), some_targets(rows, vocab), top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("pattern", ["constant", "ascending", "descending", "two_values", "one_peak", "zeros", "late"])
@pytest.mark.parametrize("rows,vocab,top", [(2, 1000, 20), (1, 40001, 64), (520, 4099, 32), (3, 4099, 128)])
def test_scores_of_ordered_and_tied_rows(pattern, rows, vocab, top, dtype):
    i = torch.arange(vocab, dtype=torch.float64)
    x = {"constant": torch.full((vocab,), 1.5, dtype=torch.float64), "ascending": i * 1e-3, "descending": -i * 1e-3,
         "two_values": (i.long() * 7 % 3 == 0).double(), "one_peak": (i == vocab - 1) * 30.0,
         "zeros": torch.where(i.long() % 2 == 0, torch.tensor(-0.0), torch.tensor(0.0)).double(),
         "late": (i > vocab - 300) * (i - vocab) * 1e-2 - 5.0 * (i <= vocab - 300)}[pattern]
    x = x.to(DTYPES[dtype]).expand(rows, vocab).contiguous()
    check_scores(x, some_targets(rows, vocab), top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,top", [(6, 101, 7), (6, 20011, 9), (530, 3001, 6)])
def test_scores_of_masked_rows(rows, vocab, top, dtype):
    """-inf and the type's lowest value in masked places, rows that keep one token or none, +inf and NaN."""
    x = logits(rows, vocab, dtype, seed=3)
    low = torch.finfo(x.dtype).min
    x[0, 5:] = -math.inf
    x[1] = -math.inf
    x[2] = low
    x[3, : vocab - 1] = low
    x[4, vocab // 2] = math.nan
    x[5, ::2] = low
    check_scores(x, torch.tensor([0, 1, 2, 3, 4, 5] + [0] * (rows - 6)), top)
    y = logits(2, vocab, dtype, seed=4)
    y[0, 3] = math.inf
    s = ops().token_scores(y.cuda(), top=2)
    assert bool(s.lse[0].isnan()) or float(s.lse[0]) == math.inf
    assert int(s.top_ids[0, 0]) == 3 and bool(s.entropy[0].isnan()) and bool(s.lse[1].isfinite())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shift", [0, 1, 3, 5])
def test_scores_of_views(shift, dtype):
    """Sequences shifted by one, rows that start at any element, rows that are all the same row."""
    batch, seq, vocab = 3, 4, 1337
    x = logits(batch * seq, vocab, dtype, seed=5).reshape(batch, seq, vocab)
    big = torch.full((batch, seq + 1, vocab + 9), 50.0, dtype=x.dtype, device="cuda")
    view = big[:, :seq, shift:shift + vocab]
    view.copy_(x)
    flat = x.reshape(-1, vocab)
    check_scores(flat, some_targets(batch * seq, vocab), 11, view=view)
    one = x[0, :1].cuda().expand(seq, vocab)
    check_scores(x[0, :1].expand(seq, vocab).contiguous(), some_targets(seq, vocab), 4, view=one)


def test_scores_targets_outside_the_vocabulary():
    x = logits(4, 50, "f32")
    check_scores(x, torch.tensor([50, -1, 49, -100]), 3)
    s = ops().token_scores(x.cuda(), torch.tensor([7, 7, 0, 1]).cuda(), ignore_index=7)
    assert float(s.logprob[0]) == 0.0 and float(s.logprob[2]) < 0.0


def far_rows(rows, vocab, dtype, gap):
    """A [rows, vocab] device view whose rows lie `gap` elements apart."""
    buf = torch.empty(gap * (rows - 1) + vocab, dtype=DTYPES[dtype], device="cuda")
    return buf.as_strided((rows, vocab), (gap, 1))


@pytest.mark.parametrize("inner", [False, True])
def test_offsets_past_32_bits(inner):
    rows, vocab, gap = 3, 2051, (1 << 31) + 3
    x = logits(rows, vocab, "bf16", seed=6)
    view = far_rows(rows, vocab, "bf16", gap)
    view.copy_(x)
    check_scores(x, some_targets(rows, vocab), 8, view=view if inner else view[:, None, :])
    ids, lp = teacher(rows, vocab, 6)
    check_distill(x, ids, lp, 1.0, view=view if inner else view[:, None, :])


# ---- distillation ----------------------------------------------------------------------------------

def teacher(rows, vocab, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]).to(torch.int32)
    lp = torch.log_softmax(torch.randn(rows, k + 1, generator=g) * 2.5, dim=1)[:, :k].sort(dim=1, descending=True).values
    return ids, lp.contiguous()


def check_distill(x, ids, lp, tau, weight=None, row_grad=None, view=None):
    dev = x.cuda() if view is None else view
    lead = dev.shape[:-1]
    cuda = lambda t: None if t is None else t.cuda().reshape(lead + t.shape[1:])
    want_loss, want_grad, loss_tol, grad_tol = R.distill(x, ids, lp, tau, weight, row_grad)
    leaf = dev.detach().requires_grad_(True)
    loss = ops().distill_loss(leaf, cuda(ids), cuda(lp), temperature=tau, row_weight=cuda(weight))
    assert loss.shape == lead and loss.dtype == torch.float32
    R.close(loss.reshape(-1), want_loss, loss_tol, "loss")
    if row_grad is None:
        grad, = torch.autograd.grad(loss.sum(), leaf)
    else:
        grad, = torch.autograd.grad(loss, leaf, cuda(row_grad))
    assert grad.dtype == x.dtype and grad.shape == dev.shape
    R.close(grad.reshape(x.shape), want_grad, grad_tol, "grad")
    if row_grad is None:
        loss, grad = ops().distill_loss_grad(dev.detach(), cuda(ids), cuda(lp), temperature=tau, row_weight=cuda(weight))
        R.close(loss.reshape(-1), want_loss, loss_tol, "step loss")
        R.close(grad.reshape(x.shape), want_grad, grad_tol, "step grad")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,k,tau", [
    (1, 1, 1, 1.0), (3, 2, 1, 2.0), (4, 10, 4, 2.0), (7, 63, 63, 1.0), (3, 64, 5, 0.5), (5, 129, 64, 1.5),
    (2, 257, 256, 1.0), (9, 1000, 32, 4.0), (3, 4099, 128, 1.0), (2, 16383, 16, 2.0), (3, 32003, 32, 1.0),
    (2, 50261, 64, 2.0), (3, 777, 9, 1e-3), (3, 777, 9, 1e3), (1, 131073, 8, 1.0), (2, 200003, 9, 3.0), (530, 1001, 3, 1.0)])
def test_distill(rows, vocab, k, tau, dtype):
    ids, lp = teacher(rows, vocab, k, seed=rows)
    check_distill(logits(rows, vocab, dtype, seed=vocab), ids, lp, tau)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [50, 3001, 70001])
def test_distill_weights_padding_and_duplicates(vocab, dtype):
    """Rows of weight 0 (whatever they hold), short and empty lists, an id listed twice, upstream gradients."""
    rows, k = 8, 6
    x = logits(rows, vocab, dtype, seed=8)
    ids, lp = teacher(rows, vocab, k, seed=9)
    weight = torch.tensor([1.0, 0.0, 0.25, 1.0, 1.0, 2.0, 1.0, 0.5])
    x[1] = math.nan                                  # weight 0
    ids[2, 4:] = -1
    ids[3] = -1                                      # nothing to learn from
    lp[4] = -math.inf                                # neither here
    lp[5, 1:] = -math.inf                            # sure of one token
    ids[6, 3] = ids[6, 0]
    ids[6, 5] = ids[6, 0]
    row_grad = torch.tensor([1.0, 3.0, -0.5, 1.0, 2.0, 0.0, 1.5, 1e-3])
    check_distill(x, ids, lp, 2.0, weight)
    check_distill(x, ids, lp, 2.0, weight, row_grad)
    check_distill(x, ids, lp, 1.0, None, row_grad)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [40, 5003, 70001])
def test_distill_masked_logits(vocab, dtype):
    """-inf and the type's lowest value beside and under the teacher's tokens, a row with no finite logit, ids
    outside the vocabulary, NaN."""
    rows, k = 7, 4
    x = logits(rows, vocab, dtype, seed=10)
    ids, lp = teacher(rows, vocab, k, seed=11)
    low = torch.finfo(x.dtype).min
    free = [next(v for v in range(vocab) if v not in ids[r].tolist()) for r in range(rows)]
    x[0, free[0]] = -math.inf
    x[1, int(ids[1, 0])] = -math.inf                 # the teacher wants what the mask forbids
    x[2] = low
    x[3] = -math.inf
    ids[4, 2] = vocab
    x[5, free[5]] = math.nan
    x[6, free[6]] = low
    check_distill(x, ids, lp, 1.0)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [37, 2050, 66001])
def test_distill_views(vocab, dtype):
    """Shifted sequences, rows at any element, strided lists and weights, a gradient of broadcast logits."""
    batch, seq, k = 2, 3, 5
    x = logits(batch * seq, vocab, dtype, seed=12)
    ids, lp = teacher(batch * seq, vocab, k, seed=13)
    for shift in (0, 1, 2, 7):
        big = torch.zeros((batch, seq + 1, vocab + 8), dtype=x.dtype, device="cuda")
        view = big[:, :seq, shift:shift + vocab]
        view.copy_(x.reshape(batch, seq, vocab))
        check_distill(x, ids, lp, 1.0, view=view)
    wide_ids = torch.full((batch * seq, k + 3), 1 << 30, dtype=torch.int32, device="cuda")
    wide_ids[:, :k] = ids.cuda()
    weight = torch.rand(batch * seq, 2)
    loss, grad = ops().distill_loss_grad(x.cuda(), wide_ids[:, :k], lp.cuda(), row_weight=weight.cuda()[:, 0])
    want_loss, want_grad, loss_tol, grad_tol = R.distill(x, ids, lp, 1.0, weight[:, 0])
    R.close(loss, want_loss, loss_tol, "loss")
    R.close(grad, want_grad, grad_tol, "grad")
    # one row of logits against every teacher: the gradient adds up over the rows
    leaf = x[:1].cuda().requires_grad_(True)
    ops().distill_loss(leaf.expand(batch * seq, vocab), ids.cuda(), lp.cuda()).sum().backward()
    _, want_grad, _, grad_tol = R.distill(x[:1].expand(batch * seq, vocab), ids, lp, 1.0)
    # torch adds the rows up in the logits' type: each of the sums rounds once more
    total = want_grad.sum(dim=0, keepdim=True)
    tol = grad_tol.sum(dim=0, keepdim=True) + batch * seq * torch.finfo(x.dtype).eps * want_grad.abs().sum(dim=0, keepdim=True)
    R.close(leaf.grad, total, tol, "broadcast grad")


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("vocab", [33, 4001, 70003])
def test_step_in_place_and_into_out(vocab, dtype):
    """The gradient over the logits, into a buffer of other alignment, nothing written beside it."""
    rows, k = 5, 7
    x = logits(rows, vocab, dtype, seed=14)
    ids, lp = teacher(rows, vocab, k, seed=15)
    weight = torch.tensor([1.0, 0.5, 0.0, 2.0, 1.0])
    want_loss, want_grad, loss_tol, grad_tol = R.distill(x, ids, lp, 1.5, weight)
    dev = x.cuda()
    loss, grad = ops().distill_loss_grad(dev, ids.cuda(), lp.cuda(), 1.5, weight.cuda(), out=dev)
    assert grad is dev
    R.close(loss, want_loss, loss_tol, "loss")
    R.close(dev, want_grad, grad_tol, "in place")
    buf = torch.full((rows, vocab + 11), 77.0, dtype=x.dtype, device="cuda")
    loss, grad = ops().distill_loss_grad(x.cuda(), ids.cuda(), lp.cuda(), 1.5, weight.cuda(), out=buf[:, 5:5 + vocab])
    R.close(grad, want_grad, grad_tol, "out")
    assert bool((buf[:, :5] == 77.0).all()) and bool((buf[:, 5 + vocab:] == 77.0).all())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", [(1, 102401), (2, 700003), (7, 131072), (128, 102407), (129, 102407)])
def test_step_of_few_long_rows(rows, vocab, dtype):
    """Rows cut in parts, and one row more than that takes."""
    x = logits(rows, vocab, dtype, seed=13)
    ids, lp = teacher(rows, vocab, 9, seed=14)
    ids[0, :4] = torch.tensor([0, vocab - 1, vocab // 2, 0])          # the ends, and one twice
    weight = torch.rand(rows) + 0.5
    if rows > 6:
        weight[1] = 0.0
        ids[2, 0] = vocab                                            # outside: NaN
        x[3, vocab // 3] = math.nan
        ids[4] = -1                                                  # no entry
        x[5] = -math.inf
        x[6, ::2] = -math.inf
    want_loss, want_grad, loss_tol, grad_tol = R.distill(x, ids, lp, 1.5, weight, None)
    dev = x.cuda()
    big = torch.full((rows, vocab + 3), 7.0, dtype=x.dtype, device="cuda")
    for out in (None, big[:, 1:1 + vocab], big[:, :vocab], dev):      # aligned unlike the logits, and in place
        loss, grad = ops().distill_loss_grad(dev, ids.cuda(), lp.cuda(), 1.5, weight.cuda(), out=out)
        R.close(loss, want_loss, loss_tol, "loss")
        R.close(grad, want_grad, grad_tol, "grad")
    assert bool((big[:, vocab + 1:] == 7).all())


def test_distill_gradient_against_differences():
    rows, vocab, k = 3, 13, 5
    x = logits(rows, vocab, "f32", seed=16, scale=1.0)
    ids, lp = teacher(rows, vocab, k, seed=17)
    leaf = x.cuda().requires_grad_(True)
    f = lambda v: ops().distill_loss(v, ids.cuda(), lp.cuda(), temperature=2.0).double().sum()
    grad, = torch.autograd.grad(f(leaf), leaf)
    h = 2.0 ** -5     # truncation: h^2 / 6 times a third derivative below T^2 / T^3 = 1/2; rounding: 3 losses of about
    # 4, each off by 1e-6 at most, over 2 h
    for r in range(rows):
        for v in range(vocab):
            d = torch.zeros_like(x)
            d[r, v] = h
            slope = (f((x + d).cuda()) - f((x - d).cuda())) / (2 * h)
            assert abs(float(slope) - float(grad[r, v])) < h * h / 12 + 6e-6 / (2 * h)


# ---- merge -----------------------------------------------------------------------------------------

def answers(K, rows, k, pool, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.stack([torch.randperm(pool, generator=g)[:k] for _ in range(rows)]) for _ in range(K)])
    ids = ids.to(torch.int32) * 7 + 3
    lp = torch.log_softmax(torch.randn(K, rows, k + 1, generator=g) * 2, dim=2)[..., :k]
    return ids, lp.sort(dim=2, descending=True).values.contiguous()


def check_merge(ids, lp, weights, top, unit=None, dev=None):
    cuda = dev or (lambda t: None if t is None else t.cuda())
    got_ids, got_lp = ops().merge_tops(cuda(ids), cuda(lp), weights, top, token_weight=cuda(unit))
    want_ids, want_lp = R.merge(ids, lp, weights, top, unit)
    assert got_ids.dtype == torch.int32 and got_lp.dtype == torch.float32
    assert torch.equal(got_ids.cpu(), want_ids), (got_ids.cpu(), want_ids)
    # sums off by 2^-51 a term of up to 8192, an fp64 logarithm, rounded once to fp32
    R.close(got_lp, want_lp, 2.0 ** -24 * want_lp.abs().nan_to_num(posinf=0.0) + 1e-11, "logprobs")


@pytest.mark.parametrize("K,rows,k,pool,top", [
    (1, 1, 1, 1, 1), (1, 3, 5, 9, 5), (2, 4, 1, 2, 2), (2, 60, 8, 16, 8), (3, 5, 7, 7, 21), (5, 9, 13, 40, 20),
    (16, 20, 32, 64, 32), (16, 3, 32, 600, 64), (100, 4, 32, 64, 64), (128, 2, 64, 128, 200), (128, 2, 64, 9000, 256),
    (32, 2, 256, 300, 256), (7, 300, 9, 30, 10), (64, 3, 5, 11, 7), (4, 5, 256, 256, 250)])
def test_merge(K, rows, k, pool, top):
    ids, lp = answers(K, rows, k, pool, seed=K + rows)
    g = torch.Generator().manual_seed(2)
    sizes = torch.randint(1, 50, (K,), generator=g)
    weights = (sizes.double() / sizes.sum()).tolist()
    check_merge(ids, lp, weights, top)
    unit = torch.rand(K, rows, generator=g) * (torch.rand(K, rows, generator=g) < 0.8)
    check_merge(ids, lp, weights, top, unit)


def test_merge_empty_short_and_strange_lists():
    K, rows, k = 4, 7, 6
    ids, lp = answers(K, rows, k, 12, seed=3)
    unit = torch.ones(K, rows)
    ids[:, 0] = -1                                  # nobody answers
    ids[1:, 1] = -1                                 # one client answers
    unit[:, 2] = 0.0                                # everybody is left out
    ids[0, 3, 2:] = -5                              # a short list
    ids[1, 4, 3] = ids[1, 4, 0]                     # a token listed twice
    lp[2, 5, 1] = -math.inf                         # a token of probability zero
    ids[2, 5, 1] = 5001
    lp[3, 6, 2] = math.nan                          # a broken client shows
    ids[0, 6, 0] = 2 ** 31 - 1
    for top in (1, 6, 24):
        check_merge(ids, lp, [0.1, 0.4, 0.3, 0.2], top, unit)
    check_merge(ids, lp, [0.0, 0.4, 0.0, 0.2], 6, unit)
    check_merge(ids, lp, [0.0] * 4, 6, unit)
    unit[0, 5] = math.nan
    unit[1, 5] = -1.0
    check_merge(ids, lp, [0.1, 0.4, 0.3, 0.2], 6, unit)


def test_merge_ties_go_to_the_lowest_id():
    ids = torch.tensor([[[9, 4, 7, 1]], [[4, 9, 2, 7]]], dtype=torch.int32)
    lp = torch.full((2, 1, 4), -2.0)
    check_merge(ids, lp, [0.5, 0.5], 5)
    got, _ = ops().merge_tops(ids.cuda(), lp.cuda(), torch.tensor([0.5, 0.5]), 5)
    assert got.cpu().tolist() == [[4, 7, 9, 1, 2]]


def test_merge_of_strided_lists():
    K, rows, k = 3, 11, 5
    ids, lp = answers(K, rows, k, 20, seed=4)
    unit = torch.rand(rows, K)

    def spread(t):
        if t is None:
            return None
        if t.dim() == 2:
            return unit.cuda().t()                   # [K, rows] with the rows' stride in front
        big = torch.zeros(rows + 2, K, k + 3, dtype=t.dtype, device="cuda")
        view = big[1:1 + rows, :, 2:2 + k].transpose(0, 1)
        view.copy_(t)
        return view
    check_merge(ids, lp, [1.0, 2.0, 0.5], 9, unit.t().contiguous(), dev=spread)
    same = ids[:, :1].cuda().expand(K, rows, k)       # every row the same answers
    got, _ = ops().merge_tops(same, lp[:, :1].cuda().expand(K, rows, k), [1.0, 1.0, 1.0], 4)
    want, _ = R.merge(ids[:, :1], lp[:, :1], [1.0] * 3, 4)
    assert torch.equal(got.cpu(), want.expand(rows, 4))


def test_merge_of_lists_with_strides_of_their_own():
    K, rows, k = 3, 11, 5
    ids, lp = answers(K, rows, k, 20, seed=6)
    for wide in (torch.int32, torch.float32):         # the ids' or the values' lists lie wider

        def spread(t):
            if t is None or t.dtype != wide:
                return None if t is None else t.cuda()
            big = torch.zeros(K, rows + 2, k, dtype=t.dtype, device="cuda")
            big[:, 1:1 + rows] = t.cuda()
            return big[:, 1:1 + rows]
        check_merge(ids, lp, [1.0, 2.0, 0.5], 9, dev=spread)


@pytest.mark.parametrize("client", [2**30 // 3 - 1, 2**30 // 3, 2**31 + 5])
def test_merge_of_clients_far_apart(client):
    K, rows, k = 3, 4, 5
    ids, lp = answers(K, rows, k, 20, seed=7)

    def spread(t):
        if t is None:
            return None
        big = torch.empty((K - 1) * client + rows * k, dtype=t.dtype, device="cuda")
        view = big.as_strided((K, rows, k), (client, k, 1))
        view.copy_(t)
        return view
    check_merge(ids, lp, [1.0, 2.0, 0.5], 9, dev=spread)


def test_more_rows_than_a_launch_takes():
    """Two classes, 2^22 + 3 rows: rows beyond the first launch's, against torch in 64 bits.

    Log probabilities here are below 32, 46 in log2 units, where fp32 steps by 2^-18: the distance and the
    difference with log2 s are each off by half of that (2^-19, times ln 2), the factor back to natural units by
    2^-24 of 32 (2^-19), the result by 2^-20: 2.9 * 2^-19 together."""
    o = ops()
    rows = (1 << 22) + 3
    x = torch.randn(rows, 2, device="cuda") * 2
    want = torch.log_softmax(x.double(), 1)
    assert float(want.min()) > -32.0
    s = o.token_scores(x, torch.ones(rows, dtype=torch.int64, device="cuda"), top=1)
    assert torch.equal(s.top_ids[:, 0], (x[:, 1] > x[:, 0]).int())
    assert float((s.logprob - want[:, 1]).abs().max()) < 3 * 2.0 ** -19
    ids = torch.ones(rows, 1, dtype=torch.int32, device="cuda")
    lp = torch.zeros(rows, 1, device="cuda")
    target = torch.tensor([0.0, 1.0], device="cuda")
    leaf = x.clone().requires_grad_(True)
    loss = o.distill_loss(leaf, ids, lp)
    grad, = torch.autograd.grad(loss.sum(), leaf)
    step_loss, step_grad = o.distill_loss_grad(x, ids, lp)
    for l, g in ((loss.detach(), grad), (step_loss, step_grad)):
        assert float((l + want[:, 1]).abs().max()) < 3 * 2.0 ** -19
        assert float((g - (want.exp() - target)).abs().max()) < 2.0 ** -20
    got, _ = o.merge_tops(ids[None], lp[None], [1.0], 1)
    assert torch.equal(got, ids)


def test_hooks_on_saved_tensors():
    """The backward pass works on what the hooks hand back: copies elsewhere, of other strides."""
    rows, vocab, k = 4, 301, 5
    x = logits(rows, vocab, "f32", seed=70)
    ids, lp = teacher(rows, vocab, k, seed=71)
    wide = torch.zeros(rows, vocab + 7, device="cuda")[:, 3:3 + vocab]
    wide.copy_(x)
    leaf = wide.requires_grad_(True)
    weight = torch.tensor([1.0, 0.5, 2.0, 0.0])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach().cpu().contiguous(), lambda t: t.cuda()):
        loss = ops().distill_loss(leaf, ids.cuda(), lp.cuda(), 2.0, weight.cuda())
    with torch.no_grad():
        wide.fill_(math.nan)                         # saved on the host long since
    grad, = torch.autograd.grad(loss.sum(), leaf)
    _, want, _, tol = R.distill(x, ids, lp, 2.0, weight)
    R.close(grad, want, tol, "grad")


def test_backward_leaves_the_forward_call_as_it_was():
    """A second backward pass of the same graph may be under way in another thread."""
    x = logits(3, 50, "f32", seed=80).cuda().requires_grad_(True)
    ids, lp = teacher(3, 50, 4, seed=81)
    weight = torch.rand(3).cuda()
    held = []

    def elsewhere(t):
        held.append(t.clone())
        return held[-1]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, elsewhere):
        loss = ops().distill_loss(x, ids.cuda(), lp.cuda(), row_weight=weight)
    call = loss.grad_fn.call[:2]
    before = [bytes(c) for c in call]
    grads = [torch.autograd.grad(loss.sum(), x, retain_graph=True)[0] for _ in range(2)]
    assert [bytes(c) for c in call] == before
    _, want, _, tol = R.distill(x.detach().cpu(), ids, lp, 1.0, weight.cpu())
    for g in grads:
        R.close(g, want, tol, "grad")


def test_a_step_over_saved_logits_is_noticed():
    """The gradient written over logits that an earlier loss saved: that loss's backward pass must refuse."""
    x = torch.randn(3, 17, device="cuda")
    ids, lp = teacher(3, 17, 2)
    leaf = x.clone().requires_grad_(True)
    held = leaf * 1.0
    loss = ops().distill_loss(held, ids.cuda(), lp.cuda())
    ops().distill_loss_grad(held.detach(), ids.cuda(), lp.cuda(), out=held.detach())
    with pytest.raises(RuntimeError):
        loss.sum().backward()


def test_backward_twice_and_of_the_second_order():
    x = torch.randn(3, 17, device="cuda", requires_grad=True)
    ids, lp = teacher(3, 17, 2)
    loss = ops().distill_loss(x, ids.cuda(), lp.cuda())
    first, = torch.autograd.grad(loss.sum(), x, retain_graph=True)
    again, = torch.autograd.grad(loss.sum(), x, create_graph=True)
    assert torch.equal(first, again)
    with pytest.raises(RuntimeError):
        again.sum().backward()


# ---- the operators as a user runs them -------------------------------------------------------------

def test_no_rows():
    o = ops()
    s = o.token_scores(torch.zeros(0, 9, device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda"), top=2)
    assert s.top_ids.shape == (0, 2) and s.lse.shape == (0,)
    ids, lp = torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, device="cuda")
    leaf = torch.zeros(0, 9, device="cuda", requires_grad=True)
    o.distill_loss(leaf, ids, lp).sum().backward()
    assert leaf.grad.shape == (0, 9)
    loss, grad = o.distill_loss_grad(torch.zeros(2, 0, 9, device="cuda"), ids.reshape(2, 0, 3), lp.reshape(2, 0, 3))
    assert loss.shape == (2, 0) and grad.shape == (2, 0, 9)
    got, _ = o.merge_tops(ids.reshape(1, 0, 3), lp.reshape(1, 0, 3), [1.0], 2)
    assert got.shape == (0, 2)


def test_results_do_not_change_from_call_to_call():
    o = ops()
    x = logits(40, 20011, "bf16", seed=20).cuda()
    ids, lp = teacher(40, 20011, 16, seed=21)
    ids, lp = ids.cuda(), lp.cuda()
    first = o.token_scores(x, top=32)
    loss, grad = o.distill_loss_grad(x, ids, lp)
    many = answers(16, 40, 32, 64, seed=22)
    merged = o.merge_tops(many[0].cuda(), many[1].cuda(), [1.0 / 16] * 16, 32)
    for _ in range(3):
        again = o.token_scores(x, top=32)
        assert all(torch.equal(a, b) for a, b in zip(first[1:], again[1:]))
        l2, g2 = o.distill_loss_grad(x, ids, lp)
        assert torch.equal(loss, l2) and torch.equal(grad, g2)
        m2 = o.merge_tops(many[0].cuda(), many[1].cuda(), [1.0 / 16] * 16, 32)
        assert torch.equal(merged[0], m2[0]) and torch.equal(merged[1], m2[1])


@pytest.mark.parametrize("rows,vocab", [(2, 40009), (64, 1009), (3, 110017)])
def test_captured_and_replayed(rows, vocab):
    """The whole path in one graph, replayed on new inputs with eager work in between."""
    o = ops()
    K, k = 3, 8
    x = logits(rows, vocab, "bf16", seed=30).cuda()
    clients = torch.stack([logits(rows, vocab, "bf16", seed=31 + c) for c in range(K)]).cuda()
    weights = [0.5, 0.3, 0.2]

    def path():
        s = o.token_scores(clients, top=k)
        ids, lp = o.merge_tops(s.top_ids, s.top_logprobs, weights, k)
        return [s.entropy, s.lse, s.top_ids, s.top_logprobs, ids, lp, *o.distill_loss_grad(x, ids, lp, 2.0)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        path()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = path()
    for step in range(4):
        x.copy_(logits(rows, vocab, "bf16", seed=40 + step))
        clients.copy_(torch.stack([logits(rows, vocab, "bf16", seed=50 + 7 * step + c) for c in range(K)]))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, path()):
            assert torch.equal(a, b)


def test_two_streams_at_once():
    o = ops()
    xs = [logits(3, 60013, "bf16", seed=60 + i).cuda() for i in range(2)]
    want = [o.token_scores(x, top=16) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(o.token_scores(xs[i], top=16))
    torch.cuda.synchronize()
    for i in range(2):
        for s in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(s[1:], want[i][1:]))


def test_steps_in_parts_on_two_streams_at_once():
    o = ops()
    x = [logits(3, 120011, "bf16", seed=70 + i).cuda() for i in range(2)]
    ids, lp = [t.cuda() for t in teacher(3, 120011, 8, seed=72)]
    want = [o.distill_loss_grad(v, ids, lp) for v in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(o.distill_loss_grad(x[i], ids, lp))
    torch.cuda.synchronize()
    for i in range(2):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))


def test_refusals():
    o = ops()
    x = torch.zeros(3, 9, device="cuda")
    ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    lp = torch.zeros(3, 2, device="cuda")
    from appfl_amd._native import NativeLibraryError
    bad = [
        (NativeLibraryError, lambda: o.token_scores(x.cpu())),
        (TypeError, lambda: o.token_scores(x.double())),
        (TypeError, lambda: o.token_scores(x, torch.zeros(3, dtype=torch.int32, device="cuda"))),
        (TypeError, lambda: o.token_scores(x, top=1.0)),
        (ValueError, lambda: o.token_scores(x[0])),
        (ValueError, lambda: o.token_scores(x.t())),
        (ValueError, lambda: o.token_scores(x[:, :0])),
        (ValueError, lambda: o.token_scores(x, torch.zeros(4, dtype=torch.int64, device="cuda"))),
        (ValueError, lambda: o.token_scores(x, top=10)),
        (ValueError, lambda: o.token_scores(x, top=-1)),
        (ValueError, lambda: o.token_scores(torch.zeros(2, 300, device="cuda"), top=129)),
        (TypeError, lambda: o.distill_loss(x, ids.long(), lp)),
        (TypeError, lambda: o.distill_loss(x, ids, lp.half())),
        (TypeError, lambda: o.distill_loss(x, ids, lp, row_weight=torch.ones(3, device="cuda").double())),
        (NativeLibraryError, lambda: o.distill_loss(x, ids.cpu(), lp)),
        (ValueError, lambda: o.distill_loss(x, ids[:2], lp[:2])),
        (ValueError, lambda: o.distill_loss(x, ids, lp[:, :1])),
        (ValueError, lambda: o.distill_loss(x, ids[:, :0], lp[:, :0])),
        (ValueError, lambda: o.distill_loss(x, ids, lp, temperature=0.0)),
        (ValueError, lambda: o.distill_loss(x, ids, lp, temperature=-1.0)),
        (ValueError, lambda: o.distill_loss(x, ids, lp, temperature=math.nan)),
        (ValueError, lambda: o.distill_loss(x, ids, lp, temperature=math.inf)),
        (ValueError, lambda: o.distill_loss(x, ids, lp, temperature=1e7)),
        (ValueError, lambda: o.distill_loss(x, ids, lp, row_weight=torch.ones(2, device="cuda"))),
        (ValueError, lambda: o.distill_loss(x, ids.t().contiguous().t(), lp)),
        (ValueError, lambda: o.distill_loss_grad(x, ids, lp, out=torch.zeros(3, 8, device="cuda"))),
        (TypeError, lambda: o.distill_loss_grad(x, ids, lp, out=torch.zeros(3, 9, device="cuda").half())),
        (ValueError, lambda: o.distill_loss_grad(x, ids, lp, out=torch.zeros(1, 9, device="cuda").expand(3, 9))),
        (ValueError, lambda: o.distill_loss_grad(x, ids, lp, out=torch.zeros(9, 3, device="cuda").t())),
        (ValueError, lambda: o.distill_loss_grad(torch.zeros(4, 9, device="cuda")[1:], ids, lp,
                                                 out=torch.zeros(4, 9, device="cuda").expand(2, 4, 9)[0, :3].t())),
        (ValueError, lambda: o.merge_tops(ids, lp, [1.0], 1)),
        (ValueError, lambda: o.merge_tops(ids[None], lp[None], [1.0, 1.0], 1)),
        (ValueError, lambda: o.merge_tops(ids[None], lp[None], [-1.0], 1)),
        (ValueError, lambda: o.merge_tops(ids[None], lp[None], [math.nan], 1)),
        (ValueError, lambda: o.merge_tops(ids[None], lp[None], [1.0], 0)),
        (ValueError, lambda: o.merge_tops(ids[None], lp[None], [1.0], 3)),
        (ValueError, lambda: o.merge_tops(
            torch.zeros(2, 3, 200, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, 200, device="cuda"), [1.0, 1.0], 257)),
        (ValueError, lambda: o.merge_tops(ids[None].expand(129, 3, 2), lp[None].expand(129, 3, 2), [1.0] * 129, 1)),
        (ValueError, lambda: o.merge_tops(ids[None], lp[None], [1.0], 1, token_weight=torch.ones(3, 1, device="cuda"))),
        (TypeError, lambda: o.merge_tops(ids[None], lp[None], [1.0], 1, token_weight=torch.ones(1, 3, device="cuda").half())),
    ]
    for i, (error, call) in enumerate(bad):
        with pytest.raises(error):
            call()
            raise RuntimeError(f"call {i} was not refused")
    buf = torch.zeros(6, 9, device="cuda")
    with pytest.raises(ValueError):
        o.distill_loss_grad(buf[:3], ids, lp, out=buf[2:5])


# ---- finite masks ------------------------------------------------------------------------------------

MASKS = {"f32": [-1e9, -2.5e9, -1e10, -1e18, -1e30], "bf16": [-1e9, -1.66e9, -2.5e9, -1e10, -1e30], "f16": [-1e4, -6e4]}
PLACES = ["front", "back", "groups", "all but one"]


def finite_masks(rows, vocab, dtype, seed, keep=None):
    """Ordinary logits, of which every row masks a run, whole lanes' elements or all but one, by another finite value;
    the elements `keep` [rows, k] stay."""
    x = logits(rows, vocab, dtype, seed=seed)
    i = torch.arange(vocab)
    for r in range(rows):
        place = PLACES[r // len(MASKS[dtype]) % len(PLACES)]
        out = {"front": i < vocab // 2, "back": i >= vocab // 2, "groups": i // 64 % 2 == 0, "all but one": i != vocab // 3}[place]
        if keep is not None:
            out = out.scatter(0, keep[r].long(), False)
        x[r, out] = MASKS[dtype][r % len(MASKS[dtype])]
    return x


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,top", [(20, 1024, 8), (20, 1023, 64), (20, 20011, 128), (520, 5003, 128), (520, 5003, 0)])
def test_scores_behind_finite_masks(rows, vocab, top, dtype):
    check_scores(finite_masks(rows, vocab, dtype, seed=90), some_targets(rows, vocab), top)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", [(20, 1024), (20, 5003), (20, 110017), (20, 70001)])
def test_distill_behind_finite_masks(rows, vocab, dtype):
    """The mask beside the teacher's tokens, and over some of them."""
    ids, lp = teacher(rows, vocab, 6, seed=91)
    for keep in (ids, None):
        for tau in (1.0, 0.5, 4.0):
            check_distill(finite_masks(rows, vocab, dtype, seed=92, keep=keep), ids, lp, tau)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab", [(6, 1000), (6, 20011), (520, 5003)])
def test_scores_of_rows_masked_throughout(rows, vocab, dtype):
    """Every element the same finite value: all tokens alike.

    x log2(e) below 2^31 is at most 64 away from the whole number beside it, so a row's terms are 2^r, |r| <= 64: log2 s
    (below 2^7 here) rounds by 2^-18, e / s by r times what a sum is off (a rounding of 2^-24 each of vocab / 64 + 64
    additions, one multiply-add a term) and 2^-18 more; in natural units all of it times ln 2 < 1."""
    for mask in MASKS[dtype]:
        x = torch.full((rows, vocab), mask).to(DTYPES[dtype])
        s = ops().token_scores(x.cuda(), torch.arange(rows).cuda() % vocab, top=min(vocab, 128))
        even = math.log(vocab)
        tol = 2.0 ** -16 + (64 + 1) * (vocab / 64 + 66) * 2.0 ** -24
        for name, want in (("entropy", even), ("logprob", -even), ("top_logprobs", -even)):
            assert float((getattr(s, name).double() - want).abs().max()) <= tol, (mask, name)
        want = float(x[0, 0]) + even
        assert float((s.lse.double() - want).abs().max()) <= 2.0 ** -22 * abs(want) + tol, mask
        assert torch.equal(s.top_ids.cpu(), torch.arange(min(vocab, 128), dtype=torch.int32).expand(rows, -1))


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,vocab,top", [(6, 1000, 64), (6, 1000, 128), (6, 20011, 128), (520, 9001, 128), (520, 9001, 5)])
def test_lists_of_padding_rows(rows, vocab, top, dtype):
    """Rows whose sums are taken a second time (nothing but -inf, the type's lowest or largest value) among rows whose
    lists have to be as well (NaN, +inf) and ordinary ones, over several chunks and with long lists."""
    x = logits(rows, vocab, dtype, seed=93)
    x[0] = -math.inf
    x[1] = torch.finfo(x.dtype).min
    x[2, ::3] = torch.finfo(x.dtype).max
    x[3, 1::2] = -math.inf
    x[3, ::2] = torch.finfo(x.dtype).min
    x[4, vocab - 2] = math.nan
    check_scores(x, some_targets(rows, vocab), top)
    x[5, vocab - 3] = math.inf
    x[5, 7] = math.inf
    s = ops().token_scores(x.cuda(), top=top)
    assert s.top_ids[5, :2].tolist() == [7, vocab - 3]


def test_merge_of_the_most_entries_of_one_token():
    """Every entry of every list the same token, its terms the largest below a power of two."""
    K, k = 32, 256
    ids = torch.full((K, 2, k), 5, dtype=torch.int32)
    ids[:, 1, 0] = 9                                # 8160 of them, and another token
    lp = torch.zeros(K, 2, k)
    weights = [1.0 - 2.0 ** -53] * K
    check_merge(ids, lp, weights, 3)
    check_merge(ids, lp, weights, 3, torch.ones(K, 2))


@pytest.mark.parametrize("power", [1023, 900, -900, -1070])
def test_merge_with_weights_at_the_ends_of_their_type(power):
    """Only the weights' ratios count: the same bits at any power of two, up to fp64's largest and down to its least."""
    K, rows, k = 3, 5, 7
    ids, lp = answers(K, rows, k, 20, seed=8)
    unit = torch.rand(K, rows) + 0.5
    base = [1.5, 1.25, 1.75]
    check_merge(ids, lp, base, 9, unit)
    want = ops().merge_tops(ids.cuda(), lp.cuda(), base, 9, token_weight=unit.cuda())
    got = ops().merge_tops(ids.cuda(), lp.cuda(), [math.ldexp(b, power) for b in base], 9, token_weight=unit.cuda())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_merge_with_weights_of_all_sizes():
    """A client whose weight is nothing beside another's still answers: its tokens come behind."""
    ids = torch.tensor([[[3, 4]], [[5, 4]]], dtype=torch.int32)
    lp = torch.log(torch.tensor([[[0.5, 0.25]], [[0.5, 0.25]]]))
    got_ids, got_lp = ops().merge_tops(ids.cuda(), lp.cuda(), [1e308, 5e-324], 4)
    assert got_ids.cpu().tolist() == [[3, 4, 5, -1]]
    R.close(got_lp[0, :2], lp[0, 0].double(), 2.0 ** -24 * 2 + 1e-11)
    assert float(got_lp[0, 2]) < -700.0


@pytest.mark.parametrize("dtype", list(DTYPES))
# The lists' least t is 3e-20 at T = 1/4 (below 2^-126 an entry is none); T * 3.4e38 fits fp32 up to 1.
@pytest.mark.parametrize("tau", [0.25, 0.5, 1.0])
@pytest.mark.parametrize("vocab", [40, 5003, 110017])
def test_distill_with_the_lowest_value_under_the_teacher(vocab, tau, dtype):
    """T^2 t (m - x) / T is finite where x / T is not; beside -inf it is inf."""
    rows, k = 6, 5
    x = logits(rows, vocab, dtype, seed=94)
    ids, lp = teacher(rows, vocab, k, seed=95)
    low = torch.finfo(x.dtype).min
    x[0, int(ids[0, 1])] = low
    x[1, ids[1].long()] = low
    x[2] = low
    x[2, int(ids[2, 0])] = 1.0
    x[3, ids[3].long()] = low
    x[3, int(ids[3, 0])] = -math.inf                # the best entry
    x[4] = -math.inf
    x[4, :2] = low
    weight = torch.tensor([1.0, 0.25, -1.0, 1.0, 1.0, 0.5])
    check_distill(x, ids, lp, tau, weight)


@pytest.mark.parametrize("vocab", [40, 5003, 110017])
def test_distill_rows_without_an_entry_whatever_their_ids(vocab):
    """Nothing of probability above 0: loss and gradient 0, also where an id is outside the vocabulary; NaN shows."""
    rows, k = 5, 3
    x = logits(rows, vocab, "f32", seed=96)
    ids, lp = teacher(rows, vocab, k, seed=97)
    ids[0], lp[0] = vocab + 5, -math.inf
    ids[1], lp[1] = torch.tensor([-1, vocab, 2]), torch.tensor([0.5, -math.inf, -math.inf])
    ids[2, 1], lp[2, 1] = vocab, -math.inf           # beside entries that count: NaN
    lp[3] = math.nan
    x[0] = math.nan
    check_distill(x, ids, lp, 1.0)
