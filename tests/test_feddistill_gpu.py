"""FedDistillAggregator: a federation of small models that exchange answers, through the serial harness,
against the operators' definitions in 64 bits."""

import math

import pytest
import torch

import token_reference as R
from appfl_amd.harness import SerialSyncHarness

pytestmark = pytest.mark.gpu


def aggregator(model=None, **cfg):
    import appfl_amd.aggregator as A
    return A.FedDistillAggregator(model, cfg, None)


def model(seed, hidden, vocab, out):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Embedding(vocab, hidden), torch.nn.Linear(hidden, out)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_round_of_answers(dtype):
    """Clients of different sizes answer a public set, the server merges, its model's gradient is the formula's."""
    vocab, batch, seq, top, tau = 301, 3, 8, 6, 2.0
    tokens = torch.randint(0, vocab, (batch, seq), generator=torch.Generator().manual_seed(1)).cuda()
    agg = aggregator(client_weights_mode="sample_size", top=top, temperature=tau)
    harness = SerialSyncHarness(agg, 3)
    sizes = [30, 10, 60]
    answers, futures = [], []
    for c in range(3):
        harness.set_sample_size(f"c{c}", sizes[c])
        with torch.no_grad():
            logits = (4.0 * model(c, 8 + 8 * c, vocab, vocab)(tokens)).to(dtype)[:, :-1]     # predicts the next token
        a = agg.answer(logits, targets=tokens[:, 1:])
        flat = logits.reshape(-1, vocab).cpu()
        want, tol = R.scores(flat, tokens[:, 1:].reshape(-1).cpu(), top)
        assert torch.equal(a["top_ids"].cpu(), want["top_ids"])
        for name in ("top_logprobs", "entropy", "logprob"):
            R.close(a[name], want[name], tol[name], name)
        answers.append({k: v.cpu() for k, v in a.items()})
        futures.append(harness.global_update(f"c{c}", dict(answers[-1])))
    teacher = futures[0].result()
    assert all(f.result() is teacher for f in futures) and harness.get_num_global_epochs() == 1
    assert not teacher["top_ids"].is_cuda and teacher["top_ids"].shape == (batch * (seq - 1), top)
    ids = torch.stack([a["top_ids"] for a in answers])
    lp = torch.stack([a["top_logprobs"] for a in answers])
    want_ids, want_lp = R.merge(ids, lp, [0.3, 0.1, 0.6], top)
    assert torch.equal(teacher["top_ids"], want_ids)
    R.close(teacher["top_logprobs"], want_lp, 2.0 ** -24 * want_lp.abs() + 1e-11)
    again = agg.get_parameters()
    assert torch.equal(again["top_ids"], teacher["top_ids"])

    student = model(9, 16, vocab, vocab).to(dtype)
    logits = student(tokens)[:, :-1]
    losses = agg.loss(logits)
    leaf = logits.detach().contiguous()
    want_loss, want_grad, loss_tol, grad_tol = R.distill(leaf.reshape(-1, vocab).cpu(), teacher["top_ids"],
                                                         teacher["top_logprobs"], tau)
    R.close(losses.reshape(-1), want_loss, loss_tol, "loss")
    step_loss, grad = agg.loss_grad(leaf)
    R.close(step_loss.reshape(-1), want_loss, loss_tol, "step loss")
    R.close(grad.reshape(-1, vocab), want_grad, grad_tol, "grad")
    # what reaches the logits is the formula's; what torch's layers below make of it is theirs (their sums
    # over positions have an order of their own, and the two kernels add a row up in different orders)
    whole = student(tokens)
    whole.retain_grad()
    agg.loss(whole[:, :-1]).sum().backward()
    R.close(whole.grad[:, :-1].reshape(-1, vocab), want_grad, grad_tol, "gradient at the logits")
    assert not whole.grad[:, -1].any() and all(bool(p.grad.abs().sum() > 0) for p in student.parameters())
    # part of the positions, weighted
    part = agg.loss(leaf[1:2], first=seq - 1, row_weight=torch.full((1, seq - 1), 0.5, device="cuda"))
    want_part, _, part_tol, _ = R.distill(leaf[1].cpu(), teacher["top_ids"][seq - 1:2 * (seq - 1)],
                                          teacher["top_logprobs"][seq - 1:2 * (seq - 1)], tau, torch.full((seq - 1,), 0.5))
    R.close(part[0], want_part, part_tol, "part")


def test_lists_of_different_lengths_and_left_out_positions():
    agg = aggregator()
    ids = [torch.tensor([[5, 2, 9], [1, 2, 3], [7, 8, 9]]), torch.tensor([[5, 4], [-1, -1], [7, 1]])]
    lp = [torch.log_softmax(torch.randn(3, 4), 1)[:, :3], torch.log_softmax(torch.randn(3, 3), 1)[:, :2]]
    unit = torch.tensor([1.0, 1.0, 0.0])
    got = agg.aggregate({"a": {"top_ids": ids[0], "top_logprobs": lp[0], "token_weight": unit},
                         "b": {"top_ids": ids[1].int(), "top_logprobs": lp[1].double()}})
    full_ids = torch.stack([ids[0].int(), torch.cat([ids[1].int(), torch.full((3, 1), -1, dtype=torch.int32)], 1)])
    full_lp = torch.stack([lp[0], torch.cat([lp[1], torch.full((3, 1), -math.inf)], 1)])
    want_ids, want_lp = R.merge(full_ids, full_lp, [0.5, 0.5], 3, torch.stack([unit, torch.ones(3)]))
    assert torch.equal(got["top_ids"], want_ids)
    R.close(got["top_logprobs"], want_lp, 2.0 ** -24 * want_lp.abs().nan_to_num(posinf=0.0) + 1e-11)


def test_before_the_first_round_and_refusals():
    net = torch.nn.Linear(3, 2)
    agg = aggregator(net, top=2)
    assert torch.equal(agg.get_parameters()["weight"], net.weight.detach())
    with pytest.raises(ValueError):
        aggregator().get_parameters()
    with pytest.raises(ValueError):
        agg.loss(torch.zeros(2, 5, device="cuda"))
    with pytest.raises(ValueError):
        agg.aggregate({})
    ids, lp = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    good = {"top_ids": ids, "top_logprobs": lp}
    for error, bad in ((KeyError, {"top_ids": ids}), (ValueError, {"top_ids": ids[:3], "top_logprobs": lp[:3]}),
                       (ValueError, {"top_ids": ids, "top_logprobs": lp[:, :1]}), (TypeError, {"top_ids": lp, "top_logprobs": lp}),
                       (TypeError, {"top_ids": ids, "top_logprobs": ids}),
                       (ValueError, {"top_ids": ids.long() + (1 << 31), "top_logprobs": lp}),
                       (ValueError, dict(good, token_weight=torch.ones(3)))):
        with pytest.raises(error):
            agg.aggregate({"a": good, "b": bad})
    with pytest.raises(ValueError):
        aggregator().answer(torch.zeros(2, 5, device="cuda"))
    agg.aggregate({"a": good, "b": good})
    for first, rows in ((3, 2), (-1, 2), (5, 1)):
        with pytest.raises(ValueError):
            agg.loss(torch.zeros(rows, 5, device="cuda"), first=first)


def test_registration():
    import types

    from appfl_amd import plugin
    m = types.ModuleType("appfl.algorithm.aggregator")

    class BaseAggregator:
        pass
    m.BaseAggregator = BaseAggregator
    cls = plugin.register_distillation(m)["FedDistillAggregator"]
    assert m.FedDistillAggregator is cls and issubclass(cls, BaseAggregator)
    assert cls(None, {"top": 2}, None).top == 2


@pytest.mark.parametrize("sizes,top", [((3,), 8), ((2, 3, 1), 16), ((4, 4), 256)])
def test_more_entries_asked_for_than_clients_send(sizes, top):
    """`top` above what the clients of a round list together: the lists end with absent entries."""
    vocab, rows = 31, 4
    agg = aggregator(top=top, temperature=2.0)
    updates, ids, lps = {}, [], []
    longest = max(sizes)
    for c, k in enumerate(sizes):
        g = torch.Generator().manual_seed(c)
        i = torch.stack([torch.randperm(vocab, generator=g)[:k] for _ in range(rows)]).int()
        v = torch.log_softmax(torch.randn(rows, k + 1, generator=g), 1)[:, :k]
        updates[f"c{c}"] = {"top_ids": i, "top_logprobs": v}
        ids.append(torch.nn.functional.pad(i, (0, longest - k), value=-1))
        lps.append(torch.nn.functional.pad(v, (0, longest - k), value=-math.inf))
    got = agg.aggregate(updates)
    want_ids, want_lp = R.merge(torch.stack(ids), torch.stack(lps), [1.0 / len(sizes)] * len(sizes), top)
    assert got["top_ids"].shape == (rows, top) and torch.equal(got["top_ids"], want_ids)
    R.close(got["top_logprobs"], want_lp, 2.0 ** -24 * want_lp.abs().nan_to_num(posinf=0.0) + 1e-11)
    assert bool((got["top_ids"][:, sum(sizes):] == -1).all())
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(9))
    want_loss, want_grad, loss_tol, grad_tol = R.distill(x, got["top_ids"], got["top_logprobs"], 2.0)
    loss, grad = agg.loss_grad(x.cuda())
    assert bool(loss.isfinite().all())
    R.close(loss, want_loss, loss_tol, "loss")
    R.close(grad, want_grad, grad_tol, "grad")


def test_losses_of_no_rows():
    agg = aggregator(top=2)
    agg.aggregate({"a": {"top_ids": torch.zeros(4, 2, dtype=torch.int32), "top_logprobs": torch.zeros(4, 2)}})
    for shape in ((0, 5), (2, 0, 5), (0, 3, 5)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        loss = agg.loss(x, first=4)
        loss.sum().backward()
        assert loss.shape == shape[:-1] and x.grad.shape == shape
        loss, grad = agg.loss_grad(x.detach())
        assert loss.shape == shape[:-1] and grad.shape == shape


@pytest.mark.parametrize("classes,top", [(10, 32), (10, 10), (1, 5), (300, 200)])
def test_answers_of_fewer_classes_than_entries(classes, top):
    """`top` above the classes there are, or above one call's lists: an answer holds what there is."""
    agg = aggregator(top=top)
    x = torch.randn(6, classes, generator=torch.Generator().manual_seed(3))
    a = agg.answer(x.cuda())
    n = min(classes, top, 128)
    want, tol = R.scores(x, None, n)
    assert torch.equal(a["top_ids"].cpu(), want["top_ids"])
    R.close(a["top_logprobs"], want["top_logprobs"], tol["top_logprobs"])
