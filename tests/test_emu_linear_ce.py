"""Cross entropy of a vocabulary head without logits (csrc/linear_ce.hip) on the host emulator, against torch in 64 bits
(tests/vocab_reference.py says what results may be off by), and its refusals."""
import pytest
import torch

from open_flamingo_amd.train.vocab import linear_cross_entropy
from tests import vocab_reference as R
from tests.emu import harness


def run(x, w, y, up, reduction="mean", piece=0, scale=1.0, table=True, **kw):
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_(table)
    loss = linear_cross_entropy(x, w, y, reduction=reduction, logit_scale=scale, piece=piece, ops=harness.emu_ops(), **kw)
    loss.backward(up)
    return loss.detach(), x.grad, w.grad


@pytest.mark.parametrize("rows,d,vocab,piece,reduction,drop,scale", [
    (1, 64, 1, 0, "mean", 0.0, 1.0),             # one row, one class: loss 0, no gradient
    (3, 64, 5, 0, "none", 0.4, 0.5),
    (5, 64, 30, 0, "mean", 1.1, 1.0),            # every label ignored
    (70, 128, 300, 256, "mean", 0.3, 1.0),       # two pieces, the second hangs over the table's end
    (70, 72, 513, 256, "sum", 0.3, 2.0),         # a depth that is no multiple of 64; three pieces, one column in the last
    (260, 64, 256, 0, "none", 0.0, 1.0),         # rows over a tile's end, a vocabulary of exactly one tile
])
def test_loss_and_gradients(rows, d, vocab, piece, reduction, drop, scale):
    R.ce_check(lambda x, w, y, up: run(x, w, y, up, reduction, piece, scale), rows, d, vocab, reduction, drop, scale)


@pytest.mark.parametrize("rows,d,vocab,piece,reduction,drop,scale", [
    (1, 64, 1, 0, "mean", 0.0, 1.0),
    (5, 64, 30, 0, "mean", 1.1, 1.0),
    (70, 72, 513, 256, "sum", 0.3, 2.0),
    (260, 64, 700, 512, "none", 0.2, 1.0),
    (7, 64, 300, 256, "none", 0.3, 60.0),        # losses far above what the early form's range holds: the form with a maximum takes over
])
def test_frozen_table(rows, d, vocab, piece, reduction, drop, scale):
    R.ce_check(lambda x, w, y, up: run(x, w, y, up, reduction, piece, scale, table=False), rows, d, vocab, reduction, drop, scale, early=True)


@pytest.mark.parametrize("rows,d,vocab,reduction,drop", [(1, 8, 1, "mean", 0.0), (2, 72, 9, "none", 0.0), (3, 520, 50, "sum", 0.5), (8, 64, 2051, "mean", 0.4),
                                                          (16, 136, 33, "none", 0.3), (9, 24, 7, "mean", 1.1)])
def test_a_handful_of_rows_without_a_gradient(rows, d, vocab, reduction, drop):
    def no_grad(x, w, y, up):
        return linear_cross_entropy(x, w, y, reduction=reduction, ops=harness.emu_ops()), None, None
    R.ce_check(no_grad, rows, d, vocab, reduction, drop)


def test_strided_operands_and_labels_outside_the_vocabulary():
    x, w, y = R.ce_inputs(9, 64, 40, drop=0.2)
    y[4] = 2
    wide, tall = torch.full((9, 80), float("nan")).bfloat16(), torch.full((40, 72), float("nan")).bfloat16()
    wide[:, 8:72], tall[:, :64] = x, w
    plain = run(x, w, y, torch.ones(()))
    views = run(wide[:, 8:72], tall[:, :64], y, torch.ones(()))
    odd = run(wide[:, 8:72], torch.nn.functional.pad(w, (1, 3))[:, 1:65], y, torch.ones(()))      # rows that begin at odd addresses
    for a, b, c in zip(plain, views, odd):
        assert torch.equal(a, b) and torch.equal(a, c)
    bad = y.clone()
    bad[4] = 40                                  # one past the last class, and not the ignored value: a caller's mistake
    loss, gx, gw = run(x, w, bad, torch.ones(9), "none")
    assert torch.isnan(loss[4]) and torch.isfinite(loss[torch.arange(9) != 4]).all()
    assert (gx[4] == 0).all() and torch.isfinite(gw.float()).all()
    few = linear_cross_entropy(x, w, bad, reduction="none", ops=harness.emu_ops())
    assert torch.isnan(few[4]) and torch.allclose(few, loss, equal_nan=True)
    none = linear_cross_entropy(x[:0], w, y[:0], reduction="none", ops=harness.emu_ops())
    assert none.shape == (0,) and torch.isnan(linear_cross_entropy(x[:0], w, y[:0], ops=harness.emu_ops()))


def test_only_the_gradients_that_are_asked_for():
    x, w, y = R.ce_inputs(6, 64, 50, drop=0.2)
    b = w.clone().requires_grad_()
    linear_cross_entropy(x, b, y, ops=harness.emu_ops()).backward()
    assert torch.equal(b.grad, run(x, w, y, torch.ones(()))[2]) and x.grad is None


@pytest.mark.parametrize("change,error", [
    (dict(reduction="avg"), ValueError), (dict(piece=-1), ValueError), (dict(hidden=lambda x, w, y: x.float()), TypeError),
    (dict(table=lambda x, w, y: w[:, :56]), ValueError), (dict(labels=lambda x, w, y: y[:-1]), ValueError), (dict(labels=lambda x, w, y: y.int()), TypeError),
    (dict(table=lambda x, w, y: w.half()), TypeError), (dict(table=lambda x, w, y: w[:0]), ValueError),
])
def test_refusals(change, error):
    x, w, y = R.ce_inputs(6, 64, 50)
    args = {k: (change[k](x, w, y) if k in change else v) for k, v in dict(hidden=x, table=w, labels=y).items()}
    kw = {k: v for k, v in change.items() if k not in args}
    with pytest.raises(error):
        linear_cross_entropy(args["hidden"], args["table"], args["labels"], ops=harness.emu_ops(), **kw)
    with pytest.raises(RuntimeError):            # the product has no CPU path
        linear_cross_entropy(x, w, y)
    with pytest.raises(ValueError):
        linear_cross_entropy(x[:, :60], w[:, :60], y, ops=harness.emu_ops())
