"""Cross entropy of a vocabulary head without logits on the GPU, against torch in 64 bits (tests/vocab_reference.py)."""
import pytest
import torch

from tests import vocab_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def run(x, w, y, up, reduction="mean", piece=0, scale=1.0, need=(True, True)):
    from open_flamingo_amd.train.vocab import linear_cross_entropy
    x, w = x.detach().requires_grad_(need[0]), w.detach().requires_grad_(need[1])
    loss = linear_cross_entropy(x, w, y, reduction=reduction, logit_scale=scale, piece=piece)
    if any(need):
        loss.backward(up)
    return loss.detach(), x.grad, w.grad


@pytest.mark.parametrize("rows,d,vocab,piece,reduction,drop,scale", [
    (1, 64, 1, 0, "mean", 0.0, 1.0),
    (1, 256, 1003, 0, "none", 0.0, 1.0),
    (3, 8, 5, 0, "none", 0.4, 0.5),
    (5, 64, 30, 0, "mean", 1.1, 1.0),
    (16, 2048, 5003, 0, "mean", 0.0, 1.0),
    (17, 136, 5003, 0, "sum", 0.1, 1.0),
    (64, 256, 1003, 256, "mean", 0.2, 1.0),
    (255, 320, 2049, 512, "none", 0.3, 2.0),
    (257, 512, 4096, 0, "sum", 0.0, 1.0),
    (1999, 2560, 3001, 1024, "mean", 0.5, 1.0),
    (2048, 1024, 50435, 0, "mean", 0.1, 1.0),
])
def test_loss_and_gradients(rows, d, vocab, piece, reduction, drop, scale):
    R.ce_check(lambda x, w, y, up: run(x, w, y, up, reduction, piece, scale), rows, d, vocab, reduction, drop, scale, device=DEV)


@pytest.mark.parametrize("rows,d,vocab,reduction", [(1, 2048, 50435, "none"), (2, 4096, 1003, "mean"), (4, 2560, 9001, "sum"), (7, 1024, 5000, "mean"),
                                                     (16, 2048, 50435, "none"), (16, 2056, 3001, "mean"), (40, 512, 3001, "none")])
def test_a_handful_of_rows_without_a_gradient(rows, d, vocab, reduction):
    from open_flamingo_amd.train.vocab import linear_cross_entropy
    R.ce_check(lambda x, w, y, up: (linear_cross_entropy(x, w, y, reduction=reduction), None, None), rows, d, vocab, reduction, 0.2, device=DEV)


def test_no_gradient_and_one_gradient():
    x, w, y = R.ce_inputs(300, 512, 2000, device=DEV)
    both = run(x, w, y, torch.ones((), device=DEV))
    assert torch.equal(run(x, w, y, None, need=(False, False))[0], both[0])
    for i, need in enumerate([(True, False), (False, True)]):
        got = run(x, w, y, torch.ones((), device=DEV), need=need)
        assert torch.equal(got[1 + i], both[1 + i]) and got[2 - i] is None
