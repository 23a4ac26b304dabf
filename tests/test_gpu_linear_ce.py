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


def test_no_gradient_and_the_tables_alone():
    x, w, y = R.ce_inputs(300, 512, 2000, device=DEV)
    both = run(x, w, y, torch.ones((), device=DEV))
    assert torch.equal(run(x, w, y, None, need=(False, False))[0], both[0])
    got = run(x, w, y, torch.ones((), device=DEV), need=(False, True))
    assert torch.equal(got[2], both[2]) and got[1] is None


@pytest.mark.parametrize("rows,d,vocab,piece,reduction,drop,scale", [
    (1, 64, 1, 0, "mean", 0.0, 1.0),
    (5, 64, 30, 0, "mean", 1.1, 1.0),
    (64, 256, 1003, 0, "mean", 0.2, 1.0),
    (255, 320, 2049, 512, "none", 0.3, 2.0),
    (1999, 2560, 3001, 1024, "sum", 0.5, 1.0),
    (2048, 1024, 50435, 0, "mean", 0.1, 1.0),
    (300, 512, 3001, 0, "none", 0.2, 40.0),        # losses beyond the early form's range
])
def test_frozen_table(rows, d, vocab, piece, reduction, drop, scale):
    R.ce_check(lambda x, w, y, up: run(x, w, y, up, reduction, piece, scale, need=(True, False)), rows, d, vocab, reduction, drop, scale, device=DEV, early=True)


def test_a_table_of_more_than_four_gigabytes():
    """byte offsets beyond 32 bits: the last classes' logits and gradient rows (the whole in fp32 chunks as the reference)"""
    g = torch.Generator(device=DEV).manual_seed(0)
    vocab, d, rows = 600_001, 4096, 40
    w = torch.empty(vocab, d, dtype=torch.bfloat16, device=DEV)
    for k in range(0, vocab, 1 << 16):
        w[k:k + (1 << 16)] = (torch.randn(min(1 << 16, vocab - k), d, generator=g, device=DEV) / 32).bfloat16()
    x = torch.randn(rows, d, generator=g, device=DEV).bfloat16()
    y = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    y[:4] = torch.arange(vocab - 4, vocab, device=DEV)
    y[7] = -100
    z = torch.cat([x.float() @ w[k:k + (1 << 16)].float().t() for k in range(0, vocab, 1 << 16)], 1)
    want = torch.nn.functional.cross_entropy(z, y)
    D = torch.softmax(z, 1)
    D[torch.arange(rows, device=DEV), y.clamp(min=0)] -= 1
    D = torch.where((y >= 0)[:, None], D / (rows - 1), 0.0)
    for need in ((True, True), (True, False), (False, False)):
        loss, gx, gw = run(x, w, y, torch.ones((), device=DEV), need=need)
        assert abs(loss - want) <= 1e-5 * want
        if gw is not None:
            tail = D[:, -1000:].t() @ x.float()
            assert (gw[-1000:].float() - tail).norm() <= 1e-2 * tail.norm()
            del gw
        if gx is not None:
            dx = sum(D[:, k:k + (1 << 16)] @ w[k:k + (1 << 16)].float() for k in range(0, vocab, 1 << 16))
            assert (gx.float() - dx).norm() <= 1e-2 * dx.norm()
    few = run(x[:3], w, y[:3], None, need=(False, False))[0]
    assert abs(few - torch.nn.functional.cross_entropy(z[:3], y[:3])) <= 1e-5 * few
