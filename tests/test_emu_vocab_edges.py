"""Calls of the vocabulary table's operators that the documentation allows and ordinary batches do not make, on the host emulator."""
import types

import pytest
import torch
from torch.autograd import forward_ad

from open_flamingo_amd.train import vocab as V
from tests import vocab_reference as R
from tests.emu import harness


@pytest.mark.parametrize("grads", [True, False])
def test_forward_mode_is_refused_and_no_tangent_dropped(grads):
    x, w, y = R.ce_inputs(3, 64, 20)
    some = torch.tensor([3, 19, -100])
    table, ids = torch.randn(5, 8, generator=torch.Generator().manual_seed(0)), torch.tensor([1, 4, 4])
    plain = V.linear_cross_entropy(x, w, some, ops=harness.emu_ops()), V.embedding_lookup(ids, table, ops=harness.emu_ops())
    with torch.set_grad_enabled(grads), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))          # noqa: E731
        for call in (lambda: V.linear_cross_entropy(dual(x), w, y, ops=harness.emu_ops()), lambda: V.linear_cross_entropy(x, dual(w), y, ops=harness.emu_ops()),
                     lambda: V.embedding_lookup(ids, dual(table), ops=harness.emu_ops())):
            with pytest.raises(NotImplementedError):
                call()
        # operands without a tangent are as before
        assert torch.equal(V.linear_cross_entropy(x, w, some, ops=harness.emu_ops()), plain[0]) and torch.isfinite(plain[0])
        assert torch.equal(V.embedding_lookup(ids, table, ops=harness.emu_ops()), plain[1])


def test_the_lm_s_own_modules_serve_forward_mode_and_function_transforms(monkeypatch):
    monkeypatch.setattr(V.helpers, "_require_hip", lambda t, what: None)
    monkeypatch.setattr(V.Ops, "default", staticmethod(harness.emu_ops))
    emb = torch.nn.Embedding(5, 8)
    emb._of_eager_forward = emb.forward
    emb.forward = types.MethodType(V._embedding_forward, emb)
    ids, w = torch.tensor([[0, 4, 4]]), emb.weight.detach()
    through = lambda t: torch.func.functional_call(emb, {"weight": t}, (ids,))          # noqa: E731
    with forward_ad.dual_level():
        tangent = forward_ad.unpack_dual(through(forward_ad.make_dual(w, 2 * w))).tangent
    assert torch.equal(tangent, 2 * w[ids])
    assert torch.equal(torch.func.jvp(through, (w,), (2 * w,))[1], 2 * w[ids])
    want = torch.zeros(5, 8).index_add_(0, ids[0], torch.ones(3, 8))
    assert torch.equal(torch.func.grad(lambda t: through(t).sum())(w), want)
    emb(ids).sum().backward()          # outside of both: the operator and its own gradient
    assert torch.equal(emb.weight.grad, want) and type(emb(ids).grad_fn).__name__.startswith(("_EmbeddingLookup", "View"))


@pytest.mark.parametrize("table_grad", [None, False, True])          # None: no gradient at all
@pytest.mark.parametrize("rows,vocab", [(1, 30), (3, 1), (1, 1)])
def test_matrices_of_one_row_with_any_stride(rows, vocab, table_grad):
    """torch calls a matrix of one row contiguous whatever its row stride is"""
    x, w, _ = R.ce_inputs(rows, 64, vocab, drop=0.0)
    y = torch.arange(rows) % vocab
    one = lambda t, stride: t if t.shape[0] > 1 else torch.nn.functional.pad(t, (0, stride - 64)).as_strided(t.shape, (stride, 1))          # noqa: E731

    def run(x, w):
        x, w = x.detach().requires_grad_(table_grad is not None), w.detach().requires_grad_(bool(table_grad))
        loss = V.linear_cross_entropy(x, w, y, ops=harness.emu_ops())
        if table_grad is None:
            return loss.detach(), None, None
        loss.backward()
        return loss.detach(), x.grad, w.grad

    want = run(x, w)
    for stride in (65, 72, 1000001):
        got = run(one(x, stride), one(w, stride))
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, want)), stride


@pytest.mark.parametrize("vocab,ids", [(7, [1, 4, 4]), (7, [6]), (1, [0]), (1, [0, 0]), (300, list(range(0, 300, 3)))])
def test_a_table_of_one_column_with_any_stride(vocab, ids):
    """torch calls a matrix of one column contiguous whatever its column stride is; the gradient of a sum has none at all"""
    ids, k = torch.tensor(ids), len(ids)
    values = torch.arange(1.0, vocab + 1)
    for table in (values[None].t(), values[:, None].clone(), values.repeat_interleave(3).as_strided((vocab, 1), (3, 7))):
        for grad in (torch.ones(()).expand(k, 1), torch.ones(1, k).t(), torch.ones(k, 3)[:, :1]):
            t = table.detach().requires_grad_()
            y = V.embedding_lookup(ids, t, scale=2.0, ops=harness.emu_ops())
            assert torch.equal(y.detach(), 2.0 * values[ids][:, None])
            dt = torch.autograd.grad(y, t, grad)[0]
            assert torch.equal(dt[:, 0], 2.0 * torch.bincount(ids, minlength=vocab).float())


@pytest.mark.parametrize("shape", [(0,), (0, 5), (2, 0)])
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_no_rows_have_torch_s_values_and_zero_gradients(reduction, shape):
    x, w = torch.zeros(*shape, 64).bfloat16().requires_grad_(), torch.ones(30, 64).bfloat16().requires_grad_()
    y = torch.zeros(shape, dtype=torch.int64)
    loss = V.linear_cross_entropy(x, w, y, reduction=reduction, ops=harness.emu_ops())
    want = torch.nn.functional.cross_entropy(torch.zeros(0, 30), y.reshape(-1), reduction=reduction)
    assert loss.dtype == want.dtype and loss.shape == (shape if reduction == "none" else ())
    assert torch.equal(loss.detach().isnan().reshape(-1), want.isnan().reshape(-1)) and (loss.isnan() | (loss == 0)).all()
    loss.sum().backward()
    assert x.grad.shape == x.shape and w.grad.dtype == w.dtype and (w.grad == 0).all()
    with torch.no_grad():
        assert not V.linear_cross_entropy(x, w, y, reduction=reduction, ops=harness.emu_ops()).requires_grad


@pytest.mark.parametrize("rows,d", [(2 ** 23 - 255, 8), (2 ** 23 - 255, 128), (2 ** 23, 64), (2 ** 19 - 255, 4096)])
def test_batches_beyond_32_bit_offsets_are_refused_by_name(rows, d):
    x, y = torch.zeros(1, d).bfloat16().expand(rows, d), torch.zeros(1, dtype=torch.int64).expand(rows)
    with pytest.raises(ValueError, match="split the batch"):
        V.linear_cross_entropy(x, torch.zeros(3, d).bfloat16(), y, ops=harness.emu_ops())
