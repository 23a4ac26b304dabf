"""Scaled lookup and its gradient by sorted tokens (csrc/embedding.hip) on the host emulator, against sums in 64 bits, and its refusals."""
import pytest
import torch

from open_flamingo_amd.train.vocab import embedding_lookup
from tests import vocab_reference as R
from tests.emu import harness


def run(ids, table, dy, **kw):
    t = table.detach().requires_grad_()
    y = embedding_lookup(ids, t, ops=harness.emu_ops(), **kw)
    y.backward(dy)
    return y.detach(), t.grad


@pytest.mark.parametrize("n,d,vocab,dtype,scale,padding_idx,kind", [
    (1, 1, 1, torch.float32, 1.0, None, "uniform"),
    (1, 8, 5, torch.bfloat16, 1.0, None, "uniform"),
    (40, 20, 7, torch.float32, 0.5, 3, "uniform"),           # every token crosses a chunk
    (64, 8, 9, torch.float32, 1.0, None, "one"),             # 64: the longest without a sort
    (64, 24, 40, torch.bfloat16, -2.0, 1, "bad"),
    (63, 7, 5, torch.bfloat16, 1.0, None, "uniform"),
    (65, 8, 5, torch.float32, 1.0, None, "one"),
    (300, 8, 50, torch.bfloat16, 45.25, -1, "skew"),
    (333, 12, 9, torch.float32, 1.0, None, "one"),           # one token over all chunks
    (333, 7, 9, torch.bfloat16, 2.0, None, "two"),           # columns that are no whole vectors
    (200, 4, 30, torch.float32, 1.0, 0, "bad"),              # ids outside the table
    (70, 4, 600, torch.float32, 1.0, None, "uniform"),       # two sorting passes
])
def test_lookup_and_gradient(n, d, vocab, dtype, scale, padding_idx, kind):
    R.emb_check(lambda ids, t, dy: run(ids, t, dy, scale=scale, padding_idx=padding_idx), n, d, vocab, dtype, scale, padding_idx, kind)


def test_the_launches_for_many_positions_and_for_large_vocabularies():
    R.emb_check(lambda ids, t, dy: run(ids, t, dy), 16385, 1, 700, torch.float32, kind="skew")
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 1 << 18, (50,), generator=g)
    ids[10:20] = ids[0]
    dy = torch.randn(50, 1, generator=g)
    dw = torch.full((1 << 18, 1), float("nan"))
    harness.emu_ops().embedding_bwd(ids, dy, dw)
    assert torch.allclose(dw, torch.zeros(1 << 18, 1).index_add_(0, ids, dy))


def test_strides_shapes_and_empty_ids():
    g = torch.Generator().manual_seed(0)
    table, ids = torch.randn(11, 24, generator=g), torch.randint(0, 11, (3, 5), generator=g)
    wide = torch.full((11, 40), float("nan"))
    wide[:, 3:27] = table
    dy = torch.randn(3, 5, 24, generator=g)
    plain, view = run(ids, table, dy), run(ids, wide[:, 3:27], dy)
    assert plain[0].shape == (3, 5, 24) and torch.equal(plain[0], view[0]) and torch.equal(plain[1], view[1])
    back = run(ids, table, dy.transpose(0, 1).contiguous().transpose(0, 1))
    across = run(ids.t().contiguous().t(), table, dy.permute(2, 0, 1).contiguous().permute(1, 2, 0))
    assert torch.equal(back[1], plain[1]) and torch.equal(across[1], plain[1])
    t = table.clone().requires_grad_()
    y = embedding_lookup(ids[:0], t, ops=harness.emu_ops())
    y.sum().backward()
    assert y.shape == (0, 5, 24) and (t.grad == 0).all()


@pytest.mark.parametrize("change,error", [
    (dict(ids=lambda i, t: i.int()), TypeError), (dict(table=lambda i, t: t.half()), TypeError), (dict(table=lambda i, t: t[0]), ValueError),
    (dict(table=lambda i, t: t[:0]), ValueError), (dict(padding_idx=11), ValueError), (dict(padding_idx=-12), ValueError),
])
def test_refusals(change, error):
    ids, table = torch.zeros(4, dtype=torch.int64), torch.zeros(11, 8)
    args = [change[k](ids, table) if k in change else v for k, v in (("ids", ids), ("table", table))]
    with pytest.raises(error):
        embedding_lookup(*args, ops=harness.emu_ops(), **{k: v for k, v in change.items() if k not in ("ids", "table")})
    with pytest.raises(RuntimeError):
        embedding_lookup(ids, table)
