"""Scaled lookup and its gradient by sorted tokens on the GPU, against sums in 64 bits (tests/vocab_reference.py)."""
import pytest
import torch

from tests import vocab_reference as R

pytestmark = pytest.mark.gpu


def run(ids, table, dy, **kw):
    from open_flamingo_amd.train.vocab import embedding_lookup
    t = table.detach().requires_grad_()
    y = embedding_lookup(ids, t, **kw)
    y.backward(dy)
    return y.detach(), t.grad


@pytest.mark.parametrize("n,d,vocab,dtype,scale,padding_idx,kind", [
    (1, 1, 1, torch.float32, 1.0, None, "uniform"),
    (1, 4096, 50435, torch.bfloat16, 1.0, None, "uniform"),
    (40, 20, 7, torch.float32, 0.5, 3, "uniform"),
    (1000, 2048, 1003, torch.bfloat16, 45.25, -1, "skew"),
    (3333, 1025, 900, torch.float32, 1.0, None, "one"),
    (3333, 72, 9, torch.bfloat16, 2.0, None, "two"),
    (2000, 100, 300, torch.float32, 1.0, 0, "bad"),
    (8192, 256, 50435, torch.float32, 1.0, 50434, "skew"),
    (16384, 64, 2000, torch.float32, 1.0, None, "skew"),
    (16385, 64, 2000, torch.bfloat16, 1.0, None, "skew"),
    (70000, 40, 66000, torch.float32, 1.0, None, "uniform"),
    (100000, 8, 300000, torch.float32, 1.0, None, "skew"),
    (50001, 16, 11, torch.float32, 1.0, 4, "one"),
    (131072, 8, 5000, torch.float32, 1.0, None, "skew"),
    (4194305, 1, 600000, torch.float32, 1.0, None, "uniform"),          # the counts are added up by a launch of their own
    (300000, 8, 700000, torch.bfloat16, 1.0, 5, "skew"),
])
def test_lookup_and_gradient(n, d, vocab, dtype, scale, padding_idx, kind):
    R.emb_check(lambda ids, t, dy: run(ids, t, dy, scale=scale, padding_idx=padding_idx), n, d, vocab, dtype, scale, padding_idx, kind, device="cuda")


def test_the_same_bits_every_time():
    g = torch.Generator().manual_seed(0)
    ids = R.emb_ids("skew", 30000, 500, g).cuda()
    table, dy = torch.randn(500, 264, generator=g).cuda(), torch.randn(30000, 264, generator=g).cuda()
    first = run(ids, table, dy)[1]
    for _ in range(5):
        assert torch.equal(run(ids, table, dy)[1], first)


@pytest.mark.parametrize("n", [1, 64])
def test_few_positions_of_a_wide_table(n):
    R.emb_check(lambda ids, t, dy: run(ids, t, dy, scale=0.5, padding_idx=3), n, 2560, 3461, torch.float32, 0.5, 3, "bad", device="cuda")


@pytest.mark.parametrize("n", [40, 300])
def test_offsets_behind_32_bits(n):
    vocab, d = 530001, 4096          # 2.2e9 elements, 4.3 GB
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, vocab, (n,), generator=g).cuda()
    ids[:4] = torch.tensor([vocab - 1, 0, vocab - 2, vocab - 1], device="cuda")
    table = torch.empty(vocab, d, dtype=torch.bfloat16, device="cuda")
    table[:] = torch.arange(d, device="cuda") % 64
    table[:, 0] = (torch.arange(vocab, device="cuda") // 256).to(torch.bfloat16)
    table[:, 1] = (torch.arange(vocab, device="cuda") % 256).to(torch.bfloat16)
    dy = torch.randint(-8, 9, (n, d), generator=g).to(torch.bfloat16).cuda()          # sums of small whole numbers: exact
    y, dt = run(ids, table, dy)
    assert torch.equal(y, table[ids])
    rows = ids.unique()
    want = torch.zeros(rows.numel(), d, device="cuda").index_add_(0, torch.searchsorted(rows, ids), dy.float())
    assert torch.equal(dt[rows].float(), want)
    dt[rows] = 0
    assert not dt.view(torch.int64).any()
