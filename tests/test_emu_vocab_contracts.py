"""What the vocabulary table's operators promise around their results, on the host emulator: no byte outside their buffers, backwards that can be
repeated, one derivative and no more, gradients that are the loss's differences."""
import pytest
import torch

from open_flamingo_amd.train import vocab as V
from open_flamingo_amd.train.optim import adamw_step
from tests import vocab_reference as R
from tests.emu import harness

PAD = 4096


class Guarded:
    """torch with ``empty`` between two zones of a known byte"""

    def __init__(self):
        self.bufs = []

    def __getattr__(self, name):
        return getattr(torch, name)

    def empty(self, *shape, dtype=torch.float32, device="cpu"):
        shape = torch.Size(shape[0] if len(shape) == 1 and not isinstance(shape[0], int) else shape)
        size = shape.numel() * dtype.itemsize
        buf = torch.full((size + 2 * PAD,), 0xA5, dtype=torch.uint8)
        self.bufs.append((buf, size))
        return buf[PAD:PAD + size].view(dtype).view(shape)

    def check(self):
        assert self.bufs
        for buf, size in self.bufs:
            assert (buf[:PAD] == 0xA5).all() and (buf[PAD + size:] == 0xA5).all(), size


@pytest.fixture
def guarded(monkeypatch):
    g = Guarded()
    monkeypatch.setattr("open_flamingo_amd.hip.ops.torch", g)
    monkeypatch.setattr("open_flamingo_amd.train.vocab.torch", g)
    return g


@pytest.mark.parametrize("rows,d,vocab,piece,table,grad,reduction", [
    (1, 8, 1, 0, True, True, "mean"), (3, 72, 257, 0, False, False, "sum"), (16, 64, 300, 0, False, False, "none"), (17, 64, 300, 0, True, False, "mean"),
    (70, 72, 513, 256, True, True, "none"), (70, 72, 513, 256, False, True, "none"), (300, 8, 255, 0, False, True, "mean"), (1100, 8, 30, 0, True, True, "sum"),
])
def test_the_loss_stays_inside_its_buffers(guarded, rows, d, vocab, piece, table, grad, reduction):
    x, w, y = (t if t.dtype == torch.int64 else t.to(torch.bfloat16) for t in R.ce_inputs(rows, d, vocab)[:3])
    x, w = x.detach().requires_grad_(grad), w.detach().requires_grad_(table and grad)
    loss = V.linear_cross_entropy(x, w, y, reduction=reduction, piece=piece, ops=harness.emu_ops())
    if grad:
        loss.sum().backward()
    guarded.check()


@pytest.mark.parametrize("n,d,vocab", [(1, 4, 3), (64, 5, 9), (65, 4, 9), (1000, 12, 70000), (20000, 2, 300), (17000, 1, 1), (131073, 1, 300)])
def test_the_lookup_stays_inside_its_buffers(guarded, n, d, vocab):
    ops = harness.emu_ops()
    ids = torch.randint(-1, vocab + 1, (n,), generator=torch.Generator().manual_seed(0))
    table, y, dy, dw = guarded.empty(vocab, d).zero_(), guarded.empty(n, d), torch.ones(n, d), guarded.empty(vocab, d)
    ops.embedding_fwd(ids, table, y, 1.0)
    ops.embedding_bwd(ids, dy, dw, 1.0, -1)
    guarded.check()
    assert torch.equal(dw[:, 0], torch.bincount(ids[(ids >= 0) & (ids < vocab)], minlength=vocab).float())


@pytest.mark.parametrize("bits", [8, 32])
def test_adamw_stays_inside_its_tensors(guarded, bits):
    sizes = [1, 255, 256, 257, 4097, 3]
    dt = torch.float32 if bits == 32 else torch.float8_e4m3fn
    ps, gs = ([guarded.empty(k).fill_(0.5) for k in sizes] for _ in range(2))
    ms, vs = ([guarded.empty(k, dtype=torch.uint8 if bits == 8 else dt).zero_().view(dt) for k in sizes] for _ in range(2))
    sc = [[guarded.empty(-(-k // 256)).zero_() for k in sizes] for _ in range(2)] if bits == 8 else [None, None]
    adamw_step(ps, gs, ms, vs, step=1, max_norm=1.0, exp_avg_scales=sc[0], exp_avg_sq_scales=sc[1], ops=harness.emu_ops())
    guarded.check()
    assert all((p != 0.5).all() for p in ps)


@pytest.mark.parametrize("table,scale", [(True, 1.0), (False, 1.0), (False, 60.0)])
def test_a_backward_can_be_repeated(table, scale):
    x, w, y = (t if t.dtype == torch.int64 else t.to(torch.bfloat16) for t in R.ce_inputs(40, 64, 300)[:3])
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_(table)
    leaves = [x, w] if table else [x]
    loss = V.linear_cross_entropy(x, w, y, logit_scale=scale, ops=harness.emu_ops())
    other = V.linear_cross_entropy(x * 2, w, y, logit_scale=scale, ops=harness.emu_ops())          # between the two: a call of its own
    first = torch.autograd.grad(loss, leaves, retain_graph=True)
    torch.autograd.grad(other, leaves)
    for a, b in zip(first, torch.autograd.grad(loss, leaves)):
        assert torch.equal(a, b)


def test_one_derivative_and_no_more():
    x, w, y = (t if t.dtype == torch.int64 else t.to(torch.bfloat16) for t in R.ce_inputs(5, 64, 30)[:3])
    x = x.detach().requires_grad_()
    plain = torch.autograd.grad(V.linear_cross_entropy(x, w, y, ops=harness.emu_ops()), x)[0]
    got = torch.autograd.grad(V.linear_cross_entropy(x, w, y, ops=harness.emu_ops()), x, create_graph=True)[0]
    assert torch.equal(got, plain)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got.float().sum(), x)
    table = torch.ones(5, 4, requires_grad=True)
    got = torch.autograd.grad(V.embedding_lookup(torch.tensor([1, 1, 4]), table, ops=harness.emu_ops()).square().sum(), table, create_graph=True)[0]
    assert torch.equal(got.detach()[:, 0], torch.tensor([0.0, 4.0, 0.0, 0.0, 2.0]))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(got.sum(), table)


@pytest.mark.parametrize("table", [True, False])
def test_the_gradient_is_the_loss_s_difference(table):
    """Central differences with h = 2^-6 along single elements (multiples of 1/8 below 2: exact in bf16 before and behind the step).  Third
    derivatives are below the third power of the logits' range per unit, 2 |w| <= 4 for x and 2 |x| <= 4 for the table: h^2/6 * 64 = 2.6e-3;
    the loss's fp32 rounding, 2^-22 of at most 16, over 2h: 1.3e-4; the gradient's own rounding, 2^-8 of it, and 2^-8 of every entry of D (two in
    all) times at most 2: 1.6e-2."""
    g = torch.Generator().manual_seed(0)
    pick = lambda *s: torch.randint(-8, 9, s, generator=g) / 8          # noqa: E731
    x, w, y = pick(6, 8), pick(20, 8), torch.tensor([3, 19, -100, 0, 7, 7])
    f = lambda x, w: float(V.linear_cross_entropy(x.to(torch.bfloat16), w.to(torch.bfloat16), y, reduction="sum", ops=harness.emu_ops()))          # noqa: E731
    a, b = x.to(torch.bfloat16).requires_grad_(), w.to(torch.bfloat16).requires_grad_(table)
    V.linear_cross_entropy(a, b, y, reduction="sum", ops=harness.emu_ops()).backward()
    for t, grad, many in ((x, a.grad, 12), (w, b.grad, 12 if table else 0)):
        for i in torch.randperm(t.numel(), generator=g)[:many].tolist():
            at, h = t.view(-1), 2.0 ** -6
            old = float(at[i])
            at[i] = old + h
            up = f(x, w)
            at[i] = old - h
            down = f(x, w)
            at[i] = old
            want, got = (up - down) / (2 * h), float(grad.reshape(-1)[i])
            rows = 1 if t is x else 5          # a table's element sums over the rows
            assert abs(got - want) <= rows * (2.6e-3 + 1.6e-2) + 1.3e-4 + 2.0 ** -8 * abs(got), (i, got, want)


def test_moments_are_not_made_inside_a_capture(monkeypatch):
    from open_flamingo_amd.train import optim
    p = torch.nn.Parameter(torch.ones(8))
    opt = optim.MultiTensorAdamW([p], lr=0.1, ops=harness.emu_ops())
    p.grad = torch.ones(8)
    monkeypatch.setattr(optim, "_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="before capturing"):
        opt.step()
    monkeypatch.setattr(optim, "_capturing", lambda: False)
    opt.step()
    monkeypatch.setattr(optim, "_capturing", lambda: True)
    opt.step()
    assert opt.applied_steps() == 2


def test_a_table_of_another_type_keeps_the_module_s_own_lookup(monkeypatch):
    import types
    emb = torch.nn.Embedding(5, 8).to(torch.float16)
    emb._of_eager_forward = emb.forward
    emb.forward = types.MethodType(V._embedding_forward, emb)
    monkeypatch.setattr(V, "_runs_here", lambda t: True)
    ids = torch.tensor([[0, 4, 4]])
    assert torch.equal(emb(ids), emb.weight[ids])
