"""Calls of the vocabulary table's operators that ordinary batches do not make, and what one training step of the whole table leaves in moments and
parameters, on the GPU."""
import pytest
import torch
from torch.autograd import forward_ad

from tests import vocab_reference as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("need", [(False, False), (True, False), (True, True)])
@pytest.mark.parametrize("rows,vocab", [(1, 3001), (3, 1), (1, 1)])
def test_matrices_of_one_row_with_any_stride(rows, vocab, need):
    from open_flamingo_amd.train.vocab import linear_cross_entropy
    x, w, _ = R.ce_inputs(rows, 264, vocab, drop=0.0, device=DEV)
    y = (torch.arange(rows) % vocab).to(DEV)
    one = lambda t, stride: t if t.shape[0] > 1 else t.as_strided(t.shape, (stride, 1))          # noqa: E731

    def run(x, w):
        x, w = x.detach().requires_grad_(need[0]), w.detach().requires_grad_(need[1])
        loss = linear_cross_entropy(x, w, y)
        if need[0]:
            loss.backward()
        return loss.detach(), x.grad, w.grad

    want = run(x, w)
    for stride in (265, 272):
        got = run(one(x, stride), one(w, stride))
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(got, want)), stride


@pytest.mark.parametrize("vocab,n", [(7, 3), (1, 1), (50435, 1), (50435, 3000)])
def test_a_table_of_one_column_with_any_stride(vocab, n):
    from open_flamingo_amd.train.vocab import embedding_lookup
    ids = (torch.arange(n) * 3 % vocab).to(DEV)
    values = torch.arange(1.0, vocab + 1, device=DEV)
    for table in (values[None].t(), values[:, None].clone()):
        t = table.detach().requires_grad_()
        y = embedding_lookup(ids, t, scale=2.0)
        assert torch.equal(y.detach(), 2.0 * values[ids][:, None])
        y.sum().backward()
        assert torch.equal(t.grad[:, 0], 2.0 * torch.bincount(ids, minlength=vocab).float())


def test_forward_mode_is_refused_and_no_tangent_dropped():
    from open_flamingo_amd.train.vocab import embedding_lookup, linear_cross_entropy
    x, w, y = R.ce_inputs(30, 64, 200, device=DEV)
    table, ids = torch.randn(5, 8, device=DEV), torch.tensor([1, 4, 4], device=DEV)
    with torch.no_grad(), forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))          # noqa: E731
        for call in (lambda: linear_cross_entropy(dual(x), w, y), lambda: linear_cross_entropy(x, dual(w), y), lambda: embedding_lookup(ids, dual(table))):
            with pytest.raises(NotImplementedError):
                call()


@pytest.mark.parametrize("bits", [8, 32])
def test_a_squared_norm_beyond_fp32_skips_the_step_and_says_so(bits):
    from open_flamingo_amd.train.optim import MultiTensorAdamW
    p = torch.nn.Parameter(torch.ones(5000, device=DEV))
    opt = MultiTensorAdamW([p], lr=1e-2, state_bits=bits)
    every = lambda: [p.detach()] + [t for t in opt.state[p].values()]          # noqa: E731
    for value, applied in ((1.0, 1), (1e21, 1), (1.7e19, 2), (1.0, 3)):
        before = [t.clone() for t in every()]
        p.grad = torch.ones_like(p)
        p.grad[77] = value
        opt.step()
        assert opt.applied_steps() == applied and bool(torch.isfinite(opt.grad_norm())) == (value < 1e20)
        assert all(torch.isfinite(t.float()).all() for t in every())
        assert value < 1e20 or all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(before, every()))


@pytest.mark.parametrize("bits", [32, 8])
def test_one_step_of_the_whole_table_against_the_loss_with_logits(bits):
    """Moments, decay and update of one clipped step, from gradients that the loss over materialised logits gives on a second model of the same
    seed.  Its logits are bf16 (half a step, 2^-8 relative: of values up to 4 an error of a probability below 2^-6, 2e-2 of a gradient's norm)."""
    from open_flamingo_amd.train import step, synthetic, towers
    from open_flamingo_amd.train.reducer import GradReducer
    lr, clip = 1e-3, 0.25
    models = []
    for lm_loss in ("libofhip", "libofhip_vocab"):
        model, info = towers.build_flamingo("OF-tiny", device=DEV, seed=0, gates=0.5, lm_loss=lm_loss)
        models.append(model.train())
    batch = synthetic.make_batch(4, 2, 64, info, DEV, seed=5)
    step.forward_loss(models[0], batch, info, amp=True).backward()
    ref = {k: p.grad.double() for k, p in models[0].named_parameters() if p.grad is not None}
    coef = min(1.0, clip / (sum(float(g.square().sum()) for g in ref.values()) ** 0.5 + 1e-6))
    assert coef < 1.0          # the clip is part of what is looked at
    model = models[1]
    red = GradReducer(model, embedding_rows=None)
    opt = step.build_optimizer(model, lr=lr, reducer=red, multi_tensor=True, state_bits=bits)
    start = {k: p.detach().clone() for k, p in model.named_parameters()}
    step.train_step(model, red, opt, batch, info, mask_embedding_rows=False, nan_check="device", clip_norm=clip)
    params = {k: p for k, p in model.named_parameters() if p in opt.state}
    assert set(params) == set(ref) and any(k.endswith("wte.weight") for k in params)
    for k, p in params.items():
        g, st = ref[k] * coef, opt.state[p]
        if g.numel() == 1:          # (a gate's gradient is what is left of one sum of both signs)
            continue
        m, r = st["exp_avg"].double(), st["exp_avg_sq"].double().sqrt()
        if bits == 8:
            m = (R.blocks256(st["exp_avg"].float()).double() * st["exp_avg_scale"][:, None]).reshape(-1)[:p.numel()].view(p.shape)
            r = (R.blocks256(st["exp_avg_sq"].float()).double() * st["exp_avg_sq_scale"][:, None]).reshape(-1)[:p.numel()].view(p.shape)
        # 2e-2 of the gradients' norm; 8 bits: half a code (1/16 of a value) to the nearest, a whole one (1/8) at random, 2^-9 of a block's
        # largest / 448 and less for what lies below the normal codes
        tol = 2e-2 + (0.0 if bits == 32 else 1 / 16 + 2.0 ** -9)
        assert (m - 0.1 * g).norm() <= tol * 0.1 * g.norm(), k
        tol = 2e-2 + (0.0 if bits == 32 else 1 / 8 + 2.0 ** -8)
        assert (r - 0.001 ** 0.5 * g.abs()).norm() <= tol * 0.001 ** 0.5 * g.norm(), k
        # The first update is lr towards the gradient's sign, plus the decay of the gated blocks alone.  Errors of 2e-2 of the norm turn the
        # sign of an element above half the root mean square in (2e-2 / 0.5)^2 of all elements at most.  (The decay of the gated blocks' LayerNorm weights, ones, is a tenth of lr.)
        clear = g.abs() > 0.5 * g.norm() / g.numel() ** 0.5
        wd = 0.1 if "gated_cross_attn" in k else 0.0
        change = p.detach().double() - start[k].double()
        want = -lr * g.sign() * (g.abs() / (g.abs() + 1e-8)) - lr * wd * start[k].double()
        wrong = ((change - want).abs() > 1e-2 * lr + 2.0 ** -22 * start[k].abs()) & clear
        assert int(wrong.sum()) <= (2e-2 / 0.5) ** 2 * g.numel(), (k, int(wrong.sum()), g.numel())
