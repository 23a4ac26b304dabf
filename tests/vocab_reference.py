"""Plain 64-bit forms of the vocabulary-table operators, and what a kernel's result may be off by, shared by the emulator and GPU tests."""
import torch

BF16_HALF = 2.0 ** -8          # half a unit in the last place of a bf16 value, relative to the value


def ce_inputs(rows, d, vocab, seed=0, drop=0.3, ignore=-100, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d, generator=g).bfloat16()
    w = (torch.randn(vocab, d, generator=g) * 2 / d ** 0.5).bfloat16()
    y = torch.randint(0, vocab, (rows,), generator=g)
    y[torch.rand(rows, generator=g) < drop] = ignore
    return x.to(device), w.to(device), y.to(device)


def ce_reference(x, w, y, upstream, reduction, ignore=-100, scale=1.0):
    """(loss, dx, dw, how far dx may be off, how far dw) in 64 bits.

    The operands are bf16 values, products exact in fp32, sums in fp32: that part is below 1e-5 of the sums of magnitudes.  An entry of
    D = softmax - onehot is rounded to bf16 once (half a step, 2^-8 of itself) and each gradient once more at its end."""
    xd, wd = x.double(), w.double()
    z = scale * xd @ wd.t()
    keep = y != ignore
    n = int(keep.sum())
    lp = torch.log_softmax(z, 1)
    rows = torch.where(keep, -lp.gather(1, y.clamp(min=0)[:, None])[:, 0], 0.0)
    loss = rows if reduction == "none" else rows.sum() / (n if reduction == "mean" else 1)
    D = lp.exp()
    D[torch.arange(len(y), device=y.device), y.clamp(min=0)] -= 1
    g = upstream.double()[:, None] if reduction == "none" else upstream.double() / (max(n, 1) if reduction == "mean" else 1)
    D = torch.where(keep[:, None], D * g * scale, 0.0)
    dx, dw = D @ wd, D.t() @ xd
    tol = BF16_HALF + 1e-5
    return loss, dx, dw, tol * (dx.abs() + D.abs() @ wd.abs()) + 1e-30, tol * (dw.abs() + D.abs().t() @ xd.abs()) + 1e-30


def ce_check(run, rows, d, vocab, reduction, drop, scale=1.0, seed=0, device="cpu"):
    """run(x, w, y, upstream) -> (loss, dx, dw)"""
    x, w, y = ce_inputs(rows, d, vocab, drop=drop, seed=seed, device=device)
    up = torch.rand(rows, generator=torch.Generator().manual_seed(1)).to(device) + 0.5 if reduction == "none" else torch.tensor(0.75, device=device)
    loss, dx, dw, bx, bw = ce_reference(x, w, y, up, reduction, scale=scale)
    got, gx, gw = run(x, w, y, up)
    if bool((y != -100).any()) or reduction != "mean":
        assert ((got.double() - loss).abs() <= 1e-5 * loss.abs().clamp(min=1)).all(), (got, loss)
    else:
        assert torch.isnan(got)
    if gx is not None:
        assert gx.dtype == torch.bfloat16 and ((gx.double() - dx).abs() <= bx).all(), float(((gx.double() - dx).abs() / bx).max())
        assert (gx[y == -100] == 0).all()
    if gw is not None:
        assert gw.dtype == torch.bfloat16 and ((gw.double() - dw).abs() <= bw).all(), float(((gw.double() - dw).abs() / bw).max())
