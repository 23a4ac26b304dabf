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


def ce_reference(x, w, y, upstream, reduction, ignore=-100, scale=1.0, early=False):
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
    one = torch.zeros_like(D)
    one[torch.arange(len(y), device=y.device), y.clamp(min=0)] = 1
    D, one = (torch.where(keep[:, None], t * g * scale, 0.0) for t in (D, one))
    dx, dw = D @ wd, D.t() @ xd
    tol = BF16_HALF + 1e-5
    bx = tol * (dx.abs() + D.abs() @ wd.abs()) + 1e-30
    if early:          # the label's p - 1 is formed in fp32 from a logit and a log-sum-exp of z log2 e: 8 half steps of 2^-24 of those
        bx = bx + 2.0 ** -21 * (z.abs().amax(1, keepdim=True) * 1.4427).clamp(min=1) * (one.abs() @ wd.abs())
    return loss, dx, dw, bx, tol * (dw.abs() + D.abs().t() @ xd.abs()) + 1e-30


def ce_check(run, rows, d, vocab, reduction, drop, scale=1.0, seed=0, device="cpu", early=False):
    """run(x, w, y, upstream) -> (loss, dx, dw); early: dx alone was asked for"""
    x, w, y = ce_inputs(rows, d, vocab, drop=drop, seed=seed, device=device)
    up = torch.rand(rows, generator=torch.Generator().manual_seed(1)).to(device) + 0.5 if reduction == "none" else torch.tensor(0.75, device=device)
    loss, dx, dw, bx, bw = ce_reference(x, w, y, up, reduction, scale=scale, early=early)
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


# ------------------------------------------------------------------------------------------------ lookup
def emb_ids(kind, n, vocab, g):
    if kind == "one":          # every position the same token
        return torch.full((n,), vocab // 2)
    if kind == "two":          # long runs of two tokens, interleaved
        return torch.arange(n) % 2 * (vocab - 1)
    if kind == "skew":
        return (torch.rand(n, generator=g).double() ** 4 * vocab).long().clamp(max=vocab - 1)
    if kind == "bad":          # some ids outside the table
        return torch.randint(-2, vocab + 2, (n,), generator=g)
    return torch.randint(0, vocab, (n,), generator=g)


def emb_check(run, n, d, vocab, dtype, scale=1.0, padding_idx=None, kind="uniform", seed=0, device="cpu"):
    """run(ids, table, dy) -> (y, dtable).  y: one multiplication and one rounding (none of either for scale 1).  dtable: k terms added in
    fp32 (k half steps of 2^-24 of the sum of magnitudes) and one multiplication, one rounding to the table's type."""
    g = torch.Generator().manual_seed(seed)
    ids = emb_ids(kind, n, vocab, g).to(device)
    table = torch.randn(vocab, d, generator=g).to(dtype).to(device)
    dy = torch.randn(n, d, generator=g).to(dtype).to(device)
    half = torch.finfo(dtype).eps / 2
    inside = (ids >= 0) & (ids < vocab)
    want = table.double()[ids.clamp(0, vocab - 1)] * scale
    y, dt = run(ids, table, dy)
    assert y.dtype == dtype and y.shape == (n, d) and torch.isnan(y[~inside]).all()
    assert ((y.double() - want).abs()[inside] <= (half + 2.0 ** -24) * want.abs()[inside]).all()
    if scale == 1.0:
        assert torch.equal(y[inside], table[ids[inside]])
    live = inside & (ids != (padding_idx if padding_idx is None or padding_idx >= 0 else padding_idx + vocab)) if padding_idx is not None else inside
    acc, mag = (torch.zeros(vocab, d, dtype=torch.float64, device=device) for _ in range(2))
    acc.index_add_(0, ids[live], dy.double()[live] * scale)
    mag.index_add_(0, ids[live], dy.double()[live].abs() * scale)
    count = torch.bincount(ids[live], minlength=vocab)[:, None]
    assert dt.dtype == dtype and dt.shape == (vocab, d)
    assert ((dt.double() - acc).abs() <= half * acc.abs() + (count + 2) * 2.0 ** -24 * mag).all()
    assert (dt[count[:, 0] == 0] == 0).all()


# ------------------------------------------------------------------------------------------------ AdamW
def uniform20(ordinal, index, step):
    """the 20 random bits of (tensor, element, step), in 64-bit integers"""
    m = 0xFFFFFFFF
    x = ((index ^ ((step * 0x9E3779B1 + ordinal * 0x85157AF5) & m)) * 0x9E3779B1) & m
    x = ((x ^ (x >> 15)) * 0x85157AF5) & m
    x = ((x ^ (x >> 13)) * 0x9E3779B1) & m
    return (x ^ (x >> 16)) & 0xFFFFF


E4M3 = torch.tensor([(m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)) for e in range(16) for m in range(8) if (e, m) != (15, 7)], dtype=torch.float64)


def neighbours(q):
    """the e4m3 values at and above / at and below q >= 0"""
    up = torch.searchsorted(E4M3.to(q.device), q.clamp(max=448.0)).clamp(max=len(E4M3) - 1)
    hi = E4M3.to(q.device)[up]
    lo = torch.where(hi == q, hi, E4M3.to(q.device)[(up - 1).clamp(min=0)])
    return lo, hi


def blocks256(x):
    n = x.numel()
    return torch.nn.functional.pad(x.reshape(-1), (0, -n % 256)).view(-1, 256)


def adamw_check(step_fn, sizes, bits, grad_dtype, *, max_norm=1.0, wd=0.1, steps=3, lr=1e-2, seed=0, device="cpu", offset=0, big=1.0):
    """step_fn(ps, gs, ms, vs, m_scales, v_scales, step) -> squared norm; several steps, each against 64 bits from the state in front of it."""
    b1, b2, eps = 0.9, 0.999, 1e-8
    g = torch.Generator().manual_seed(seed)
    rnd = lambda n: torch.randn(n + offset, generator=g)[offset:]          # noqa: E731
    f8 = torch.float8_e4m3fn
    put = lambda t: torch.cat([t.new_zeros(offset), t]).to(device)[offset:] if offset else t.to(device)          # noqa: E731
    ps = [put(rnd(n)) for n in sizes]
    dt = torch.float32 if bits == 32 else f8
    ms, vs = ([torch.zeros(n + offset, dtype=torch.float32, device=device).to(dt)[offset:] for n in sizes] for _ in range(2))
    sc = [[torch.zeros(-(-n // 256), device=device) for n in sizes] for _ in range(2)] if bits == 8 else None
    for t in range(1, steps + 1):
        gs = [put((rnd(n) * torch.rand(n, generator=g) ** 4 * big).to(grad_dtype)) for n in sizes]
        norm2 = sum(float(x.double().square().sum()) for x in gs)
        coef = min(1.0, max_norm / (norm2 ** 0.5 + 1e-6)) if max_norm > 0 else 1.0
        old = [[x.double().clone() if x.dtype != f8 else x.float().double() for x in xs] for xs in (ps, ms, vs)]
        osc = [[x.double().clone() for x in xs] for xs in sc] if sc else None
        got = step_fn(ps, gs, ms, vs, sc[0] if sc else None, sc[1] if sc else None, t)
        assert abs(float(got) - norm2) <= 1e-5 * norm2
        for i, n in enumerate(sizes):
            p, m, v = (o[i] for o in old)
            if bits == 8:
                m = (blocks256(m) * osc[0][i][:, None]).reshape(-1)[:n]
                v = (blocks256(v) * osc[1][i][:, None]).reshape(-1)[:n] ** 2
            ge = gs[i].double() * coef
            m, v = b1 * m + (1 - b1) * ge, b2 * v + (1 - b2) * ge * ge
            upd = lr / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + eps)
            p = p * (1 - lr * wd) - upd
            # ten operations in fp32 and the clip factor (a square root, a sum of squares within 1e-5): 2e-5 of each term
            assert ((ps[i].double() - p).abs() <= 2e-5 * upd.abs() + 1e-6 * p.abs() + 1e-9).all(), (t, i)
            if bits == 32:
                assert ((ms[i].double() - m).abs() <= 2e-5 * (m.abs() + ge.abs())).all() and ((vs[i].double() - v).abs() <= 4e-5 * v + 2.0 ** -126).all()      # (the smallest normal fp32 value)
                continue
            r = v.sqrt()
            for codes, scales, val, signed in ((ms[i], sc[0][i], m, True), (vs[i], sc[1][i], r, False)):
                top = blocks256(val.abs()).amax(1)
                assert ((scales.double() - top / 448).abs() <= 2e-5 * (top + blocks256(ge.abs()).amax(1)) / 448).all()
                q = (blocks256(val.abs()) / (top / 448).clamp(min=1e-300)[:, None]).reshape(-1)[:n]
                c = codes.float().double()
                if signed:
                    assert (c * val >= 0).all()
                c = c.abs()
                lo, hi = neighbours(q)
                slack = 3e-5 * q + 3e-5 * (ge.abs() / (top.repeat_interleave(256)[:n] / 448).clamp(min=1e-300) if signed else 0) + 1e-12
                assert ((c >= lo - slack) & (c <= hi + slack) | ((c - q).abs() <= slack) | (~torch.as_tensor(signed) & (q > 0) & (q < 2.0 ** -9) & (c == 2.0 ** -9))).all()
                if signed:          # to the nearest
                    assert ((c - q).abs() <= torch.minimum((q - lo).abs(), (hi - q).abs()) + 2 * slack).all()
                else:               # at random in proportion: the reference's own bits, where q is not at the border of its draw
                    u = uniform20(i, torch.arange(n, device=device), t).double() / 2 ** 20
                    frac = torch.where(hi > lo, (q - lo) / (hi - lo).clamp(min=1e-300), 0.0)
                    want = torch.where(frac + u >= 1.0, hi, lo)
                    some = v >= 2.0 ** -126          # smaller values are no normal numbers in fp32, in which the update is held: zero, or nearly
                    want = torch.where(some, want.clamp(min=2.0 ** -9), want)
                    sure = (frac + u - 1.0).abs() > 1e-3
                    assert ((c == want) | ~sure | ~some | ((c - q).abs() <= slack)).all()
                    assert (c[some] > 0).all()
